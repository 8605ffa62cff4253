"""GPU tests of the expert-layer operators against their definitions in 64 bits.

Bounds.  u is the output type's unit roundoff (bf16 2^-8, fp16 2^-11, fp32
2^-24).  A sum of n products formed in fp32 in any order is off by at most
n * 2^-22 * (sum of the products' magnitudes), which leaves a factor of 4 over
round-to-nearest for adders that truncate.  Errors then follow the formula:
 * activation: slope at most 1.13, plus 2^-20 * (1 + |z|) for its own fp32
   evaluation (fast exponential and erf included);
 * gradient of the activation: z is stored rounded, so act' moves by at most
   max|act''| * u * |z| (GELU 0.80, SiLU 0.50), and dz is rounded once; ReLU's
   slope is unknown where |z| is below the product's own error;
 * every result is rounded once: u * |result| (plus the smallest subnormal).
"""
import math

import pytest
import torch

import efficient_linear_assignment_b200 as ela

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.80, "silu": 0.50}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def choices(T, k, E, seed, left_out=0.1, dtype=torch.int64, skew=False):
    g = gen(seed)
    e = torch.randint(0, E, (T, k), generator=g)
    if skew:  # most tokens to expert 0, half of the experts empty
        e = torch.where(torch.rand(T, k, generator=g) < 0.7, torch.zeros_like(e), e // 2 * 2 % max(E, 1))
    gone = torch.rand(T, k, generator=g) < left_out
    e = torch.where(gone, torch.where(torch.rand(T, k, generator=g) < 0.5, -1, E + 3), e)
    return e.to(dtype)


def plan_by_definition(e, E):
    flat = e.reshape(-1).tolist()
    lists = [[] for _ in range(E + 1)]
    for s, v in enumerate(flat):
        lists[v if 0 <= v < E else E].append(s)
    source = [s for li in lists for s in li]
    position = [0] * len(flat)
    for r, s in enumerate(source):
        position[s] = r
    offsets = [0]
    for li in lists[:E]:
        offsets.append(offsets[-1] + len(li))
    return (torch.tensor(offsets, dtype=torch.int32), torch.tensor(position, dtype=torch.int32).view(e.shape),
            torch.tensor(source, dtype=torch.int32))


def close(got, ref, bound, what=""):
    got = got.detach().double().cpu()
    off = (got - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3g} over the bound, largest difference {off.max().item():.3g}"


# ---------------------------------------------------------------- plan

@pytest.mark.parametrize("T,k,E", [(0, 1, 3), (0, 2, 1), (1, 1, 1), (1, 2, 16), (31, 1, 2), (33, 3, 7), (1000, 1, 1),
                                   (1000, 2, 64), (5003, 1, 128), (4096, 8, 64), (777, 4, 1000), (3000, 2, 4096),
                                   (20011, 8, 160), (70001, 3, 5)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_plan_is_the_stable_sort(T, k, E, dtype):
    for seed, (left, skew) in enumerate([(0.0, False), (0.15, False), (0.1, True), (1.0, False)]):
        e = choices(T, k, E, 100 * seed + T, left, dtype, skew)
        got = ela.expert_plan(e.cuda(), E)
        for a, b in zip(got, plan_by_definition(e, E)):
            assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)


def test_plan_takes_one_dimension_strides_and_extreme_ids():
    e = torch.tensor([2 ** 40, -2 ** 62, 1, 0, -1, 1, 2, 3, 2 ** 32])  # 2^32 must not wrap to expert 0
    got = ela.expert_plan(e.cuda(), 3)
    want = plan_by_definition(e.view(-1, 1), 3)
    assert got.position.shape == (9, 1) and all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    wide = choices(100, 6, 5, 1).cuda()
    got, want = ela.expert_plan(wide[:, ::2], 5), plan_by_definition(wide[:, ::2].cpu(), 5)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


# ---------------------------------------------------------------- dispatch and combine

ROUTES = [(1, 1, 1, 1), (1, 2, 16, 1024), (8, 2, 16, 1024), (5, 3, 4, 7), (64, 1, 8, 33), (129, 2, 5, 1000),
          (501, 8, 64, 136), (1030, 1, 128, 2050), (77, 6, 3, 4096), (257, 4, 12, 8200)]


@pytest.mark.parametrize("T,k,E,H", ROUTES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_dispatch_and_its_gradient(T, k, E, H, dtype):
    e = choices(T, k, E, T + H)
    off, pos, src = plan_by_definition(e, E)
    V = int(off[-1])
    g = gen(7 * T + H)
    x = torch.randn(T, H, generator=g).to(dtype)
    drows = torch.randn(T * k, H, generator=g).to(dtype)
    drows[V:] = float("nan")  # rows of no expert: their gradient must not count
    xg = x.cuda().requires_grad_()
    plan = ela.expert_plan(e.cuda(), E)
    rows = ela.expert_dispatch(xg, plan)
    want = x[src.long() // k].clone()
    want[V:] = 0
    assert rows.dtype == dtype and torch.equal(rows.detach().cpu(), want)
    (dx,) = torch.autograd.grad(rows, xg, drows.cuda())
    ref, mag = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for j in range(k):
        has = pos[:, j] < V
        v = drows[pos[has, j].long()].double()
        ref[has] += v
        mag[has] += v.abs()
    close(dx, ref, U[dtype] * ref.abs() + k * 2.0 ** -22 * mag + TINY[dtype], "dx")


@pytest.mark.parametrize("T,k,E,H", ROUTES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.float16, torch.float32),
                                          (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float16), (torch.bfloat16, None)])
def test_combine_and_its_gradients(T, k, E, H, dtype, wdtype):
    e = choices(T, k, E, 3 * T + H)
    off, pos, src = plan_by_definition(e, E)
    V = int(off[-1])
    g = gen(11 * T + H)
    y = torch.randn(T * k, H, generator=g).to(dtype)
    y[V:] = float("inf")  # rows of no expert may hold anything
    w = torch.randn(T, k, generator=g).to(wdtype or torch.float32)
    if wdtype is not None:
        w[pos >= V] = float("nan")  # and so may the weights of their slots
    dout = torch.randn(T, H, generator=g).to(dtype)
    yg, wg = y.cuda().requires_grad_(), w.cuda().requires_grad_()
    plan = ela.expert_plan(e.cuda(), E)
    out = ela.expert_combine(yg, plan, wg if wdtype is not None else None)
    f64 = torch.float64
    ref, mag = torch.zeros(T, H, dtype=f64), torch.zeros(T, H, dtype=f64)
    dy, dw, dwm = torch.zeros(T * k, H, dtype=f64), torch.zeros(T, k, dtype=f64), torch.zeros(T, k, dtype=f64)
    for j in range(k):
        has = pos[:, j] < V
        at = pos[has, j].long()
        wj = w[has, j].double()[:, None] if wdtype is not None else torch.ones(int(has.sum()), 1, dtype=f64)
        ref[has] += wj * y[at].double()
        mag[has] += (wj * y[at].double()).abs()
        dy[at] = wj * dout[has].double()
        p = y[at].double() * dout[has].double()
        dw[has, j], dwm[has, j] = p.sum(1), p.abs().sum(1)
    u = U[dtype]
    assert out.dtype == dtype
    close(out, ref, u * ref.abs() + k * 2.0 ** -22 * mag + TINY[dtype], "out")
    wanted = (yg, wg) if wdtype is not None else (yg,)
    got = torch.autograd.grad(out, wanted, dout.cuda())
    close(got[0], dy, 1.01 * max(u, 2.0 ** -23) * dy.abs() + TINY[dtype], "dy")
    assert (got[0][V:] == 0).all()
    if wdtype is not None:
        assert got[1].dtype == wdtype
        close(got[1], dw, U[wdtype] * dw.abs() + H * 2.0 ** -22 * dwm + TINY[wdtype], "dw")


def test_combine_gradient_against_differences():
    """out is linear in y and in w, so a difference quotient has only rounding error."""
    T, k, E, H = 40, 3, 6, 65
    g = gen(5)
    plan = ela.expert_plan(choices(T, k, E, 5).cuda(), E)
    y, w, d = (torch.randn(s, generator=g).cuda() for s in ((T * k, H), (T, k), (T, H)))
    vy, vw = (torch.randn(s, generator=g).cuda() for s in ((T * k, H), (T, k)))
    yr, wr = y.clone().requires_grad_(), w.clone().requires_grad_()
    gy, gw = torch.autograd.grad(ela.expert_combine(yr, plan, wr), (yr, wr), d)

    def f(a, b):
        return (ela.expert_combine(a, plan, b).double() * d.double()).sum()

    for a, b, want in ((vy, torch.zeros_like(w), (gy.double() * vy.double()).sum()),
                       (torch.zeros_like(y), vw, (gw.double() * vw.double()).sum())):
        quotient = (f(y + a, w + b) - f(y - a, w - b)) / 2
        # about 1e4 terms of size about 1 to 10, each off by a few 2^-24
        assert abs((quotient - want).item()) < 1e4 * 10 * 8 * 2.0 ** -24


def test_strided_rows_empty_and_offsets_beyond_32_bits_of_bytes():
    plan = ela.expert_plan(torch.tensor([[1], [0], [-1], [1]], device="cuda"), 2)
    wide = torch.randn(4, 50, device="cuda")
    for x in (wide[:, 3:20], wide[:, :16], wide[::2].repeat(2, 1)[:, 1::2], torch.randn(30, 4, device="cuda").t(),
              torch.randn(1, 8, device="cuda").expand(4, 8)):
        rows = ela.expert_dispatch(x, plan)
        assert torch.equal(rows, torch.stack([x[1], x[0], x[3], torch.zeros_like(x[0])]))
        back = ela.expert_combine(rows, plan)
        assert torch.equal(back, torch.stack([x[0], x[1], torch.zeros_like(x[0]), x[3]]))
        assert torch.equal(ela.expert_combine(x, plan), torch.stack([x[1], x[0], torch.zeros_like(x[0]), x[2]]))
    none = ela.expert_plan(torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 2)
    assert ela.expert_dispatch(torch.zeros(0, 8, device="cuda"), none).shape == (0, 8)
    assert ela.expert_combine(torch.zeros(0, 8, device="cuda"), none).shape == (0, 8)
    assert ela.expert_dispatch(torch.zeros(4, 0, device="cuda"), plan).shape == (4, 0)
    # more than 2^32 bytes of rows: the last row is where it should be
    T, k, H = 1100, 8, 260 * 1024
    e = torch.zeros(T, k, dtype=torch.int64, device="cuda")
    plan = ela.expert_plan(e, 1)
    x = torch.zeros(T, H, device="cuda", dtype=torch.bfloat16)
    x[:, -1] = torch.arange(T, device="cuda").to(torch.bfloat16)
    rows = ela.expert_dispatch(x, plan)
    assert torch.equal(rows[:, -1], x[:, -1].repeat_interleave(k)) and (rows[:, 0] == 0).all()
    out = ela.expert_combine(rows, plan, torch.full((T, k), 0.125, device="cuda"))
    assert torch.equal(out, x)


def test_plans_with_values_out_of_range_stay_inside_their_buffers():
    pos = torch.tensor([[0], [-5], [2 ** 31 - 1], [9]], dtype=torch.int32, device="cuda")
    x = torch.randn(4, 16, device="cuda")
    for last in (4, -7, 2 ** 31 - 1):
        off = torch.tensor([0, last], dtype=torch.int32, device="cuda")
        plan = ela.ExpertPlan(off, pos, pos.view(-1))
        rows = ela.expert_dispatch(x, plan)
        assert torch.equal(rows[0], x[0] if last > 0 else torch.zeros_like(x[0]))
        out = ela.expert_combine(x, plan)
        assert (out[1:] == 0).all() and torch.equal(out[0], x[0] if last > 0 else torch.zeros_like(x[0]))


# ---------------------------------------------------------------- linear

def act64(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        q = torch.sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    return z, torch.ones_like(z)


def linear_case(R, E, K, N, dtype, seed, counts=None, bias=True, residual=True, first=0):
    g = gen(seed)
    if counts is None:
        cut = torch.randint(0, R + 1, (E,), generator=g).sort().values.tolist()
        off = [0] + cut
    else:
        off = [first]
        for c in counts:
            off.append(off[-1] + c)
    assert off[-1] <= R
    t = {"x": torch.randn(R, K, generator=g).to(dtype), "weight": (torch.randn(E, N, K, generator=g) * K ** -0.5).to(dtype),
         "bias": torch.randn(E, N, generator=g).to(dtype) if bias else None,
         "residual": torch.randn(R, N, generator=g).to(dtype) if residual else None}
    return t, off, torch.randn(R, N, generator=g).to(dtype)


def linear_definition(t, off, act, dy, dtype):
    """Results and their bounds, expert by expert, in 64 bits on the GPU."""
    d = lambda v: None if v is None else v.cuda().double()  # noqa: E731
    x, w, b, res, dy = d(t["x"]), d(t["weight"]), d(t["bias"]), d(t["residual"]), d(dy)
    (R, K), (E, N, _) = x.shape, w.shape
    u, tiny = U[dtype], TINY[dtype]
    y = res.clone() if res is not None else torch.zeros(R, N, dtype=torch.float64, device="cuda")
    ref = {"y": y, "x": torch.zeros_like(x), "weight": torch.zeros_like(w),
           "bias": torch.zeros(E, N, dtype=torch.float64, device="cuda")}
    bound = {k: torch.zeros_like(v) for k, v in ref.items()}
    for e in range(E):
        a, c = off[e], off[e + 1]
        if a == c:
            continue
        z = x[a:c] @ w[e].t()
        ez = (K + 1) * 2.0 ** -22 * (x[a:c].abs() @ w[e].abs().t())
        if b is not None:
            z = z + b[e]
            ez = ez + 2.0 ** -22 * (z.abs() + b[e].abs())
        v, slope = act64(z, act)
        y[a:c] += v
        bound["y"][a:c] = 1.13 * ez + 2.0 ** -20 * (1 + z.abs()) + 2.0 ** -23 * y[a:c].abs()
        dz = dy[a:c] * slope
        edz = dy[a:c].abs() * (CURVE[act] * (1.01 * u * z.abs() + ez + tiny) + 2.0 ** -20)
        if act == "relu":
            edz = edz + dy[a:c].abs() * (z.abs() <= ez + tiny)
        ebias = edz  # the bias gradient sums dz before it is rounded
        if act != "none":
            edz = edz + u * dz.abs() + tiny
        ref["x"][a:c] = dz @ w[e]
        bound["x"][a:c] = edz @ w[e].abs() + N * 2.0 ** -22 * (dz.abs() @ w[e].abs())
        ref["weight"][e] = dz.t() @ x[a:c]
        bound["weight"][e] = edz.t() @ x[a:c].abs() + (c - a) * 2.0 ** -22 * (dz.abs().t() @ x[a:c].abs())
        ref["bias"][e] = dz.sum(0)
        bound["bias"][e] = ebias.sum(0) + (c - a) * 2.0 ** -22 * dz.abs().sum(0)
    for k in ref:
        bound[k] += 1.01 * u * (ref[k].abs() + bound[k]) + tiny
    return {k: v.cpu() for k, v in ref.items()}, {k: v.cpu() for k, v in bound.items()}


def check_linear(t, off, act, dy, dtype, two_d=False, give_offsets=True):
    c = {k: v.cuda() if v is not None else None for k, v in t.items()}
    if two_d:
        c["weight"] = c["weight"][0]
        c["bias"] = None if c["bias"] is None else c["bias"][0]
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda") if give_offsets else None
    ref, bound = linear_definition(t, off, act, dy, dtype)
    quiet = ela.expert_linear(c["x"], c["weight"], c["bias"], c["residual"], act, offsets)
    close(quiet, ref["y"], bound["y"], "y")
    leaf = {k: v.clone().requires_grad_() for k, v in c.items() if v is not None}
    y = ela.expert_linear(leaf["x"], leaf["weight"], leaf.get("bias"), leaf.get("residual"), act, offsets)
    assert torch.equal(y.detach(), quiet)
    names = [k for k in ("x", "weight", "bias", "residual") if k in leaf]
    for k, g in zip(names, torch.autograd.grad(y, [leaf[k] for k in names], dy.cuda())):
        assert g.dtype == dtype and g.shape == leaf[k].shape
        if k == "residual":
            assert torch.equal(g.cpu(), dy)
        else:
            close(g.reshape(ref[k].shape), ref[k], bound[k], "d" + k)


LINEAR = [(1, 1, 1, 1), (1, 2, 16, 8), (3, 4, 40, 24), (16, 16, 1024, 512), (17, 3, 64, 128), (64, 1, 128, 256),
          (100, 5, 136, 264), (129, 2, 257, 130), (300, 7, 1032, 520), (513, 3, 72, 1000), (1000, 64, 128, 192),
          (2048, 1, 512, 640), (1531, 4, 2056, 264)]


@pytest.mark.parametrize("R,E,K,N", LINEAR)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_and_its_gradients(R, E, K, N, dtype, act):
    t, off, dy = linear_case(R, E, K, N, dtype, R + K + N)
    check_linear(t, off, act, dy, dtype)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_epilogues(act, bias, residual):
    for R, E, K, N, dtype in ((200, 3, 96, 160, torch.bfloat16), (7, 2, 64, 48, torch.float16)):
        t, off, dy = linear_case(R, E, K, N, dtype, 5, bias=bias, residual=residual)
        check_linear(t, off, act, dy, dtype)


@pytest.mark.parametrize("counts,first,R", [([0, 0, 0], 0, 40), ([40, 0, 0], 0, 40), ([0, 0, 40], 0, 40),
                                            ([1, 255, 256, 257, 31, 33, 0, 128, 127], 0, 1100), ([5, 0, 70], 9, 120),
                                            ([1] * 30, 0, 30), ([15, 16, 17, 1, 63, 64, 65], 3, 250)])
def test_linear_group_sizes(counts, first, R):
    t, off, dy = linear_case(R, len(counts), 200, 264, torch.bfloat16, 17, counts, first=first)
    check_linear(t, off, "silu", dy, torch.bfloat16)


def test_linear_one_matrix():
    for R, K, N in ((1, 64, 64), (130, 264, 392), (700, 512, 256)):
        t, off, dy = linear_case(R, 1, K, N, torch.bfloat16, R, [R])
        check_linear(t, off, "gelu", dy, torch.bfloat16, two_d=True, give_offsets=False)
        check_linear(t, off, "none", dy, torch.bfloat16, give_offsets=False)
    t, off, dy = linear_case(50, 1, 64, 64, torch.float16, 3, [20], first=10)
    check_linear(t, off, "gelu", dy, torch.float16, two_d=True)


def test_linear_large_sums():
    """Long sums: K, N and the rows of an expert past every tile."""
    for R, E, K, N in ((4096, 2, 1024, 512), (300, 2, 8200, 136), (260, 2, 136, 8200)):
        t, off, dy = linear_case(R, E, K, N, torch.bfloat16, R)
        check_linear(t, off, "gelu", dy, torch.bfloat16)


@pytest.mark.parametrize("K,N", [(1024, 96), (264, 40), (130, 33), (97, 64), (2100, 20)])
@pytest.mark.parametrize("counts", [[1, 0, 1, 1], [9, 8, 0, 3], [40, 2, 0, 1, 0, 0, 0, 0], [17, 16, 30, 1], [5]])
def test_linear_few_rows(K, N, counts):
    """The path that streams the weights once: rows past a group of 8, uneven loads, widths
    that make loads of 32, 16, 4 and 2 bytes."""
    for dtype in (torch.bfloat16, torch.float16):
        t, off, dy = linear_case(sum(counts) + 3, len(counts), K, N, dtype, K + N, counts, first=2)
        check_linear(t, off, "gelu", dy, dtype)


def test_linear_one_matrix_few_rows():
    for R in (1, 8, 9, 16, 17, 33, 64, 65):
        t, off, dy = linear_case(R, 1, 520, 136, torch.bfloat16, R, [R])
        check_linear(t, off, "silu", dy, torch.bfloat16, two_d=True, give_offsets=False)


def test_linear_many_experts():
    """More experts than a warp has lanes, most of them without rows; and the most there are."""
    g = gen(77)
    for E, R in ((70, 3000), (1000, 2000), (4096, 500)):
        cut = torch.randint(0, R + 1, (E,), generator=g).sort().values
        counts = torch.diff(torch.cat([torch.zeros(1, dtype=torch.long), cut])).tolist()
        t, off, dy = linear_case(R, E, 72, 40, torch.bfloat16, E, counts)
        check_linear(t, off, "relu", dy, torch.bfloat16)


def test_weight_gradient_of_many_short_sums():
    """Hundreds of sums of 1 to 70 rows in a row, each ending inside a block of 16, again and
    again: the two CTAs of a pair run apart by several of them."""
    g = gen(78)
    E, K, N = 700, 72, 40
    counts = torch.randint(1, 71, (E,), generator=g)
    counts[::3] = torch.randint(1, 4, counts[::3].shape, generator=g)
    R = int(counts.sum())
    t, off, dy = linear_case(R, E, K, N, torch.bfloat16, 78, counts.tolist(), bias=False, residual=False)
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    ref, bound = linear_definition(t, off, "none", dy, torch.bfloat16)
    x, w, dyc = t["x"].cuda(), t["weight"].cuda().requires_grad_(), dy.cuda()
    for _ in range(20):
        y = ela.expert_linear(x, w, None, None, "none", offsets)
        (dw,) = torch.autograd.grad(y, w, dyc)
    close(dw, ref["weight"], bound["weight"], "dweight")
    ela.expert_check()


@pytest.mark.parametrize("R,E,K,N", [(300, 1, 512, 2048), (700, 1, 256, 4096), (1100, 2, 320, 1024), (90, 1, 128, 9000)])
def test_linear_column_tiles(R, E, K, N):
    """Sizes that choose tiles of other than 256 columns."""
    t, off, dy = linear_case(R, E, K, N, torch.float16, R)
    check_linear(t, off, "none", dy, torch.float16)


def test_linear_rows_of_others_do_not_leak():
    """NaN and infinities in rows of no expert, and in one expert's rows, stay there."""
    R, E, K, N = 150, 3, 80, 72
    for bad in (float("nan"), float("inf")):
        t, off, dy = linear_case(R, E, K, N, torch.bfloat16, 23, [41, 50, 30], first=7)
        want, _ = linear_definition(t, off, "gelu", dy, torch.bfloat16)
        clean = {k: v.clone() for k, v in t.items()}
        dirty_dy = dy.clone()
        for v in (t["x"], dirty_dy):
            v[:off[0]] = bad
            v[off[-1]:] = bad
            v[off[1]:off[2]] = bad
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        grads = {}
        for name, s, d in (("clean", clean, dy), ("dirty", t, dirty_dy)):
            leaf = {k: v.cuda().requires_grad_() for k, v in s.items()}
            y = ela.expert_linear(leaf["x"], leaf["weight"], leaf["bias"], leaf["residual"], "gelu", offsets)
            grads[name] = [y.detach(), *torch.autograd.grad(y, [leaf[k] for k in ("x", "weight", "bias")], d.cuda())]
        (y0, x0, w0, b0), (y1, x1, w1, b1) = grads["clean"], grads["dirty"]
        keep = torch.ones(R, dtype=torch.bool)
        keep[off[1]:off[2]] = False
        assert torch.equal(y0[keep], y1[keep]) and torch.equal(x0[keep], x1[keep])
        for e in (0, 2):
            assert torch.equal(w0[e], w1[e]) and torch.equal(b0[e], b1[e])
        assert torch.isnan(w1[1]).any()


def test_linear_strides_and_alignment():
    R, E, K, N = 90, 2, 72, 88
    for dtype in (torch.bfloat16, torch.float16):
        t, off, dy = linear_case(R, E, K, N, dtype, 31, [50, 33])
        ref, bound = linear_definition(t, off, "relu", dy, dtype)
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        xs = [torch.zeros(R, K + 8, dtype=dtype).cuda()[:, :K], torch.zeros(R, K + 5, dtype=dtype).cuda()[:, 3:K + 3],
              torch.zeros(K, R, dtype=dtype).cuda().t(), torch.zeros(R * K + 1, dtype=dtype).cuda()[1:].view(R, K)]
        ws = [torch.zeros(E, N + 2, K + 8, dtype=dtype).cuda()[:, 1:N + 1, :K], torch.zeros(E, K, N, dtype=dtype).cuda().transpose(1, 2),
              torch.zeros(E, N, K + 1, dtype=dtype).cuda()[:, :, 1:], torch.zeros(E * N * K + 3, dtype=dtype).cuda()[3:].view(E, N, K)]
        rs = [torch.zeros(R, N + 3, dtype=dtype).cuda()[:, 3:], torch.zeros(N, R, dtype=dtype).cuda().t(),
              torch.zeros(R, N + 8, dtype=dtype).cuda()[:, :N], torch.zeros(R, N, dtype=dtype).cuda()]
        for x, w, r in zip(xs, ws, rs):
            x.copy_(t["x"])
            w.copy_(t["weight"])
            r.copy_(t["residual"])
            x.requires_grad_(), w.requires_grad_()
            y = ela.expert_linear(x, w, t["bias"].cuda(), r, "relu", offsets)
            close(y, ref["y"], bound["y"], "y")
            dyt = torch.zeros(N, R, dtype=dtype).cuda().t()
            dyt.copy_(dy)
            dx, dw = torch.autograd.grad(y, (x, w), dyt)
            close(dx, ref["x"], bound["x"], "dx")
            close(dw, ref["weight"], bound["weight"], "dw")
        # the gradient of a sum: dy of stride 0
        leaf = t["x"].cuda().requires_grad_()
        y = ela.expert_linear(leaf, t["weight"].cuda(), None, None, "none", offsets)
        y.sum().backward()
        ones, _ = linear_definition({**t, "bias": None, "residual": None}, off, "none", torch.ones_like(dy), dtype)
        _, tol = linear_definition({**t, "bias": None, "residual": None}, off, "none", torch.ones_like(dy), dtype)
        close(leaf.grad, ones["x"], tol["x"], "dx of a sum")


def test_linear_gradient_against_differences():
    """The gradient along a direction against a central difference of the 64-bit definition."""
    R, E, K, N = 60, 3, 48, 40
    for act in ("gelu", "silu"):
        t, off, dy = linear_case(R, E, K, N, torch.float16, 41, [25, 0, 30])
        leaf = {k: v.cuda().requires_grad_() for k, v in t.items()}
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        y = ela.expert_linear(leaf["x"], leaf["weight"], leaf["bias"], leaf["residual"], act, offsets)
        names = ["x", "weight", "bias"]
        grads = dict(zip(names, torch.autograd.grad(y, [leaf[k] for k in names], dy.cuda())))
        _, bound = linear_definition(t, off, act, dy, torch.float16)

        def value(shift, name, v):
            total = 0.0
            s = {k: q.double() for k, q in t.items()}
            s[name] = s[name] + shift * v
            for e in range(E):
                a, c = off[e], off[e + 1]
                z = s["x"][a:c] @ s["weight"][e].t() + s["bias"][e]
                total += (act64(z, act)[0] * dy[a:c].double()).sum().item()
            return total

        for name in names:
            v = torch.randn(t[name].shape, generator=gen(43), dtype=torch.float64)
            h = 1e-5
            quotient = (value(h, name, v) - value(-h, name, v)) / (2 * h)
            along = (grads[name].double().cpu() * v).sum().item()
            # the gradient's own bound along v, and the quotient's: h^2 curvature plus 1e-16/h cancellation
            assert abs(quotient - along) <= (bound[name] * v.abs()).sum().item() + 1e-4 * abs(quotient) + 1e-4


# ---------------------------------------------------------------- use

def layer(x, expert, E, w1, b1, w2, gate):
    plan = ela.expert_plan(expert, E)
    rows = ela.expert_dispatch(x, plan)
    h = ela.expert_linear(rows, w1, b1, activation="gelu", offsets=plan.offsets)
    h = ela.expert_linear(h, w2, offsets=plan.offsets)
    return ela.expert_combine(h, plan, gate)


def layer_inputs(T=96, k=2, E=8, H=128, F=256, dtype=torch.bfloat16):
    g = gen(3)
    return (torch.randn(T, H, generator=g).to(dtype).cuda(), choices(T, k, E, 3).cuda(), E,
            (torch.randn(E, F, H, generator=g) * H ** -0.5).to(dtype).cuda(), torch.randn(E, F, generator=g).to(dtype).cuda(),
            (torch.randn(E, H, F, generator=g) * F ** -0.5).to(dtype).cuda(), torch.rand(T, k, generator=g).cuda())


def test_same_inputs_same_bits_on_any_stream():
    a = layer_inputs()
    want = layer(*a)
    again = layer(*a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = layer(*a)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, again) and torch.equal(want, other)


def test_layer_in_a_graph():
    x, expert, E, w1, b1, w2, gate = layer_inputs()
    layer(x, expert, E, w1, b1, w2, gate)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, expert, E, w1, b1, w2, gate)
    for seed in (1, 2):  # other tokens and another routing through the same graph
        x.copy_(torch.randn(x.shape, generator=gen(seed)).to(x.dtype))
        expert.copy_(choices(*expert.shape, E, seed, 0.3))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(x, expert, E, w1, b1, w2, gate))


def test_layer_in_a_compiled_graph():
    """torch.compile traces the operators and their gradients (no graph break) to the same bits."""
    x, expert, E, w1, b1, w2, gate = layer_inputs()
    leaves = [v.requires_grad_() for v in (x, w1, b1, w2, gate)]

    def f(x, w1, b1, w2, gate):
        return layer(x, expert, E, w1, b1, w2, gate)

    traced = torch.compile(f, backend="aot_eager", fullgraph=True)
    want, got = f(*leaves), traced(*leaves)
    assert torch.equal(want, got)
    for a, b in zip(torch.autograd.grad(want, leaves, torch.ones_like(want)), torch.autograd.grad(got, leaves, torch.ones_like(got))):
        assert torch.equal(a, b)


def test_assignment_to_experts_end_to_end():
    """Tokens to expert slots by the solver, through the experts and back; tokens
    that the solver leaves out (max_iter) come back as zeros."""
    T, E, H, cap = 128, 8, 64, 16
    g = gen(9)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    score = torch.randn(T, E, generator=g).cuda()
    w = torch.randn(E, H, H, generator=g).to(torch.bfloat16).cuda()
    for max_iter in (1000, 3):
        slot, _ = ela.AuctionB200(epsilon=1e-2, max_iter=max_iter).solve((-score).repeat_interleave(cap, 1)[None])
        expert = torch.where(slot[0] >= 0, slot[0] // cap, slot[0])
        plan = ela.expert_plan(expert, E)
        counts = (plan.offsets[1:] - plan.offsets[:-1]).cpu()
        assert counts.max() <= cap and counts.sum() == (expert >= 0).sum()
        gate = torch.sigmoid(score.gather(1, expert.clamp(min=0)[:, None]))
        out = ela.expert_combine(ela.expert_linear(ela.expert_dispatch(x, plan), w, offsets=plan.offsets), plan, gate)
        ref = torch.einsum("th,tnh->tn", x.double(), w.double()[expert.clamp(min=0)])
        ref = torch.where((expert >= 0)[:, None], ref * gate.double(), 0 * ref)
        # two roundings to bf16 and a sum of 64 products of size about 1
        assert ((out.double() - ref).abs() <= 2.1 * 2.0 ** -8 * ref.abs() + 64 * 2.0 ** -20 * 8).all()
        assert max_iter == 1000 or (expert < 0).any()


# ---------------------------------------------------------------- refusals

def test_refusals():
    bf = torch.bfloat16
    e = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    x = torch.zeros(4, 8, device="cuda")
    plan = ela.expert_plan(e, 2)
    for call, error in [
            (lambda: ela.expert_plan(e.float(), 2), TypeError), (lambda: ela.expert_plan(e, 0), ValueError),
            (lambda: ela.expert_plan(e, 4097), ValueError), (lambda: ela.expert_plan(e[None], 2), ValueError),
            (lambda: ela.expert_plan(e.cpu(), 2), RuntimeError),
            (lambda: ela.expert_dispatch(x[:3], plan), ValueError), (lambda: ela.expert_dispatch(x[0], plan), ValueError),
            (lambda: ela.expert_dispatch(x.double(), plan), TypeError), (lambda: ela.expert_dispatch(x.cpu(), plan), RuntimeError),
            (lambda: ela.expert_dispatch(x, plan._replace(position=plan.position.long())), ValueError),
            (lambda: ela.expert_combine(x, plan), ValueError),
            (lambda: ela.expert_combine(x.repeat(2, 1), plan, torch.zeros(4, 1, device="cuda")), ValueError),
            (lambda: ela.expert_combine(x.repeat(2, 1), plan, torch.zeros(4, 2, device="cuda").half()), TypeError),
            (lambda: ela.expert_combine(x.repeat(2, 1), plan, torch.zeros(4, 2)), ValueError)]:
        with pytest.raises(error):
            call()
    a, w = torch.zeros(4, 8, device="cuda", dtype=bf), torch.zeros(2, 16, 8, device="cuda", dtype=bf)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for call, error in [
            (lambda: ela.expert_linear(a.float(), w.float(), offsets=off), TypeError),
            (lambda: ela.expert_linear(a, w.half(), offsets=off), TypeError),
            (lambda: ela.expert_linear(a, w), ValueError), (lambda: ela.expert_linear(a, w[:, :, :4], offsets=off), ValueError),
            (lambda: ela.expert_linear(a, w, offsets=off.long()), ValueError),
            (lambda: ela.expert_linear(a, w, offsets=off[:2]), ValueError),
            (lambda: ela.expert_linear(a, w, offsets=off.cpu()), ValueError),
            (lambda: ela.expert_linear(a, w, activation="tanh", offsets=off), ValueError),
            (lambda: ela.expert_linear(a, w, bias=torch.zeros(16, device="cuda", dtype=bf), offsets=off), ValueError),
            (lambda: ela.expert_linear(a, w, residual=a, offsets=off), ValueError),
            (lambda: ela.expert_linear(a, w[:, :0], offsets=off), ValueError),
            (lambda: ela.expert_linear(a[:, :0], w[:, :, :0], offsets=off), ValueError),
            (lambda: ela.expert_linear(a.cpu(), w, offsets=off), RuntimeError),
            (lambda: ela.expert_linear(a, w.cpu(), offsets=off), ValueError)]:
        with pytest.raises(error):
            call()
    y = ela.expert_linear(a.requires_grad_(), w, offsets=off)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), a, create_graph=True)


def test_no_wait_gave_up():
    """After everything above: no kernel ended a wait at its limit."""
    ela.expert_check()


def test_example_trains():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "balanced_experts.py")
    spec = importlib.util.spec_from_file_location("balanced_experts", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.train(steps=30, tokens=512, hidden=128, width=256, experts=8, verbose=False)
    assert losses[-1] < 0.7 * losses[0]
    assert mod.generate(steps=3, tokens=4, hidden=128, width=256, experts=8, verbose=False)


def test_linear_without_rows():
    w = torch.randn(2, 16, 8, device="cuda", dtype=torch.bfloat16).requires_grad_()
    b = torch.randn(2, 16, device="cuda", dtype=torch.bfloat16).requires_grad_()
    x = torch.zeros(0, 8, device="cuda", dtype=torch.bfloat16).requires_grad_()
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    for act in ("none", "gelu"):
        y = ela.expert_linear(x, w, b, None, act, off)
        assert y.shape == (0, 16)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 16, device="cuda", dtype=torch.bfloat16))
        assert gx.shape == (0, 8) and (gw == 0).all() and (gb == 0).all()
