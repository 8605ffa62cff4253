"""GPU tests of the 4-bit experts against their definitions in 64 bits.

Scales and whole numbers are equal: quotients of 16-bit floats are either exactly halfway
between two whole numbers or further from it than fp32 rounds.  Products follow the bounds of
the 16-bit experts' tests, on the dequantized weights: a sum of n products formed in fp32
in any order is off by at most n * 2^-22 * (sum of the products' magnitudes); the
activation's slope is at most 1.13, its own evaluation off by 2^-20 * (1 + |z|); the result is
rounded once.
"""
import math

import pytest
import torch

import efficient_linear_assignment_b200 as ela

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def quantize_by_definition(w, group):
    """q (…, N, K) and scales (…, parts, N) in 64 bits."""
    K = w.shape[-1]
    q, scales = [], []
    for a in range(0, K, group):
        part = w[..., a:a + group].double()
        s = (part.abs().amax(-1) / 7).to(w.dtype)
        d = s.double().unsqueeze(-1)
        q.append(torch.where((d > 0) & (d < math.inf), torch.round(part / d).clamp(-8, 7), torch.zeros_like(part)))
        scales.append(s)
    return torch.cat(q, -1), torch.stack(scales, -2)


def unpack_by_definition(packed, K):
    """The whole numbers, from the layout that is documented."""
    words = packed.cpu().long() & 0xffffffff
    out = torch.empty(*words.shape, 8, dtype=torch.int64)
    for j in range(8):
        out[..., j] = ((words >> (4 * (j // 2) + 16 * (j % 2))) & 15) - 8
    return out.flatten(-2)


def weights_by_definition(q, scales, group):
    s = scales.double().transpose(-1, -2).repeat_interleave(group, -1)[..., :q.shape[-1]]
    return (q.double() * s).to(scales.dtype)


def random_weight(E, N, K, dtype, seed):
    g = gen(seed)
    return (torch.randn(E, N, K, generator=g) * K ** -0.5 * torch.exp(torch.randn(E, N, 1, generator=g))).to(dtype)


SHAPES = [(1, 1, 1), (1, 1, 33), (2, 3, 31), (1, 5, 64), (3, 33, 96), (2, 40, 129), (1, 64, 1000), (4, 31, 256), (2, 100, 1027), (1, 257, 2056)]


@pytest.mark.parametrize("E,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_and_back(E, N, K, dtype, group):
    w = random_weight(E, N, K, dtype, E + N + K)
    q, s = quantize_by_definition(w, group)
    got = ela.expert_quantize(w.cuda(), group)
    assert got.features == K and got.group == group and got.packed.shape == (E, N, 8 * -(-K // 64)) and got.scales.shape == (E, -(-K // group), N)
    assert torch.equal(got.scales.cpu(), s)
    unpacked = unpack_by_definition(got.packed, K)
    assert torch.equal(unpacked[..., :K], q.long()) and (unpacked[..., K:] == 0).all()
    back = ela.expert_dequantize(got)
    assert back.dtype == dtype and torch.equal(back.cpu(), weights_by_definition(q, s, group))
    one = ela.expert_quantize(w[0].cuda(), group)
    assert one.packed.shape == got.packed.shape[1:] and torch.equal(one.packed, got.packed[0]) and torch.equal(one.scales, got.scales[0])
    assert torch.equal(ela.expert_dequantize(one), back[0])


def test_quantize_halves_extremes_and_zeros():
    for dtype in (torch.bfloat16, torch.float16):
        w = torch.zeros(1, 6, 64).to(dtype)
        w[0, 0, :15] = torch.arange(-7, 8).to(dtype) / 2          # halfway cases: scale 0.5
        w[0, 1, :15] = torch.arange(-7, 8).to(dtype)               # scale 1
        w[0, 1, 15:20] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5]).to(dtype)
        w[0, 2] = torch.finfo(dtype).max
        w[0, 3] = torch.finfo(dtype).smallest_normal
        w[0, 4, 5] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest subnormal: its scale is 0
        w[0, 5, ::2] = -1.0
        q, s = quantize_by_definition(w, 32)
        got = ela.expert_quantize(w.cuda(), 32)
        assert torch.equal(got.scales.cpu(), s) and torch.equal(unpack_by_definition(got.packed, 64), q.long())
        assert torch.equal(ela.expert_dequantize(got).cpu(), weights_by_definition(q, s, 32))


def test_groups_that_are_not_finite_show_it():
    w = random_weight(1, 4, 128, torch.bfloat16, 1)
    w[0, 1, 40], w[0, 2, 70] = math.nan, math.inf
    got = ela.expert_quantize(w.cuda(), 64)
    assert got.scales[0, 0, 1].isnan() and got.scales[0, 1, 2].isinf() and got.scales.isfinite().sum() == 6
    back = ela.expert_dequantize(got).isfinite().cpu()
    assert not back[0, 1, :64].any() and not back[0, 2, 64:].any() and back[0, [0, 3]].all() and back[0, 1, 64:].all()
    x = torch.ones(3, 128, dtype=torch.bfloat16, device="cuda")
    for R in (3, 300):
        y = ela.expert_linear_4bit(x[:1].expand(R, -1), got, offsets=torch.tensor([0, R], dtype=torch.int32, device="cuda"))
        assert y[:, [1, 2]].isnan().all() and y[:, [0, 3]].isfinite().all()


def test_quantize_strides():
    w = random_weight(4, 50, 300, torch.bfloat16, 2).cuda()
    for view in (w[1:3], w[:, 3:40], w[:, :, 8:200], w[:, :, 1:130], w[:, :, ::2], w[::2, ::3], w.transpose(1, 2), w[0], w[2, :, 5:64].t()):
        got, want = ela.expert_quantize(view, 32), ela.expert_quantize(view.contiguous(), 32)
        assert torch.equal(got.packed, want.packed) and torch.equal(got.scales, want.scales)


# ---------------------------------------------------------------- product

def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z * torch.special.expit(z) if act == "silu" else z


def product_by_definition(x, w, bias, residual, act, off):
    """The result and its bound, in 64 bits on the GPU; w: the dequantized weights."""
    dtype, u = x.dtype, U[x.dtype]
    x, w = x.cuda().double(), w.cuda().double()
    (R, K), (E, N, _) = x.shape, w.shape
    y = residual.cuda().double().clone() if residual is not None else torch.zeros(R, N, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(y)
    for e in range(E):
        a, c = off[e], off[e + 1]
        if a == c:
            continue
        z = x[a:c] @ w[e].t()
        ez = (K + 1) * 2.0 ** -22 * (x[a:c].abs() @ w[e].abs().t())
        if bias is not None:
            b = bias[e].cuda().double()
            z = z + b
            ez = ez + 2.0 ** -22 * (z.abs() + b.abs())
        y[a:c] += act64(z, act)
        bound[a:c] = 1.13 * ez + 2.0 ** -20 * (1 + z.abs()) + 2.0 ** -23 * y[a:c].abs()
    return y, bound + 1.01 * u * (y.abs() + bound) + TINY[dtype]


def product_case(R, E, K, N, dtype, seed, counts=None, first=0, bias=True, residual=True, group=32):
    g = gen(seed)
    if counts is None:
        off = [0] + torch.randint(0, R + 1, (E,), generator=g).sort().values.tolist()
    else:
        off = [first]
        for c in counts:
            off.append(off[-1] + c)
    assert off[-1] <= R
    x = torch.randn(R, K, generator=g).to(dtype)
    b = torch.randn(E, N, generator=g).to(dtype) if bias else None
    r = torch.randn(R, N, generator=g).to(dtype) if residual else None
    return x, ela.expert_quantize(random_weight(E, N, K, dtype, seed + 1).cuda(), group), b, r, off


def close(got, ref, bound):
    assert got.isfinite().all()
    worst = ((got.double() - ref).abs() - bound).max().item() if got.numel() else -1.0
    assert worst <= 0, f"{worst:.3g} over the bound"


def check(x, w, b, r, off, act, offsets=True):
    ref, bound = product_by_definition(x, ela.expert_dequantize(w), b, r, act, off)
    c = lambda v: None if v is None else v.cuda()  # noqa: E731
    y = ela.expert_linear_4bit(c(x), w, c(b), c(r), act, torch.tensor(off, dtype=torch.int32, device="cuda") if offsets else None)
    assert y.dtype == x.dtype and y.shape == (x.shape[0], w.packed.shape[1])
    close(y, ref, bound)
    return y


PRODUCTS = [(1, 1, 1, 1), (1, 1, 4096, 512), (1, 2, 16, 8), (3, 4, 40, 24), (8, 1, 300, 33), (16, 16, 1024, 512), (17, 3, 64, 128), (64, 1, 128, 256),
            (100, 5, 136, 264), (129, 2, 257, 130), (300, 7, 1032, 520), (513, 3, 72, 1000), (1000, 64, 128, 192), (2048, 1, 512, 640),
            (1531, 4, 2056, 264), (700, 2, 1027, 517)]


@pytest.mark.parametrize("R,E,K,N", PRODUCTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_product(R, E, K, N, dtype, group):
    check(*product_case(R, E, K, N, dtype, R + K + N, group=group), "gelu")


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
def test_epilogues(act, bias, residual):
    for R, E, K, N, dtype in ((200, 3, 96, 160, torch.bfloat16), (7, 2, 64, 48, torch.float16), (400, 2, 200, 131, torch.float16)):
        check(*product_case(R, E, K, N, dtype, 5, bias=bias, residual=residual, group=64), act)


@pytest.mark.parametrize("counts,first,R", [([0, 0, 5], 0, 5), ([1, 0, 0, 7], 0, 8), ([0, 0, 0], 0, 4), ([3, 300, 0, 2], 2, 320), ([128, 256, 32, 33], 0, 449),
                                            ([1, 1, 1, 1], 3, 12), ([700, 0, 1], 1, 720), ([9, 8, 7, 17], 0, 60)])
def test_group_sizes(counts, first, R):
    """Experts without rows, rows before the first and behind the last expert."""
    for dtype in (torch.bfloat16, torch.float16):
        x, w, b, r, off = product_case(R, len(counts), 200, 136, dtype, R, counts, first)
        y = check(x, w, b, r, off, "silu")
        gone = torch.ones(R, dtype=torch.bool)
        gone[off[0]:off[-1]] = False
        assert torch.equal(y.cpu()[gone], r[gone])
        assert (check(x, w, b, None, off, "silu").cpu()[gone] == 0).all()


def test_one_matrix():
    for R, K, N in ((1, 512, 768), (5, 96, 40), (33, 200, 64), (500, 264, 1000)):
        x, w, b, r, off = product_case(R, 1, K, N, torch.bfloat16, R, [R], group=64)
        y = check(x, w, b, r, off, "gelu", offsets=False)
        flat = ela.Expert4Bit(w.packed[0], w.scales[0], w.features, w.group)
        assert torch.equal(y, ela.expert_linear_4bit(x.cuda(), flat, b[0].cuda(), r.cuda(), "gelu"))


@pytest.mark.parametrize("K", [1, 31, 32, 33, 63, 65, 127, 128, 160, 1000, 1056, 5000, 16384])
@pytest.mark.parametrize("rows", [1, 40, 400])
def test_lengths_of_the_sum(K, rows):
    for group in (32, 128):
        check(*product_case(rows, 1, K, 72, torch.bfloat16, K, [rows], group=group), "none")


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 63, 65, 127, 129, 255, 257])
def test_feature_counts(N):
    for rows in (2, 30, 200):
        check(*product_case(rows, 2, 96, N, torch.float16, N, [rows // 2, rows - rows // 2]), "none")


def test_agrees_with_the_16_bit_product():
    """Few rows and many: the weights are those that dequantizing writes."""
    for R, E, K, N in ((24, 6, 512, 256), (900, 3, 512, 384)):
        x, w, b, r, off = product_case(R, E, K, N, torch.bfloat16, 3, [R // E] * E)
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        y4 = ela.expert_linear_4bit(x.cuda(), w, b.cuda(), r.cuda(), "none", o)
        y16 = ela.expert_linear(x.cuda(), ela.expert_dequantize(w), b.cuda(), r.cuda(), "none", o)
        _, bound = product_by_definition(x, ela.expert_dequantize(w), b, r, "none", off)
        assert ((y4.double() - y16.double()).abs() <= 2 * bound).all()


def test_rows_of_others_do_not_leak():
    """NaN in rows of no expert, in other experts' rows and in their weights stays there."""
    for counts, R in (([5, 3, 4], 20), ([100, 300, 40], 600)):
        x, w, b, r, off = product_case(R, 3, 160, 96, torch.bfloat16, 8, counts, 2)
        want = ela.expert_linear_4bit(x.cuda(), w, b.cuda(), r.cuda(), "gelu", torch.tensor(off, dtype=torch.int32, device="cuda"))
        x2 = x.clone()
        x2[:off[0]] = math.nan
        x2[off[1]:off[2]] = math.inf
        x2[off[3]:] = math.nan
        s2 = w.scales.clone()
        s2[1] = math.nan
        got = ela.expert_linear_4bit(x2.cuda(), w._replace(scales=s2), b.cuda(), r.cuda(), "gelu", torch.tensor(off, dtype=torch.int32, device="cuda"))
        keep = torch.ones(R, dtype=torch.bool)
        keep[off[1]:off[2]] = False
        assert torch.equal(got.cpu()[keep], want.cpu()[keep]) and got.cpu()[~keep].isnan().all()


def test_strides_and_alignment():
    for rows in (6, 350):
        for dtype in (torch.bfloat16, torch.float16):
            x, w, b, r, off = product_case(rows, 2, 130, 77, dtype, 4, [rows // 2, rows - rows // 2])
            o = torch.tensor(off, dtype=torch.int32, device="cuda")
            ref, bound = product_by_definition(x, ela.expert_dequantize(w), b, r, "silu", off)
            wide, res = torch.full((rows, 160), 7.0, dtype=dtype, device="cuda"), torch.full((rows, 99), 5.0, dtype=dtype, device="cuda")
            for at in (0, 1, 8, 13):
                xv, rv = wide[:, at:at + 130], res[:, at:at + 77]
                xv.copy_(x)
                rv.copy_(r)
                close(ela.expert_linear_4bit(xv, w, b.cuda(), rv, "silu", o), ref, bound)
            close(ela.expert_linear_4bit(x.cuda().t().contiguous().t(), w, b.cuda(), r.cuda().t().contiguous().t(), "silu", o), ref, bound)
            # packed words off their 16 bytes, scales off their place, both out of a larger tensor
            buf = torch.zeros(w.packed.numel() + 1, dtype=torch.int32, device="cuda")
            buf[1:] = w.packed.view(-1)
            sbuf = torch.zeros(w.scales.numel() + 1, dtype=dtype, device="cuda")
            sbuf[1:] = w.scales.reshape(-1)
            off16 = w._replace(packed=buf[1:].view(w.packed.shape), scales=sbuf[1:].view(w.scales.shape))
            close(ela.expert_linear_4bit(x.cuda(), off16, b.cuda(), r.cuda(), "silu", o), ref, bound)
            assert torch.equal(ela.expert_dequantize(off16), ela.expert_dequantize(w))


def test_one_expert_of_many_and_slices():
    """Weights cut out of a larger model by expert."""
    w = ela.expert_quantize(random_weight(6, 40, 96, torch.bfloat16, 9).cuda(), 32)
    part = w._replace(packed=w.packed[2:5], scales=w.scales[2:5])
    x = torch.randn(9, 96, generator=gen(1)).to(torch.bfloat16)
    check(x, part, None, None, [0, 2, 5, 9], "none")


def test_offsets_out_of_range_stay_inside():
    x, w, _, r, _ = product_case(40, 3, 64, 48, torch.bfloat16, 6, [10, 10, 20])
    for off in ([-5, 3, 2 ** 30, 2 ** 30], [30, 10, 5, 40], [2 ** 31 - 1] * 4, [-2 ** 31] * 4, [0, 0, 0, 0]):
        y = ela.expert_linear_4bit(x.cuda(), w, None, r.cuda(), "none", torch.tensor(off, dtype=torch.int32, device="cuda"))
        assert y.shape == (40, 48)
    torch.cuda.synchronize()
    ela.expert_check()


@pytest.mark.parametrize("E,R", [(700, 9000), (4096, 40000)])
def test_many_experts_in_tiles(E, R):
    """More experts than fit beside many stages; every expert a few rows, some none."""
    g = gen(E)
    counts = torch.multinomial(torch.rand(E, generator=g) * (torch.rand(E, generator=g) < 0.9), R - 50, replacement=True, generator=g).bincount(minlength=E)
    assert R > 8 * E
    x, w, b, r, off = product_case(R, E, 200, 40, torch.bfloat16, 3, counts.tolist(), 20)
    check(x, w, b, r, off, "silu")


def test_wide_offsets_out_of_range_in_tiles():
    x, w, _, r, _ = product_case(500, 3, 200, 300, torch.bfloat16, 6, [100, 100, 300])
    for off in ([-5, 300, 2 ** 30, 2 ** 30], [300, 100, 50, 400], [2 ** 31 - 1] * 4, [-2 ** 31] * 4, [0, 0, 0, 0], [0, 500, 0, 500]):
        y = ela.expert_linear_4bit(x.cuda(), w, None, r.cuda(), "none", torch.tensor(off, dtype=torch.int32, device="cuda"))
        assert y.shape == (500, 300)
    torch.cuda.synchronize()
    ela.expert_check()


def test_two_calls_at_once_with_workspaces():
    """Odd widths, whose operands are copied into a workspace, on two streams, over and over."""
    cases = []
    for seed in (1, 2):
        x, w, b, r, off = product_case(900, 3, 205, 333, torch.bfloat16, seed, [300, 0, 600])
        cases.append((x.cuda(), w, b.cuda(), r.cuda(), "gelu", torch.tensor(off, dtype=torch.int32, device="cuda")))
    want = [ela.expert_linear_4bit(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(ela.expert_linear_4bit(*c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_activations_of_extreme_sums():
    """Sums from the far tails: what rounds to 0 may be 0, infinities and NaN come out as the formula has them."""
    K, N = 64, 32
    w = ela.expert_quantize(torch.eye(N, K).to(torch.bfloat16).mul(7).cuda(), 32)  # feature n: 7 x_n
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 0.5, -0.5, 3.0, -3.0, 6.0, -6.0, 12.0, -12.0, 14.0, -14.0, 80.0, -80.0, 100.0, -100.0, 1e4, -1e4,
                      1e18, -1e18, 1e20, -1e20, 3e37, -3e37, math.inf, -math.inf, math.nan, 1.0, -1.0, 2.0])
    x = torch.zeros(300, K)
    x[:, :N] = z / 7
    x[:, 26:29] = 0  # (an infinity times the other features' zeros would be NaN everywhere)
    x = x.to(torch.bfloat16).cuda()
    bias = torch.zeros(N)
    bias[26:29] = z[26:29]
    bias = bias.to(torch.bfloat16).cuda()
    s = (x[0, :N].double() * 7 + bias.double()).cpu()
    for act in ("relu", "gelu", "silu"):
        want = act64(s, act)
        for rows in (2, 300):
            y = ela.expert_linear_4bit(x[:rows], w, bias, None, act).double().cpu()
            assert torch.equal(y[0], y[-1]) or y[0].isnan().any()
            y, fin = y[0], want.isfinite()
            assert y[28].isnan() and y[26] == math.inf and (y[27] == 0 if act == "relu" else y[27].isnan())  # -inf * 0
            own = torch.where(want != 0, 2.0 ** -20 * (1 + s.abs()), torch.zeros_like(s))[fin]  # (a product with 0 would be NaN at -inf)
            assert ((y - want).abs()[fin] <= own + 2.0 ** -8 * 1.01 * want.abs()[fin] + 2.0 ** -20).all()


def test_large_sums_and_large_values():
    """Values whose sums pass fp16's range come out as infinities, as rounding makes them."""
    x = torch.full((3, 256), 200.0).half()
    w = ela.expert_quantize(torch.full((1, 16, 256), 7.0).half().cuda(), 64)
    for rows in (3, 400):
        y = ela.expert_linear_4bit(x[:1].expand(rows, -1).cuda(), w, offsets=torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
        assert y.isinf().all()
        assert not ela.expert_linear_4bit(x[:1].expand(rows, -1).cuda() / 100, w, offsets=torch.tensor([0, rows], dtype=torch.int32, device="cuda")).isinf().any()


def test_without_rows():
    w = ela.expert_quantize(random_weight(2, 8, 32, torch.bfloat16, 1).cuda(), 32)
    y = ela.expert_linear_4bit(torch.zeros(0, 32, dtype=torch.bfloat16, device="cuda"), w, offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert y.shape == (0, 8)


def layer(logits, x, w1, b1, w2, b2, bias):
    expert, weights = ela.expert_route(logits, 2, "sigmoid", bias, 4, 2, "top2", True, 1.5)
    plan = ela.expert_plan(expert, logits.shape[1])
    rows = ela.expert_dispatch(x, plan)
    h = ela.expert_linear_4bit(rows, w1, b1, activation="gelu", offsets=plan.offsets)
    return expert, ela.expert_combine(ela.expert_linear_4bit(h, w2, b2, offsets=plan.offsets), plan, weights)


def layer_case(T, dtype=torch.bfloat16, E=8, H=128, F=320):
    g = gen(T)
    w1, w2 = random_weight(E, F, H, dtype, 1).cuda(), random_weight(E, H, F, dtype, 2).cuda()
    return [torch.randn(T, E, generator=g).cuda(), torch.randn(T, H, generator=g).to(dtype).cuda(), ela.expert_quantize(w1, 32),
            (torch.randn(E, F, generator=g) * 0.2).to(dtype).cuda(), ela.expert_quantize(w2, 64), (torch.randn(E, H, generator=g) * 0.2).to(dtype).cuda(),
            (torch.randn(E, generator=g) * 0.1).cuda()]


@pytest.mark.parametrize("T", [1, 8, 300, 3000])
def test_routed_layer(T):
    """Route, plan, dispatch, two 4-bit products and combine, against the layer in 64 bits."""
    case = layer_case(T)
    logits, x, w1, b1, w2, b2, bias = case
    logits[T // 2, 1:] = -math.inf  # a token with one expert
    expert, out = layer(*case)
    s = torch.special.expit(logits.double())
    w = torch.where(expert >= 0, s.gather(1, expert.long().clamp(min=0)), torch.zeros((), dtype=torch.float64, device="cuda"))
    w = 1.5 * w / w.sum(1, keepdim=True)
    d1, d2 = ela.expert_dequantize(w1).double(), ela.expert_dequantize(w2).double()
    u = U[torch.bfloat16]
    ref, bound = torch.zeros(x.shape, dtype=torch.float64, device="cuda"), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for j in range(2):
        e = expert[:, j].long()
        for i in range(8):
            at = torch.nonzero(e == i).view(-1)
            if not len(at):
                continue
            z = x[at].double() @ d1[i].t() + b1[i].double()
            h = act64(z, "gelu")
            eh = u * h.abs() + 1.13 * 200 * 2.0 ** -22 * (x[at].double().abs() @ d1[i].abs().t() + b1[i].double().abs()) + 2.0 ** -20 * (1 + z.abs())
            y = h @ d2[i].t() + b2[i].double()
            ey = (eh @ d2[i].abs().t()) * 1.01 + 400 * 2.0 ** -22 * (h.abs() @ d2[i].abs().t() + b2[i].double().abs())
            ey = ey + 1.01 * u * (y.abs() + ey)
            ref[at] += w[at, j, None] * y
            bound[at] += w[at, j, None] * (ey + 2.0 ** -18 * y.abs())
    close(out, ref, bound * 1.01 + 1.01 * u * (ref.abs() + bound) + 2.0 ** -100)
    ela.expert_check()


def test_routed_layer_in_a_graph_and_on_two_streams():
    for T in (8, 900):
        case = layer_case(T)
        want = layer(*case)
        torch.cuda.synchronize()
        graphs, outs = [], []
        for _ in range(2):  # two graphs that share nothing but their inputs
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(layer(*case))
            graphs.append(graph)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        other = layer_case(T + 1)
        case[0].copy_(other[0][:T])
        case[1].copy_(other[1][:T])
        graphs[0].replay()
        want = layer(*case)
        assert all(torch.equal(a, b) for a, b in zip(outs[0], want))


def test_routed_layer_in_a_compiled_graph():
    case = layer_case(64)
    want = layer(*case)

    def flat(logits, x, p1, s1, b1, p2, s2, b2, bias):
        return layer(logits, x, ela.Expert4Bit(p1, s1, 128, 32), b1, ela.Expert4Bit(p2, s2, 320, 64), b2, bias)

    got = torch.compile(flat, backend="aot_eager", fullgraph=True)(case[0], case[1], case[2].packed, case[2].scales, case[3], case[4].packed, case[4].scales,
                                                                 case[5], case[6])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_router_trains_through_the_layer():
    """Gradients of the logits through combine and 16-bit experts, against differences of the 64-bit layer."""
    T, E, H = 40, 6, 64
    g = gen(21)
    logits, x = torch.randn(T, E, generator=g).cuda().requires_grad_(), torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    w = random_weight(E, H, H, torch.bfloat16, 3).cuda()
    dout = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    expert, weights = ela.expert_route(logits, 2)
    plan = ela.expert_plan(expert, E)
    y = ela.expert_linear(ela.expert_dispatch(x, plan), w, offsets=plan.offsets)
    (d,) = torch.autograd.grad(ela.expert_combine(y, plan, weights), logits, dout)
    rows = y.detach().double()[plan.position.long()]  # (T, 2, H)
    gain = (rows * dout.double()[:, None, :]).sum(2)
    l = logits.detach().double().requires_grad_()
    r = torch.softmax(l.gather(1, expert.long()), 1)
    (ref,) = torch.autograd.grad(r, l, gain)
    size = (rows.abs() * dout.double().abs()[:, None, :]).sum(2).amax(1, keepdim=True)
    assert ((d.double() - ref).abs() <= 2.0 ** -16 * size + 2.0 ** -18 * gain.abs().amax(1, keepdim=True)).all()


def test_refusals():
    w = torch.zeros(2, 16, 64, dtype=torch.bfloat16, device="cuda")
    q = ela.expert_quantize(w, 32)
    x, off = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda"), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for bad in (16, 48, 256, 0, -32):
        with pytest.raises(ValueError):
            ela.expert_quantize(w, bad)
        with pytest.raises(ValueError):
            ela.expert_dequantize(q._replace(group=bad))
    for bad in (w.float(), w.double(), w.int()):
        with pytest.raises(TypeError):
            ela.expert_quantize(bad)
    for bad in (w[0, 0], w[None], w[:0], w[:, :0], w[:, :, :0]):
        with pytest.raises(ValueError):
            ela.expert_quantize(bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        ela.expert_quantize(w.cpu())
    with pytest.raises(RuntimeError, match="CUDA"):
        ela.expert_linear_4bit(x.cpu(), q, offsets=off)

    def call(x=x, w=q, b=None, r=None, act="none", off=off):
        return ela.expert_linear_4bit(x, w, b, r, act, off)

    call()
    bf = dict(dtype=torch.bfloat16, device="cuda")
    for bad in (dict(x=x[:, :63]), dict(x=x[0]), dict(off=None), dict(off=off[:2]), dict(off=off.long()), dict(off=off.cpu()), dict(act="tanh"),
                dict(b=torch.zeros(16, **bf)), dict(b=torch.zeros(2, 15, **bf)), dict(r=torch.zeros(4, 15, **bf)), dict(r=torch.zeros(5, 16, **bf)),
                dict(w=q._replace(features=65)), dict(w=q._replace(features=0)), dict(w=q._replace(group=64)), dict(w=q._replace(scales=q.scales[:1])),
                dict(w=q._replace(packed=q.packed[:, :8])), dict(w=q._replace(group=100))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(x=x.half()), dict(x=x.float()), dict(b=torch.zeros(2, 16, device="cuda")), dict(r=torch.zeros(4, 16, device="cuda")),
                dict(w=q._replace(packed=q.packed.long())), dict(w=q._replace(scales=q.scales.float()))):
        with pytest.raises(TypeError):
            call(**bad)
    # gradients that would be lost
    for bad in (dict(x=x.clone().requires_grad_()), dict(b=torch.zeros(2, 16, requires_grad=True, **bf)), dict(r=torch.zeros(4, 16, requires_grad=True, **bf))):
        with pytest.raises(RuntimeError, match="no gradient"):
            call(**bad)
        with torch.no_grad():
            call(**bad)
    leaf = w.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ela.expert_quantize(leaf)
    with torch.no_grad():
        ela.expert_quantize(leaf)


def test_no_wait_gave_up():
    ela.expert_check()
