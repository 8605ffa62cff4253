"""GPU tests of the expert-layer operators where ordinary data does not lead:
signs next to 0, the ends of fp16's range, sizes at a limit, derivatives that
are not there."""
import os
import subprocess
import sys

import pytest
import torch

import efficient_linear_assignment_b200 as ela

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def slopes_of(x, w, b, counts, act):
    """act'(z) of every row and feature, as the operator rounds it: the rows get a
    column each that no weight reads, dy is 1, and dW's entry there is that row's dz."""
    R, E = x.shape[0], len(counts)
    tag = torch.eye(R, dtype=x.dtype)
    xt = torch.cat([x, tag], 1).cuda()
    wt = torch.cat([w, torch.zeros(*w.shape[:2], R, dtype=w.dtype)], 2).cuda().requires_grad_()
    off = torch.tensor([0] + list(counts)).cumsum(0)
    y = ela.expert_linear(xt, wt, None if b is None else b.cuda(), None, act, off.int().cuda())
    (dw,) = torch.autograd.grad(y, wt, torch.ones_like(y))
    e = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    return dw.cpu()[e, :, x.shape[1] + torch.arange(R)]


def exact_z(x, w, b, counts):
    out = []
    for e, part in enumerate(x.split(list(counts))):
        out.append(part.double() @ w[e].double().t() + (0 if b is None else b[e].double()))
    return torch.cat(out)


def cancelling(counts, half, N, dtype, every, seed, bias=False):
    """Every so-and-so-many-th feature's sum is the two halves of K against each other plus one
    product of size 2^-23 to 2^-16 (with a bias: a sum that the bias takes away but for its
    rounding): z is next to 0 with a sign that the order of an fp32 sum would decide."""
    g = gen(seed)
    R, E = sum(counts), len(counts)
    p = torch.randn(R, half, generator=g)
    sign = torch.randint(0, 2, (R, 1), generator=g) * 2.0 - 1
    x = torch.cat([p, p, sign * 2.0 ** -6], 1).to(dtype)
    w = (torch.randn(E, N, 2 * half + 1, generator=g) * half ** -0.5).to(dtype)
    w[:, ::every, half:2 * half] = -w[:, ::every, :half]
    w[:, ::every, 2 * half] = (torch.exp2(-torch.randint(10, 18, (E, w[:, ::every].shape[1]), generator=g).float())).to(dtype)
    b = None
    if bias:
        b = torch.randn(E, N, generator=g).to(dtype)
        # feature 1's sum: x's first column is 1, its weight there the bias's opposite
        x[:, 0] = 1
        x[:, half] = 1
        w[:, ::every, 0] = -b[:, ::every]
        w[:, ::every, half] = 0
    return x, w, b


# ---------------------------------------------------------------- ReLU's slope next to 0

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("counts,half,N,every", [([100, 87, 63], 96, 136, 8), ([300], 500, 264, 32), ([70, 66, 65], 40, 520, 4),
                                                 ([17] * 40, 64, 72, 8)])
def test_relu_slope_next_to_zero(counts, half, N, every, bias, dtype):
    """The slope is the sign of the 64-bit sum, in every row, the last of an expert's too."""
    x, w, b = cancelling(counts, half, N, dtype, every, 5 * half + N, bias)
    z = exact_z(x, w, b, counts)
    near = z.abs() < 2.0 ** -15
    assert near.float().mean() > 0.5 / every and (z[near] != 0).all()
    got = slopes_of(x, w, b, counts, "relu")
    assert torch.equal(got.double(), (z > 0).double())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("counts,half,N,every", [([1, 0, 2, 1], 96, 64, 8), ([9, 8, 20, 3], 250, 48, 8), ([4, 1], 33, 136, 16),
                                                 ([40], 500, 96, 32)])
def test_relu_slope_next_to_zero_few_rows(counts, half, N, every, bias, dtype):
    x, w, b = cancelling(counts, half, N, dtype, every, 7 * half + N, bias)
    z = exact_z(x, w, b, counts)
    assert (z.abs() < 2.0 ** -15).any()
    assert torch.equal(slopes_of(x, w, b, counts, "relu").double(), (z > 0).double())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[300, 61, 0, 150], [9, 1, 0, 5]])
@pytest.mark.parametrize("kind", ["rows", "features", "blocks", "signs", "mixed"])
def test_relu_slope_of_sums_that_are_zero(kind, counts, dtype):
    """Sums of nothing but zeros, and of whole numbers that cancel, are 0 and have slope 0; what
    is next to them, and next to 0, has its sign."""
    g = gen(21)
    x, w, b = cancelling(counts, 130, 72, dtype, 24, 22)
    if kind == "rows":
        x[::3] = 0
    elif kind == "features":
        w[:, 1::5] = 0
    elif kind == "blocks":
        x *= (torch.rand(x.shape[0], 9, generator=g) < 0.3).to(dtype).repeat_interleave(29, 1)[:, :261]
        w *= (torch.rand(*w.shape[:2], 9, generator=g) < 0.3).to(dtype).repeat_interleave(29, 2)[:, :, :261]
    elif kind == "signs":
        x, w = x.sign(), w.sign()
        x[:, -1] = 0  # (an even number of terms)
    else:
        x[::7] = 0
        w[:, 2::9] = 0
        b = torch.randn(w.shape[:2], generator=g).to(dtype)
        b[:, ::2] = 0
    z = exact_z(x, w, b, counts)
    assert (z == 0).any()
    assert torch.equal(slopes_of(x, w, b, counts, "relu").double(), (z > 0).double())


@pytest.mark.parametrize("K,N", [(67, 1), (130, 3), (96, 7), (101, 33), (264, 131)])
@pytest.mark.parametrize("rows", [5, 230])
def test_relu_slope_next_to_zero_odd_sizes(rows, K, N):
    """Operands off 16 bytes, features stored one by one, and too few of them to fill a warp."""
    x, w, b = cancelling([rows], K // 2, N, torch.bfloat16, 4, K + N)
    if N < 4:  # (a feature next to 0 needs one beside it that is not)
        w[:, :1] = torch.randn(w[:, :1].shape, generator=gen(K)).to(w.dtype)
    z = exact_z(x, w, b, [rows])
    assert torch.equal(slopes_of(x, w, b, [rows], "relu").double(), (z > 0).double())


@pytest.mark.parametrize("R,E,K,N", [(8192, 4, 512, 2048), (4096, 1, 2048, 4096)])
def test_relu_signs_of_ordinary_values(R, E, K, N):
    """Tens of millions of sums of normal values: every sign is that of the 64-bit sum."""
    g = torch.Generator(device="cuda").manual_seed(R)
    x = torch.randn(R, K, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(E, N, K, generator=g, device="cuda") * K ** -0.5).to(torch.bfloat16)
    b = (torch.randn(E, N, generator=g, device="cuda") * 0.3).to(torch.bfloat16)
    off = torch.arange(E + 1, device="cuda", dtype=torch.int32) * (R // E)
    _, z = torch.ops.ela_native.expert_linear_z(x, w, b, None, off, 1, True)
    for e in range(E):
        a, c = e * (R // E), (e + 1) * (R // E)
        want = x[a:c].double() @ w[e].double().t() + b[e].double()
        assert torch.equal(z[a:c] > 0, want > 0)


def test_relu_gradients_same_bits():
    """More sums next to 0 than any CTA could list, the same gradients every time."""
    counts = [700, 801, 523]
    x, w, b = cancelling(counts, 120, 512, torch.bfloat16, 4, 3)
    off = torch.tensor([0] + counts).cumsum(0).int().cuda()
    leaf = [v.cuda().requires_grad_() for v in (x, w)]
    dy = torch.randn(sum(counts), 512, generator=gen(4)).to(torch.bfloat16).cuda()
    first = None
    for _ in range(20):
        y = ela.expert_linear(*leaf, None, None, "relu", off)
        grads = torch.autograd.grad(y, leaf, dy)
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(first, grads))


# ---------------------------------------------------------------- fp16's range

@pytest.mark.parametrize("rows", [3, 300])
def test_relu_slope_below_fp16(rows):
    """A sum too small for fp16 still has its sign."""
    g = gen(8)
    x = torch.randn(rows, 64, generator=g).half()
    w = torch.randn(1, 40, 64, generator=g).half()
    w[0, ::4] = 0
    x[:, 0] = 2.0 ** -12 * (torch.randint(0, 2, (rows,), generator=g) * 2 - 1)
    w[0, ::4, 0] = 2.0 ** -14
    z = exact_z(x, w, None, [rows])
    assert (z[:, ::4].abs() == 2.0 ** -26).all()
    assert torch.equal(slopes_of(x, w, None, [rows], "relu").double(), (z > 0).double())


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows", [3, 300])
def test_gradients_past_fp16_are_finite(rows, act):
    """z beyond +-65504: the slope there is 0 or 1, as the forward pass's value says."""
    g = gen(9)
    x = torch.randn(rows, 64, generator=g).half()
    w = (torch.randn(1, 48, 64, generator=g) * 0.125).half()
    w[0, 5] = 0
    w[0, 5, 3] = 300.0
    x[:, 3] = torch.where(torch.arange(rows) % 2 == 0, 300.0, -300.0)  # z = +-90000
    w[0, :5, 3] = w[0, 6:, 3] = 0
    z = exact_z(x, w, None, [rows])
    assert z[:, 5].abs().min() > 65504
    got = slopes_of(x, w, None, [rows], act)
    assert torch.isfinite(got).all()
    assert torch.equal(got[:, 5].double(), (z[:, 5] > 0).double())
    leaf = [v.cuda().requires_grad_() for v in (x, w)]
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    y = ela.expert_linear(*leaf, None, None, act, off)
    dy = torch.ones_like(y)
    dy[:, 5] = 2.0 ** -10  # (dx holds 300 * dy)
    for grad in torch.autograd.grad(y, leaf, dy):
        assert torch.isfinite(grad).all()


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[3, 0, 4], [300, 301]])
def test_slope_of_unrounded_z(counts, dtype, act):
    """dz = dy * act'(z) is off by its own rounding, u |dz|, and not by the rounding of z, which
    would be up to 0.8 u |z| (a sum's own error, 66 * 2^-22 of its terms, and the fast
    exponential's 2^-20 besides)."""
    g = gen(10)
    x = torch.randn(sum(counts), 64, generator=g).to(dtype)
    w = (torch.randn(len(counts), 40, 64, generator=g) * 0.3).to(dtype)
    z = exact_z(x, w, None, counts)
    if act == "gelu":
        ref = torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    else:
        ref = torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))
    terms = exact_z(x.abs(), w.abs(), None, counts)
    bound = 1.01 * U[dtype] * ref.abs() + 0.8 * 66 * 2.0 ** -22 * terms + 2.0 ** -20 * (1 + z.abs())
    if dtype == torch.float16:
        bound += 2.0 ** -24
    off = (slopes_of(x, w, None, counts, act).double() - ref).abs()
    assert (off <= bound).all(), (off - bound).max()


# ---------------------------------------------------------------- the plan's limits

def test_plan_at_the_default_shared_memory():
    """Counts that take 48 KB of shared memory but for the kernel's own, as the first plans of a
    process (a larger one before them would have asked the driver for more)."""
    code = """
import torch, efficient_linear_assignment_b200 as ela
for E, T in ((371, 2000), (720, 1000), (1363, 400), (2455, 200), (3070, 100), (4095, 100)):
    for dtype in (torch.int32, torch.int64):
        e = torch.randint(-1, E, (T,), generator=torch.Generator().manual_seed(1)).to(dtype)
        p = ela.expert_plan(e.cuda(), E)
        want = torch.sort(torch.where(e < 0, E, e), stable=True).indices
        assert torch.equal(p.source.cpu().long(), want)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_plan_of_the_most_choices():
    """2^31 - 1 choices: the last step of a warp's range is inside the buffers and the plan right."""
    n = 2 ** 31 - 1
    e = torch.zeros(n, dtype=torch.int32, device="cuda")
    e[0] = 1
    e[-5:] = 1
    plan = ela.expert_plan(e, 2)
    del e
    assert plan.offsets.tolist() == [0, n - 6, n]
    pos = plan.position.view(-1)
    assert pos[0].item() == n - 6 and pos[-5:].tolist() == list(range(n - 5, n))
    assert plan.source[n - 6:].tolist() == [0] + list(range(n - 5, n))
    for a in (1, n // 3, n - 2 ** 26 - 5):
        want = torch.arange(a, a + 2 ** 26, device="cuda", dtype=torch.int32)
        assert torch.equal(pos[a:a + 2 ** 26], want - 1) and torch.equal(plan.source[a - 1:a - 1 + 2 ** 26], want)
    del plan, pos, want
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- derivatives that are not there

def layer_parts():
    bf = torch.bfloat16
    plan = ela.expert_plan(torch.tensor([[0], [1], [1], [-1]], device="cuda"), 2)
    x, w = torch.randn(4, 8, device="cuda").to(bf), torch.randn(2, 16, 8, device="cuda").to(bf)
    g = torch.rand(4, 1, device="cuda")
    return [(lambda v: ela.expert_dispatch(v, plan), x), (lambda v: ela.expert_combine(v, plan, g), x),
            (lambda v: ela.expert_combine(x, plan, v), g), (lambda v: ela.expert_linear(v, w, offsets=plan.offsets), x),
            (lambda v: ela.expert_linear(x, v, offsets=plan.offsets), w),
            (lambda v: ela.expert_linear(x, w, v, offsets=plan.offsets), w[:, :, 0].contiguous())]


def test_forward_mode_is_refused():
    """A tangent is not dropped: forward-mode derivatives raise."""
    import torch.autograd.forward_ad as fwd
    for f, v in layer_parts():
        for needs in (False, True):
            with fwd.dual_level():
                dual = fwd.make_dual(v.clone().requires_grad_(needs), torch.ones_like(v))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    f(dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(f, (v,), (torch.ones_like(v),))
        f(v)  # (and nothing else does)


def test_compiled_gradient_of_gates_without_a_second_dimension():
    g = gen(12)
    expert = torch.randint(-1, 4, (50,), generator=g).cuda()
    plan = ela.expert_plan(expert, 4)
    leaves = [torch.randn(50, 16, generator=g).cuda().requires_grad_(), torch.rand(50, generator=g).cuda().requires_grad_()]

    def f(y, w):
        return ela.expert_combine(y, plan, w) * 2

    want, got = f(*leaves), torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(want, got)
    for a, b in zip(torch.autograd.grad(want, leaves, torch.ones_like(want)), torch.autograd.grad(got, leaves, torch.ones_like(got))):
        assert a.shape == b.shape and torch.equal(a, b)
