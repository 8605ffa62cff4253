"""The expert-layer operators as a user's program calls them, with their plain forms.

``dispatch``  tokens sorted by their expert: the plan (stable order, offsets,
              positions) and the rows gathered into that order.
``combine``   the experts' rows back to their tokens, weighted and summed.
``linear``    the product with each expert's weights; bias, activation and
              residual in the same pass (one weight matrix for all rows when
              the case has one expert).

A case with ``train`` also returns the gradients.  Token-to-expert choices
come from noisy router scores with a preference per expert (skewed loads), or
are balanced exactly, as an assignment of tokens to expert slots makes them
(``balanced``); a share ``left_out`` of the choices has expert -1, as rows
that an assignment leaves without a slot have.
"""
import math

import torch

own = False  # True: the framework's operators; False: their plain forms

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases

def _route(name, op, dtype, tokens, k, experts, hidden, train=False, balanced=False, left_out=0.0):
    return {"name": name, "op": op, "dtype": dtype, "tokens": tokens, "k": k, "experts": experts, "hidden": hidden,
            "train": train, "balanced": balanced, "left_out": left_out}


def _linear(name, dtype, rows, experts, n_in, n_out, activation, bias=True, residual=False, train=False,
            balanced=False, left_out=0.0):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "experts": experts, "in": n_in, "out": n_out,
            "activation": activation, "bias": bias, "residual": residual, "train": train, "balanced": balanced,
            "left_out": left_out}


def listed():
    return [
        # one step of 8 sequences that generate, two experts each: pure latency
        _route("dispatch step of 8", "dispatch", "bf16", 8, 2, 16, 1024),
        # a prompt of 4096 tokens over many small experts, 8 each: the write of eight copies
        _route("dispatch prompt 4096 x 8", "dispatch", "bf16", 4096, 8, 64, 4096, left_out=0.02),
        # training with an exactly balanced assignment, odd token count and width, 32-bit activations
        _route("dispatch train balanced", "dispatch", "fp32", 5003, 1, 128, 2050, train=True, balanced=True,
               left_out=0.05),
        # the way back of a step of 8 sequences
        _route("combine step of 8", "combine", "fp16", 8, 2, 16, 1024),
        # the way back of the prompt: the read of eight rows a token
        _route("combine prompt 4096 x 8", "combine", "bf16", 4096, 8, 64, 4096, left_out=0.02),
        # training, top-2: output, gradient of rows and of weights
        _route("combine train top-2", "combine", "bf16", 8192, 2, 32, 2048, train=True, left_out=0.01),
        # a generating step's product: 16 rows spread over 16 experts, the read of their weights
        _linear("linear step of 16 rows", "bf16", 16, 16, 1024, 4096, "gelu", balanced=True),
        # a short prompt, ragged in every size, with residual
        _linear("linear short ragged", "fp16", 1003, 8, 1032, 2056, "silu", residual=True, left_out=0.03),
        # a long prompt through large experts
        _linear("linear prompt 8192", "bf16", 8192, 8, 2048, 8192, "gelu"),
        # one weight matrix for all rows: a transformer's output projection with its residual
        _linear("linear one matrix 4096", "bf16", 4096, 1, 4096, 4096, "none", residual=True),
        # training of many small experts, loads balanced by an assignment
        _linear("linear train 64 experts", "bf16", 8192, 64, 1024, 1024, "relu", train=True, balanced=True),
        # training of large experts: the largest work here
        _linear("linear train 8 experts", "bf16", 16384, 8, 2048, 8192, "gelu", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature count: mostly a multiple of 8, one in six any number."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < 1 / 6 else max(8, v // 8 * 8)


def draw(rng):
    op = rng.choice(["dispatch", "combine", "linear", "linear"])
    balanced, left_out = rng.random() < 0.3, rng.choice([0.0, 0.0, 0.01, 0.1])
    train = rng.random() < 0.4
    experts = _log_int(rng, 1, 160)
    if op != "linear":
        k = rng.choice([1, 1, 2, 2, 3, 4, 6, 8])
        hidden = _width(rng, 64, 8192)
        most = min(16384, 4096 * 8 * 4096 // (k * hidden * (2 if train else 1)))
        tokens = _log_int(rng, 1, max(1, most))
        case = _route("", op, rng.choice(["bf16", "bf16", "fp16", "fp32"]), tokens, k, experts, hidden, train,
                      balanced, left_out)
    else:
        n_in, n_out = _width(rng, 64, 8192), _width(rng, 64, 8192)
        experts = max(1, min(experts, 8 * 2048 * 8192 // (n_in * n_out)))
        most = min(16384, 16384 * 2048 * 8192 // (n_in * n_out))
        case = _linear("", rng.choice(["bf16", "bf16", "fp16"]), _log_int(rng, 1, most), experts, n_in, n_out,
                       rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.7, rng.random() < 0.4, train,
                       balanced, left_out)
    del case["name"]
    return {key: v + 8 if type(v) is int and v == 3072 else v for key, v in case.items()}


# ---------------------------------------------------------------- inputs

def _choices(g, tokens, k, experts, balanced, left_out):
    """(tokens, k) int64 experts, -1 for the share left out."""
    if balanced:  # every expert equally often, in random order
        slots = torch.randperm(tokens * k, generator=g, device="cuda")
        expert = (slots % experts).view(tokens, k)
    else:
        score = torch.randn(experts, generator=g, device="cuda") * 0.7
        u = torch.rand(tokens, experts, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
        noisy = score - torch.log(-torch.log(u))
        expert = noisy.topk(min(k, experts), dim=1).indices
        expert = expert.repeat(1, -(-k // expert.shape[1]))[:, :k].contiguous()
    if left_out:
        gone = torch.rand(tokens, k, generator=g, device="cuda") < left_out
        expert = expert.masked_fill(gone, -1)
    return expert


def _sorted_plan(expert, experts):
    """offsets, position, source of a stable sort by expert, those of no expert last."""
    flat = expert.reshape(-1)
    bucket = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    source = torch.sort(bucket, stable=True).indices
    position = torch.empty_like(source)
    position[source] = torch.arange(source.numel(), device=source.device)
    counts = torch.bincount(bucket, minlength=experts + 1)[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return offsets.int(), position.view(expert.shape).int(), source.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    s = {"case": case}
    if case["op"] == "linear":
        R, E, K, N = case["rows"], case["experts"], case["in"], case["out"]
        expert = _choices(g, R, 1, E, case["balanced"], case["left_out"])
        s["offsets"] = _sorted_plan(expert, E)[0]
        s["x"] = randn(R, K)
        s["weight"] = randn(E, N, K, scale=K ** -0.5)
        s["bias"] = randn(E, N, scale=0.3) if case["bias"] else None
        s["residual"] = randn(R, N) if case["residual"] else None
        s["dy"] = randn(R, N) if case["train"] else None
        return s
    T, k, H = case["tokens"], case["k"], case["hidden"]
    s["expert"] = _choices(g, T, k, case["experts"], case["balanced"], case["left_out"])
    if case["op"] == "dispatch":
        s["x"] = randn(T, H)
        s["drows"] = randn(T * k, H) if case["train"] else None
    else:  # the plan is the one that the way there made
        s["offsets"], s["position"], s["source"] = _sorted_plan(s["expert"], case["experts"])
        s["y"] = randn(T * k, H)
        s["weights"] = torch.rand(T, k, generator=g, device="cuda").softmax(1) if k > 1 else \
            torch.rand(T, k, generator=g, device="cuda")
        s["dout"] = randn(T, H) if case["train"] else None
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_dispatch(s):
    import efficient_linear_assignment_b200 as ela
    plan = ela.expert_plan(s["expert"], s["case"]["experts"])
    if not s["case"]["train"]:
        return [plan.offsets, plan.position, plan.source, ela.expert_dispatch(s["x"], plan)]
    x = s["x"].detach().requires_grad_()
    rows = ela.expert_dispatch(x, plan)
    return [plan.offsets, plan.position, plan.source, rows.detach(), *torch.autograd.grad(rows, x, s["drows"])]


def _own_combine(s):
    import efficient_linear_assignment_b200 as ela
    plan = ela.ExpertPlan(s["offsets"], s["position"], s["source"])
    if not s["case"]["train"]:
        return [ela.expert_combine(s["y"], plan, s["weights"])]
    y, w = s["y"].detach().requires_grad_(), s["weights"].detach().requires_grad_()
    out = ela.expert_combine(y, plan, w)
    return [out.detach(), *torch.autograd.grad(out, (y, w), s["dout"])]


def _own_linear(s):
    import efficient_linear_assignment_b200 as ela
    keys = [n for n in ("x", "weight", "bias", "residual") if s[n] is not None]
    t = {n: s[n].detach().requires_grad_() if s["case"]["train"] else s[n] for n in keys}
    y = ela.expert_linear(t["x"], t["weight"], t.get("bias"), t.get("residual"), s["case"]["activation"],
                          s["offsets"])
    if not s["case"]["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [t[n] for n in keys], s["dy"])]


def _plain_dispatch(s):
    c = s["case"]
    x, k = s["x"], c["k"]
    offsets, position, source = _sorted_plan(s["expert"], c["experts"])
    valid = torch.arange(source.numel(), device=x.device) < offsets[-1]
    rows = x[(source // k).long()].masked_fill(~valid[:, None], 0)
    out = [offsets, position, source, rows]
    if c["train"]:
        taken = s["drows"].float()[position.long().view(-1)].view(c["tokens"], k, -1)
        taken = taken.masked_fill((position >= offsets[-1])[:, :, None], 0)
        out.append(taken.sum(1).to(x.dtype))
    return out


def _plain_combine(s):
    c = s["case"]
    T, k = c["tokens"], c["k"]
    at = s["position"].long().view(-1)
    gone = (s["position"] >= s["offsets"][-1])[:, :, None]
    taken = s["y"].float()[at].view(T, k, -1).masked_fill(gone, 0)
    out = [(taken * s["weights"].float()[:, :, None]).sum(1).to(s["y"].dtype)]
    if c["train"]:
        d = s["dout"].float()[:, None, :]
        dy = torch.empty_like(s["y"])
        dy[at] = (d * s["weights"].float()[:, :, None]).masked_fill(gone, 0).to(dy.dtype).view(T * k, -1)
        out += [dy, (taken * d).sum(2).to(s["weights"].dtype)]
    return out


def _plain_linear(s):
    c = s["case"]
    x, E = s["x"], c["experts"]
    R, N = c["rows"], c["out"]
    offsets = s["offsets"].long()
    r = torch.arange(R, device=x.device)
    e = torch.bucketize(r, offsets[1:], right=True)  # expert of a row; E: none
    most = max(1, int((offsets[1:] - offsets[:-1]).max()))
    mine = torch.nonzero(e < E).view(-1)
    at = e[mine] * most + mine - offsets[e[mine]]  # rows padded to the largest expert's
    w = s["weight"].float()

    def pad(v):
        p = torch.zeros(E * most, v.shape[1], device=x.device)
        p[at] = v[mine].float()
        return p.view(E, most, -1)

    xp = pad(x)
    z = torch.matmul(xp, w.transpose(1, 2))
    if s["bias"] is not None:
        z = z + s["bias"].float()[:, None, :]
    act = c["activation"]
    if act == "none":
        a = z
    elif act == "relu":
        a = z.clamp(min=0)
    elif act == "gelu":
        a = 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    else:
        a = z / (1 + torch.exp(-z))
    y = s["residual"].float() if s["residual"] is not None else torch.zeros(R, N, device=x.device)
    y = y.index_add(0, mine, a.reshape(E * most, N)[at])
    out = [y.to(x.dtype)]
    if c["train"]:
        dz = pad(s["dy"])
        if act == "relu":
            dz = dz * (z > 0)
        elif act == "gelu":
            dz = dz * (0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5)
        elif act == "silu":
            q = 1 / (1 + torch.exp(-z))
            dz = dz * q * (1 + z * (1 - q))
        dx = torch.zeros_like(x)
        dx[mine] = torch.matmul(dz, w).view(E * most, -1)[at].to(x.dtype)
        out += [dx, torch.matmul(dz.transpose(1, 2), xp).to(x.dtype)]
        if s["bias"] is not None:
            out.append(dz.sum(1).to(x.dtype))
        if s["residual"] is not None:
            out.append(s["dy"])
    return out


_own = {"dispatch": _own_dispatch, "combine": _own_combine, "linear": _own_linear}
_plain = {"dispatch": _plain_dispatch, "combine": _plain_combine, "linear": _plain_linear}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definitions, expert by expert and choice by choice, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(case, s)
    T, k, E, H = case["tokens"], case["k"], case["experts"], case["hidden"]
    ids = s["expert"].cpu().view(-1)
    lists = [torch.nonzero(ids == e).view(-1) for e in range(E)]
    kept = torch.cat(lists)
    source = torch.cat([kept, torch.nonzero((ids < 0) | (ids >= E)).view(-1)])
    V = kept.numel()
    position = torch.empty(T * k, dtype=torch.int64)
    position[source] = torch.arange(T * k)
    offsets = torch.tensor([0] + [len(v) for v in lists]).cumsum(0)
    at, kept = position.cuda().view(T, k), kept.cuda()
    if case["op"] == "dispatch":
        rows = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
        rows[:V] = s["x"].double()[kept // k]
        out = [offsets.int(), position.view(T, k).int(), source.int(), rows]
        if case["train"]:
            dx = torch.zeros(T, H, dtype=torch.float64, device="cuda")
            for j in range(k):
                has = at[:, j] < V
                dx[has] += s["drows"][at[has, j]].double()
            out.append(dx)
        return out
    w = s["weights"].double()
    res = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    dy = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
    dw = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        has = at[:, j] < V
        y = s["y"][at[has, j]].double()
        res[has] += w[has, j, None] * y
        if case["train"]:
            d = s["dout"][has].double()
            dy[at[has, j]] = w[has, j, None] * d
            dw[has, j] = (d * y).sum(1)
    return [res, dy, dw] if case["train"] else [res]


def _exact_linear(case, s):
    E, act = case["experts"], case["activation"]
    off = s["offsets"].tolist()
    x = s["x"].double()
    y = s["residual"].double().clone() if case["residual"] else torch.zeros(case["rows"], case["out"],
                                                                           dtype=torch.float64, device="cuda")
    dx = torch.zeros_like(x)
    dw = torch.zeros(s["weight"].shape, dtype=torch.float64, device="cuda") if case["train"] else None
    db = torch.zeros(E, case["out"], dtype=torch.float64, device="cuda")
    for e in range(E):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        w = s["weight"][e].double()
        z = x[a:b] @ w.t()
        if case["bias"]:
            z += s["bias"][e].double()
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        sig = torch.special.expit(z)
        one = torch.ones_like(z)
        value, slope = {"none": (z, one), "relu": (torch.where(z > 0, z, 0 * z), (z > 0).double()),
                        "gelu": (z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)),
                        "silu": (z * sig, sig + z * sig * (1 - sig))}[act]
        y[a:b] += value
        if case["train"]:
            dz = s["dy"][a:b].double() * slope
            dx[a:b] = dz @ w
            dw[e] = dz.t() @ x[a:b]
            db[e] = dz.sum(0)
    if not case["train"]:
        return [y]
    return [y, dx, dw] + ([db] if case["bias"] else []) + ([s["dy"].double()] if case["residual"] else [])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "linear":
        R, E, K, N = case["rows"], case["experts"], case["in"], case["out"]
        V = R * (1 - case["left_out"])  # rows that have an expert, and the experts that have a row:
        used = min(E, V) if case["balanced"] else E * (1 - (1 - 1 / E) ** V)
        b = size * (V * K + used * N * K + R * N * (2 if case["residual"] else 1)) + 4 * (E + 1)
        b += size * used * N if case["bias"] else 0
        if case["train"]:  # dy in; dx, the weights' and the bias's gradient out
            b += size * (V * N + R * K + E * N * K + (E * N if case["bias"] else 0))
        return {"bytes": b, "flops": 2 * V * N * K * (3 if case["train"] else 1)}
    T, k, H = case["tokens"], case["k"], case["hidden"]
    there = size * (T + T * k) * H
    if case["op"] == "dispatch":
        ids = T * k * (8 + 4 + 4) + 4 * (case["experts"] + 1)
        return {"bytes": there * (2 if case["train"] else 1) + ids, "flops": T * k * H if case["train"] else 0}
    b = there + T * k * (4 + 4) + 4
    if case["train"]:  # the gradient in, the rows' and the weights' out
        b += size * (T + T * k) * H + 4 * T * k
    return {"bytes": b, "flops": T * k * H * (5 if case["train"] else 2)}
