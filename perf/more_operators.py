"""Routing and 4-bit experts, as a user's program calls them, with their plain forms.

``route``     a router's logits to the k experts of each token and their
              weights: softmax or sigmoid scores, a bias that balances the
              choice, groups of experts, weights that sum to ``scale``.  A case
              with ``train`` also returns the gradient of the logits.
``quantize``  experts' weights to 4 bits with a scale per group of inputs, and
              the weights that these stand for.
``linear``    the product with each expert's 4-bit weights; bias, activation
              and residual in the same pass (one matrix for all rows when the
              case has one expert).

A logit of -inf takes an expert away from a token (``masked``), and all of a
padding token's are (``padding``): it has expert -1 and weight 0 wherever no
expert is left.  Rows come in expert order with the offsets that a plan gives;
a share ``left_out`` of them has no expert.
"""
import math

import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain forms

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases

def _route(name, dtype, tokens, experts, k, score, bias=False, groups=1, kept=1, group_score="max", renormalize=True,
           scale=1.0, train=False, masked=0.0, padding=0.0):
    return {"name": name, "op": "route", "dtype": dtype, "tokens": tokens, "experts": experts, "k": k, "score": score,
            "bias": bias, "groups": groups, "kept": kept, "group_score": group_score, "renormalize": renormalize,
            "scale": scale, "train": train, "masked": masked, "padding": padding}


def _quantize(name, dtype, experts, n_in, n_out, group):
    return {"name": name, "op": "quantize", "dtype": dtype, "experts": experts, "in": n_in, "out": n_out, "group": group}


def _linear(name, dtype, rows, experts, n_in, n_out, group, activation, bias=True, residual=False, balanced=False,
            left_out=0.0):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "experts": experts, "in": n_in, "out": n_out,
            "group": group, "activation": activation, "bias": bias, "residual": residual, "balanced": balanced,
            "left_out": left_out}


def listed():
    return [
        # one step of 8 sequences that generate: pure latency
        _route("route step of 8", "bf16", 8, 16, 2, "softmax"),
        # a long prompt over many small experts: balanced by a bias, half of the groups, padding at its end
        _route("route prompt 8192 x 256", "fp32", 8192, 256, 8, "sigmoid", bias=True, groups=8, kept=4,
               group_score="top2", scale=2.5, padding=0.02),
        # training, top-2 of few experts, weights as the softmax gives them: the gradient is dense
        _route("route train 32768 x 32", "bf16", 32768, 32, 2, "softmax", renormalize=False, train=True),
        # training, odd sizes, some experts closed to some tokens
        _route("route train 5003 x 120", "fp16", 5003, 120, 6, "softmax", bias=True, train=True, masked=0.1),
        # a checkpoint's experts brought to 4 bits
        _quantize("quantize 16 experts", "bf16", 16, 1024, 4096, 32),
        # one matrix of odd sizes
        _quantize("quantize odd matrix", "fp16", 1, 1027, 2051, 64),
        # one token through one matrix: the read of its weights, mostly latency
        _linear("linear single token", "bf16", 1, 1, 4096, 4096, 128, "none", bias=False, residual=True),
        # a generating step's product: 16 rows spread over 16 experts
        _linear("linear step of 16 rows", "bf16", 16, 16, 1024, 4096, 32, "gelu", balanced=True),
        # a batch of sequences that generate: 256 rows over 16 experts, the read of their weights still counts
        _linear("linear step of 256 rows", "bf16", 256, 16, 2048, 4096, 64, "silu"),
        # a short prompt, ragged in every size, with residual
        _linear("linear short ragged", "fp16", 1003, 8, 1032, 2056, 64, "silu", residual=True, left_out=0.03),
        # a long prompt through large experts: the largest work here
        _linear("linear prompt 8192", "bf16", 8192, 8, 2048, 8192, 64, "gelu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature count: mostly a multiple of 8, one in six any number."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < 1 / 6 else max(8, v // 8 * 8)


def draw(rng):
    op = rng.choice(["route", "route", "quantize", "linear", "linear"])
    if op == "route":
        experts = _log_int(rng, 2, 512)
        if rng.random() < 0.6:
            experts = max(8, experts // 8 * 8)
        parts = [g for g in range(2, 33) if experts % g == 0 and experts // g >= 2]
        groups, kept, group_score = 1, 1, "max"
        if parts and rng.random() < 0.5:
            groups = rng.choice(parts)
            kept, group_score = rng.randint(1, groups), rng.choice(["max", "top2"])
        k = min(rng.choice([1, 2, 2, 3, 4, 6, 8, 8, 16]), kept * (experts // groups))
        tokens = _log_int(rng, 1, min(32768, 8192 * 256 // experts))
        case = _route("", rng.choice(["fp32", "fp32", "bf16", "fp16"]), tokens, experts, k,
                      rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, kept, group_score,
                      rng.random() < 0.6, rng.choice([1.0, 1.0, 2.5]), rng.random() < 0.5,
                      rng.choice([0.0, 0.0, 0.1, 0.5]), rng.choice([0.0, 0.05]))
    else:
        n_in, n_out = _width(rng, 32, 8192), _width(rng, 16, 8192)
        experts = max(1, min(_log_int(rng, 1, 64), 4 * 2048 * 8192 // (n_in * n_out)))
        dtype, group = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([32, 64, 128])
        if op == "quantize":
            case = _quantize("", dtype, experts, n_in, n_out, group)
        else:
            most = min(8192, 8192 * 2048 * 8192 // (n_in * n_out))
            case = _linear("", dtype, _log_int(rng, 1, most), experts, n_in, n_out, group,
                           rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.7, rng.random() < 0.4,
                           rng.random() < 0.3, rng.choice([0.0, 0.0, 0.01, 0.1]))
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs

def _offsets(g, rows, experts, balanced, left_out):
    """int32 (E+1,): the experts' rows in order, skewed loads or equal ones, the rest left out."""
    if balanced:
        e = torch.arange(rows, device="cuda") % experts
    else:
        share = (torch.randn(experts, generator=g, device="cuda") * 0.7).softmax(0)
        e = torch.multinomial(share, rows, replacement=True, generator=g)
    if left_out:
        e = e[torch.rand(rows, generator=g, device="cuda") >= left_out]
    counts = torch.bincount(e, minlength=experts)
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()


def _rounded(weight, group):
    """(E, N, K) weights to whole numbers -8..7 and a scale per group of inputs, (E, groups, N)."""
    E, N, K = weight.shape
    parts = -(-K // group)
    w = torch.zeros(E, N, parts * group, dtype=weight.dtype, device=weight.device)
    w[:, :, :K] = weight
    w = w.view(E, N, parts, group).float()
    scale = (w.abs().amax(3) / 7).to(weight.dtype)
    q = (w / scale.float()[..., None]).nan_to_num(0.0).round().clamp(-8, 7)
    return q.view(E, N, -1)[:, :, :K].to(torch.int8), scale.transpose(1, 2).contiguous()


def _weights_of(q, scale, group):
    """The weights that they stand for, rounded to the scales' type."""
    s = scale.transpose(1, 2).float().repeat_interleave(group, 2)[:, :, :q.shape[2]]
    return (q.float() * s).to(scale.dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    s = {"case": case}
    if case["op"] == "route":
        T, E = case["tokens"], case["experts"]
        liked = torch.randn(E, generator=g, device="cuda") * 0.7
        logits = torch.randn(T, E, generator=g, device="cuda") * 1.5 + liked
        if case["masked"]:
            gone = torch.rand(T, E, generator=g, device="cuda") < case["masked"]
            logits = logits.masked_fill(gone, float("-inf"))
        if case["padding"]:
            logits[T - int(T * case["padding"]):] = float("-inf")
        s["logits"] = logits.to(dt)
        # the balancing bias works against what is liked, in the scores' size
        size = 0.1 if case["score"] == "sigmoid" else 0.3 / E
        s["bias"] = (torch.randn(E, generator=g, device="cuda") * 0.3 - liked) * size if case["bias"] else None
        s["dweights"] = torch.randn(T, case["k"], generator=g, device="cuda") if case["train"] else None
        return s
    E, K, N = case["experts"], case["in"], case["out"]
    weight = randn(E, N, K, scale=K ** -0.5)
    if case["op"] == "quantize":
        s["weight"] = weight
        return s
    R = case["rows"]
    s["offsets"] = _offsets(g, R, E, case["balanced"], case["left_out"])
    s["x"] = randn(R, K)
    s["bias"] = randn(E, N, scale=0.3) if case["bias"] else None
    s["residual"] = randn(R, N) if case["residual"] else None
    if own:  # quantized once, when the model is loaded
        import efficient_linear_assignment_b200 as ela
        s["weight"] = ela.expert_quantize(weight, case["group"])
    else:
        s["q"], s["scale"] = _rounded(weight, case["group"])
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_route(s):
    import efficient_linear_assignment_b200 as ela
    c = s["case"]
    logits = s["logits"].detach().requires_grad_() if c["train"] else s["logits"]
    expert, weights = ela.expert_route(logits, c["k"], c["score"], s["bias"], c["groups"], c["kept"], c["group_score"],
                                       c["renormalize"], c["scale"])
    if not c["train"]:
        return [expert, weights]
    return [expert, weights.detach(), *torch.autograd.grad(weights, logits, s["dweights"])]


def _own_quantize(s):
    import efficient_linear_assignment_b200 as ela
    packed = ela.expert_quantize(s["weight"], s["case"]["group"])
    return [packed.scales, ela.expert_dequantize(packed)]


def _own_linear(s):
    import efficient_linear_assignment_b200 as ela
    return [ela.expert_linear_4bit(s["x"], s["weight"], s["bias"], s["residual"], s["case"]["activation"], s["offsets"])]


def _plain_route(s):
    c = s["case"]
    T, E, k, G = c["tokens"], c["experts"], c["k"], c["groups"]
    lowest = float("-inf")
    there = s["logits"] != lowest
    none = ~there.any(1, keepdim=True)
    # the choice, in 64 bits: next to a border 32 do not tell
    l64 = s["logits"].double()
    e64 = torch.exp(l64 - l64.amax(1, keepdim=True).masked_fill(none, 0.0))
    score = e64 / e64.sum(1, keepdim=True).masked_fill(none, 1.0) if c["score"] == "softmax" else 1 / (1 + torch.exp(-l64))
    if s["bias"] is not None:
        score = score + s["bias"].double()
    score = score.masked_fill(~there, lowest)
    key = l64 if s["bias"] is None else score
    if G > 1:
        best = (key if c["group_score"] == "max" else score).view(T, G, E // G).topk(1 if c["group_score"] == "max" else 2, 2)
        rank = torch.sort(best.values.sum(2), dim=1, descending=True, stable=True).indices
        out = torch.ones(T, G, dtype=torch.bool, device=key.device).scatter_(1, rank[:, :c["kept"]], False)
        key = key.masked_fill(out.repeat_interleave(E // G, 1), lowest)
    key, expert = torch.sort(key, dim=1, descending=True, stable=True)
    gone = key[:, :k] == lowest
    at = expert[:, :k]
    # their weights, and the gradient of the logits
    l = s["logits"].float()
    mine = l.gather(1, at).masked_fill(gone, lowest)
    empty = gone.all(1, keepdim=True)
    if c["score"] == "softmax":
        p = torch.exp(l - l.amax(1, keepdim=True).masked_fill(none, 0.0))
        p = p / p.sum(1, keepdim=True).masked_fill(none, 1.0)
        r = torch.exp(mine - mine.amax(1, keepdim=True).masked_fill(empty, 0.0))
    else:
        p = 1 / (1 + torch.exp(-l))
        low = mine.clamp(max=0)
        r = torch.exp(low - low.amax(1, keepdim=True).masked_fill(empty, 0.0)) / (1 + torch.exp(-mine.abs()))
    chosen = p.gather(1, at).masked_fill(gone, 0.0)
    r = r / r.sum(1, keepdim=True).masked_fill(empty, 1.0) if c["renormalize"] else chosen
    out = [at.masked_fill(gone, -1).int(), c["scale"] * r]
    if c["train"]:
        g = c["scale"] * s["dweights"].masked_fill(gone, 0.0)
        d = torch.zeros_like(l)
        if c["renormalize"]:
            mean = (g * r).sum(1, keepdim=True)
            slope = r * (g - mean) if c["score"] == "softmax" else r * (g - mean) / (1 + torch.exp(mine))
            d.scatter_add_(1, at, slope.masked_fill(gone, 0.0))
        elif c["score"] == "softmax":
            d = p * (d.scatter_add_(1, at, g) - (g * chosen).sum(1, keepdim=True))
        else:
            d.scatter_add_(1, at, (g * chosen / (1 + torch.exp(mine))).masked_fill(gone, 0.0))
        out.append(d.to(s["logits"].dtype))
    return out


def _plain_quantize(s):
    q, scale = _rounded(s["weight"], s["case"]["group"])
    return [scale, _weights_of(q, scale, s["case"]["group"])]


def _plain_linear(s):
    c = s["case"]
    x, E, R, N = s["x"], c["experts"], c["rows"], c["out"]
    offsets = s["offsets"].long()
    r = torch.arange(R, device=x.device)
    e = torch.bucketize(r, offsets[1:], right=True)  # expert of a row; E: none
    most = max(1, int((offsets[1:] - offsets[:-1]).max()))
    mine = torch.nonzero(e < E).view(-1)
    at = e[mine] * most + mine - offsets[e[mine]]  # rows padded to the largest expert's
    xp = torch.zeros(E * most, c["in"], device=x.device)
    xp[at] = x[mine].float()
    z = torch.matmul(xp.view(E, most, -1), _weights_of(s["q"], s["scale"], c["group"]).float().transpose(1, 2))
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
    return [y.index_add(0, mine, a.reshape(E * most, N)[at]).to(x.dtype)]


_own = {"route": _own_route, "quantize": _own_quantize, "linear": _own_linear}
_plain = {"route": _plain_route, "quantize": _plain_quantize, "linear": _plain_linear}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definitions in 64 bits, token by token or expert by expert where that is quick enough."""
    global own
    here, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = here
    return {"route": _exact_route, "quantize": _exact_quantize, "linear": _exact_linear}[case["op"]](case, s)


def _descending(key):
    """Row by row: the places of the keys from the largest on, equal ones in order of place."""
    return np.argsort(-key, axis=1, kind="stable")


def _exact_route(case, s):
    T, E, k, G = case["tokens"], case["experts"], case["k"], case["groups"]
    l = s["logits"].double().cpu()
    closed = torch.isneginf(l)
    log_score = torch.log_softmax(l, 1) if case["score"] == "softmax" else torch.nn.functional.logsigmoid(l)
    value = torch.exp(log_score).masked_fill(closed, 0.0)
    key = value if s["bias"] is None else value + s["bias"].double().cpu()
    key = key.masked_fill(closed, -math.inf).numpy()
    order_key = l.numpy() if s["bias"] is None else key  # a score grows with its logit
    order_key = order_key.copy()
    if G > 1:
        by_size = np.sort(key.reshape(T, G, E // G), 2)
        total = by_size[:, :, -1] if case["group_score"] == "max" else by_size[:, :, -1] + by_size[:, :, -2]
        if case["group_score"] == "max":
            total = order_key.reshape(T, G, E // G).max(2)
        for t, dropped in enumerate(_descending(total)[:, case["kept"]:]):
            order_key[t].reshape(G, E // G)[dropped] = -math.inf
    at = _descending(order_key)[:, :k].copy()
    gone = np.take_along_axis(order_key, at, 1) == -math.inf
    at, gone = torch.from_numpy(at), torch.from_numpy(gone)
    log_mine = log_score.gather(1, at).masked_fill(gone, -math.inf)
    if case["renormalize"]:
        r = torch.softmax(log_mine, 1).masked_fill(gone, 0.0)
    else:
        r = torch.exp(log_mine).masked_fill(gone, 0.0)
    out = [at.masked_fill(gone, -1).int(), r * case["scale"]]
    if case["train"]:
        # w = scale * softmax of the chosen log scores, or scale * their exponentials;
        # d log softmax_i / d l_j = [i = j] - p_j, d log sigmoid_i / d l_i = 1 - p_i
        g = s["dweights"].double().cpu().masked_fill(gone, 0.0) * case["scale"] * r
        dlog = g - r * g.sum(1, keepdim=True) if case["renormalize"] else g
        if case["score"] == "softmax":
            d = -value * dlog.sum(1, keepdim=True)
            d.scatter_add_(1, at, dlog)
        else:
            d = torch.zeros_like(l)
            d.scatter_add_(1, at, (dlog * torch.special.expit(-l.gather(1, at))).masked_fill(gone, 0.0))
        out.append(d)
    return out


def _exact_quantize(case, s):
    scales, values = [], []
    K, group = case["in"], case["group"]
    for w in s["weight"].double():
        columns, back = [], torch.empty_like(w)
        for a in range(0, K, group):
            part = w[:, a:a + group]
            scale = (part.abs().max(1).values / 7).to(s["weight"].dtype).double()
            q = torch.where(scale[:, None] > 0, torch.round(part / scale[:, None]), 0.0).clamp(-8, 7)
            back[:, a:a + group] = (q * scale[:, None]).to(s["weight"].dtype).double()
            columns.append(scale)
        scales.append(torch.stack(columns))
        values.append(back)
    return [torch.stack(scales), torch.stack(values)]


def _exact_linear(case, s):
    act, group = case["activation"], case["group"]
    off = s["offsets"].tolist()
    x = s["x"].double()
    y = s["residual"].double().clone() if case["residual"] else torch.zeros(case["rows"], case["out"],
                                                                           dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        z = torch.zeros(b - a, case["out"], dtype=torch.float64, device="cuda")
        w = s["q"][e].double()
        for i, scale in enumerate(s["scale"][e].double()):
            w[:, i * group:(i + 1) * group] *= scale[:, None]
        z += x[a:b] @ w.to(s["scale"].dtype).double().t()
        if case["bias"]:
            z += s["bias"][e].double()
        y[a:b] += {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0 * z),
                   "gelu": lambda: z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0)),
                   "silu": lambda: z * torch.special.expit(z)}[act]()
    return [y]


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        b = size * T * E + T * k * (4 + 4) + (4 * E if case["bias"] else 0)
        if case["train"]:  # the weights' gradient in, the logits' out
            b += T * k * 4 + size * T * E
        # a score is about four operations, a choice one comparison per expert
        return {"bytes": b, "flops": T * E * (4 + k) + (4 * T * E if case["train"] else 0)}
    E, K, N, group = case["experts"], case["in"], case["out"], case["group"]
    parts = -(-K // group)
    if case["op"] == "quantize":  # the weights in, the 4 bits and scales out, the weights they stand for out
        return {"bytes": E * N * (2 * size * K + K / 2 + size * parts), "flops": 4 * E * N * K}
    R = case["rows"]
    V = R * (1 - case["left_out"])  # rows that have an expert, and the experts that have a row:
    used = min(E, V) if case["balanced"] else E * (1 - (1 - 1 / E) ** V)
    b = size * (V * K + R * N * (2 if case["residual"] else 1)) + used * N * (K / 2 + size * parts) + 4 * (E + 1)
    b += size * used * N if case["bias"] else 0
    return {"bytes": b, "flops": 2 * V * N * K}
