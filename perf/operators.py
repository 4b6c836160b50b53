"""The measured cases of the encoder-block operators: attention over packed sequences, layer norm, and the dense layer with
its activation and residual in the epilogue.

``run`` computes a case either in plain form (``own = False``: elementary torch operations in 32 bits, rounded once at the
end) or through the framework's entry points (``own = True``); both take the same inputs from ``prepare`` and return the
same outputs.  ``exact`` gives those outputs from the definition in 64 bits.

* attention: ``o = softmax(scale q k^T + mask) v`` per sequence and head; query head ``i`` of ``heads`` reads key / value
  head ``i // (heads / kv_heads)``; causal rows see keys up to their own.  Rows behind the last sequence give zeros.
* norm: ``y = (x - mean) / sqrt(var + eps) * w + b`` per row, variance over all columns.
* linear: ``y = act(x W^T + b) + residual``.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}


# ---- cases --------------------------------------------------------------------------------------------------------------

def _attention(name, lengths, heads, kv_heads, dk, dv, dtype, causal, train, rows=0):
    text = ",".join(str(n) for n in lengths)
    return {"name": name, "op": "attention", "lengths": text, "rows": max(rows, sum(lengths)), "heads": heads,
            "kv_heads": kv_heads, "dk": dk, "dv": dv, "dtype": dtype, "causal": causal, "train": train}


def _norm(name, rows, cols, dtype, param_dtype, train):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "param_dtype": param_dtype, "train": train}


def _linear(name, rows, in_features, out_features, dtype, activation, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "in_features": in_features, "out_features": out_features,
            "dtype": dtype, "activation": activation, "residual": residual, "train": train}


def listed():
    windows = [200, 129, 500, 173, 200, 96, 311, 50, 200, 1000, 64, 257, 333, 200, 140, 200]
    documents = [2048, 1, 777, 1500, 64, 130, 2011, 1024, 333, 17, 1900, 640, 255, 1333, 2, 900, 1201, 700, 405, 1000]
    return [
        # a handful of short requests in one forward pass: launch and latency
        _attention("attention-requests", [1, 37, 96, 5, 64, 18, 128, 50], 8, 2, 64, 64, "bf16", True, False),
        # training on ragged windows in the search's default precision, every window past or below 128 tokens, both directions
        # of time visible, half-width keys (key_dim_scaling 0.5)
        _attention("attention-windows-train", windows, 8, 8, 32, 64, "f32", False, True),
        # documents of very different lengths packed into one training batch, the batch padded to a round number of rows
        _attention("attention-documents-train", documents, 16, 4, 128, 128, "bf16", True, True, rows=16384),
        # one long prompt with two key / value heads
        _attention("attention-prompt", [16383], 16, 2, 128, 128, "bf16", True, False),
        # the last row of every sequence of a small batch: latency
        _norm("norm-last-rows", 32, 512, "f32", "f32", False),
        # the widest model of the full search, batch 256 of 500 tokens
        _norm("norm-encoder-train", 128000, 512, "f32", "f32", True),
        # a wide residual stream in bf16 with f32 parameters
        _norm("norm-wide-train", 16384, 4096, "bf16", "f32", True),
        # rows of an odd number of columns
        _norm("norm-odd-train", 5001, 10007, "bf16", "bf16", True),
        # single rows of a few requests through a wide layer: the weight has to be read once
        _linear("linear-requests", 7, 4096, 8192, "bf16", "relu", False, False),
        # an encoder layer's first dense layer in the search's default precision, batch 64 of 200 tokens
        _linear("linear-encoder-train", 12800, 512, 2048, "f32", "gelu", False, True),
        # a layer of the width-8192 network
        _linear("linear-wide-train", 8192, 8192, 8192, "bf16", "gelu", False, True),
        # the projection back to the residual stream on a ragged number of rows
        _linear("linear-residual-train", 5003, 8192, 2048, "bf16", "none", True, True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_attention(rng):
    heads_per_kv, kv_heads = rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    dk = rng.choice([16, 20, 32, 40, 64, 64, 80, 96, 128, 128])
    dv = dk if rng.random() < 0.7 else rng.choice([16, 32, 48, 64, 128])
    count = _log_int(rng, 1, 64)
    longest = _log_int(rng, 1, 16384)
    lengths = [max(0, min(longest, int(longest * rng.random() ** 2) + rng.randint(0, 2))) for _ in range(count)]
    lengths[rng.randrange(count)] = longest
    rows = sum(lengths) + (rng.randint(1, 300) if rng.random() < 0.3 else 0)
    return _attention("", lengths, heads_per_kv * kv_heads, kv_heads, dk, dv, rng.choice(["f32", "bf16", "bf16"]),
                      rng.random() < 0.7, rng.random() < 0.6, rows)


def _draw_norm(rng):
    cols = _log_int(rng, 8, 16384)
    rows = _log_int(rng, 1, max(2, min(200000, (1 << 26) // cols)))
    dtype = rng.choice(["f32", "bf16"])
    return _norm("", rows, cols, dtype, "f32" if dtype == "f32" else rng.choice(["f32", "bf16"]), rng.random() < 0.6)


def _draw_linear(rng):
    in_features, out_features = _log_int(rng, 8, 8192), _log_int(rng, 1, 8192)
    if rng.random() < 0.6:
        in_features, out_features = (in_features + 7) // 8 * 8, (out_features + 7) // 8 * 8
    train = rng.random() < 0.6
    rows = _log_int(rng, 1, 16384)
    # relu's slope steps at zero, where two orders of summation may fall on different sides: forward passes only
    return _linear("", rows, in_features, out_features, rng.choice(["f32", "bf16", "bf16"]),
                   rng.choice(["none", "gelu"] if train else ["none", "relu", "gelu"]), rng.random() < 0.5, train)


def _cost(case):
    """A rough time: the plain form's flops at the f32 rate and its bytes, a dozen passes over the widest tensor."""
    w = work(case)
    return w["flops"] / 1e14 + 6 * w["bytes"] / 4e12


def draw(rng):
    make = {"attention": _draw_attention, "norm": _draw_norm, "linear": _draw_linear}[rng.choice(["attention", "norm", "linear"])]
    limit = max(_cost(c) for c in listed() if c["op"] == make.__name__[len("_draw_"):])
    while True:
        case = make(rng)
        if _cost(case) <= limit and case["rows"] > 0:
            del case["name"]
            return case


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "attention":
        h, hk, dk, dv, rows = case["heads"], case["kv_heads"], case["dk"], case["dv"], case["rows"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))
        flops = 2 * h * pairs * (dk + dv)
        tensors = rows * (h * (dk + dv) + hk * (dk + dv))                     # q, o, k, v
        if case["train"]:
            flops += 2 * h * pairs * (3 * dk + 2 * dv)
            tensors += rows * (h * (dk + dv) + hk * (dk + dv))                # do, dq, dk, dv
        return {"bytes": tensors * size, "flops": flops}
    if case["op"] == "norm":
        cells, psize = case["rows"] * case["cols"], SIZES[case["param_dtype"]]
        if case["train"]:
            return {"bytes": 4 * cells * size + 4 * case["cols"] * psize, "flops": 20 * cells}
        return {"bytes": 2 * cells * size + 2 * case["cols"] * psize, "flops": 8 * cells}
    m, k, n = case["rows"], case["in_features"], case["out_features"]
    tensors = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
    flops = 2 * m * n * k
    if case["train"]:
        tensors += m * n + m * k + n * k + n                                 # dy, dx, dw, db (the residual's gradient is dy)
        flops *= 3
    return {"bytes": tensors * size, "flops": flops}


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


# ---- inputs -------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    state = {"case": case}
    if case["op"] == "attention":
        rows, h, hk, dk, dv = (case[n] for n in ("rows", "heads", "kv_heads", "dk", "dv"))
        state.update(q=normal(rows, h, dk), k=normal(rows, hk, dk), v=normal(rows, hk, dv))
        if case["train"]:
            state["do"] = normal(rows, h, dv, scale=0.1)
        if own:
            from mitune.ops.attention import SequencePack
            state["pack"] = SequencePack(_lengths(case), rows=rows, device="cuda")
    elif case["op"] == "norm":
        rows, cols, pdtype = case["rows"], case["cols"], DTYPES[case["param_dtype"]]
        spread = torch.rand(rows, 1, device="cuda", generator=g) + 0.5
        shift = torch.randn(rows, 1, device="cuda", generator=g) * 0.5
        state["x"] = (torch.randn(rows, cols, device="cuda", generator=g) * spread + shift).to(dtype)
        state["w"] = normal(cols, scale=0.2, dtype=torch.float32).add_(1.0).to(pdtype)
        state["b"] = normal(cols, scale=0.2, dtype=pdtype)
        if case["train"]:
            state["dy"] = normal(rows, cols, scale=0.1)
    else:
        m, k, n = case["rows"], case["in_features"], case["out_features"]
        state["x"] = normal(m, k)
        state["w"] = normal(n, k, scale=1.0 / math.sqrt(k))
        state["b"] = normal(n, scale=0.1)
        state["r"] = normal(m, n) if case["residual"] else None
        if case["train"]:
            state["dy"] = normal(m, n, scale=0.1)
    return state


# ---- the operators ------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    kind = case["op"] + ("_train" if case["train"] else "")
    return globals()[("_own_" if own else "_plain_") + kind](state, case)


def _leaves(*tensors):
    return [t.detach().requires_grad_() for t in tensors]


def _own_attention(state, case):
    from mitune.ops.attention import packed_attention
    return packed_attention(state["q"], state["k"], state["v"], state["pack"], causal=case["causal"])


def _own_attention_train(state, case):
    from mitune.ops.attention import packed_attention
    q, k, v = _leaves(state["q"], state["k"], state["v"])
    o = packed_attention(q, k, v, state["pack"], causal=case["causal"])
    return (o.detach(),) + torch.autograd.grad(o, (q, k, v), state["do"])


def _own_norm(state, case):
    from mitune.ops.layernorm import layer_norm
    return layer_norm(state["x"], state["w"], state["b"], EPS)


def _own_norm_train(state, case):
    from mitune.ops.layernorm import layer_norm
    x, w, b = _leaves(state["x"], state["w"], state["b"])
    y = layer_norm(x, w, b, EPS)
    return (y.detach(),) + torch.autograd.grad(y, (x, w, b), state["dy"])


def _own_linear(state, case):
    from mitune.ops.linear import linear
    act = None if case["activation"] == "none" else case["activation"]
    return linear(state["x"], state["w"], state["b"], activation=act, residual=state["r"])


def _own_linear_train(state, case):
    from mitune.ops.linear import linear
    act = None if case["activation"] == "none" else case["activation"]
    x, w, b = _leaves(state["x"], state["w"], state["b"])
    leaves = (x, w, b)
    r = state["r"]
    if r is not None:
        (r,) = _leaves(r)
        leaves += (r,)
    y = linear(x, w, b, activation=act, residual=r)
    return (y.detach(),) + torch.autograd.grad(y, leaves, state["dy"])


def _spans(case, chunk):
    """(first row, rows, query offset, queries, keys) of every piece of at most ``chunk`` queries of every sequence."""
    start = 0
    for n in _lengths(case):
        for a in range(0, n, chunk):
            b = min(n, a + chunk)
            yield start, n, a, b - a, (b if case["causal"] else n)
        start += n


def _chunk(case):
    longest = max(_lengths(case) + [1])
    return max(64, min(2048, (1 << 28) // (case["heads"] * longest)))


def _scores(case, q, k, a, dtype):
    """softmax weights [kv_heads, group, queries, keys] of ``q`` [queries, heads, dk] at offset ``a`` over ``k`` [keys, kv_heads, dk]."""
    hk, dk = case["kv_heads"], case["dk"]
    qs = q.to(dtype).view(q.shape[0], hk, -1, dk).permute(1, 2, 0, 3)                     # [kv, group, queries, dk]
    group, nq = qs.shape[1], qs.shape[2]
    kt = k.to(dtype).permute(1, 2, 0).contiguous()                                        # [kv, dk, keys]
    s = torch.matmul(qs.reshape(hk, group * nq, dk).contiguous(), kt).view(hk, group, nq, -1) * (1.0 / math.sqrt(dk))
    if case["causal"]:
        hidden = torch.arange(k.shape[0], device=q.device)[None, :] > (a + torch.arange(nq, device=q.device))[:, None]
        s = s.masked_fill_(hidden, float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    return s.div_(s.sum(-1, keepdim=True)), qs


def _heads_first(t, hk, dtype):
    """[queries, heads, d] -> [kv_heads, group * queries, d]."""
    n, _, d = t.shape
    return t.to(dtype).view(n, hk, -1, d).permute(1, 2, 0, 3).reshape(hk, -1, d).contiguous()


def _heads_last(t, group, n):
    """[kv_heads, group * queries, d] -> [queries, heads, d]."""
    hk, d = t.shape[0], t.shape[2]
    return t.view(hk, group, n, d).permute(2, 0, 1, 3).reshape(n, hk * group, d)


def _attend(state, case, dtype):
    q, k, v = state["q"], state["k"], state["v"]
    hk = case["kv_heads"]
    out = torch.zeros(q.shape[0], case["heads"], case["dv"], device=q.device, dtype=dtype)
    for start, _, a, n, keys in _spans(case, _chunk(case)):
        p, qs = _scores(case, q[start + a:start + a + n], k[start:start + keys], a, dtype)
        vv = v[start:start + keys].to(dtype).permute(1, 0, 2).contiguous()
        o = torch.matmul(p.view(hk, -1, keys), vv)
        out[start + a:start + a + n] = _heads_last(o, qs.shape[1], n)
    return out


def _attend_train(state, case, dtype):
    q, k, v, do = state["q"], state["k"], state["v"], state["do"]
    hk, scale = case["kv_heads"], 1.0 / math.sqrt(case["dk"])
    zeros = lambda t: torch.zeros(t.shape, device=t.device, dtype=dtype)                  # noqa: E731
    out, dq, dk, dv = zeros(do), zeros(q), zeros(k), zeros(v)
    for start, _, a, n, keys in _spans(case, _chunk(case)):
        rows, cols = slice(start + a, start + a + n), slice(start, start + keys)
        p, qs = _scores(case, q[rows], k[cols], a, dtype)
        group = qs.shape[1]
        p = p.view(hk, group * n, keys)
        vv = v[cols].to(dtype).permute(1, 0, 2).contiguous()
        dd = _heads_first(do[rows], hk, dtype)
        o = torch.matmul(p, vv)
        out[rows] = _heads_last(o, group, n)
        dv[cols] += torch.matmul(p.transpose(1, 2).contiguous(), dd).permute(1, 0, 2)
        ds = torch.matmul(dd, vv.transpose(1, 2).contiguous()).sub_((dd * o).sum(-1, keepdim=True)).mul_(p)
        kk = k[cols].to(dtype).permute(1, 0, 2).contiguous()
        dq[rows] = _heads_last(torch.matmul(ds, kk).mul_(scale), group, n)
        dk[cols] += torch.matmul(ds.transpose(1, 2).contiguous(), _heads_first(q[rows], hk, dtype)).mul_(scale).permute(1, 0, 2)
    return out, dq, dk, dv


def _plain_attention(state, case):
    return _attend(state, case, torch.float32).to(DTYPES[case["dtype"]])


def _plain_attention_train(state, case):
    return tuple(t.to(DTYPES[case["dtype"]]) for t in _attend_train(state, case, torch.float32))


def _plain_norm(state, case):
    x = state["x"].float()
    c = x - x.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return (c * rstd * state["w"].float() + state["b"].float()).to(DTYPES[case["dtype"]])


def _plain_norm_train(state, case):
    x, w, b, dy = (state[n].float() for n in ("x", "w", "b", "dy"))
    c = x - x.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xhat = c * rstd
    y = xhat * w + b
    gw = dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    dw, db = (dy * xhat).sum(0), dy.sum(0)
    dtype, pdtype = DTYPES[case["dtype"]], DTYPES[case["param_dtype"]]
    return y.to(dtype), dx.to(dtype), dw.to(pdtype), db.to(pdtype)


def _activate(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_linear(state, case):
    y = _activate(state["x"].float() @ state["w"].float().t() + state["b"].float(), case["activation"])
    if state["r"] is not None:
        y = y + state["r"].float()
    return y.to(DTYPES[case["dtype"]])


def _plain_linear_train(state, case):
    x, w, dy = state["x"].float(), state["w"].float(), state["dy"].float()
    z = x @ w.t() + state["b"].float()
    y = _activate(z, case["activation"])
    if state["r"] is not None:
        y = y + state["r"].float()
    dz = dy if case["activation"] == "none" else dy * _slope(z, case["activation"])
    outs = [y, dz @ w, dz.t() @ x, dz.sum(0)] + ([dy] if state["r"] is not None else [])
    return tuple(t.to(DTYPES[case["dtype"]]) for t in outs)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return globals()["_exact_" + case["op"]](state, case)


def _exact_attention(state, case):
    """One key / value head and one piece of a sequence at a time: weights from the shifted exponentials, gradients from
    the softmax's Jacobian applied to the upstream product."""
    names = ("q", "k", "v") + (("do",) if case["train"] else ())
    t = {n: state[n].double().transpose(0, 1).contiguous() for n in names}                # [heads, rows, d]
    h, hk = case["heads"], case["kv_heads"]
    group, scale = h // hk, case["dk"] ** -0.5
    o = torch.zeros(h, case["rows"], case["dv"], device="cuda", dtype=torch.float64)
    grads = {n: torch.zeros_like(t[n]) for n in ("q", "k", "v")} if case["train"] else {}
    first = 0
    for n in _lengths(case):
        for i in range(h):
            j = i // group
            for a in range(0, n, 4096):
                b = min(n, a + 4096)
                end = b if case["causal"] else n
                q, k, v = t["q"][i, first + a:first + b], t["k"][j, first:first + end], t["v"][j, first:first + end]
                s = (q @ k.T) * scale
                if case["causal"]:
                    s += torch.full_like(s, float("-inf")).triu_(a + 1)
                p = torch.softmax(s, dim=-1)
                del s
                o[i, first + a:first + b] = p @ v
                if case["train"]:
                    do = t["do"][i, first + a:first + b]
                    dp = do @ v.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                    grads["q"][i, first + a:first + b] = ds @ k * scale
                    grads["k"][j, first:first + end] += ds.T @ q * scale
                    grads["v"][j, first:first + end] += p.T @ do
        first += n
    outs = [o] + [grads[n] for n in ("q", "k", "v") if case["train"]]
    outs = [u.transpose(0, 1) for u in outs]
    return tuple(outs) if case["train"] else outs[0]


def _exact_norm(state, case):
    x, w, b = (state[n].double() for n in ("x", "w", "b"))
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    inv = 1.0 / torch.sqrt(var + EPS)
    unit = (x - mean) * inv
    if not case["train"]:
        return unit * w + b
    dy = state["dy"].double()
    du = dy * w
    m = case["cols"]
    dx = inv / m * (m * du - du.sum(1, keepdim=True) - unit * (du * unit).sum(1, keepdim=True))
    return unit * w + b, dx, (dy * unit).sum(0), dy.sum(0)


def _exact_linear(state, case):
    x, w = state["x"].double(), state["w"].double()
    z = torch.addmm(state["b"].double(), x, w.t())
    normal = torch.distributions.Normal(torch.zeros((), device="cuda", dtype=torch.float64),
                                        torch.ones((), device="cuda", dtype=torch.float64), validate_args=False)
    if case["activation"] == "relu":
        y, slope = z.clamp(min=0.0), (z > 0).double()
    elif case["activation"] == "gelu":
        cdf = normal.cdf(z)
        y, slope = z * cdf, cdf + z * normal.log_prob(z).exp()
    else:
        y, slope = z.clone(), None
    if state["r"] is not None:
        y += state["r"].double()
    if not case["train"]:
        return y
    dy = state["dy"].double()
    dz = dy if slope is None else dy * slope
    outs = [y, dz @ w, dz.t() @ x, dz.sum(0)]
    return tuple(outs + ([dy] if state["r"] is not None else []))
