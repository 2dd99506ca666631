"""Cases of the operators around a decoder block's feed-forward half, and their plain forms.

Three kinds, which follow each other in such a block:

``norm``    layer norm over the last dimension, forward, or the backward pass of a training step: the gradient of the input, and of weight and
            bias, which are sums over all rows.
``linear``  ``act(x @ w.T + bias) + residual`` of a dense fp16 / bf16 weight [n, k]: an up-projection with its activation, a
            down-projection with the block's residual.
``moe``     a whole mixture-of-experts layer for a few tokens: router (softmax over all experts, the top_k largest, divided by their
            sum where ``renormalize``), gated experts ``silu(gate) * up``, down-projection, weighted sum.  Expert weights are dense
            (``nbits`` 16) or group-quantized codes of 8 or 4 bits with an fp16 scale per ``group`` of a row, and a zero point where ``zero``.

Sizes are those of the benchmark configurations (hidden 640 to 4096, intermediate 2048 to 14336) and what lies between them.
"""

import math

import torch

own = False
DEVICE = "cuda"
EPS = 1e-5
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
MAX_FLOPS = 2.0 * 4096 * 14336 * 4096  # of a product
MAX_NORM = 8192 * 4096  # elements of a normed activation
MAX_PAIR_WEIGHTS = 32 * 3 * 4096 * 14336  # weights that the (token, expert) pairs of a moe layer meet
MAX_EXPERT_BYTES = 3 * 10**9  # of all experts of a layer


def _norm(name, rows, width, dtype, backward):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype, "backward": backward}


def _linear(name, m, n, k, dtype, act, bias, residual):
    return {"name": name, "kind": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "bias": bias, "residual": residual}


def _moe(name, m, experts, top_k, hidden, inter, dtype, nbits, group=32, zero=False, renormalize=True):
    return {"name": name, "kind": "moe", "m": m, "experts": experts, "top_k": top_k, "hidden": hidden, "inter": inter, "dtype": dtype,
            "nbits": nbits, "group": group, "zero": zero, "renormalize": renormalize}  # fmt: skip


def listed():
    return [
        # One decode token of a small model: nothing but latency.
        _norm("norm-m1", 1, 2048, "bfloat16", False),
        # The norm in front of a long prompt's feed-forward half.
        _norm("norm-m4096", 4096, 4096, "bfloat16", False),
        # The backward pass of an odd batch with odd rows: nothing is aligned.
        _norm("norm-back-ragged", 509, 3003, "float16", True),
        # The backward pass of a training step's batch: 8 sequences of 1024 tokens.
        _norm("norm-back-m8192", 8192, 4096, "bfloat16", True),
        # A decode step's down-projection and the residual it is added to.
        _linear("linear-down-m1", 1, 4096, 14336, "bfloat16", "none", False, True),
        # A decode step of 17 sequences, an up-projection with bias and activation.
        _linear("linear-up-m17", 17, 8192, 2048, "float16", "gelu_tanh", True, False),
        # Nothing a multiple of a tile.
        _linear("linear-ragged-m77", 77, 3003, 2184, "float16", "relu", True, True),
        # A long prompt's up-projection, the largest product.
        _linear("linear-up-m4096", 4096, 14336, 4096, "bfloat16", "gelu", True, False),
        # One decode token through two of eight large int4 experts.
        _moe("moe-int4-m1", 1, 8, 2, 4096, 14336, "bfloat16", 4),
        # A decode step of 16 sequences: nearly every expert is met, the most bytes of all.
        _moe("moe-int4-m16", 16, 8, 2, 4096, 14336, "float16", 4, group=128, zero=True),
        # Many small int8 experts, seven tokens.
        _moe("moe-int8-m7", 7, 64, 8, 2048, 1024, "bfloat16", 8, group=64, renormalize=False),
        # Dense experts, four tokens of a draft that are verified together.
        _moe("moe-dense-m4", 4, 16, 4, 2048, 2048, "bfloat16", 16),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, step):
    return max(step, int(round(_log(rng, lo, hi) / step)) * step)


def draw(rng):
    kind = rng.choice(["norm", "linear", "moe"])
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "norm":
        rows, width = int(round(_log(rng, 1, 8192))), _size(rng, 64, 8192, rng.choice([1, 8, 64, 128]))
        case = _norm("", min(rows, MAX_NORM // width), width, rng.choice([dtype, dtype, "float32"]), rng.random() < 0.5)
    elif kind == "linear":
        m, n = int(round(_log(rng, 1, 4096))), _size(rng, 64, 14336, rng.choice([1, 16, 64, 128]))
        k = _size(rng, 64, 14336, rng.choice([1, 8, 64, 128]))
        case = _linear("", max(1, min(m, int(MAX_FLOPS / (2.0 * n * k)))), n, k, dtype, rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                       rng.random() < 0.5, rng.random() < 0.5)  # fmt: skip
    else:
        m, experts = int(round(_log(rng, 1, 32))), rng.choice([4, 8, 16, 32, 60, 64, 128])
        top_k = rng.randint(1, min(8, experts))
        nbits, group = rng.choice([4, 4, 8, 16]), rng.choice([32, 64, 128])
        hidden, inter = _size(rng, 256, 4096, 128), _size(rng, 256, 14336, 128)
        while hidden * inter * 3 * experts * nbits / 8 > MAX_EXPERT_BYTES or m * top_k * 3 * hidden * inter > MAX_PAIR_WEIGHTS:
            hidden, inter = max(256, hidden // 256 * 128), max(256, inter // 256 * 128)
            m = max(1, m - 1)
        case = _moe("", m, experts, top_k, hidden, inter, dtype, nbits, group, nbits < 16 and rng.random() < 0.4, rng.random() < 0.7)
    case.pop("name")
    return case


# ----------------------------------------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------------------------------------


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std + mean).to(to)

    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        # Activations of a residual stream: a mean of their own per row, a few features far larger than the others.
        x = torch.randn(rows, width, generator=g, device=DEVICE) + torch.randn(rows, 1, generator=g, device=DEVICE)
        x[:, :: max(1, width // 4)] *= 12.0
        s = {"x": x.to(dtype), "weight": normal(width, std=0.2, mean=1.0), "bias": normal(width, std=0.1)}
        if case["backward"]:
            xf = s["x"].double()
            mean = xf.mean(-1)
            s["mean"], s["rstd"] = mean.float(), torch.rsqrt((xf - mean[:, None]).square().mean(-1) + EPS).float()  # as the forward pass left them
            s["dy"] = normal(rows, width)
        return s
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"x": normal(m, k), "w": normal(n, k, std=k**-0.5), "bias": normal(n, std=0.5) if case["bias"] else None,
                "residual": normal(m, n) if case["residual"] else None}  # fmt: skip
    m, e, h, i, nbits = case["m"], case["experts"], case["hidden"], case["inter"], case["nbits"]
    # A trained router tells experts apart: logits with a standard deviation of two.
    s = {"x": normal(m, h), "router": normal(e, h, std=2.0 * h**-0.5)}
    for name, rows, cols in (("gate_up", 2 * i, h), ("down", h, i)):
        if nbits == 16:
            s[name] = normal(e, rows, cols, std=cols**-0.5)
            continue
        groups, top = cols // case["group"], 1 << nbits
        s[name] = torch.randint(0, 256, (e, rows, cols * nbits // 8), generator=g, device=DEVICE, dtype=torch.uint8)
        s[name + "_scale"] = ((torch.rand(e, rows, groups, generator=g, device=DEVICE) + 0.5) * 3.5 / top * cols**-0.5).half()
        if case["zero"]:
            s[name + "_zero"] = (top / 2 + torch.randn(e, rows, groups, generator=g, device=DEVICE) * top / 16).half()
    return s


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    if own and case["kind"] == "moe":
        from neuropress_amd import kernels

        s["handle"] = kernels.MoEExperts(s["router"], s["gate_up"], s["down"], nbits=s["nbits"], group_size=s["group"],
                                         gate_up_scale=s.get("gate_up_scale"), gate_up_zero=s.get("gate_up_zero"),
                                         down_scale=s.get("down_scale"), down_zero=s.get("down_zero"))  # fmt: skip
    return s


# ----------------------------------------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    return {"norm": _norm_plain, "linear": _linear_plain, "moe": _moe_plain}[s["kind"]](s)


def _own(s):
    from neuropress_amd import kernels

    if s["kind"] == "norm":
        if s["backward"]:
            return kernels.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
        return kernels.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if s["kind"] == "linear":
        act = None if s["act"] == "none" else s["act"]
        return kernels.dense_linear_act(s["x"], s["w"], bias=s["bias"], activation=act, residual=s["residual"])
    return kernels.moe_layer(s["x"], s["handle"], s["top_k"], renormalize=s["renormalize"])


def _norm_plain(s):
    x, w = s["x"].float(), s["weight"].float()
    if not s["backward"]:
        mean = x.mean(-1, keepdim=True)
        d = x - mean
        y = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS) * w + s["bias"].float()
        return y.to(s["x"].dtype)
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    to = s["x"].dtype
    # sums over thousands of rows of either sign: in 64 bits
    return dx.to(to), (dy * xhat).sum(0, dtype=torch.float64).to(to), dy.sum(0, dtype=torch.float64).to(to)


def _act(name, v):
    if name == "relu":
        return torch.maximum(v, torch.zeros_like(v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    return v / (1.0 + torch.exp(-v)) if name == "silu" else v


def _linear_plain(s):
    v = torch.mm(s["x"].float(), s["w"].float().t())
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(s["act"], v)
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["x"].dtype)


def _weights(s, name, ids):
    """The weights of the experts *ids*, in 32 bits."""
    w, nbits = s[name][ids], s["nbits"]
    if nbits == 16:
        return w.float()
    if nbits == 4:  # the low nibble is the even column
        w = torch.stack((w & 15, w >> 4), -1).flatten(-2)
    zero = s[name + "_zero"][ids].float()[..., None] if s["zero"] else float(1 << (nbits - 1))
    w = w.float().unflatten(-1, (-1, s["group"]))
    return ((w - zero) * s[name + "_scale"][ids].float()[..., None]).flatten(-2)


def _moe_plain(s):
    x, k = s["x"], s["top_k"]
    logits = torch.mm(x.double(), s["router"].double().t())  # in 64 bits: neighbours decide which expert is met
    p = torch.exp(logits - logits.max(-1, keepdim=True).values)
    p, ids = torch.sort(p / p.sum(-1, keepdim=True), dim=-1, descending=True, stable=True)
    p, ids = p[:, :k].float(), ids[:, :k].reshape(-1)
    if s["renormalize"]:
        p = p / p.sum(-1, keepdim=True)
    xs = x.float().repeat_interleave(k, 0)[..., None]
    gate, up = torch.bmm(_weights(s, "gate_up", ids), xs).squeeze(-1).chunk(2, -1)
    h = _act("silu", gate) * up
    y = torch.bmm(_weights(s, "down", ids), h[..., None]).squeeze(-1)
    return (y.unflatten(0, (-1, k)) * p[..., None]).sum(1).to(x.dtype)


# ----------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without, and its value in 64 bits
# ----------------------------------------------------------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "norm":
        n, width = case["rows"] * case["width"], case["width"]
        if case["backward"]:
            return {"bytes": size * (3.0 * n + 3 * width) + 8.0 * case["rows"], "flops": 14.0 * n}
        return {"bytes": size * (2.0 * n + 2 * width), "flops": 8.0 * n}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        outs = m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        return {"bytes": size * (1.0 * m * k + 1.0 * n * k + outs), "flops": 2.0 * m * n * k}
    m, e, h, i, k = case["m"], case["experts"], case["hidden"], case["inter"], case["top_k"]
    met = e * (1.0 - (1.0 - k / e) ** m)  # experts that m tokens meet, on average
    per_weight = case["nbits"] / 8 + (0 if case["nbits"] == 16 else (4 if case["zero"] else 2) / case["group"])
    return {"bytes": met * 3 * h * i * per_weight + 2.0 * (e * h + 2 * m * h), "flops": 2.0 * m * (k * 3 * h * i + e * h)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "norm":
        x = s["x"].double()
        if not case["backward"]:
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            return (x - mean) / torch.sqrt(var + EPS) * s["weight"].double() + s["bias"].double()
        # the gradient of sum(dy * (xhat * w + b)) through xhat = (x - mean) * rstd, by its Jacobian (I - 1 1^T / n - xhat xhat^T / n) * rstd
        dy, rstd, n = s["dy"].double(), s["rstd"].double()[:, None], case["width"]
        xhat = (x - s["mean"].double()[:, None]) * rstd
        v = dy * s["weight"].double()
        dx = v - v.sum(-1, keepdim=True) / n - xhat * torch.linalg.vecdot(v, xhat).unsqueeze(-1) / n
        return dx * rstd, torch.linalg.vecdot(dy, xhat, dim=0), torch.ones(case["rows"], dtype=torch.float64, device=DEVICE) @ dy
    if case["kind"] == "linear":
        if 2.0 * case["m"] * case["n"] * case["k"] > 1e12:
            return None
        y = torch.nn.functional.linear(s["x"].double(), s["w"].double(), None if s["bias"] is None else s["bias"].double())
        f = torch.nn.functional
        y = {"none": lambda t: t, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"), "silu": f.silu}[case["act"]](y)
        return y if s["residual"] is None else y + s["residual"].double()
    x, top_k = s["x"].double(), case["top_k"]
    logits = x @ s["router"].double().T
    # rank of every expert: how many are ahead of it, ties to the lower index
    order = torch.arange(case["experts"], device=DEVICE)
    ahead = (logits[:, None, :] > logits[:, :, None]) | ((logits[:, None, :] == logits[:, :, None]) & (order[None, None, :] < order[None, :, None]))
    taken = ahead.sum(-1) < top_k
    share = torch.softmax(logits, -1) * taken
    if case["renormalize"]:
        share = share / share.sum(-1, keepdim=True)

    def weights(name, expert):
        w = s[name][expert]
        if case["nbits"] == 16:
            return w.double()
        rows, cols = w.shape[0], w.shape[1] * 8 // case["nbits"]
        column = torch.arange(cols, device=DEVICE)
        codes = w[:, column * case["nbits"] // 8].to(torch.int32)
        codes = (codes >> (column * case["nbits"] % 8).to(torch.int32)) & ((1 << case["nbits"]) - 1)
        group = column // case["group"]
        z = s[name + "_zero"][expert].double()[:, group] if case["zero"] else torch.full((rows, cols), 2.0 ** (case["nbits"] - 1), device=DEVICE, dtype=torch.float64)
        return (codes.double() - z) * s[name + "_scale"][expert].double()[:, group]

    y = torch.zeros_like(x)
    for expert in range(case["experts"]):
        rows = taken[:, expert].nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        both = x[rows] @ weights("gate_up", expert).T
        gate, up = both[:, : case["inter"]], both[:, case["inter"] :]
        y[rows] += ((gate * torch.sigmoid(gate) * up) @ weights("down", expert).T) * share[rows, expert : expert + 1]
    return y
