"""Cases of the operators that join the halves of a decoder block, and their plain forms.

Three kinds, which follow each other in such a block:

``norm``     where one half of a block ends and the next begins: the half's output y is normed (where ``post``), gated (``gate``) and scaled, added to the
             residual stream x, and the sum is normed for the next half.  ``r = x + scale * gate * rmsnorm(y, post_weight)``, ``z = rmsnorm(r, weight)``; both
             are outputs.  A gate is one vector for all rows ("channel"), one for each sequence or one for each token.  Backward: the gradients of x, y, both
             weights and the gate from those of r and z.
``gated``    the first half of a gated feed-forward block, ``act(x @ gate.T + bias) * (x @ up.T + bias)`` with the weights one behind the other in
             ``gate_up`` [2 * inter, hidden].  Backward: the gradients of x, the weights and the bias, from the rounded sums that the forward pass left.
``adapter``  low-rank adapters of many requests beside a projection that they share: ``base + scale[a] * (x @ A[a].T) @ B[a].T``, a the adapter of a token's
             request, none for some.  ``base`` is what the projection gave.

Sizes are those of the benchmark configurations (hidden 640 to 4096, intermediate 2048 to 14336) and what lies between them.
"""

import math
import random

import torch

own = False
DEVICE = "cuda"
EPS = 1e-6
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
MAX_NORM = 8192 * 4096  # elements of a residual stream
MAX_FLOPS = 8.0 * 4096 * 14336 * 4096  # of the products of a gated block
MAX_ADAPTER_ELEMENTS = 4096 * (4096 + 2 * 14336)  # of x, base and the output together
MAX_ADAPTER_WEIGHTS = 1 << 28


def _norm(name, seqs, tokens, width, dtype, post, gate, scale, backward):
    return {"name": name, "kind": "norm", "seqs": seqs, "tokens": tokens, "width": width, "dtype": dtype, "post": post, "gate": gate, "scale": scale,
            "backward": backward}  # fmt: skip


def _gated(name, m, inter, hidden, dtype, act, bias, backward):
    return {"name": name, "kind": "gated", "m": m, "inter": inter, "hidden": hidden, "dtype": dtype, "act": act, "bias": bias, "backward": backward}


def _adapter(name, m, requests, adapters, rank, n, k, dtype):
    return {"name": name, "kind": "adapter", "m": m, "requests": requests, "adapters": adapters, "rank": rank, "n": n, "k": k, "dtype": dtype}


def listed():
    return [
        # One decode token of a small model, a plain residual add and the next norm: nothing but latency.
        _norm("norm-m1", 1, 1, 2048, "bfloat16", False, "none", 1.0, False),
        # A long prompt of a model that norms before and after each half and scales what a half adds.
        _norm("norm-m4096", 1, 4096, 4096, "bfloat16", True, "channel", 0.22, False),
        # The backward pass of an odd batch with odd rows, gates of each sequence's own: nothing is aligned.
        _norm("norm-back-ragged", 3, 171, 3003, "float16", False, "sequence", 1.0, True),
        # The backward pass of a training step's batch: 8 sequences of 1024 tokens.
        _norm("norm-back-m8192", 8, 1024, 4096, "bfloat16", True, "channel", 0.22, True),
        # One decode token: both weights are all that counts.
        _gated("gated-m1", 1, 14336, 4096, "bfloat16", "silu", False, False),
        # A decode step of 17 sequences with bias.
        _gated("gated-m17", 17, 8192, 2048, "float16", "gelu_tanh", True, False),
        # A long prompt.
        _gated("gated-m4096", 4096, 14336, 4096, "bfloat16", "silu", False, False),
        # The backward pass of a small batch, nothing a multiple of a tile.
        _gated("gated-back-m1000", 1000, 2739, 2184, "float16", "gelu", True, True),
        # The backward pass of a training step's batch, the largest products.
        _gated("gated-back-m4096", 4096, 14336, 4096, "bfloat16", "silu", False, True),
        # One decode token of one request.
        _adapter("adapter-m1", 1, 1, 8, 16, 4096, 4096, "bfloat16"),
        # A decode step of 32 requests with 64 adapters loaded, an up-projection.
        _adapter("adapter-m32", 32, 32, 64, 16, 14336, 4096, "bfloat16"),
        # The prompts of five requests, one behind the other.
        _adapter("adapter-prompts", 4096, 5, 16, 64, 14336, 4096, "float16"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi, step):
    return max(step, int(round(_log(rng, lo, hi) / step)) * step)


def draw(rng):
    kind = rng.choice(["norm", "gated", "adapter"])
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "norm":
        rows, width = int(round(_log(rng, 1, 8192))), _size(rng, 64, 8192, rng.choice([1, 8, 64, 128]))
        rows = min(rows, MAX_NORM // width)
        seqs = rng.randint(1, min(rows, 8))
        case = _norm("", seqs, rows // seqs, width, rng.choice([dtype, dtype, "float32"]), rng.random() < 0.5, rng.choice(["none", "none", "channel", "sequence", "token"]),
                     rng.choice([1.0, round(rng.uniform(0.1, 1.5), 3)]), rng.random() < 0.5)  # fmt: skip
    elif kind == "gated":
        backward = rng.random() < 0.5
        m, step = int(round(_log(rng, 1, 4096))), rng.choice([1, 8, 64, 128])
        inter, hidden = _size(rng, 64, 14336, step), _size(rng, 64, 8192, rng.choice([1, 8, 64, 128]))
        m = max(1, min(m, int(MAX_FLOPS / ((8.0 if backward else 4.0) * inter * hidden))))
        case = _gated("", m, inter, hidden, dtype, rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]), rng.random() < 0.4, backward)
    else:
        m, adapters, rank = int(round(_log(rng, 1, 4096))), int(round(_log(rng, 1, 256))), rng.choice([4, 8, 16, 16, 24, 32, 64, 128])
        n, k = _size(rng, 64, 14336, rng.choice([1, 16, 64, 128])), _size(rng, 64, 14336, rng.choice([1, 8, 64, 128]))
        m = max(1, min(m, MAX_ADAPTER_ELEMENTS // (k + 2 * n)))
        adapters = max(1, min(adapters, MAX_ADAPTER_WEIGHTS // (rank * (n + k))))
        requests = m if m <= 64 and rng.random() < 0.7 else rng.randint(1, min(m, 64))
        case = _adapter("", m, requests, adapters, rank, n, k, dtype)
    case.pop("name")
    return case


# ----------------------------------------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------------------------------------


def _requests(case, seed):
    """(first token, past the last, adapter) of every request; adapter -1: none."""
    rng = random.Random(seed)
    m, count = case["m"], case["requests"]
    ends = sorted(rng.sample(range(1, m), count - 1)) + [m]
    adapters = [-1 if count > 1 and rng.random() < 0.125 else rng.randrange(case["adapters"]) for _ in range(count)]
    return list(zip([0] + ends[:-1], ends, adapters))


def _rms(v):
    """The reciprocal root of the mean square of each row, in 64 bits."""
    return torch.rsqrt(v.square().mean(-1) + EPS)


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std + mean).to(to)

    if case["kind"] == "norm":
        seqs, tokens, width = case["seqs"], case["tokens"], case["width"]
        # A residual stream, a few features far larger than the others, and what a half of the block adds to it.
        x = torch.randn(seqs, tokens, width, generator=g, device=DEVICE) * 2.0
        x[..., :: max(1, width // 4)] *= 12.0
        s = {"x": x.to(dtype), "y": normal(seqs, tokens, width, std=0.7), "weight": normal(width, std=0.2, mean=1.0)}
        s["post_weight"] = normal(width, std=0.2, mean=1.0) if case["post"] else None
        shape = {"none": None, "channel": (width,), "sequence": (seqs, 1, width), "token": (seqs, tokens, width)}[case["gate"]]
        s["gate"] = None if shape is None else normal(*shape, std=0.5, mean=0.5)
        if case["backward"]:  # as the forward pass left them
            b = s["y"].double()
            s["post_rstd"] = None
            if case["post"]:
                rstd = _rms(b)
                s["post_rstd"], b = rstd.float(), b * rstd[..., None] * s["post_weight"].double()
            if s["gate"] is not None:
                b = b * s["gate"].double()
            stream = s.pop("x").double() + case["scale"] * b
            s["stream"], s["rstd"] = stream.to(dtype), _rms(stream).float()
            s["dstream"], s["dnormed"] = normal(seqs, tokens, width), normal(seqs, tokens, width)
        return s
    if case["kind"] == "gated":
        m, inter, hidden = case["m"], case["inter"], case["hidden"]
        s = {"x": normal(m, hidden), "gate_up": normal(2 * inter, hidden, std=hidden**-0.5), "bias": normal(2 * inter, std=0.5) if case["bias"] else None}
        if case["backward"]:
            pre = torch.mm(s["x"], s["gate_up"].t())  # as the forward pass left them
            s["pre"] = pre if s["bias"] is None else pre + s["bias"]
            s["dh"] = normal(m, inter)
        return s
    m, count, rank, n, k = case["m"], case["adapters"], case["rank"], case["n"], case["k"]
    requests = _requests(case, seed)
    ids = [a for first, last, a in requests for _ in range(last - first)]
    return {"x": normal(m, k), "base": normal(m, n), "a": normal(count, rank, k, std=k**-0.5), "b": normal(count, n, rank, std=0.3 * rank**-0.5),
            "alpha": torch.rand(count, generator=g, device=DEVICE) * 1.5 + 0.5, "ids": torch.tensor(ids, dtype=torch.int32).to(DEVICE), "spans": requests}  # fmt: skip


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    if own and case["kind"] == "adapter":
        from neuropress_amd import kernels

        s["handle"] = kernels.LowRankAdapters(s["a"], s["b"], s["alpha"])
    return s


# ----------------------------------------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    return {"norm": _norm_plain, "gated": _gated_plain, "adapter": _adapter_plain}[s["kind"]](s)


def _own(s):
    from neuropress_amd import kernels

    if s["kind"] == "norm":
        if s["backward"]:
            out = kernels.residual_norm_backward(s["dstream"], s["dnormed"], s["y"], s["stream"], s["weight"], s["post_weight"], s["gate"], s["scale"],
                                                 s["post_rstd"], s["rstd"])  # fmt: skip
            return [t for t in out if t is not None]
        return kernels.residual_norm(s["x"], s["y"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], scale=s["scale"], eps=EPS)
    if s["kind"] == "gated":
        if s["backward"]:
            out = kernels.gated_linear_backward(s["dh"], s["x"], s["gate_up"], s["pre"], s["act"], needs=(True, True, s["bias"] is not None))
            return [t for t in out if t is not None]
        return kernels.gated_linear(s["x"], s["gate_up"], bias=s["bias"], activation=s["act"])
    return kernels.adapter_linear(s["x"], s["handle"], s["ids"], s["base"])


def _sum_to(t, shape):
    """The sums of *t* over what *shape* does not have, in 64 bits: thousands of rows of either sign."""
    lead = [i for i in range(t.dim() - 1) if len(shape) < t.dim() or shape[i] == 1]
    return t.sum(lead, dtype=torch.float64).reshape(shape) if lead else t


def _norm_plain(s):
    to, w, y, scale = s["y"].dtype, s["weight"].float(), s["y"].float(), s["scale"]
    wp = None if s["post_weight"] is None else s["post_weight"].float()
    gate = None if s["gate"] is None else s["gate"].float()
    if not s["backward"]:
        if wp is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * wp
        if gate is not None:
            y = y * gate
        r = s["x"].float() + scale * y
        return r.to(to), (r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * w).to(to)
    dz, rstd = s["dnormed"].float(), s["rstd"][..., None]
    rh = s["stream"].float() * rstd
    v = dz * w
    dr = s["dstream"].float() + rstd * (v - rh * (v * rh).mean(-1, keepdim=True))
    out = [dr.to(to), None, _sum_to(dz * rh, w.shape).to(to)]
    db = scale * dr
    bh = y if wp is None else y * s["post_rstd"][..., None]
    if gate is not None:
        dgate = _sum_to(db * (bh if wp is None else bh * wp), gate.shape).to(to)
        db = db * gate
    if wp is not None:
        out.append(_sum_to(db * bh, wp.shape).to(to))
        v = db * wp
        db = s["post_rstd"][..., None] * (v - bh * (v * bh).mean(-1, keepdim=True))
    out[1] = db.to(to)
    return out if gate is None else [*out, dgate]


def _act(name, v):
    """The activation and its derivative."""
    if name == "relu":
        return torch.maximum(v, torch.zeros_like(v)), (v > 0).float()
    if name == "gelu":
        phi = 0.5 * (1.0 + torch.erf(v * 0.7071067811865476))
        return v * phi, phi + v * torch.exp(-0.5 * v * v) * 0.3989422804014327
    if name == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v))
        return 0.5 * v * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * v * v)
    p = 1.0 / (1.0 + torch.exp(-v))
    return v * p, p * (1.0 + v * (1.0 - p))


def _gated_plain(s):
    x, w, to = s["x"].float(), s["gate_up"].float(), s["x"].dtype
    if not s["backward"]:
        pre = torch.mm(x, w.t())
        if s["bias"] is not None:
            pre = pre + s["bias"].float()
        gate, up = pre.chunk(2, -1)
        return (_act(s["act"], gate)[0] * up).to(to)
    gate, up = s["pre"].float().chunk(2, -1)
    dh = s["dh"].float()
    value, slope = _act(s["act"], gate)
    dpre = torch.cat((dh * up * slope, dh * value), -1)
    out = [torch.mm(dpre, w).to(to), torch.mm(dpre.t(), x).to(to)]
    if s["bias"] is not None:
        out.append(dpre.sum(0, dtype=torch.float64).to(to))
    return out


def _adapter_plain(s):
    x, base, a, b = s["x"], s["base"], s["a"], s["b"]
    if s["m"] <= 64 and s["m"] * s["rank"] * max(s["n"], s["k"]) <= 1 << 28:  # each token with weights of its own
        ids = s["ids"].long()
        met = ids.clamp(min=0)
        t = (a[met].float() * x.float()[:, None, :]).sum(-1)
        delta = (b[met].float() * t[:, None, :]).sum(-1) * (s["alpha"][met] * (ids >= 0))[:, None]
        return (base.float() + delta).to(x.dtype)
    out = torch.empty_like(base)
    for first, last, i in s["spans"]:
        rows = base[first:last].float()
        if i >= 0:
            rows = rows + s["alpha"][i] * torch.mm(torch.mm(x[first:last].float(), a[i].float().t()), b[i].float().t())
        out[first:last] = rows.to(x.dtype)
    return out


# ----------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without, and its value in 64 bits
# ----------------------------------------------------------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "norm":
        rows, width = case["seqs"] * case["tokens"], case["width"]
        n = rows * width
        gate = {"none": 0, "channel": width, "sequence": case["seqs"] * width, "token": n}[case["gate"]]
        weights = width * (2 if case["post"] else 1)
        if case["backward"]:
            return {"bytes": size * (6.0 * n + 2 * weights + 2 * gate) + 4.0 * rows * (2 if case["post"] else 1), "flops": (30.0 if case["post"] else 18.0) * n}
        return {"bytes": size * (4.0 * n + weights + gate), "flops": (13.0 if case["post"] else 8.0) * n}
    if case["kind"] == "gated":
        m, inter, hidden = case["m"], case["inter"], case["hidden"]
        bias = 2 * inter if case["bias"] else 0
        if case["backward"]:
            return {"bytes": size * (3.0 * m * inter + 2.0 * m * hidden + 4.0 * inter * hidden + bias), "flops": 8.0 * m * inter * hidden}
        return {"bytes": size * (1.0 * m * hidden + 2.0 * inter * hidden + 1.0 * m * inter + bias), "flops": 4.0 * m * inter * hidden}
    m, count, requests, rank, n, k = (case[name] for name in ("m", "adapters", "requests", "rank", "n", "k"))
    some = 1.0 if requests == 1 else 0.875  # of the requests have an adapter
    met = count * (1.0 - (1.0 - 1.0 / count) ** (some * requests))  # adapters that they meet, on average
    return {"bytes": size * (some * m * k + 2.0 * m * n + met * rank * (n + k)) + 4.0 * (m + met), "flops": 2.0 * some * m * rank * (n + k)}


def _leaf(t):
    return None if t is None else t.double().requires_grad_(True)


def exact(case, seed):
    s = _inputs(case, seed)
    f = torch.nn.functional
    if case["kind"] == "norm":
        if not case["backward"]:
            b = s["y"].double()
            if case["post"]:
                b = f.rms_norm(b, (case["width"],), s["post_weight"].double(), EPS)
            r = s["x"].double() + case["scale"] * b * (1.0 if s["gate"] is None else s["gate"].double())
            return r, f.rms_norm(r, (case["width"],), s["weight"].double(), EPS)
        # The Jacobian of v * rstd(v) is (I - vh vh^T / n) * rstd, vh = v * rstd; the sums over rows as products with ones.
        n = case["width"]

        def through(v, vh, rstd):
            return (v - vh * (torch.linalg.vecdot(v, vh) / n).unsqueeze(-1)) * rstd

        def total(t, like):
            if like.dim() == 1:
                return torch.ones(t.shape[0] * t.shape[1], dtype=torch.float64, device=DEVICE) @ t.reshape(-1, n)
            return t.sum(1, keepdim=True) if like.shape[1] == 1 else t

        rstd = s["rstd"].double().unsqueeze(-1)
        rh = s["stream"].double() * rstd
        dr = s["dstream"].double() + through(s["dnormed"].double() * s["weight"].double(), rh, rstd)
        dweight = total(s["dnormed"].double() * rh, s["weight"])
        y = s["y"].double()
        gate = torch.ones((), dtype=torch.float64, device=DEVICE) if s["gate"] is None else s["gate"].double()
        out, tail = [dr], []
        if case["post"]:
            post_rstd, wp = s["post_rstd"].double().unsqueeze(-1), s["post_weight"].double()
            yh = y * post_rstd
            out += [through(case["scale"] * dr * gate * wp, yh, post_rstd), dweight, total(case["scale"] * dr * gate * yh, s["post_weight"])]
            b = yh * wp
        else:
            out += [case["scale"] * dr * gate, dweight]
            b = y
        if s["gate"] is not None:
            tail = [total(case["scale"] * dr * b, s["gate"])]
        return out + tail
    if case["kind"] == "gated":
        act = {"relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"), "silu": f.silu}[case["act"]]
        if not case["backward"]:
            inter = case["inter"]
            bias = [None, None] if s["bias"] is None else [s["bias"][:inter].double(), s["bias"][inter:].double()]
            x = s["x"].double()
            return act(f.linear(x, s["gate_up"][:inter].double(), bias[0])) * f.linear(x, s["gate_up"][inter:].double(), bias[1])
        pre = _leaf(s["pre"])
        gate, up = pre.chunk(2, -1)
        dpre = torch.autograd.grad(act(gate) * up, pre, s["dh"].double())[0]
        out = [dpre @ s["gate_up"].double(), dpre.T @ s["x"].double()]
        return out if s["bias"] is None else [*out, torch.ones(case["m"], dtype=torch.float64, device=DEVICE) @ dpre]
    y = s["base"].double()
    for i in range(case["adapters"]):
        rows = (s["ids"] == i).nonzero()[:, 0]
        if rows.numel():
            y[rows] += s["alpha"][i].double() * f.linear(f.linear(s["x"][rows].double(), s["a"][i].double()), s["b"][i].double())
    return y
