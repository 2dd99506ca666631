"""The mixture-of-experts layer against the formulas in 64 bits.

Tolerances: half a step of the output type; the rounding of silu(gate) * up, half a step e / 2 of each value, independent of each other: eight standard deviations of
their sum through the down-projection, 8 (e / 2) / sqrt(3) sqrt(sum (p w h)^2); what f32 adds to sums of n terms, n 2^-24 of the sum of magnitudes with n at
most K / 16 + 40 -- for codes times 2^7, as they are summed with an offset of up to 128 times their spread."""

import pytest
import torch

from neuropress_amd.t2n.packing import BitPacking
from tests import cases

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
FORMATS = [(16, 32, False), (4, 32, False), (4, 128, True), (8, 64, False), (8, 32, True), (4, 64, False)]


def _layer(seed, e, h, i, dtype, nbits, group=32, zero=False):
    g = cases.gen(seed)
    layer = {"router": (torch.randn(e, h, generator=g) * 2 * h**-0.5).to(dtype), "nbits": nbits, "group_size": group}
    dense = {}
    for name, rows, cols in (("gate_up", 2 * i, h), ("down", h, i)):
        if nbits == 16:
            layer[name] = (torch.randn(e, rows, cols, generator=g) * cols**-0.5).to(dtype)
            dense[name] = layer[name].double()
            continue
        codes = torch.randint(0, 1 << nbits, (e * rows, cols), generator=g, dtype=torch.int64).to(torch.uint8)
        layer[name] = BitPacking(nbits).compress(codes).reshape(e, rows, -1)
        s = ((torch.rand(e, rows, cols // group, generator=g) + 0.5) * 3.5 / (1 << nbits) * cols**-0.5).half()
        layer[name + "_scale"] = s
        z = torch.full_like(s, float(1 << (nbits - 1)))
        if zero:
            z = layer[name + "_zero"] = (torch.randn(e, rows, cols // group, generator=g) * (1 << nbits) / 16 + (1 << (nbits - 1))).half()
        wide = lambda t: t.double().repeat_interleave(group, -1)
        dense[name] = (codes.reshape(e, rows, cols).double() - wide(z)) * wide(s)
    return layer, dense


def _experts(layer):
    from neuropress_amd import kernels

    return kernels.MoEExperts(**{k: v.to("cuda") if isinstance(v, torch.Tensor) else v for k, v in layer.items()})


def _reference(x, layer, dense, top_k, renormalize):
    """The result and how far f32 sums and the rounding of h may take it, all in 64 bits on the CPU."""
    xd, dtype = x.double(), x.dtype
    logits = xd @ layer["router"].double().T
    p = torch.softmax(logits, -1)
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top_k]
    p = p.gather(1, order)
    if renormalize:
        p = p / p.sum(-1, keepdim=True)
    h, i = dense["down"].shape[1:]
    wide = 1.0 if layer["nbits"] == 16 else 128.0
    y, rounding, slack = (torch.zeros_like(xd) for _ in range(3))
    for m in range(x.shape[0]):
        for t in range(top_k):
            e = int(order[m, t])
            both, spread = dense["gate_up"][e] @ xd[m], dense["gate_up"][e].abs() @ xd[m].abs()
            gate, up = both[:i], both[i:]
            v = torch.nn.functional.silu(gate) * up
            dv = 2.0**-24 * wide * (h / 16 + 40) * (1.1 * spread[:i] * up.abs() + gate.abs() * spread[i:]) + 2.0**-20 * v.abs()
            w, share = dense["down"][e], p[m, t]
            y[m] += share * (w @ v)
            rounding[m] += share**2 * (w.square() @ v.square())
            # the router's own sum moves p by 2 n 2^-24 sum |x r| relative
            moved = 2.0**-23 * (h / 16 + 40) * (xd[m].abs() @ layer["router"][e].double().abs())
            slack[m] += share * (w.abs() @ (dv + 2.0**-24 * wide * (i / 16 + 40) * v.abs())) + moved * share * (w @ v).abs()
    eps = torch.finfo(dtype).eps
    return y, y.abs() * eps / 2 * 1.0001 + 8 * eps / 2 / 3**0.5 * rounding.sqrt() + slack + torch.finfo(dtype).smallest_normal * eps * (1 + i**0.5)


def _check(y, ref, tol, dtype):
    assert y.dtype == dtype and y.shape == ref.shape
    err = (y.double().cpu() - ref).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1, f"{worst:.2f} of the tolerance"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nbits,group,zero", FORMATS)
@pytest.mark.parametrize("m,top_k", [(1, 2), (2, 1), (7, 3), (16, 2), (17, 4), (32, 8)])
def test_formats_and_tokens(gpu, dtype, nbits, group, zero, m, top_k):
    from neuropress_amd import kernels

    e, h, i = 8, 256, 384
    layer, dense = _layer(m + nbits, e, h, i, dtype, nbits, group, zero)
    x = torch.randn(m, h, generator=cases.gen(m)).to(dtype)
    experts = _experts(layer)
    for renormalize in (True, False):
        y = kernels.moe_layer(x.to(gpu), experts, top_k, renormalize)
        _check(y, *_reference(x, layer, dense, top_k, renormalize), dtype)
    assert torch.equal(kernels.moe_layer(x.to(gpu), experts, top_k, False), y), "the same inputs, other bits"


@pytest.mark.parametrize("nbits,group,zero", FORMATS[:4])
@pytest.mark.parametrize("e,top_k,h,i,m", [(1, 1, 64, 64, 3), (1, 1, 128, 128, 32), (3, 3, 128, 640, 5), (64, 8, 384, 128, 9), (60, 4, 128, 1408, 2), (130, 5, 192, 192, 31),
                                           (512, 16, 128, 128, 4), (4, 2, 1152, 2304, 1)])  # fmt: skip
def test_sizes(gpu, nbits, group, zero, e, top_k, h, i, m):
    from neuropress_amd import kernels

    if nbits != 16 and (h % group or i % group):
        group = 64
    layer, dense = _layer(e, e, h, i, torch.bfloat16, nbits, group, zero)
    x = torch.randn(m, h, generator=cases.gen(m)).to(torch.bfloat16)
    _check(kernels.moe_layer(x.to(gpu), _experts(layer), top_k), *_reference(x, layer, dense, top_k, True), torch.bfloat16)


@pytest.mark.parametrize("nbits,group", [(16, 32), (4, 64)])
@pytest.mark.parametrize("m", [1, 8, 32])
def test_every_token_to_the_same_experts(gpu, nbits, group, m):
    """One row of tokens: two experts take all of them, the others none; then each token an expert of its own."""
    from neuropress_amd import kernels

    e, h, i = 32, 256, 256
    layer, dense = _layer(5, e, h, i, torch.float16, nbits, group)
    x = torch.randn(1, h, generator=cases.gen(9)).half()
    y = kernels.moe_layer(x.to(gpu).expand(m, h), _experts(layer), 2)
    _check(y, *(t.expand(m, h) for t in _reference(x, layer, dense, 2, True)), torch.float16)
    layer["router"] = torch.zeros(e, h).half()
    layer["router"][:, :e] = torch.eye(e).half()
    x = torch.randn(m, h, generator=cases.gen(9)).half()
    x[:, :e] = 0
    x[torch.arange(m), torch.arange(m)] = 12.0
    _check(kernels.moe_layer(x.to(gpu), _experts(layer), 1), *_reference(x, layer, dense, 1, True), torch.float16)


def test_ties_go_to_the_lower_index(gpu):
    from neuropress_amd import kernels

    e, h, i = 70, 128, 64
    layer, dense = _layer(6, e, h, i, torch.bfloat16, 16)
    for row in (torch.zeros(h), torch.ones(h) / 16):  # every expert has the same logit, zero or not
        layer["router"] = row.to(torch.bfloat16).expand(e, h).contiguous()
        x = torch.randn(4, h, generator=cases.gen(2)).to(torch.bfloat16)
        for top_k in (1, 5, 16):
            _check(kernels.moe_layer(x.to(gpu), _experts(layer), top_k, False), *_reference(x, layer, dense, top_k, False), torch.bfloat16)


def test_values_that_are_not_finite_stay_where_they_are(gpu):
    from neuropress_amd import kernels

    for nbits in (16, 4):
        layer, dense = _layer(7, 8, 128, 128, torch.float16, nbits)
        x = torch.randn(6, 128, generator=cases.gen(4)).half()
        clean = kernels.moe_layer(x.to(gpu), _experts(layer), 2)
        order = torch.sort(x.double() @ layer["router"].double().T, dim=-1, descending=True, stable=True).indices[:, :2]
        # an expert with infinite weights or scales reaches only the tokens that meet it
        bad = int(order[0, 0])
        if nbits == 16:
            layer["down"][bad, 3, 5] = float("inf")
        else:
            layer["down_scale"][bad, 3, 1] = float("inf")
        y = kernels.moe_layer(x.to(gpu), _experts(layer), 2).cpu()
        meets = (order == bad).any(-1)
        assert torch.equal(y[~meets], clean.cpu()[~meets]) and not y[meets][:, 3].isfinite().any()
        others = [c for c in range(128) if c != 3]
        assert torch.equal(y[:, others], clean.cpu()[:, others])
        # a token that is not a number: its own row, and it picks experts that exist
        x[2, 7] = float("nan")
        y = kernels.moe_layer(x.to(gpu), _experts(_layer(7, 8, 128, 128, torch.float16, nbits)[0]), 2).cpu()
        assert y[2].isnan().all() and torch.equal(y[[0, 1, 3, 4, 5]], clean.cpu()[[0, 1, 3, 4, 5]])


def test_shapes_strides_and_no_tokens(gpu):
    from neuropress_amd import kernels

    layer, dense = _layer(8, 8, 128, 192, torch.bfloat16, 4)
    experts = _experts(layer)
    x = torch.randn(2, 6, 128, generator=cases.gen(1)).to(torch.bfloat16).to(gpu)
    y = kernels.moe_layer(x, experts, 2)
    assert y.shape == x.shape and torch.equal(y.view(12, 128), kernels.moe_layer(x.view(12, 128), experts, 2))
    assert torch.equal(kernels.moe_layer(x[0, 0], experts, 2), kernels.moe_layer(x[0, :1], experts, 2)[0])
    assert kernels.moe_layer(x[:, :0], experts, 2).shape == (2, 0, 128)
    wide = torch.full((12, 136 + 3), float("nan"), dtype=torch.bfloat16, device=gpu)
    for ld in (136, 139):
        view = wide.view(-1)[: 12 * ld].view(12, ld)[:, :128]
        view.copy_(x.view(12, 128))
        assert torch.equal(kernels.moe_layer(view, experts, 2), y.view(12, 128))
        wide.fill_(float("nan"))
    odd = torch.empty(12 * 128 + 1, dtype=torch.bfloat16, device=gpu)[1:].view(12, 128)  # rows between two 16-byte addresses
    odd.copy_(x.view(12, 128))
    assert torch.equal(kernels.moe_layer(odd, experts, 2), y.view(12, 128))

    def shifted(v):
        if not isinstance(v, torch.Tensor):
            return v
        return torch.cat([v.reshape(-1)[:1], v.reshape(-1)]).to(gpu)[1:].view(v.shape)

    assert torch.equal(kernels.moe_layer(x, kernels.MoEExperts(**{k: shifted(v) for k, v in layer.items()}), 2), y)


def test_refusals(gpu):
    from neuropress_amd import kernels

    layer, _ = _layer(1, 4, 128, 128, torch.float16, 4)
    experts = _experts(layer)
    x = torch.randn(2, 128, device=gpu).half()
    with pytest.raises(RuntimeError, match="at most 32 tokens"):
        kernels.moe_layer(x[:1].expand(33, 128), experts, 2)
    for top_k in (0, 5, -1, (1 << 32) + 2):
        with pytest.raises(RuntimeError, match="bad shape"):
            kernels.moe_layer(x, experts, top_k)
    with pytest.raises(RuntimeError, match="x must be"):
        kernels.moe_layer(x.float(), experts, 2)
    with pytest.raises(RuntimeError, match="x must be"):
        kernels.moe_layer(x[:, :64], experts, 2)
    with pytest.raises(RuntimeError, match="inference only"):
        kernels.moe_layer(x.clone().requires_grad_(), experts, 2)
    odd = {k: v.to(gpu) if isinstance(v, torch.Tensor) else v for k, v in layer.items()}
    with pytest.raises(RuntimeError, match="scales"):
        kernels.MoEExperts(**{**odd, "down_scale": None})
    with pytest.raises(RuntimeError, match="must be"):
        kernels.MoEExperts(**{**odd, "down": odd["down"][:, :64].contiguous()})
    with pytest.raises(RuntimeError, match="zero points"):
        kernels.MoEExperts(**odd, gate_up_zero=odd["gate_up_scale"])
    with pytest.raises(RuntimeError, match="nbits"):
        kernels.MoEExperts(**{**odd, "nbits": 2})
    dense, _ = _layer(1, 4, 96, 128, torch.float16, 16)
    with pytest.raises(RuntimeError, match="multiples of 64"):
        kernels.moe_layer(x[:, :96], _experts(dense), 2)


@pytest.mark.parametrize("m,experts,top_k", [(9, 9, 4), (10, 9, 4), (16, 8, 2), (17, 8, 2), (32, 32, 4), (32, 31, 4), (5, 20, 4), (5, 19, 4), (32, 128, 4)])
@pytest.mark.parametrize("nbits", [4, 8, 16])
def test_all_tokens_meet_in_the_same_experts(gpu, nbits, m, experts, top_k):
    """More tokens at an expert than one pass over its weights takes, on both sides of the number of pairs from which a pass takes more."""
    from neuropress_amd import kernels

    layer, dense = _layer(m + experts, experts, 128, 192, torch.float16, nbits, 64, nbits == 8)
    x = torch.randn(m, 128, generator=cases.gen(m)).abs().half()  # positive, so the first experts' positive rows are far ahead
    layer["router"][:top_k] = layer["router"][:top_k].abs() + 0.05 * torch.arange(1, top_k + 1)[:, None]
    assert ((x.double() @ layer["router"].double().T).topk(top_k).indices < top_k).all()
    _check(kernels.moe_layer(x.to(gpu), _experts(layer), top_k), *_reference(x, layer, dense, top_k, True), torch.float16)


@pytest.mark.parametrize("nbits,group,zero", [(4, 64, True), (8, 64, True), (8, 128, False), (16, 32, False)])
@pytest.mark.parametrize("e,top_k,h,i,m", [(2, 2, 256, 4480, 2), (14, 7, 128, 2688, 2), (4, 4, 640, 192, 19), (4, 4, 128, 128, 32), (6, 2, 2304, 128, 3), (6, 2, 1152, 128, 1),
                                           (8, 8, 64, 1024, 32)])  # fmt: skip
def test_few_row_tiles_many_columns_and_the_other_way_round(gpu, nbits, group, zero, e, top_k, h, i, m):
    """Columns in many parts, blocks of three waves, entries of sixteen pairs whose items are too few to share tokens."""
    from neuropress_amd import kernels

    if nbits != 16 and (h % group or i % group):
        group = 64
    layer, dense = _layer(e + m, e, h, i, torch.float16, nbits, group, zero)
    x = torch.randn(m, h, generator=cases.gen(m)).half()
    _check(kernels.moe_layer(x.to(gpu), _experts(layer), top_k), *_reference(x, layer, dense, top_k, True), torch.float16)


@pytest.mark.parametrize("e,top_k", [(1, 1), (2, 1), (16, 1), (17, 1), (32, 2), (33, 2), (63, 4), (64, 4), (64, 3), (65, 5), (64, 16), (128, 8)])
def test_routing(gpu, e, top_k):
    """Equal logits go to the lower index, NaN above all, infinities in their order; shares against the softmax in 64 bits.  Expert k answers in column k % 64,
    so y tells which experts were met, at which share."""
    from neuropress_amd import kernels

    h = i = 64
    g = cases.gen(e + top_k)
    router = torch.zeros(e, h).half()
    router[:, :4] = torch.randint(-2, 3, (e, 4), generator=g).half()  # sums of small whole numbers: many equal logits
    gate_up, down = torch.zeros(e, 2 * i, h).half(), torch.zeros(e, h, i).half()
    gate_up[:, 0, 4], gate_up[:, i, 4] = 4.0, 1.0
    down[:, torch.arange(64), 0] = 0
    down[torch.arange(e), torch.arange(e) % 64, 0] = 1.0
    x = torch.zeros(7, h).half()
    x[:, :4] = torch.randint(-1, 2, (7, 4), generator=g).half()
    x[:, 4] = 1.0
    layer = kernels.MoEExperts(router.to(gpu), gate_up.to(gpu), down.to(gpu))
    logits = x.double() @ router.double().T
    p = torch.softmax(logits, -1)
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top_k]
    answer = float(torch.nn.functional.silu(torch.tensor(4.0, dtype=torch.float64)))
    for renormalize in (True, False):
        share = p.gather(1, ids)
        share = share / share.sum(-1, keepdim=True) if renormalize else share
        want = torch.zeros(7, h, dtype=torch.float64)
        for m in range(7):
            for t in range(top_k):
                want[m, ids[m, t] % 64] += share[m, t] * answer
        y = kernels.moe_layer(x.to(gpu), layer, top_k, renormalize).double().cpu()
        # silu(4) and y are rounded to half a step each, 2^-11, f32 far less
        assert bool(((y - want).abs() <= 2.0**-9.9 * want + 2.0**-24).all())
    bad = router.clone()
    bad[e - 1, 5] = float("nan")  # this expert's logit is NaN whatever x holds: it is met first and every share is NaN
    y = kernels.moe_layer(x.to(gpu), kernels.MoEExperts(bad.to(gpu), gate_up.to(gpu), down.to(gpu)), top_k)
    assert bool(y.isnan().all(0)[(e - 1) % 64])


def _single_products(m, e, dtype, nbits, zero):
    """One expert takes all tokens; token t has one value that is not zero, in column t, and row t of the expert's gate and up rows meets nothing else: y[t, n] is one
    product of a weight and silu(gate) * up."""
    h = i = 64
    g = cases.gen(m + nbits + e)
    rand = lambda *s: torch.rand(*s, generator=g)
    sign = lambda *s: torch.randint(0, 2, s, generator=g) * 2 - 1
    x = torch.zeros(m, h, dtype=dtype)
    x[torch.arange(m), torch.arange(m)] = ((rand(m) + 0.5) * sign(m)).to(dtype)
    layer, dense = {"router": torch.zeros(e, h, dtype=dtype), "nbits": nbits, "group_size": 32}, {}
    for name, rows, cols in (("gate_up", 2 * i, h), ("down", h, i)):
        full = torch.ones(e, rows, cols, dtype=torch.bool) if name == "down" else (torch.arange(rows)[:, None] % i == torch.arange(cols)).expand(e, rows, cols)
        if nbits == 16:
            layer[name] = (torch.where(full, (rand(e, rows, cols) + 0.5) * sign(e, rows, cols), 0.0)).to(dtype)
            dense[name] = layer[name].double()
            continue
        half = 1 << (nbits - 1)
        codes = torch.where(full, half + sign(e, rows, cols) * torch.randint(half // 2, half, (e, rows, cols), generator=g), half).to(torch.uint8)
        layer[name] = BitPacking(nbits).compress(codes.reshape(e * rows, cols)).reshape(e, rows, -1)
        s = layer[name + "_scale"] = ((rand(e, rows, cols // 32) + 0.5) / half).half()
        if zero:
            layer[name + "_zero"] = torch.full_like(s, half)
        dense[name] = (codes.double() - half) * s.double().repeat_interleave(32, -1)
    return x, layer, dense


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nbits,zero", [(16, False), (4, False), (4, True), (8, False), (8, True)])
@pytest.mark.parametrize("m,e", [(1, 1), (3, 8), (5, 1), (9, 2), (32, 1), (32, 8)])
def test_the_hidden_values_are_not_rounded_to_sixteen_bits(gpu, dtype, nbits, zero, m, e):
    """y is rounded once.  What else there is: 2^-16 of the hidden values' two parts, 2^-20 of SiLU, and f32 sums of codes with an offset of up to 1032 on values of at
    least four, 2^-24 1032 / 4 = 2^-16 each for gate, up and down: 2^-13 is more than all of it."""
    from neuropress_amd import kernels

    x, layer, dense = _single_products(m, e, dtype, nbits, zero)
    both = x.double() @ dense["gate_up"][0].T
    ref = (torch.nn.functional.silu(both[:, :64]) * both[:, 64:]) @ dense["down"][0].T
    y = kernels.moe_layer(x.to(gpu), _experts(layer), 1).double().cpu()
    assert bool(((y - ref).abs() <= ref.abs() * (torch.finfo(dtype).eps / 2 * 1.0001 + 2.0**-13) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all())


@pytest.mark.parametrize("nbits,group,zero", FORMATS)
@pytest.mark.parametrize("m,e,top_k", [(1, 8, 2), (7, 8, 3), (32, 4, 2)])
def test_hidden_values_past_the_range_of_fp16(gpu, nbits, group, zero, m, e, top_k):
    """silu(gate) * up past 65504 where y is not."""
    from neuropress_amd import kernels

    layer, dense = _layer(m + nbits, e, 256, 384, torch.float16, nbits, group, zero)
    layer["gate_up" if nbits == 16 else "gate_up_scale"] *= 128  # exact
    dense["gate_up"] = dense["gate_up"] * 128
    x = torch.randn(m, 256, generator=cases.gen(m)).half()
    both = torch.einsum("erc,mc->emr", dense["gate_up"], x.double())
    assert (torch.nn.functional.silu(both[..., :384]) * both[..., 384:]).abs().max() > 65504
    ref, tol = _reference(x, layer, dense, top_k, True)
    y, inside = kernels.moe_layer(x.to(gpu), _experts(layer), top_k).cpu(), ref.abs() + tol < 65504  # a few results are past it themselves
    assert inside.double().mean() > 0.99 and not y.isnan().any()
    _check(y[inside], ref[inside], tol[inside], torch.float16)


@pytest.mark.parametrize("e,h,i", [(0, 64, 64), (2, 0, 64), (2, 64, 0)])
def test_experts_of_no_size_are_refused(gpu, e, h, i):
    from neuropress_amd import kernels

    with pytest.raises(RuntimeError, match="at least one expert"):
        kernels.MoEExperts(*(torch.zeros(*s, device=gpu).half() for s in ((e, h), (e, 2 * i, h), (e, h, i))))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["weight", "hidden"])
@pytest.mark.parametrize("m,top_k", [(1, 1), (5, 2), (32, 3)])
def test_infinite_weights_and_hidden_values(gpu, dtype, kind, m, top_k):
    """Dense experts: an infinite weight of the down-projection leaves an infinity of the product's sign, and so do weights that meet an infinite hidden value."""
    from neuropress_amd import kernels

    layer, _ = _layer(17, 4, 128, 128, dtype, 16)
    x = torch.randn(m, 128, generator=cases.gen(m)).to(dtype)
    x[:, 0] = 1.0
    down, gate_up = layer["down"], layer["gate_up"]
    down[down == 0] = 1.0
    if kind == "weight":
        down[:, 3, 5], down[:, 7, 9], down[:, 64:, 11] = float("inf"), float("-inf"), float("inf")
    else:
        gate_up[:, 20] = 0
        gate_up[:, 20, 0] = float("inf")
    logits = x.double() @ layer["router"].double().T
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top_k]
    p = torch.softmax(logits, -1).gather(1, order)
    ref = torch.zeros(m, 128, dtype=torch.float64)
    for t in range(m):
        for e, share in zip(order[t], p[t]):
            gate, up = (gate_up[e].double() @ x[t].double()).chunk(2)
            ref[t] += share * (down[e].double() @ (torch.nn.functional.silu(gate) * up))
    y = kernels.moe_layer(x.to(gpu), _experts(layer), top_k, False).double().cpu()
    assert ref.isinf().any() and torch.equal(y.isnan(), ref.isnan()) and torch.equal(y == float("inf"), ref == float("inf")) and torch.equal(y == float("-inf"), ref == float("-inf"))
