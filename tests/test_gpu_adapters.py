"""Low-rank adapters of many requests against the formula in 64 bits.

Tolerances: half a step of the output type, plus what f32 adds: a sum of K products is off by at most n 2^-24 of the sum of their absolute values, n = K / 16 + 40; x A^T is held to 2^-16 of itself
with bfloat16, with float16 to 2^-21 and 2^-28 of its row's largest value."""

import pytest
import torch

from tests import cases

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
U = 2.0**-24


def _make(m, n, k, rank, adapters, dtype, seed=0, scaled=True):
    g = cases.gen(seed + m + 7 * n + 13 * k + rank)
    make = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).to(dtype).cuda()
    a, b = make(adapters, rank, k, std=k**-0.5), make(adapters, n, rank, std=rank**-0.5)
    scale = (torch.rand(adapters, generator=g) * 2 + 0.25).cuda() if scaled else None
    return make(m, k), a, b, scale, make(m, n)


def _ids(m, adapters, how, seed=0):
    g = cases.gen(seed + m)
    ids = torch.randint(-1, adapters, (m,), generator=g)
    if how == "runs":
        ids = ids.sort().values
        ids = torch.cat((ids[m // 3 :], ids[: m // 3]))
    elif how == "one":
        ids[:] = adapters - 1
    elif how == "none":
        ids[:] = -1
    elif how == "odd":  # numbers that are no adapter's
        ids = torch.where(torch.rand(m, generator=g) < 0.5, ids, torch.tensor([-(2**31), -2, adapters, 2**31 - 1])[torch.randint(0, 4, (m,), generator=g)])
    return ids.int().cuda()


def _check(x, a, b, scale, base, ids, y, what=""):
    dtype = x.dtype
    m, k = x.shape
    rank = a.shape[1]
    ref = torch.zeros(m, b.shape[1], dtype=torch.float64, device="cuda") if base is None else base.double()
    tol = ref.abs() * 2 * U
    assert y.dtype == dtype and y.shape == ref.shape
    none = (ids < 0) | (ids >= a.shape[0])
    assert torch.equal(y[none], torch.zeros_like(y[none]) if base is None else base[none]), f"{what}: tokens without an adapter"
    for i in ids.unique().tolist():
        if not 0 <= i < a.shape[0]:
            continue
        rows = ids == i
        xd, ad, bd, s = x[rows].double(), a[i].double(), b[i].double(), 1.0 if scale is None else scale[i].double()
        t = xd @ ad.T
        et = (k / 16 + 40) * U * (xd.abs() @ ad.abs().T)
        if dtype == torch.bfloat16:
            et = et + 2.0**-16 * t.abs()
        else:
            et = et + 2.0**-21 * t.abs() + 2.0**-28 * t.abs().amax(-1, keepdim=True)
        delta = s * (t @ bd.T)
        ref[rows] += delta
        tol[rows] += s * (et @ bd.abs().T + (rank / 16 + 40) * U * (t.abs() @ bd.abs().T)) + 3 * U * delta.abs()
    eps = torch.finfo(dtype).eps
    bad = (y.double() - ref).abs() / (tol + ref.abs() * (eps / 2) * 1.0001 + torch.finfo(dtype).smallest_normal * eps / 2)
    assert bool((bad <= 1).all()), f"{what}: {bad.max().item():.2f} of the tolerance"


def _run(x, a, b, scale, ids, base):
    from neuropress_amd import kernels

    return kernels.adapter_linear(x, kernels.LowRankAdapters(a, b, scale), ids, base)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["any", "runs", "one", "none", "odd"])
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 33, 63, 64, 65, 100, 129, 300, 1100])
def test_tokens(gpu, dtype, how, m):
    x, a, b, scale, base = _make(m, 200, 136, 16, 7, dtype)
    ids = _ids(m, 7, how)
    for s in (scale, None):
        for r in (base, None):
            _check(x, a, b, s, r, ids, _run(x, a, b, s, ids, r), f"scale {s is not None} base {r is not None}")
    assert torch.equal(_run(x, a, b, scale, ids, base), _run(x, a, b, scale, ids.long(), base)), "the same inputs, other bits"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 40, 70, 200])
@pytest.mark.parametrize("rank", [1, 4, 8, 12, 16, 24, 31, 32, 33, 40, 48, 64, 72, 100, 128, 136, 200, 256])
def test_ranks(gpu, dtype, m, rank):
    x, a, b, scale, base = _make(m, 150, 264, rank, 5, dtype)
    ids = _ids(m, 5, "any")
    _check(x, a, b, scale, base, ids, _run(x, a, b, scale, ids, base))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [2, 20, 90])
@pytest.mark.parametrize("n,k", [(1, 1), (7, 5), (8, 8), (64, 9), (65, 31), (63, 33), (72, 1000), (1001, 40), (130, 4095), (70, 4104), (640, 14336), (14336, 640)])
def test_sizes(gpu, dtype, m, n, k):
    x, a, b, scale, base = _make(m, n, k, 8, 6, dtype)
    ids = _ids(m, 6, "any")
    _check(x, a, b, scale, base, ids, _run(x, a, b, scale, ids, base))


@pytest.mark.parametrize("m,n,k,rank,adapters,how", [(1, 4096, 4096, 16, 8, "one"), (32, 14336, 4096, 16, 64, "any"), (4096, 2048, 1024, 64, 16, "runs"), (4096, 4096, 512, 128, 3, "any"),
                                                     (5000, 72, 136, 8, 8192, "any"), (50, 72, 136, 8, 8192, "any"), (3000, 640, 2048, 256, 2, "runs")])  # fmt: skip
def test_large(gpu, m, n, k, rank, adapters, how):
    x, a, b, scale, base = _make(m, n, k, rank, adapters, torch.bfloat16)
    ids = _ids(m, adapters, how)
    y = _run(x, a, b, scale, ids, base)
    _check(x, a, b, scale, base, ids, y)
    for _ in range(3):
        assert torch.equal(_run(x, a, b, scale, ids, base), y), "the same inputs, other bits"


@pytest.mark.parametrize("m", [3, 64, 65, 200])
def test_a_tokens_result_is_its_own(gpu, m):
    """Whatever the other tokens are and wherever it stands."""
    x, a, b, scale, base = _make(m, 300, 520, 16, 4, torch.bfloat16)
    ids = _ids(m, 4, "any")
    y = _run(x, a, b, scale, ids, base)
    order = torch.randperm(m, generator=cases.gen(m)).cuda()
    assert torch.equal(_run(x[order], a, b, scale, ids[order], base[order]), y[order])


@pytest.mark.parametrize("m", [3, 40, 130])
def test_rows_at_any_distance_and_address(gpu, m):
    x, a, b, scale, base = _make(m, 139, 203, 16, 4, torch.float16)
    ids = _ids(m, 4, "any")
    y = _run(x, a, b, scale, ids, base)

    def spread(v, at, room):
        wide = torch.full((v.shape[0], v.shape[1] + room), float("nan"), device="cuda", dtype=v.dtype)
        wide[:, at : at + v.shape[1]] = v
        return wide[:, at : at + v.shape[1]]

    for at, room in ((0, 5), (1, 13), (3, 8)):
        assert torch.equal(_run(spread(x, at, room), a, b, scale, ids, spread(base, at, room)), y)
    assert torch.equal(_run(x, a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(0, 1).contiguous().transpose(0, 1), scale, ids, base), y)


def test_ids_of_sequences(gpu):
    from neuropress_amd import kernels

    x, a, b, scale, base = _make(60, 72, 64, 8, 4, torch.bfloat16)
    adapters = kernels.LowRankAdapters(a, b, scale)
    ids = torch.tensor([2, -1, 0], device="cuda")
    want = kernels.adapter_linear(x, adapters, ids.repeat_interleave(20), base)
    assert torch.equal(kernels.adapter_linear(x.view(3, 20, 64), adapters, ids, base.view(3, 20, 72)).view(60, 72), want)
    assert torch.equal(kernels.adapter_linear(x.view(3, 4, 5, 64), adapters, ids[:, None].expand(3, 4), base.view(3, 4, 5, 72)).view(60, 72), want)
    assert torch.equal(kernels.adapter_linear(x[0], adapters, ids[0], base[0]), want[0])
    assert kernels.adapter_linear(x[:0], adapters, ids[:0], base[:0]).shape == (0, 72)


def test_output_in_the_place_of_the_base(gpu):
    from neuropress_amd import _lib

    for m in (5, 100):
        x, a, b, scale, base = _make(m, 77, 64, 16, 4, torch.bfloat16)
        ids = _ids(m, 4, "any")
        y = _run(x, a, b, scale, ids, base)
        need = _lib.load().npamd_adapter_linear_workspace_bytes(m, 77, 64, 16, 4)
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        wide = torch.full((m, 90), 3.0, device="cuda", dtype=torch.bfloat16)
        wide[:, :77] = base
        _lib.call("npamd_adapter_linear", x.data_ptr(), 64, ids.data_ptr(), 32, a.data_ptr(), b.data_ptr(), scale.data_ptr(), wide.data_ptr(), 90, wide.data_ptr(), 90, m, 77, 64, 16, 4,
                  _lib.BF16, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)  # fmt: skip
        assert torch.equal(wide[:, :77], y) and bool((wide[:, 77:] == 3.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [4, 70])
def test_special_values(gpu, dtype, m):
    """Large, tiny and infinite values of x A^T, infinite weights, and what other tokens and adapters hold."""
    big = 3e4 if dtype == torch.float16 else 1e30
    x, a, b, scale, base = _make(m, 80, 64, 16, 3, dtype)
    ids = torch.arange(m, device="cuda", dtype=torch.int32) % 3
    x[0], x[1], x[2] = big, 1e-6, 0.0
    a.abs_()
    b.abs_()
    b[0, 5, 3] = float("inf")
    b[1, 7, 0] = float("nan")
    x[3, 0] = float("inf")
    y = _run(x, a, b, scale, ids, torch.zeros_like(base))
    finite = torch.ones_like(y, dtype=torch.bool)
    finite[ids == 0, 5] = False
    finite[ids == 1, 7] = False
    finite[3] = False
    if dtype == torch.float16:
        finite[0] = False  # past the type's range
    assert bool(y[finite].isfinite().all()) and bool(y[ids == 1, 7].isnan().all())
    assert bool((y[0, 5] == float("inf")).all()) and bool(y[3].isinf().all())
    live = [i for i in range(1, m) if i != 3 and i % 3 != 1]
    bb = b.clone()
    bb[0, 5, 3] = 0.0
    z = _run(x, a, bb, scale, ids, torch.zeros_like(base))
    keep = torch.arange(80, device="cuda") != 5
    _check(x[live], a, bb, scale, None, ids[live], z[live])
    assert torch.equal(z[live][:, keep], y[live][:, keep])


def test_module(gpu):
    from neuropress_amd.kernels import LowRankAdapters, adapter_linear
    from neuropress_amd.nn import NPAdapterLinear, attach_adapters, set_adapter_ids

    model = torch.nn.Sequential(torch.nn.Linear(256, 96), torch.nn.Linear(96, 64)).half().to(gpu)
    a = [LowRankAdapters(*_make(1, n, k, 8, 3, torch.float16)[1:4]) for n, k in ((96, 256), (64, 96))]
    x = torch.randn(6, 256, generator=cases.gen(7)).half().to(gpu)
    plain = model(x)
    assert attach_adapters(model, {"0": a[0], "1": a[1]}) == 2 and isinstance(model[0], NPAdapterLinear)
    assert torch.equal(model(x), plain)
    ids = torch.tensor([0, -1, 2, 1, 0, 5], device=gpu)
    set_adapter_ids(model, ids)
    with torch.no_grad():
        mid = adapter_linear(x, a[0], ids, model[0].base(x))
        want = adapter_linear(mid, a[1], ids, model[1].base(mid))
        assert torch.equal(model(x), want) and torch.equal(model[0](x, ids), mid)
    assert not torch.equal(want[0], plain[0])
    with pytest.raises(RuntimeError, match="inference only"):
        model(x.clone().requires_grad_())
    attach_adapters(model, {"0": a[0]})
    assert not isinstance(model[0].base, NPAdapterLinear)
    set_adapter_ids(model, None)
    assert torch.equal(model(x), plain)


def test_refusals(gpu):
    from neuropress_amd import kernels

    x, a, b, scale, base = _make(6, 72, 64, 8, 4, torch.float16)
    ids = _ids(6, 4, "any")
    for args, match in [((a.float(), b.float()), "float16 or bfloat16"), ((a, b.bfloat16()), "float16 or bfloat16"), ((a, b[:3]), "L, r, K"), ((a[0], b[0]), "L, r, K"),
                        ((a, b[:, :, :7]), "L, r, K"), ((a[:, :, :0], b), "at least one"), ((a, b, scale.half()), "scale"), ((a, b, scale[:3]), "scale"), ((a, b.cpu()), "GPU")]:  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            kernels.LowRankAdapters(*args)
    with pytest.raises(RuntimeError, match="up to 256"):
        kernels.LowRankAdapters(*_make(1, 8, 8, 257, 1, torch.float16)[1:3])
    with pytest.raises(RuntimeError, match="8192 adapters"):
        kernels.LowRankAdapters(a[:1].expand(8193, -1, -1), b[:1].expand(8193, -1, -1))
    ad = kernels.LowRankAdapters(a, b, scale)
    for args, match in [((x.bfloat16(), ad, ids, base), "x must be"), ((x[:, :32], ad, ids, base), "x must be"), ((x, ad, ids[:5], base), "ids"), ((x, ad, ids.float(), base), "ids"),
                        ((x, ad, ids[None], base), "ids"), ((x, ad, ids, base[:, :8]), "base"), ((x, ad, ids, base.float()), "base"), ((x, ad, ids.cpu(), base), "GPU"),
                        ((x.clone().requires_grad_(), ad, ids, base), "inference only")]:  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            kernels.adapter_linear(*args)
    narrow = kernels.LowRankAdapters(a[:, :, :5], b)
    with pytest.raises(RuntimeError, match="x must be"):
        kernels.adapter_linear(x[:, :8], narrow, ids, base)


def test_more_entries_than_rows_of_a_grid(gpu):
    """Entries of 32 tokens, more than 65535 of them."""
    m, adapters = 2_200_000, 5
    x, a, b, scale, base = _make(m, 8, 8, 136, adapters, torch.bfloat16)
    ids = _ids(m, adapters, "any")
    _check(x, a, b, scale, base, ids, _run(x, a, b, scale, ids, base))


@pytest.mark.parametrize("m", [4, 80])
def test_broadcast_inputs(gpu, m):
    """One row for all tokens, one number for all, and rows that lie the other way round."""
    from neuropress_amd import kernels

    x, a, b, scale, base = _make(m, 72, 64, 8, 4, torch.float16)
    ids = _ids(m, 4, "any")
    ad = kernels.LowRankAdapters(a, b, scale)
    for xs, bs, i in ((x[:1].expand(m, -1), base[:1].expand(m, -1), ids), (x.T.contiguous().T, base.T.contiguous().T, ids), (x, base, ids[:1].expand(m)), (x, base, torch.tensor(2, device=gpu))):
        y = kernels.adapter_linear(xs, ad, i, bs)
        _check(xs.contiguous(), a, b, scale, bs.contiguous(), i.expand(m).contiguous(), y)


@pytest.mark.parametrize("tokens", [1, 20, 90])
def test_module_beside_quantized_layers(gpu, tokens):
    """The base of a module is what its projection gives, int4 or codebook, whatever kernels take it."""
    from neuropress_amd.kernels import LowRankAdapters
    from neuropress_amd.nn import NPAdapterLinear, NPLinear

    q = cases.q4_layer(5, 96, 128)
    base = NPLinear(q["blob"], q["scale"], 96, 128, 32, 4, "sym", "cuda", compute_dtype=torch.float16).to(gpu)
    x, a, b, scale, _ = _make(tokens, 96, 128, 12, 3, torch.float16)
    layer = NPAdapterLinear(base, LowRankAdapters(a, b, scale))
    ids = _ids(tokens, 3, "any")
    with torch.no_grad():
        _check(x, a, b, scale, base(x), ids, layer(x, ids), "tokens")
        twice = x[None].expand(2, -1, -1)
        y, per_sequence = base(twice), layer(twice, torch.tensor([1, -1], device=gpu))  # of so many tokens: the projection's kernels may be others
    _check(x, a, b, scale, y[0], torch.ones_like(ids), per_sequence[0], "sequences")
    assert torch.equal(per_sequence[1], y[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,rank", [(1030, 8192 + 8, 128), (1030, 8192 + 3, 66), (4100, 4096, 100), (300, 4096, 128), (4100, 2048, 200)])
def test_wide_ranks_of_long_prompts(gpu, dtype, m, n, rank):
    """Both widths of a lane's columns past rank 64, entries of 32 to 128 tokens."""
    x, a, b, scale, base = _make(m, n, 72, rank, 5, dtype)
    for how in ("runs", "any"):
        ids = _ids(m, 5, how)
        _check(x, a, b, scale, base, ids, _run(x, a, b, scale, ids, base), how)


@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("rank", [8, 24, 60, 128, 200])
def test_small_values_beside_large_ones(gpu, m, rank):
    """float16, values of x A^T of one token 2^22 apart, and columns of y that meet only the small ones: x A^T is held to 2^-21 of each and 2^-37 of the token's largest."""
    k, n = 256, 136
    x, a, b, _, _ = _make(m, n, k, rank, 2, torch.float16)
    a = torch.cat((a[:, :1] * 2.0**10, a[:, 1:] * 2.0**-12), 1)
    b[:, ::2, 0] = 0.0
    ids = _ids(m, 2, "random")
    scale = torch.tensor([2.0**6, 2.0**7], device="cuda")
    y = _run(x, a, b, scale, ids, None)
    tried = 0
    for i in range(2):
        rows = ids == i
        xd, ad, bd = x[rows].double(), a[i].double(), b[i, ::2].double()
        t = xd @ ad.T
        et = (k / 16 + 40) * U * (xd.abs() @ ad.abs().T) + 2.0**-21 * t.abs() + 2.0**-37 * t.abs().amax(-1, keepdim=True)
        ref = scale[i].double() * (t @ bd.T)
        tol = scale[i].double() * (et @ bd.abs().T + (rank / 16 + 40) * U * (t[:, 1:].abs() @ bd[:, 1:].abs().T)) + 3 * U * ref.abs()
        eps = torch.finfo(torch.float16).eps
        bad = (y[rows, ::2].double() - ref).abs() / (tol + ref.abs() * (eps / 2) * 1.0001 + torch.finfo(torch.float16).smallest_normal * eps / 2)
        assert bool((bad <= 1).all()), f"{bad.max().item():.2f} of the tolerance"
        tried += int(rows.sum())
    assert tried
