"""GPU: gpu_eigsh.features (embedding lookup, layer norm, edge distances) against the
definitions in 64 bits, elementwise, with error bounds counted from the arithmetic.

u = eps / 2 is the largest relative error of one rounding: ua of the accumulation
type (fp32, fp64 for fp64), ut of the element type.  A sum of n terms in any order
is off by at most n ua (1 + small) of the sum of the absolute values."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F64 = torch.float64
DT = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16, "bf16": torch.bfloat16}
SLACK = 1.01   # second-order terms of the bounds


@pytest.fixture(autouse=True)
def need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def acc(dt):
    return F64 if dt == F64 else torch.float32


def u(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Largest absolute error of a rounding that underflows."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dt, seed, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda", dtype=F64) * std + mean).to(dt)


def check(got, ref, bound, what=""):
    assert got.shape == ref.shape, (got.shape, ref.shape)
    d = (got.to(F64) - ref).abs()
    bad = ~(d <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / bound).max()):.3g} x"


# ---------------------------------------------------------------------------
# Embedding lookup
# ---------------------------------------------------------------------------
def make_ids(kind, rows, n, seed, dtype=torch.int64):
    g = gen(seed)
    if kind == "one":
        ids = torch.full((n,), rows // 2, device="cuda")
    elif kind == "zipf":
        x = torch.rand(n, generator=g, device="cuda", dtype=F64)
        ids = (torch.exp(x * math.log(rows + 1.0)).long() - 1).clamp_(0, rows - 1)
    else:
        ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    return ids.to(dtype)


def lookup_case(dt, rows, dim, n, kind, scale, pad=None, id_dtype=torch.int64, seed=0, out_of_range=False):
    """Runs forward and backward and checks all outputs."""
    from gpu_eigsh.features import embedding_lookup

    W = randn((rows, dim), dt, seed + 1).requires_grad_(True)
    ids = make_ids(kind, rows, n, seed + 2, id_dtype)
    if pad is not None and n > 1:
        ids[:: 3] = pad
    if out_of_range and n > 4:
        ids[1], ids[4] = -7, rows
    g = randn((n, dim), dt, seed + 3)
    f = None
    if scale == "number":
        f = 1.7
    elif scale == "column":
        f = randn((dim,), acc(dt), seed + 4).requires_grad_(True)
    y = embedding_lookup(W, ids, f, pad)
    assert y.dtype == dt
    leaves = [W] + ([f] if scale == "column" else [])
    grads = torch.autograd.grad(y, leaves, g)

    i64 = ids.long()
    is_pad = torch.zeros(n, dtype=torch.bool, device="cuda") if pad is None else i64 == pad
    ok = (i64 >= 0) & (i64 < rows) & ~is_pad
    s = torch.ones(dim, dtype=F64, device="cuda") if f is None else f.detach().to(F64) if scale == "column" else \
        torch.full((dim,), f, dtype=F64, device="cuda")
    Wd, gd = W.detach().to(F64), g.to(F64)
    safe = torch.where(ok, i64, 0)
    y_ref = Wd[safe] * s
    # the number rounded to the accumulation type, the product, the element type
    ua, ut = u(acc(dt)), u(dt)
    bound = y_ref.abs() * (2 * ua + ut) * SLACK + tiny(dt)
    if scale == "none":
        assert torch.equal(y.detach()[ok], W.detach()[safe][ok])
    check(y.detach()[ok], y_ref[ok], bound[ok], "y")
    assert bool((y.detach()[is_pad] == 0).all())
    assert bool(torch.isnan(y.detach()[~ok & ~is_pad]).all())

    at, gk = i64[ok], gd[ok]
    G = torch.zeros((rows, dim), dtype=F64, device="cuda").index_add_(0, at, gk)
    Ga = torch.zeros_like(G).index_add_(0, at, gk.abs())
    cnt = torch.bincount(at, minlength=rows).to(F64)[:, None]
    ref = G * s
    bound = (cnt * ua * Ga * s.abs() + ref.abs() * (2 * ua + ut)) * SLACK + tiny(dt)
    check(grads[0], ref, bound, "dW")
    assert bool((grads[0][cnt[:, 0] == 0] == 0).all())
    if scale == "column":
        m = int(ok.sum())
        ref = (Wd[at] * gk).sum(0)
        # a product, the sum of a row, the sum over rows and partial sums: at most m + 2 roundings on one path
        check(grads[1], ref, (m + 4) * ua * (Wd[at] * gk).abs().sum(0) * SLACK + 1e-300, "ds")
    again = torch.autograd.grad(embedding_lookup(W, ids, f, pad), leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "not repeatable"


@pytest.mark.parametrize("scale", ["none", "number", "column"])
@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("rows,dim,n,kind", [(1, 1, 1, "one"), (7, 1, 40, "uniform"), (50, 3, 33, "zipf"),
                                             (300, 20, 777, "zipf"), (1000, 64, 1, "uniform"),
                                             (129, 333, 500, "uniform"), (40, 1030, 260, "zipf"),
                                             (5, 24, 3000, "one"), (2000, 8, 5000, "zipf")])
def test_lookup(dt, rows, dim, n, kind, scale):
    lookup_case(DT[dt], rows, dim, n, kind, scale)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("dim", [3, 5, 6, 7, 9, 17, 25, 26, 27, 33, 47, 48, 49, 100, 132, 192, 196, 384, 392])
def test_lookup_rows_that_leave_lanes_idle(dim, dt):
    """Row lengths on both sides of the choice between a group of lanes a row and all vectors in one line."""
    for n in (1, 341, 1025):
        lookup_case(DT[dt], 60, dim, n, "uniform", "column" if n == 341 else "none", pad=5, out_of_range=True, seed=dim)


@pytest.mark.parametrize("pad", [-1, 0, 6, 49, 10 ** 12])
@pytest.mark.parametrize("scale", ["none", "column"])
def test_lookup_padding_and_out_of_range(pad, scale):
    lookup_case(torch.float32, 50, 12, 200, "zipf", scale, pad=pad, out_of_range=True)
    lookup_case(torch.bfloat16, 50, 12, 2000, "uniform", scale, pad=pad, out_of_range=True, seed=50)


def test_lookup_narrow_ids_and_many_tokens():
    lookup_case(torch.bfloat16, 1000, 40, 70001, "zipf", "number", pad=3, id_dtype=torch.int32)
    lookup_case(torch.float32, 70000, 5, 200003, "uniform", "column")
    lookup_case(torch.float32, 3, 4, 300000, "uniform", "none")


@pytest.mark.parametrize("n", [31, 32, 33, 63, 64, 65, 96, 255, 2047, 2048, 2049, 4096, 4097, 8192, 8193])
def test_lookup_runs_at_tile_borders(n):
    """Lengths around the cuts of the sorted ids; few ids, so runs cross many cuts."""
    for kind, rows in (("one", 3), ("uniform", 2), ("uniform", 9), ("zipf", 600)):
        lookup_case(torch.float32, rows, 6, n, kind, "column", seed=n)


@pytest.mark.parametrize("n", [1, 4095, 4096, 4097, 4128, 4129])
@pytest.mark.parametrize("dim", [510, 512, 513])
def test_column_scale_gradient_by_the_last_block_or_a_launch(n, dim):
    """Up to 128 blocks of 32 sorted ids a column piece add up the scale's gradient themselves."""
    lookup_case(torch.float32, 3000, dim, n, "zipf", "column", pad=1, seed=n)


@pytest.mark.parametrize("n,kind", [(3, "uniform"), (700, "zipf"), (5000, "zipf"), (20000, "uniform"), (40000, "zipf"),
                                    (140000, "zipf")])
def test_lookup_large_tables(n, kind):
    """Tables beyond what is cleared beside the sort, of odd rows too; every way of sorting."""
    lookup_case(torch.bfloat16, 70001, 1024 if n < 100000 else 8, n, kind, "number", pad=70000, seed=n)
    lookup_case(torch.float32, 60011, 601 if n < 10000 else 33, n, kind, "none", seed=n + 1)


def test_lookup_saves_only_what_its_gradient_needs():
    """The table may change between the passes unless the scale's gradient reads it."""
    from gpu_eigsh.features import embedding_lookup

    ids = make_ids("zipf", 20, 50, 1)
    W = randn((20, 6), torch.float32, 2).requires_grad_(True)
    s = randn((6,), torch.float32, 3).requires_grad_(True)
    g = randn((50, 6), torch.float32, 4)
    ref = torch.autograd.grad(embedding_lookup(W, ids, s.detach()), [W], g)[0]
    y = embedding_lookup(W, ids, s.detach())
    with torch.no_grad():
        W.add_(1.0)
    assert torch.equal(torch.autograd.grad(y, [W], g)[0], ref)
    y = embedding_lookup(W, ids, s)
    with torch.no_grad():
        W.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, [W, s], g)


def test_lookup_all_tokens_are_padding():
    from gpu_eigsh.features import embedding_lookup

    W = randn((9, 5), torch.float32, 1).requires_grad_(True)
    s = torch.ones(5, device="cuda", requires_grad=True)
    ids = torch.full((70,), 4, device="cuda")
    y = embedding_lookup(W, ids, s, 4)
    dW, ds = torch.autograd.grad(y, [W, s], torch.full_like(y, float("nan")))
    assert bool((y == 0).all()) and bool((dW == 0).all()) and bool((ds == 0).all())


def test_lookup_ignores_what_is_not_named():
    """NaN in rows that no id names and in the gradients of padding tokens stay where they are."""
    from gpu_eigsh.features import embedding_lookup

    W = randn((40, 16), torch.float32, 1)
    W[20:] = float("nan")
    W.requires_grad_(True)
    s = randn((16,), torch.float32, 2).requires_grad_(True)
    ids = make_ids("uniform", 20, 300, 3)
    ids[::5] = -1
    g = randn((300, 16), torch.float32, 4)
    g[::5] = float("inf")
    y = embedding_lookup(W, ids, s, -1)
    dW, ds = torch.autograd.grad(y, [W, s], g)
    assert all(bool(torch.isfinite(t).all()) for t in (y, dW, ds))
    with torch.no_grad():   # and a NaN that is named arrives
        W[7, 3] = float("nan")
    assert bool(torch.isnan(embedding_lookup(W, torch.tensor([7], device="cuda"))[0, 3]))


def test_lookup_shapes_strides_and_empty():
    from gpu_eigsh.features import embedding_lookup

    big = randn((30, 50), torch.float32, 1)
    ids = make_ids("uniform", 30, 24, 2).reshape(2, 3, 4)
    for W in (big[:, 3:20], big[:, ::2], big[::2].contiguous()[:, :49], big.t()[:30, :].contiguous().t()):
        idw = ids % W.shape[0]
        W = W.detach().requires_grad_(True)
        y = embedding_lookup(W, idw, 2.0)
        assert y.shape == (2, 3, 4, W.shape[1]) and torch.equal(y.detach(), W.detach()[idw] * 2.0)
        wide = randn((2, 3, 8, W.shape[1]), torch.float32, 3)
        for g in (wide[:, :, ::2], torch.ones((), device="cuda").expand(y.shape), wide[0, 0, 0].expand(y.shape)):
            (dW,) = torch.autograd.grad(y, [W], g, retain_graph=True)
            ref = torch.zeros(W.shape, dtype=F64, device="cuda").index_add_(
                0, idw.reshape(-1), 2.0 * g.reshape(-1, W.shape[1]).to(F64))
            torch.testing.assert_close(dW.to(F64), ref, rtol=1e-6, atol=24 * 6e-8 * 10)
    W = big.detach().requires_grad_(True)
    strided = torch.arange(20, device="cuda")[::2]
    assert torch.equal(embedding_lookup(W, strided).detach(), big[::2][:10])
    y = embedding_lookup(W, torch.zeros((0, 2), dtype=torch.int64, device="cuda"))
    (dW,) = torch.autograd.grad(y, [W], y.detach())
    assert y.shape == (0, 2, 50) and dW.shape == W.shape and bool((dW == 0).all())
    assert embedding_lookup(W, torch.tensor(3, device="cuda")).shape == (50,)


def test_lookup_needs_only_what_is_asked():
    from gpu_eigsh.features import embedding_lookup

    W = randn((30, 10), torch.float32, 1)
    s = randn((10,), torch.float32, 2).requires_grad_(True)
    ids = make_ids("zipf", 30, 100, 3)
    g = randn((100, 10), torch.float32, 4)
    (ds,) = torch.autograd.grad(embedding_lookup(W, ids, s), [s], g)
    W2 = W.clone().requires_grad_(True)
    dW2, ds2 = torch.autograd.grad(embedding_lookup(W2, ids, s), [W2, s], g)
    assert torch.equal(ds, ds2)
    (dW3,) = torch.autograd.grad(embedding_lookup(W2, ids, s.detach()), [W2], g)
    assert torch.equal(dW3, dW2)
    with torch.no_grad():
        assert not embedding_lookup(W2, ids, s).requires_grad


def test_lookup_offsets_beyond_32_bits():
    from gpu_eigsh.features import embedding_lookup

    rows, dim = 1_200_000, 2048   # 2.46e9 elements
    W = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([rows - 1, 0, rows - 2, rows - 1, 1_048_576], device="cuda")
    rowval = torch.arange(1, 6, device="cuda", dtype=torch.bfloat16)[:, None]
    W[ids] = torch.tensor([4.0, 2.0, 3.0, 4.0, 5.0], device="cuda", dtype=torch.bfloat16)[:, None]
    W.requires_grad_(True)
    y = embedding_lookup(W, ids)
    assert torch.equal(y.detach(), W.detach()[ids])
    (dW,) = torch.autograd.grad(y, [W], rowval.expand(5, dim))
    nz = torch.nonzero(dW[:, 0]).reshape(-1).tolist()
    assert nz == [0, 1_048_576, rows - 2, rows - 1]
    assert bool((dW[rows - 1] == 5).all()) and bool((dW[rows - 2] == 3).all()) and bool((dW[1_048_576] == 5).all())
    assert float(dW.sum(dtype=F64)) == (1 + 4 + 2 + 3 + 5) * dim


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def norm_case(dt, shape, affine="both", pdt=None, eps=1e-5, std=1.5, mean=0.25, seed=0, x=None, g=None):
    from gpu_eigsh.features import layer_norm

    dim = shape[-1]
    pdt = pdt or dt
    x = randn(shape, dt, seed + 1, std, mean) if x is None else x
    x = x.detach().requires_grad_(True)
    w = randn((dim,), pdt, seed + 2, 0.5, 1.0).requires_grad_(True) if affine in ("both", "weight") else None
    b = randn((dim,), pdt, seed + 3).requires_grad_(True) if affine in ("both", "bias") else None
    g = randn(shape, dt, seed + 4) if g is None else g
    y = layer_norm(x, w, b, eps)
    assert y.dtype == dt and y.shape == x.shape
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, g)

    ua, ut, up = u(acc(dt)), u(dt), u(pdt)
    X, Gd = x.detach().to(F64).reshape(-1, dim), g.to(F64).reshape(-1, dim)
    Wd = torch.ones(dim, dtype=F64, device="cuda") if w is None else w.detach().to(F64)
    Bd = torch.zeros(dim, dtype=F64, device="cuda") if b is None else b.detach().to(F64)
    mu = X.mean(1, keepdim=True)
    c = X - mu
    var = (c * c).mean(1, keepdim=True)
    r = 1.0 / torch.sqrt(var + eps)
    h = c * r
    # additions on one path of a row's sum: 32 in a thread (or dim / 1024), 5 in a warp, 32 over the warps
    D = min(dim, 72 + dim // 1024 + 1)
    e_mu = (D + 2) * ua * X.abs().mean(1, keepdim=True)
    rel_r = 0.5 * ((D + 5) * ua * var + e_mu ** 2 + 2 * ua * (var + eps)) / (var + eps) + 3 * ua
    e_h = r * (e_mu + ua * (c.abs() + e_mu)) + h.abs() * (rel_r + ua)
    e_h = e_h * SLACK
    Y = h * Wd + Bd
    e_y = (Wd.abs() * e_h + 2 * ua * ((h * Wd).abs() + Y.abs()) + ut * Y.abs()) * SLACK + tiny(dt)
    check(y.detach().reshape(-1, dim), Y, e_y, "y")

    wg = Gd * Wd
    m0, m1 = wg.mean(1, keepdim=True), (wg * h).mean(1, keepdim=True)
    e_m0 = (D + 3) * ua * wg.abs().mean(1, keepdim=True)
    e_m1 = (D + 4) * ua * (wg * h).abs().mean(1, keepdim=True) + (wg.abs() * e_h).mean(1, keepdim=True)
    t = wg - m0 - h * m1
    e_t = e_m0 + h.abs() * e_m1 + m1.abs() * e_h + 4 * ua * (wg.abs() + m0.abs() + (h * m1).abs())
    ref = r * t
    e = (r * e_t + ref.abs() * (rel_r + 2 * ua + ut)) * SLACK + tiny(dt)
    check(grads[0].reshape(-1, dim), ref, e, "dx")
    R = X.shape[0]
    k = 1
    if w is not None:
        ref = (Gd * h).sum(0)
        e = (R + 3) * ua * (Gd * h).abs().sum(0) + (Gd.abs() * e_h).sum(0) + up * ref.abs()
        check(grads[k], ref, e * SLACK + tiny(pdt), "dw")
        k += 1
    if b is not None:
        ref = Gd.sum(0)
        check(grads[k], ref, ((R + 1) * ua * Gd.abs().sum(0) + up * ref.abs()) * SLACK + tiny(pdt), "db")
    again = torch.autograd.grad(layer_norm(x, w, b, eps), leaves, g)
    assert all(torch.equal(p, q) for p, q in zip(grads, again)), "not repeatable"
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (1, 8), (5, 10), (2, 3, 7), (64, 16), (700, 33), (33, 128), (130, 200),
                                   (9, 256), (65, 513), (17, 1000), (4, 1024), (300, 1537), (6, 2049), (3, 4096),
                                   (2, 8192), (2, 8193)])
def test_norm(dt, shape):
    norm_case(DT[dt], shape)


@pytest.mark.parametrize("dt,shape", [("bf16", (3, 32768)), ("bf16", (3, 32776)), ("f32", (2, 16384)),
                                      ("f32", (5, 16388)), ("f64", (3, 8192)), ("f64", (3, 8195)), ("f16", (2, 40001)),
                                      ("f32", (700, 4099))])
def test_norm_long_rows(dt, shape):
    norm_case(DT[dt], shape)


@pytest.mark.parametrize("affine", ["both", "weight", "bias", "none"])
def test_norm_parameters(affine):
    norm_case(torch.float32, (40, 96), affine)
    norm_case(torch.bfloat16, (2000, 40), affine, torch.float32)
    norm_case(torch.float16, (7, 515), affine, torch.float32)
    norm_case(torch.float64, (3, 40001), affine)


def test_norm_hard_rows():
    """A mean far from the spread, tiny and large values, constant rows."""
    norm_case(torch.float32, (50, 300), std=1e-2, mean=100.0)
    norm_case(torch.float64, (50, 300), std=1e-6, mean=1.0, eps=1e-14)
    norm_case(torch.float32, (20, 64), std=1e-12, mean=0.0)
    norm_case(torch.bfloat16, (20, 64), std=1e15)
    norm_case(torch.float32, (20, 64), eps=0.0)
    from gpu_eigsh.features import layer_norm

    c = torch.full((4, 100), 3.5, device="cuda")
    assert bool((layer_norm(c) == 0).all())
    b = randn((100,), torch.float32, 1)
    assert torch.equal(layer_norm(c, None, b), b.expand(4, 100))
    assert bool(torch.isnan(layer_norm(c, eps=0.0)).all())   # 0 / 0


def test_norm_nonfinite_rows_stay_alone():
    from gpu_eigsh.features import layer_norm

    for dim in (10, 100, 700, 5000):
        x = randn((12, dim), torch.float32, dim)
        ref = layer_norm(x)
        x[3, dim // 2], x[7, 0], x[9, -1] = float("nan"), float("inf"), -float("inf")
        y = layer_norm(x)
        good = [i for i in range(12) if i not in (3, 7, 9)]
        assert torch.equal(y[good], ref[good])
        assert bool(torch.isnan(y[[3, 7, 9]]).any(1).all())


def test_norm_strides_and_empty():
    from gpu_eigsh.features import layer_norm

    big = randn((40, 60), torch.bfloat16, 1)
    for x in (big[:, 3:40], big[::2, :48], big[:, ::3], big.t(), big.reshape(5, 8, 60).transpose(0, 1)):
        norm_case(torch.bfloat16, tuple(x.shape), x=x, g=torch.ones((), device="cuda", dtype=torch.bfloat16).expand(x.shape))
        norm_case(torch.bfloat16, tuple(x.shape), x=x, g=randn((*x.shape[:-1], 2 * x.shape[-1]), torch.bfloat16, 5)[..., ::2])
    x = torch.zeros((0, 7), device="cuda", requires_grad=True)
    w = torch.ones(7, device="cuda", requires_grad=True)
    y = layer_norm(x, w, w)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 7) and bool((dw == 0).all())


def test_norm_needs_only_what_is_asked():
    from gpu_eigsh.features import layer_norm

    x, w, b = randn((90, 70), torch.float32, 1), randn((70,), torch.float32, 2), randn((70,), torch.float32, 3)
    g = randn((90, 70), torch.float32, 4)
    all_in = [t.clone().requires_grad_(True) for t in (x, w, b)]
    full = torch.autograd.grad(layer_norm(*all_in), all_in, g)
    for k in range(3):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        (one,) = torch.autograd.grad(layer_norm(*leaves), [leaves[k]], g)
        assert torch.equal(one, full[k])


# ---------------------------------------------------------------------------
# Edge distances
# ---------------------------------------------------------------------------
def make_edges(n, m, seed, hubs=False):
    g = gen(seed)
    i = torch.randint(0, n, (m,), generator=g, device="cuda")
    j = make_ids("zipf", n, m, seed + 1) if hubs else torch.randint(0, n, (m,), generator=g, device="cuda")
    return torch.stack([i, j])


def edge_case(dt, n, m, dim, hubs=False, seed=0, x=None, idx=None, narrow=False):
    from gpu_eigsh.features import EdgeDistances, edge_sqdist

    idx = make_edges(n, m, seed + 1, hubs) if idx is None else idx
    x = (randn((n, dim), dt, seed + 2) if x is None else x).detach().requires_grad_(True)
    g = randn((m,), acc(dt), seed + 3)
    graph = EdgeDistances(idx.to(torch.int32) if narrow else idx, n)
    d2 = graph(x)
    assert d2.dtype == acc(dt)
    (dx,) = torch.autograd.grad(d2, [x], g)
    ua, ut = u(acc(dt)), u(dt)
    X, (i, j) = x.detach().to(F64), idx
    diff = X[i] - X[j]
    ref = (diff ** 2).sum(1)
    # a difference, its square, a sum of dim terms
    check(d2.detach(), ref, (dim + 4) * ua * ref * SLACK + tiny(acc(dt)), "d2")
    c = 2.0 * g.to(F64)[:, None] * diff
    ref = torch.zeros_like(X).index_add_(0, i, c).index_add_(0, j, -c)
    mag = torch.zeros_like(X).index_add_(0, i, c.abs()).index_add_(0, j, c.abs())
    deg = torch.bincount(idx.reshape(-1), minlength=n).to(F64)[:, None]
    check(dx, ref, ((deg + 3) * ua * mag + ut * ref.abs()) * SLACK + tiny(dt), "dx")
    assert bool((dx[deg[:, 0] == 0] == 0).all())
    (dx2,) = torch.autograd.grad(edge_sqdist(x, idx), [x], g)
    assert torch.equal(dx, dx2), "not repeatable"


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("n,m,dim", [(1, 1, 1), (2, 1, 3), (5, 40, 2), (600, 3000, 3), (100, 17, 10), (3000, 20000, 7),
                                     (50, 300, 64), (20, 100, 129), (200, 3000, 300), (4, 9, 2050)])
def test_edges(dt, n, m, dim):
    edge_case(DT[dt], n, m, dim)


@pytest.mark.parametrize("dt", sorted(DT))
def test_edges_hubs(dt):
    edge_case(DT[dt], 500, 20000, 12, hubs=True)
    edge_case(DT[dt], 3, 5000, 5)
    edge_case(DT[dt], 70, 40000, 80, hubs=True)


@pytest.mark.parametrize("dt,n,m,dim,hubs", [("f16", 2000, 27000, 333, False), ("bf16", 700, 130000, 65, True),
                                             ("f32", 9000, 70000, 65, False), ("f32", 300, 90000, 50, True),
                                             ("f32", 400, 1450000, 3, False), ("f64", 5000, 70000, 33, True)])
def test_edges_of_rows_that_are_copied(dt, n, m, dim, hubs):
    """Rows at odd addresses and enough edges: the calls read an aligned copy."""
    x = randn((n, 2 * dim), DT[dt], 5)
    edge_case(DT[dt], n, m, dim, hubs=hubs)
    edge_case(DT[dt], n, m, dim, hubs=hubs, x=x[:, 1:dim + 1])


@pytest.mark.parametrize("m", [127, 128, 129, 255, 256, 257, 511, 512, 513, 1025])
def test_edges_list_lengths_around_a_chunk(m):
    """A star: its centre has m edges."""
    idx = torch.stack([torch.full((m,), 3, device="cuda"), torch.arange(m, device="cuda") % 40 + 4])
    edge_case(torch.float32, 50, m, 6, idx=idx)
    edge_case(torch.float32, 50, m, 6, idx=idx.flip(0), narrow=True)


def test_edges_same_edge_twice_self_edges_and_empty():
    from gpu_eigsh.features import EdgeDistances, edge_sqdist

    idx = torch.tensor([[0, 0, 2, 1, 0, 2], [1, 1, 2, 0, 1, 0]], device="cuda")
    edge_case(F64, 4, 6, 5, idx=idx)
    x = randn((4, 5), torch.float32, 1).requires_grad_(True)
    none = torch.zeros((2, 0), dtype=torch.int64, device="cuda")
    d2 = EdgeDistances(none, 4)(x)
    (dx,) = torch.autograd.grad(d2, [x], d2.detach())
    assert d2.shape == (0,) and bool((dx == 0).all())
    loops = torch.tensor([[1, 3], [1, 3]], device="cuda")
    y = edge_sqdist(x, loops)
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert bool((y == 0).all()) and bool((dx == 0).all())


def test_edges_strides_and_nonfinite():
    big = randn((90, 50), torch.float32, 1)
    for x in (big[:60, 3:20], big[30:, ::2], big[:, :48][::2][:40]):
        edge_case(torch.float32, x.shape[0], 500, x.shape[1], x=x)
    from gpu_eigsh.features import EdgeDistances

    x = randn((30, 9), torch.float32, 2)
    idx = make_edges(30, 200, 3)
    ref = EdgeDistances(idx, 30)(x)
    x[4] = float("nan")
    got = EdgeDistances(idx, 30)(x)
    at = (idx == 4).any(0)
    assert torch.equal(got[~at], ref[~at]) and bool(torch.isnan(got[at]).all())
    one = torch.ones((), device="cuda").expand(200)
    x = randn((30, 9), torch.float32, 2).requires_grad_(True)
    d = EdgeDistances(idx, 30)(x)
    a = torch.autograd.grad(d, [x], one, retain_graph=True)[0]
    b = torch.autograd.grad(d, [x], one.contiguous())[0]
    assert torch.equal(a, b)


def test_values_behind_a_pending_negation():
    """The imaginary part of a conjugate holds the negated values in memory."""
    from gpu_eigsh.features import edge_sqdist, embedding_lookup, layer_norm

    z = torch.complex(randn((40, 1), torch.float32, 1), randn((40, 1), torch.float32, 2))
    neg = z.conj().imag
    val = -z.imag
    assert neg.is_neg() and not val.is_neg()
    ids = make_ids("uniform", 40, 100, 3)
    idx = make_edges(40, 60, 4)
    assert torch.equal(embedding_lookup(neg, ids), val[ids])
    assert torch.equal(edge_sqdist(neg + 0, idx), edge_sqdist(val, idx)) and torch.equal(edge_sqdist(neg, idx), edge_sqdist(val, idx))
    x, w = randn((5, 40), torch.float32, 5), neg.reshape(40)
    assert torch.equal(layer_norm(x, w), layer_norm(x, val.reshape(40)))
    assert torch.equal(layer_norm(neg.T, None, w), layer_norm(val.T.contiguous(), None, val.reshape(40)))
    s = torch._neg_view(randn((3,), torch.float32, 6))
    W = randn((40, 3), torch.float32, 7)
    assert torch.equal(embedding_lookup(W, ids, scale=s), embedding_lookup(W, ids, scale=s.clone()))
    g = torch._neg_view(randn((100, 3), torch.float32, 8))
    W.requires_grad_(True)
    a, b = (torch.autograd.grad(embedding_lookup(W, ids), [W], h)[0] for h in (g, g.clone()))
    assert torch.equal(a, b)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad

    from gpu_eigsh.features import edge_sqdist, embedding_lookup, layer_norm

    x = randn((6, 4), torch.float32, 1)
    ids = torch.arange(6, device="cuda")
    with fwad.dual_level():
        d = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: embedding_lookup(d, ids), lambda: layer_norm(d), lambda: edge_sqdist(d, torch.stack([ids, ids]))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_layer_norm_of_the_longest_rows():
    """2^24 columns in 2-byte pieces (an odd address), with all gradients: every column
    against the formula over the row's own statistics in 64 bits."""
    from gpu_eigsh.features import layer_norm

    n = 2 ** 24
    x = randn((n + 1,), torch.bfloat16, 1)[1:].reshape(1, n).detach().requires_grad_(True)
    w = randn((n,), torch.bfloat16, 2).requires_grad_(True)
    g = randn((1, n), torch.bfloat16, 3)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], g)
    X, W, G = (t.detach().to(F64) for t in (x, w, g))
    mu = X.mean()
    r = 1 / torch.sqrt(((X - mu) ** 2).mean() + 1e-5)
    h = (X - mu) * r
    wg = W * G
    ref = r * (wg - wg.mean() - h * (wg * h).mean())
    # sums of 2^24 terms by 1024 threads (2^14 terms each, then a tree): under 2^14 + 32 roundings of
    # 2^-24 relative to the sum of magnitudes, at most 2^-9.9 of mean |.| in a mean, and one rounding
    # of 2^-8 relative to the result
    off = 2.0 ** -9.9
    err_mu = off * X.abs().mean()
    err_h = (err_mu * r + h.abs() * 2 * off) * SLACK
    check(y.detach(), h * W, err_h * W.abs() + 2.0 ** -8 * (h * W).abs() * SLACK + tiny(torch.bfloat16), "y")
    check(dw[None], h * G, err_h * G.abs() + 2.0 ** -8 * (h * G).abs() * SLACK + tiny(torch.bfloat16), "dw")
    m = (wg * h).mean().abs()
    err = r * (off * wg.abs().mean() + err_h * (m + off * (wg * h).abs().mean()) +
               h.abs() * (off * (wg * h).abs().mean() + (wg.abs() * err_h).mean())) + 3 * off * ref.abs()
    check(dx, ref, err * SLACK + 2.0 ** -8 * ref.abs() * SLACK + tiny(torch.bfloat16), "dx")


def test_edges_many():
    """The lists of a large graph, and their sort over several passes."""
    edge_case(torch.float32, 200000, 1000000, 4, seed=9)


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_refusals():
    from gpu_eigsh.features import EdgeDistances, edge_sqdist, embedding_lookup, layer_norm

    W = torch.zeros((6, 4), device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (W[0], W[:0], W[:, :0]):
        with pytest.raises(ValueError):
            embedding_lookup(bad, ids)
    for bad in (W.int(), W.to(torch.complex64)):
        with pytest.raises(TypeError):
            embedding_lookup(bad, ids)
    for bad in (ids.cpu(), ids.float(), ids.to(torch.int16), [0, 1]):
        with pytest.raises(TypeError):
            embedding_lookup(W, bad)
    for bad, err in ((torch.ones(3, device="cuda"), ValueError), (torch.ones((1, 4), device="cuda"), ValueError),
                     (torch.ones(4, device="cuda", dtype=F64), TypeError), (torch.ones(4), ValueError)):
        with pytest.raises(err):
            embedding_lookup(W, ids, bad)
    with pytest.raises(TypeError):
        embedding_lookup(W.bfloat16(), ids, torch.ones(4, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        embedding_lookup(W, ids, None, 2 ** 63)

    w = torch.ones(4, device="cuda")
    for kw, err in ((dict(weight=w[:3]), ValueError), (dict(bias=w.double()), TypeError), (dict(weight=w.cpu()), TypeError),
                    (dict(weight=w.half()), TypeError), (dict(eps=-1e-5), ValueError), (dict(eps=float("nan")), ValueError),
                    (dict(eps=float("inf")), ValueError)):
        with pytest.raises(err):
            layer_norm(W, **kw)
    with pytest.raises(TypeError):
        layer_norm(W.half(), w, w.half())
    with pytest.raises(ValueError):
        layer_norm(W[:, :0])
    with pytest.raises(ValueError):
        layer_norm(torch.zeros((), device="cuda"))

    idx = torch.tensor([[0, 1], [2, 3]], device="cuda")
    for bad, n, err in ((idx[0], 4, ValueError), (idx.float(), 4, TypeError), (idx, 3, ValueError), (idx - 1, 4, ValueError),
                        (idx, 0, ValueError), (idx + 2 ** 33, 4, ValueError), (idx.t()[:1], 4, ValueError)):
        with pytest.raises(err):
            EdgeDistances(bad, n)
    graph = EdgeDistances(idx, 4)
    for bad, err in ((W, ValueError), (W[:4, 0], ValueError), (W[:4].int(), TypeError), (W[:4, :0], ValueError),
                     (W[:4].cpu(), TypeError)):
        with pytest.raises(err):
            graph(bad)
    with pytest.raises(ValueError):
        edge_sqdist(W[0], idx)


def test_second_derivatives_are_refused():
    from gpu_eigsh.features import edge_sqdist, embedding_lookup, layer_norm

    x = randn((6, 4), torch.float32, 1).requires_grad_(True)
    ids = torch.tensor([0, 1, 1], device="cuda")
    for f in (lambda: embedding_lookup(x, ids), lambda: layer_norm(x), lambda: edge_sqdist(x, torch.stack([ids, ids + 2]))):
        (d,) = torch.autograd.grad((f() ** 2).sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            d.sum().backward()


# ---------------------------------------------------------------------------
# Gradients against differences; streams; graphs
# ---------------------------------------------------------------------------
def test_gradients_against_differences():
    from gpu_eigsh.features import EdgeDistances, embedding_lookup, layer_norm

    ids = torch.tensor([[1, 4, 1], [0, -1, 1]], device="cuda")
    W, s = randn((5, 7), F64, 1).requires_grad_(True), randn((7,), F64, 2).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda a, b: embedding_lookup(a, ids, b, -1), (W, s))
    # -1 is out of range here: its row of NaN has no difference, the others do
    assert torch.autograd.gradcheck(lambda a: embedding_lookup(a, ids, 0.3, 4).reshape(6, 7)[[0, 1, 2, 3, 5]], (W,))
    w, b = randn((7,), F64, 3).requires_grad_(True), randn((7,), F64, 4).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *t: layer_norm(*t, eps=1e-3), (W, w, b))
    assert torch.autograd.gradcheck(lambda t: layer_norm(t), (W,))
    graph = EdgeDistances(torch.tensor([[0, 1, 4, 0, 2], [1, 2, 0, 1, 2]], device="cuda"), 5)
    assert torch.autograd.gradcheck(graph, (W,))


def _pipeline(W, s, w, b, ids, graph):
    from gpu_eigsh.features import embedding_lookup, layer_norm

    return graph(layer_norm(embedding_lookup(W, ids, s, -1), w, b))


def _pipeline_inputs(seed, dt=torch.bfloat16, V=300, d=40, n=500, m=3000):
    W = randn((V, d), dt, seed).requires_grad_(True)
    s = (randn((d,), torch.float32, seed + 1) * 0.1 + 1).requires_grad_(True)
    w, b = randn((d,), dt, seed + 2, 0.2, 1.0).requires_grad_(True), randn((d,), dt, seed + 3).requires_grad_(True)
    return [W, s, w, b], make_ids("zipf", V, n, seed + 4), make_edges(n, m, seed + 5, hubs=True), randn((m,), torch.float32, seed + 6)


def test_other_streams():
    from gpu_eigsh.features import EdgeDistances

    leaves, ids, idx, g = _pipeline_inputs(1)
    graph = EdgeDistances(idx, ids.numel())
    ref = torch.autograd.grad(_pipeline(*leaves, ids, graph), leaves, g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            for _ in range(3):
                outs.append(torch.autograd.grad(_pipeline(*leaves, ids, graph), leaves, g))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, ref))


def test_captured_and_replayed():
    """Forward and backward in two graphs of their own inputs, replayed in turn with new values."""
    from gpu_eigsh.features import EdgeDistances

    cases = []
    for seed in (10, 20):
        leaves, ids, idx, g = _pipeline_inputs(seed)
        graph = EdgeDistances(idx, ids.numel())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(_pipeline(*leaves, ids, graph), leaves, g)
        torch.cuda.current_stream().wait_stream(side)
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            y = _pipeline(*leaves, ids, graph)
            grads = torch.autograd.grad(y, leaves, g)
        cases.append((cg, leaves, ids, graph, g, y, grads))
    for turn in range(3):
        for k, (cg, leaves, ids, graph, g, y, grads) in enumerate(cases):
            fresh, new_ids, _, new_g = _pipeline_inputs(100 + 10 * turn + k)
            with torch.no_grad():
                for t, v in zip(leaves, fresh):
                    t.copy_(v)
                ids.copy_(new_ids)
                g.copy_(new_g)
        for cg, *_ in cases:
            cg.replay()
        torch.cuda.synchronize()
        for cg, leaves, ids, graph, g, y, grads in cases:
            y2 = _pipeline(*leaves, ids, graph)
            assert torch.equal(y.detach(), y2.detach())
            assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(y2, leaves, g)))


# ---------------------------------------------------------------------------
# Together, with the framework's graph operators
# ---------------------------------------------------------------------------
def test_features_to_eigenvalues_to_features():
    """Token features -> layer norm -> edge distances -> Laplacian values ->
    differentiable_eigsh -> eigenvector rows scaled by a function of the
    eigenvalues -> loss, with gradients down to the table; against dense fp64
    autograd.  The eigenvectors enter the loss as constants of their sign-free
    squares, where the gradient through the eigenvalues is exact."""
    from gpu_eigsh import differentiable_eigsh
    from gpu_eigsh.features import EdgeDistances, embedding_lookup, layer_norm
    from gpu_eigsh.graph import knn

    n, V, d, k, nn = 150, 60, 6, 4, 6
    table = randn((V, d), F64, 1).requires_grad_(True)
    w, b = randn((d,), F64, 2, 0.2, 1.0).requires_grad_(True), randn((d,), F64, 3, 0.2).requires_grad_(True)
    ids = make_ids("uniform", V, n, 4)
    pts = torch.rand((n, 2), generator=gen(5), device="cuda", dtype=F64)
    nb, _ = knn(pts, nn)
    i = torch.arange(n, device="cuda").repeat_interleave(nn)
    lo, hi = torch.minimum(i, nb.reshape(-1)), torch.maximum(i, nb.reshape(-1))
    key = torch.unique(lo * n + hi)
    idx = torch.stack([key // n, key % n])
    m = idx.shape[1]
    graph = EdgeDistances(idx, n)
    # CSR of the Laplacian: values = -w_e off the diagonal, row sums on it
    rows = torch.cat([idx[0], idx[1], torch.arange(n, device="cuda")])
    cols = torch.cat([idx[1], idx[0], torch.arange(n, device="cuda")])
    order = torch.argsort(rows * n + cols)
    crow = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    crow[1:] = torch.cumsum(torch.bincount(rows, minlength=n), 0)

    def weights(x, dist):
        return torch.exp(-dist(x) / 8.0)

    def loss_own():
        x = layer_norm(embedding_lookup(table, ids, 1.5), w, b)
        we = weights(x, graph)
        diag = torch.zeros(n, dtype=F64, device="cuda").index_add(0, idx[0], we).index_add(0, idx[1], we)
        vals = torch.cat([-we, -we, diag])[order]
        A = torch.sparse_csr_tensor(crow, cols[order], vals, (n, n))
        lam, vec = differentiable_eigsh(A, k=k, tol=1e-13)
        batch = torch.arange(0, n, 3, device="cuda")
        phi = embedding_lookup(vec.detach() ** 2, batch, lam + 0.5)
        return (phi ** 2).sum() * n + (lam * torch.arange(1.0, k + 1, device="cuda", dtype=F64)).sum()

    def loss_dense():
        x = torch.nn.functional.layer_norm(table[ids] * 1.5, (d,), w, b, 1e-5)
        we = weights(x, lambda t: ((t[idx[0]] - t[idx[1]]) ** 2).sum(1))
        Ad = torch.zeros((n, n), dtype=F64, device="cuda").index_put((idx[0], idx[1]), we)
        Ad = Ad + Ad.t()
        lam, vec = torch.linalg.eigh(torch.diag(Ad.sum(1)) - Ad)
        lam, vec = lam[:k], vec[:, :k]
        phi = vec.detach()[::3] ** 2 * (lam + 0.5)
        return (phi ** 2).sum() * n + (lam * torch.arange(1.0, k + 1, device="cuda", dtype=F64)).sum()

    leaves = [table, w, b]
    a, ref = loss_own(), loss_dense()
    ga, gr = torch.autograd.grad(a, leaves), torch.autograd.grad(ref, leaves)
    assert m > n and float(gr[0].abs().max()) > 1e-4
    assert abs(float(a.detach()) - float(ref.detach())) <= 1e-8 * abs(float(ref.detach()))
    for p, q in zip(ga[:2], gr[:2]):
        assert float((p - q).abs().max()) <= 1e-7 * float(q.abs().max())
    # the same bias on every vertex moves no distance: its gradient is a sum of the vertices' gradients that is
    # zero but for their roundings, on both sides, so it is held to the size of the other gradients
    for t in (ga[2], gr[2]):
        assert float(t.abs().max()) <= 1e-7 * float(gr[1].abs().max())


def test_knn_of_normalised_points():
    """graph.knn(normalize=True) is knn of the layer-normalised points; its squared distances are
    2 dim (1 - correlation) of the points' coordinates."""
    from gpu_eigsh.features import layer_norm
    from gpu_eigsh.graph import knn, knn_laplacian

    P = randn((400, 10), F64, 1, 3.0, 5.0)
    idx, d2 = knn(P, 7, normalize=True)
    ref_i, ref_d = knn(layer_norm(P, eps=1e-12), 7)
    assert torch.equal(idx, ref_i) and torch.equal(d2, ref_d)
    corr = torch.corrcoef(P)
    # eps moves the variance by 1e-12 of itself (variances here are of order 9)
    want = 20.0 * (1.0 - torch.gather(corr, 1, idx))
    assert float((d2 - want).abs().max()) < 1e-11
    rp, col, val = knn_laplacian(P, 7, 0.5, normalize=True)
    rp2, col2, val2 = knn_laplacian(layer_norm(P, eps=1e-12), 7, 0.5)
    assert torch.equal(rp, rp2) and torch.equal(col, col2) and torch.equal(val, val2)
    with pytest.raises(ValueError):
        knn(P[:, :1], 3, normalize=True)


def test_distances_drive_the_graph_gp():
    """The distances as x_edge_dists of the IMGP operator, and their gradient through slq_logdet of a torch matvec."""
    from gpu_eigsh.features import EdgeDistances, layer_norm
    from gpu_eigsh.funm_torch import slq_logdet
    from gpu_eigsh.imgp import make_imgp_precision_matvec

    n, m, d = 80, 300, 5
    idx = make_edges(n, m, 1)
    idx = idx[:, idx[0] != idx[1]]
    x = randn((n, d), F64, 2)
    graph = EdgeDistances(idx, n)
    d2 = graph(layer_norm(x))
    assert torch.allclose(d2, ((layer_norm(x)[idx[0]] - layer_norm(x)[idx[1]]) ** 2).sum(1), rtol=1e-12)
    mv = make_imgp_precision_matvec(x_edge_dists=d2, idx=idx, operator_dim=n, nu=1)
    y = randn((n,), F64, 3)
    assert bool(torch.isfinite(mv(y, torch.tensor(1.0), torch.tensor(1.0))).all())

    def matvec(v, we):
        v2 = v.reshape(n, -1)
        t = we[:, None] * (v2[idx[0]] - v2[idx[1]])
        return (2.0 * v2 + torch.zeros_like(v2).index_add(0, idx[0], t).index_add(0, idx[1], -t)).reshape(v.shape)

    leaf = x.clone().requires_grad_(True)
    we = torch.exp(-graph(layer_norm(leaf)) / 4.0)
    ld = slq_logdet(matvec, n, (we,), m_probes=4, lanczos_m=n // 2, seed=0, device="cuda")
    (gx,) = torch.autograd.grad(ld, [leaf])
    v = randn((n, d), F64, 4)
    h = 1e-5

    def value(t):
        w_ = torch.exp(-graph(layer_norm(t)) / 4.0)
        return float(slq_logdet(matvec, n, (w_,), m_probes=4, lanczos_m=n // 2, seed=0, device="cuda"))

    diff = (value(x + h * v) - value(x - h * v)) / (2 * h)
    # the difference's own error: h^2 of a smooth function's third derivative, and rounding 1e-12 / h
    assert abs(diff - float((gx * v).sum())) <= 1e-5 * max(1.0, abs(diff))


def test_too_many_edges_are_refused():
    from gpu_eigsh.features import EdgeDistances

    idx = torch.zeros((2, 1), dtype=torch.int64, device="cuda").expand(2, 2 ** 30 - 64)   # a view: no memory
    with pytest.raises(ValueError, match="edges"):
        EdgeDistances(idx, 4)
