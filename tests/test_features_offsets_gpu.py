"""GPU: layer norm and edge distances where elements lie beyond 2^31 elements or 4 GiB, on every kernel that
forms such offsets.  (The embedding lookup has its test beside its others.)"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F64 = torch.float64


@pytest.fixture(autouse=True)
def need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    yield
    torch.cuda.empty_cache()


def randn(shape, dt, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=dt)


def u(dt):
    return torch.finfo(dt).eps / 2


# part-warp teams, a block a row, rows too long for a block's registers
@pytest.mark.parametrize("dim", [16, 4096, 32776])
def test_layer_norm(dim):
    """Every row equals the row computed alone (a part of the tensor far below 2^31 elements), bit for bit; the
    gradient of the weight and the bias, of the few rows that have one, is the formula's."""
    from gpu_eigsh.features import layer_norm

    rows = 2 ** 31 // dim + 9
    x = randn((rows, dim), torch.bfloat16, 1)
    w, b = randn((dim,), torch.bfloat16, 2), randn((dim,), torch.bfloat16, 3)
    at = [0, 1, rows // 2, 2 ** 31 // dim - 1, 2 ** 31 // dim, 2 ** 31 // dim + 1, rows - 2, rows - 1]
    g = torch.zeros_like(x)
    few = randn((len(at), dim), torch.bfloat16, 4)
    g[at] = few
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, g)
    y, X, W, B = y.detach(), x.detach(), w.detach(), b.detach()
    step = 2 ** 28 // dim
    for r in range(0, rows, step):
        assert torch.equal(y[r:r + step], layer_norm(X[r:r + step], W, B)), r
    one = X[at].requires_grad_(True)
    (want,) = torch.autograd.grad(layer_norm(one, W, B), [one], few)
    assert torch.equal(dx[at], want) and bool((want != 0).any(1).all())
    dx[at] = 0
    for r in range(0, rows, step):
        assert not bool(dx[r:r + step].any()), r
    xs = X[at].to(F64)
    c = xs - xs.mean(1, keepdim=True)
    h = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)
    G = few.to(F64)
    # rows of about standard normal values.  h: a mean's error, at most (dim / 1024 + 75) u of mean |x| < 1, and the
    # same relative to h from the variance; sums of 8 terms (and of zeros, which are exact); one rounding to bf16
    err_h = (dim // 1024 + 80) * u(torch.float32) * (1 + h.abs()) * 1.1
    ref = (G * h).sum(0)
    err = (G.abs() * err_h).sum(0) + 10 * u(torch.float32) * (G * h).abs().sum(0)
    assert bool(((dw.to(F64) - ref).abs() <= err + u(torch.bfloat16) * (ref.abs() + err)).all())
    ref = G.sum(0)
    err = 10 * u(torch.float32) * G.abs().sum(0)
    assert bool(((db.to(F64) - ref).abs() <= err + u(torch.bfloat16) * (ref.abs() + err)).all())


def edge_case(n, dim, m, seed):
    """Edges among the first, the middle and the last rows of x, the others' gradients zero."""
    from gpu_eigsh.features import EdgeDistances

    assert n * dim * 4 > 2 ** 32
    x = randn((n, dim), torch.float32, seed).requires_grad_(True)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    few = 600
    where = torch.tensor([0, n // 2, n - 20], device="cuda")
    idx = where[torch.randint(0, 3, (2, m), generator=gen, device="cuda")] + torch.randint(0, 20, (2, m), generator=gen, device="cuda")
    if m > few:   # the rest anywhere
        idx[:, few:] = torch.randint(0, n, (2, m - few), generator=gen, device="cuda")
    g = torch.zeros(m, device="cuda")
    g[:few] = randn((min(few, m),), torch.float32, seed + 2)
    d2 = EdgeDistances(idx, n)(x)
    (dx,) = torch.autograd.grad(d2, [x], g)
    X, d2 = x.detach(), d2.detach()
    step = 2 ** 28 // dim
    for e in range(0, m, step):
        i, j = idx[:, e:e + step]
        ref = ((X[i].to(F64) - X[j].to(F64)) ** 2).sum(1)
        # a difference, its square, a sum of dim terms
        assert bool(((d2[e:e + step].to(F64) - ref).abs() <= 1.01 * (dim + 4) * u(torch.float32) * ref).all()), e
    rows, back = torch.unique(idx[:, :few], return_inverse=True)
    S = X[rows].to(F64)
    c = 2.0 * g[:few].to(F64)[:, None] * (S[back[0]] - S[back[1]])
    ref = torch.zeros_like(S).index_add_(0, back[0], c).index_add_(0, back[1], -c)
    mag = torch.zeros_like(S).index_add_(0, back[0], c.abs()).index_add_(0, back[1], c.abs())
    deg = torch.bincount(idx.reshape(-1), minlength=n)[rows].to(F64)[:, None]   # the terms, those of zeros among them
    assert bool(((dx[rows].to(F64) - ref).abs() <= 1.01 * (deg + 4) * u(torch.float32) * mag).all())
    assert bool((mag[:, 0] > 0).any())
    dx[rows] = 0
    for r in range(0, n, step):
        assert not bool(dx[r:r + step].any()), r


def test_edges_of_short_rows():
    edge_case(2 ** 28 + 50, 4, 600, 1)


def test_edges_of_long_rows():
    edge_case(2 ** 20 + 50, 1100, 600, 2)


def test_edges_of_copied_rows():
    """Odd rows and enough edges that the calls read an aligned copy."""
    from gpu_eigsh import _native

    n, dim, m = 1100000, 1025, 2200000
    assert _native.lib.lg_edge_sqdist_workspace_bytes(n, m, dim, 0, 4096, dim) == n * 4112
    edge_case(n, dim, m, 3)
