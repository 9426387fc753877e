"""GPU: graph.knn(normalize=True) finds neighbours by correlation whatever the points' units, against the
definition in extended precision on the host."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
U = 2.0 ** -53


@pytest.fixture(autouse=True)
def need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def points(n=300, dim=10, seed=7):
    return np.random.default_rng(seed).normal(5.0, 3.0, (n, dim))


def exact_d2(P):
    """2 dim (1 - correlation) of all pairs as sums of squares (no cancellation), in 64-bit significands, and a bound
    on what fp64 makes of one: of the points' normalised coordinates, then of their distance."""
    X = P.astype(np.longdouble)
    n, dim = X.shape
    lo, hi = X.min(1, keepdims=True), X.max(1, keepdims=True)
    S = X / (hi - lo)
    c = S - S.mean(1, keepdims=True)
    r = 1 / np.sqrt((c * c).mean(1, keepdims=True))
    h = c * r
    # the mean: dim additions and a division, relative to the mean magnitude; 1 / deviation: half of the variance's
    # relative error (dim + 5 roundings, the mean's error squared, the eps: at most 2e-12 dim of the variance), a
    # root and a division
    e_mu = (dim + 2) * U * np.abs(S).mean(1, keepdims=True)
    rel = 0.5 * ((dim + 7) * U + (e_mu * r) ** 2 + 2e-12 * dim) + 3 * U
    e_h = r * (e_mu + U * (np.abs(c) + e_mu)) + np.abs(h) * (rel + U)
    d = h[:, None, :] - h[None, :, :]
    e = e_h[:, None, :] + e_h[None, :, :]
    d2 = (d * d).sum(2)
    return d2, 1.01 * ((2 * np.abs(d) * e + e * e).sum(2) + (dim + 4) * U * d2)


def check(P, k=7):
    from gpu_eigsh.graph import knn

    idx, d2 = (t.cpu().numpy() for t in knn(P, k, normalize=True))
    ref, bound = exact_d2(P)
    got = np.take_along_axis(ref, idx, 1)
    off = np.take_along_axis(bound, idx, 1)
    assert (np.abs(d2 - got) <= off).all(), float((np.abs(d2 - got) / off).max())
    np.fill_diagonal(ref, np.inf)
    assert (idx != np.arange(len(P))[:, None]).all()
    kth = np.sort(ref, 1)[:, k - 1:k]
    assert (got <= kth + 2 * bound.max(1, keepdims=True)).all(), "not the nearest"
    return idx


# the squares of deviations of 1e-300 and 1e307 leave fp64's range
@pytest.mark.parametrize("scale", [1.0, 1e-3, 1e-5, 1e-6, 1e-8, 1e8, 1e-30, 1e150, 1e-300, 1e307])
def test_any_unit(scale):
    P = points() * scale
    assert np.array_equal(check(P), check(points()))


def test_a_scale_per_point():
    P = points()
    rng = np.random.default_rng(8)
    check(P * 10.0 ** rng.uniform(-200, 200, (len(P), 1)))
    # powers of two change no bit of the data, and where the points are of one size none of the result
    P = P * 2.0 ** (16.0 * rng.integers(-40, 41, (len(P), 1)))
    assert np.array_equal(check(P), check(points()))


def test_small_spread_on_a_large_mean():
    P = points(60, 6)
    check(1e6 + 1e-4 * P, 3)
    check(1e-6 + 1e-9 * P, 3)


def test_laplacian_of_small_points():
    from gpu_eigsh.graph import knn_laplacian

    P = points(200, 5)
    for a, b in zip(knn_laplacian(P * 2.0 ** -32, 6, 0.5, normalize=True), knn_laplacian(P, 6, 0.5, normalize=True)):
        assert torch.equal(a, b)


def test_points_without_a_correlation_are_refused():
    from gpu_eigsh.graph import knn

    for value in (0.0, 3.25, 1e-9, -1e300):
        P = points(20, 4)
        P[13] = value
        with pytest.raises(ValueError, match="point 13"):
            knn(P, 3, normalize=True)
        knn(P, 3)
    P = points(20, 4)
    P[3, 1] = np.nan
    P[5, 2] = np.inf
    with pytest.raises(Exception):
        knn(P, 3, normalize=True)
