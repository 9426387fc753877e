"""GPU: layer norm where the definition gives exact zeros: rows of one value, and constant gradients on them.

A row's sum is exact here (the values are small multiples of powers of two), so its mean is the value itself if the
sum is divided by the row length, correctly rounded; a product with the rounded reciprocal is an ulp away for many
lengths, and 1 / sqrt(eps) = 316 enlarges that."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DT = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16, "bf16": torch.bfloat16}
DIMS = [1, 3, 7, 10, 41, 47, 55, 100, 333, 1000, 1537, 4100, 8200, 20001, 40001]


@pytest.fixture(autouse=True)
def need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("value", [100.0, 1000.0, -3.0])
def test_constant_rows(dt, value):
    from gpu_eigsh.features import layer_norm

    for dim in DIMS:
        x = torch.full((3, dim), value, device="cuda", dtype=DT[dt])
        b = torch.linspace(-1, 1, dim, device="cuda").to(DT[dt])
        assert bool((layer_norm(x) == 0).all()), dim
        assert torch.equal(layer_norm(x, None, b), b.expand(3, dim)), dim


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("value", [1.0, 3.0])
def test_constant_gradients(dt, value):
    """h = 0 in the whole row, so dx = r (g - mean(g)) = 0, dw = 0 and db = the rows' sum of g."""
    from gpu_eigsh.features import layer_norm

    for dim in DIMS:
        x = torch.full((3, dim), 100.0, device="cuda", dtype=DT[dt], requires_grad=True)
        w = torch.ones(dim, device="cuda", dtype=DT[dt], requires_grad=True)
        b = torch.zeros(dim, device="cuda", dtype=DT[dt], requires_grad=True)
        g = torch.full((3, dim), value, device="cuda", dtype=DT[dt])
        (dx,) = torch.autograd.grad(layer_norm(x), [x], g)
        assert bool((dx == 0).all()), dim
        dx, dw, db = torch.autograd.grad(layer_norm(x, w, b), [x, w, b], g)
        assert bool((dx == 0).all()) and bool((dw == 0).all()) and bool((db == 3 * value).all()), dim
