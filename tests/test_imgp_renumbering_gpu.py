"""GPU: ImgpPrecisionMatvec.to_internal and to_caller are index_select of the rows: differentiable to any order, in
forward mode and under torch.func, for any block."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
N = 60


@pytest.fixture(autouse=True)
def need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


@pytest.fixture()
def methods():
    from gpu_eigsh.imgp import make_imgp_precision_matvec

    # a path through shuffled vertices, so that the operator renumbers them
    p = torch.randperm(N, generator=torch.Generator().manual_seed(1)).cuda()
    mv = make_imgp_precision_matvec(x_edge_dists=torch.ones(N - 1, device="cuda", dtype=torch.float64),
                                    idx=torch.stack([p[:-1], p[1:]]), operator_dim=N, nu=1)
    assert mv.perm is not None and not torch.equal(mv.perm, torch.arange(N, device="cuda"))
    return [(mv.to_internal, mv.perm), (mv.to_caller, mv.pos)]


def block(b=3, seed=2):
    return torch.randn(N, b, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).cuda()


def test_rows(methods):
    for f, at in methods:
        for X in (block(), block(1), block()[:, 0], block().to(torch.float32), block().to(torch.int64),
                  block().to(torch.complex64), block()[:, :0], block(6).reshape(N, 2, 3)):
            assert torch.equal(f(X), X[at])


def test_second_derivative(methods):
    for f, at in methods:
        X = block().requires_grad_(True)
        (g,) = torch.autograd.grad((f(X) ** 3).sum(), [X], create_graph=True)
        (h,) = torch.autograd.grad(g.sum(), [X])
        assert torch.equal(h, 6 * X.detach())
        assert torch.autograd.gradgradcheck(lambda t: f(t) ** 2, (block(1).requires_grad_(True),))


def test_forward_mode(methods):
    import torch.autograd.forward_ad as fwad

    X, T = block(), block(3, 3)
    for f, at in methods:
        with fwad.dual_level():
            y, t = fwad.unpack_dual(f(fwad.make_dual(X, T)))
            assert torch.equal(y, X[at]) and torch.equal(t, T[at])


def test_torch_func(methods):
    X, T = block(), block(3, 3)
    for f, at in methods:
        y, t = torch.func.jvp(f, (X,), (T,))
        assert torch.equal(y, X[at]) and torch.equal(t, T[at])
        many = torch.stack([X, T])
        assert torch.equal(torch.func.vmap(f)(many), many[:, at])
        assert torch.equal(torch.func.hessian(lambda v: (f(v) ** 2).sum())(X[:, :1]).reshape(N, N), 2 * torch.eye(N, dtype=X.dtype, device="cuda"))


def test_blocks_without_derivatives():
    from gpu_eigsh.ordering import renumber_rows

    at = torch.randperm(N, generator=torch.Generator().manual_seed(4)).cuda()
    wide = block(8)
    for X in (block(), block(1), wide[:, 1:6], wide[:, ::2], block(6).t().contiguous().t(), wide[:, :1].expand(N, 5),
              block().to(torch.float32), block().to(torch.bfloat16), block().to(torch.int64), block()[:, 0], block()[:, :0]):
        assert torch.equal(renumber_rows(X, at), X[at])
