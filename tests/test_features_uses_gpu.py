"""GPU: the node-feature operators under what a training program puts around them: threads, saved-tensor hooks,
checkpointing, inference mode, torch.func, inputs changed in place, a graph used twice."""
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def randn(shape, seed, dt=torch.float32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)


def inputs(seed=0, V=300, d=40, n=500, m=3000):
    W = randn((V, d), seed, torch.bfloat16).requires_grad_(True)
    s = (randn((d,), seed + 1) * 0.1 + 1).requires_grad_(True)
    w, b = (randn((d,), seed + k, torch.bfloat16).requires_grad_(True) for k in (2, 3))
    gen = torch.Generator(device="cuda").manual_seed(seed + 4)
    ids = torch.randint(0, V, (n,), generator=gen, device="cuda")
    idx = torch.randint(0, n, (2, m), generator=gen, device="cuda")
    return [W, s, w, b], ids, idx, randn((m,), seed + 5)


def chain(leaves, ids, graph):
    from gpu_eigsh.features import embedding_lookup, layer_norm

    W, s, w, b = leaves
    return graph(layer_norm(embedding_lookup(W, ids, s, 7), w, b))


def reference(seed=0):
    from gpu_eigsh.features import EdgeDistances

    leaves, ids, idx, g = inputs(seed)
    graph = EdgeDistances(idx, ids.numel())
    y = chain(leaves, ids, graph)
    return leaves, ids, graph, g, y.detach(), torch.autograd.grad(y, leaves, g)


def same(a, b):
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


def test_many_threads():
    """One graph and one set of leaves, from several threads at once, each on its own stream."""
    leaves, ids, graph, g, y, grads = reference()
    torch.cuda.synchronize()
    wrong = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    out = chain(leaves, ids, graph)
                    got = torch.autograd.grad(out, leaves, g)
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(out.detach(), y) or not same(got, grads):
                        wrong.append("another result")
        except Exception as e:   # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_saved_tensors_on_the_host_and_checkpointing():
    from torch.utils.checkpoint import checkpoint

    leaves, ids, graph, g, y, grads = reference()
    for pin in (False, True):
        with torch.autograd.graph.save_on_cpu(pin_memory=pin):
            out = chain(leaves, ids, graph)
        assert same(torch.autograd.grad(out, leaves, g), grads)
    out = checkpoint(lambda *t: chain(t, ids, graph), *leaves, use_reentrant=False)
    assert same(torch.autograd.grad(out, leaves, g), grads)


def test_retained_and_used_twice():
    leaves, ids, graph, g, y, grads = reference()
    out = chain(leaves, ids, graph)
    assert same(torch.autograd.grad(out, leaves, g, retain_graph=True), grads)
    assert same(torch.autograd.grad(out, leaves, g), grads)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, g)
    one = torch.autograd.grad(chain(leaves, ids, graph), [leaves[1]], g)   # one leaf alone
    assert torch.equal(one[0], grads[1])


def test_inputs_changed_in_place_are_noticed():
    from gpu_eigsh.features import EdgeDistances, embedding_lookup, layer_norm

    leaves, ids, idx, g = inputs()
    W, s, w, b = leaves
    graph = EdgeDistances(idx, ids.numel())
    x = randn((ids.numel(), 40), 9).requires_grad_(True) * 1

    def ids_change():
        at = ids.clone()
        return embedding_lookup(W, at), at

    def norm_change():
        t = x * 2
        return layer_norm(t), t

    def edge_change():
        t = x * 3
        return graph(t), t

    for make in (ids_change, norm_change, edge_change):
        y, t = make()
        with torch.no_grad():
            t.add_(1).sub_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    table = W.detach().clone()   # needed for the scale's gradient
    y = embedding_lookup(table, ids, s)
    table.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    table = W.detach().clone().requires_grad_(True)   # not needed for its own gradient
    y = embedding_lookup(table * 1, ids)
    with torch.no_grad():
        table.add_(1)
    y.sum().backward()
    assert torch.equal(table.grad.sum(1), 40.0 * torch.bincount(ids, minlength=300).to(torch.bfloat16))


def test_inference_mode():
    from gpu_eigsh.features import EdgeDistances

    leaves, ids, graph, g, y, grads = reference()
    with torch.inference_mode():
        out = chain(leaves, ids, graph)
        other = EdgeDistances(inputs()[2], ids.numel())
    assert torch.equal(out, y) and not out.requires_grad
    assert same(torch.autograd.grad(chain(leaves, ids, other), leaves, g), grads)   # a graph built there trains too


def test_torch_func_is_refused():
    """The compiled calls have no batching rule: a wrapped tensor has no memory, which is an error and no launch."""
    from gpu_eigsh.features import EdgeDistances, embedding_lookup, layer_norm

    x, ids = randn((6, 4), 1), torch.arange(6, device="cuda")
    graph = EdgeDistances(torch.stack([ids, ids.flip(0)]), 6)
    for f in (lambda t: embedding_lookup(t, ids), layer_norm, graph):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.vmap(f)(torch.stack([x, x]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.grad(lambda t: f(t).sum())(x)
        leaf = x.clone().requires_grad_(True)
        y = f(leaf)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, [leaf], torch.stack([y.detach(), y.detach()]), is_grads_batched=True)
    assert torch.equal(layer_norm(x), layer_norm(x.clone()))   # and the calls after it work


def test_under_a_compiler_that_breaks_the_graph():
    leaves, ids, graph, g, y, grads = reference()
    f = torch.compile(lambda *t: chain(t, ids, graph) * 1.0, backend="eager")
    out = f(*leaves)
    assert torch.equal(out.detach(), y) and same(torch.autograd.grad(out, leaves, g), grads)


def test_under_autocast():
    leaves, ids, graph, g, y, grads = reference()
    with torch.autocast("cuda", dtype=torch.float16):
        out = chain(leaves, ids, graph)
    assert torch.equal(out.detach(), y) and same(torch.autograd.grad(out, leaves, g), grads)
