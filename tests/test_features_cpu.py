"""CPU: what gpu_eigsh.features and its C entry points refuse before any GPU work."""
import pytest
import torch

from gpu_eigsh import _native, features

L = _native.lib
BAD = _native.LG_ERR_INVALID
P = 4096   # an address that no refused call reads


def test_cpu_tensors_are_refused():
    W, ids = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="table"):
        features.embedding_lookup(W, ids)
    with pytest.raises(TypeError, match="x must be"):
        features.layer_norm(W)
    with pytest.raises(TypeError, match="idx"):
        features.EdgeDistances(torch.zeros(2, 3, dtype=torch.int64), 4)
    with pytest.raises(TypeError, match="x must be"):
        features.edge_sqdist(W, torch.zeros(2, 3, dtype=torch.int64))


def gather(rows=4, dim=3, dtype=0, table=P, ld=3, n=2, ids=P, mode=0, scale=None, out=P):
    return L.lg_rows_gather(rows, dim, dtype, table, ld, n, ids, 1, mode, scale, 1.0, 0, 0, out, None)


@pytest.mark.parametrize("bad", [dict(rows=0), dict(rows=2 ** 31), dict(dim=0), dict(dim=2 ** 20 + 1), dict(dtype=4),
                                 dict(dtype=-1), dict(table=None), dict(ld=2), dict(n=0), dict(n=2 ** 31),
                                 dict(ids=None), dict(mode=3), dict(mode=2), dict(out=None)])
def test_gather_refuses(bad):
    assert gather(**bad) == BAD
    assert "lg_rows_gather" in _native.last_error()


def scatter(rows=4, dim=3, dtype=0, table=P, ld=3, n=2, ids=P, mode=0, scale=None, g=P, ld_g=3, dw=P, ds=None, ws=P,
            nb=1 << 30):
    return L.lg_rows_scatter(rows, dim, dtype, table, ld, n, ids, 1, mode, scale, 1.0, 0, 0, g, ld_g, dw, ds, ws, nb,
                             None)


@pytest.mark.parametrize("bad", [dict(rows=0), dict(dim=0), dict(dtype=7), dict(n=0), dict(ids=None), dict(g=None),
                                 dict(ld_g=2), dict(dw=None), dict(ws=None), dict(nb=16), dict(ds=P),
                                 dict(ds=P, mode=2, scale=P, table=None), dict(ds=P, mode=2, scale=P, ld=1)])
def test_scatter_refuses(bad):
    assert scatter(**bad) == BAD
    assert "lg_rows_scatter" in _native.last_error()


def test_scatter_workspace():
    size = L.lg_rows_scatter_workspace_bytes
    assert size(0, 3, 0, 2, 0) == 0 and size(4, 0, 0, 2, 0) == 0 and size(4, 3, 9, 2, 0) == 0 and size(4, 3, 0, 0, 0) == 0
    assert 0 < size(4, 3, 0, 2, 0) < size(4, 3, 0, 2, 1)
    assert size(1000, 64, 0, 100000, 0) < size(1000, 64, 1, 100000, 0)


def norm_fwd(rows=4, dim=3, dtype=0, x=P, ld=3, pd=0, eps=1e-5, y=P, mean=None, rstd=None):
    return L.lg_layer_norm_forward(rows, dim, dtype, x, ld, pd, None, None, eps, y, mean, rstd, None)


@pytest.mark.parametrize("bad", [dict(rows=0), dict(dim=0), dict(dim=2 ** 24 + 1), dict(dtype=5), dict(x=None),
                                 dict(ld=2), dict(pd=1), dict(dtype=1, pd=0), dict(dtype=2, pd=3), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(y=None), dict(mean=P), dict(rstd=P)])
def test_norm_forward_refuses(bad):
    assert norm_fwd(**bad) == BAD
    assert "lg_layer_norm_forward" in _native.last_error()


@pytest.mark.parametrize("bad", [dict(rows=0), dict(dim=0), dict(dtype=5), dict(x=None), dict(g=None), dict(ld=2),
                                 dict(ldg=2), dict(mean=None), dict(rstd=None), dict(dx=None), dict(dw=P),
                                 dict(db=P)])
def test_norm_backward_refuses(bad):
    a = dict(rows=4, dim=3, dtype=0, x=P, ld=3, g=P, ldg=3, mean=P, rstd=P, dx=P, dw=None, db=None)
    a.update(bad)
    assert L.lg_layer_norm_backward(a["rows"], a["dim"], a["dtype"], a["x"], a["ld"], a["g"], a["ldg"], 0, None,
                                    a["mean"], a["rstd"], a["dx"], a["dw"], a["db"], None, 0, None) == BAD
    assert "lg_layer_norm_backward" in _native.last_error()


def test_misaligned_addresses_are_refused():
    """An address inside an element would be a fault on the device."""
    for bad in (dict(table=P + 2), dict(out=P + 2), dict(ids=P + 4), dict(mode=2, scale=P + 2), dict(dtype=1, table=P + 4),
                dict(dtype=3, out=P + 1), dict(dtype=1, mode=2, scale=P + 4)):
        assert gather(**bad) == BAD, bad
    for bad in (dict(ids=P + 4), dict(g=P + 2), dict(dw=P + 2), dict(ws=P + 8), dict(mode=2, scale=P, ds=P + 2),
                dict(mode=2, scale=P, ds=P, table=P + 2)):
        assert scatter(**bad) == BAD, bad
    for bad in (dict(x=P + 2), dict(y=P + 1), dict(mean=P + 2, rstd=P), dict(dtype=1, pd=1, mean=P, rstd=P + 4)):
        assert norm_fwd(**bad) == BAD, bad
    big = 1 << 30

    def norm_bwd(x=P, g=P, mean=P, dx=P, dw=None, ws=P):
        return L.lg_layer_norm_backward(4, 3, 0, x, 3, g, 3, 0, None, mean, P, dx, dw, None, ws, big, None)

    for bad in (dict(x=P + 2), dict(g=P + 1), dict(mean=P + 2), dict(dx=P + 2), dict(dw=P + 2), dict(ws=P + 8)):
        assert norm_bwd(**bad) == BAD, bad
    assert L.lg_edge_graph(4, 4, P + 4, P, P, P, P, P, P, big, None) == BAD
    assert L.lg_edge_graph(4, 4, P, P + 2, P, P, P, P, P, big, None) == BAD
    assert L.lg_edge_graph(4, 4, P, P, P, P, P, P, P + 8, big, None) == BAD
    for ends, x, d2 in ((P + 2, P, P), (P, P + 2, P), (P, P, P + 2)):
        assert L.lg_edge_sqdist(4, 4, 3, 0, ends, x, 3, d2, None, 0, None) == BAD
    for x, g, dx, ws in ((P + 2, P, P, P), (P, P + 2, P, P), (P, P, P + 2, P), (P, P, P, P + 8)):
        assert L.lg_edge_sqdist_grad(4, 4, 3, 0, P, P, P, 0, None, None, 0, None, None, x, 3, g, dx, ws, big, None) == BAD


def test_edge_calls_refuse():
    big = 1 << 30
    assert L.lg_edge_graph_workspace_bytes(0, 4) == 0 and L.lg_edge_graph_workspace_bytes(4, 0) == 0
    assert L.lg_edge_graph_workspace_bytes(4, 2 ** 30) == 0 and L.lg_edge_graph_workspace_bytes(4, 5) > 0
    for n, m, idx, ws, nb in ((0, 4, P, P, big), (4, 0, P, P, big), (4, 2 ** 30, P, P, big), (4, 4, None, P, big),
                              (4, 4, P, None, big), (4, 4, P, P, 8)):
        assert L.lg_edge_graph(n, m, idx, P, P, P, P, P, ws, nb, None) == BAD
    for n, m, dim, dt, ends, x, ld, d2 in ((0, 4, 3, 0, P, P, 3, P), (4, 0, 3, 0, P, P, 3, P), (4, 4, 0, 0, P, P, 3, P),
                                           (4, 4, 3, 6, P, P, 3, P), (4, 4, 3, 0, None, P, 3, P),
                                           (4, 4, 3, 0, P, None, 3, P), (4, 4, 3, 0, P, P, 2, P),
                                           (4, 4, 3, 0, P, P, 3, None)):
        assert L.lg_edge_sqdist(n, m, dim, dt, ends, x, ld, d2, None, 0, None) == BAD

    # rows of 333 halves can be read by twos only: a copy in rows of 672 bytes, where it pays
    need = L.lg_edge_sqdist_workspace_bytes(100000, 1000000, 333, 2, P, 333)
    assert need == 100000 * 672
    assert L.lg_edge_sqdist_grad_workspace_bytes(100000, 1000000, 333, 2, P, 333, 3) >= need + 3 * 333 * 4
    assert L.lg_edge_sqdist(100000, 1000000, 333, 2, P, P, 333, P, P, need - 1, None) == BAD
    assert L.lg_edge_sqdist(100000, 1000000, 333, 2, P, P, 333, P, None, need, None) == BAD
    for m, dim, ld in ((1000000, 336, 336), (30000, 333, 333), (1000000, 16, 16)):
        assert L.lg_edge_sqdist_workspace_bytes(100000, m, dim, 2, P, ld) == 0

    def grad(n=4, m=4, dim=3, dt=0, rp=P, nlong=0, lr=None, nch=0, x=P, ld=3, g=P, dx=P, ws=None, nb=0):
        return L.lg_edge_sqdist_grad(n, m, dim, dt, rp, P, P, nlong, lr, lr, nch, lr, lr, x, ld, g, dx, ws, nb, None)

    for bad in (dict(n=0), dict(m=0), dict(dim=0), dict(dt=4), dict(rp=None), dict(x=None), dict(ld=1), dict(g=None),
                dict(dx=None), dict(nlong=-1), dict(nlong=2, nch=1, lr=P, ws=P, nb=big), dict(nlong=1, nch=2),
                dict(nlong=1, nch=2, lr=P), dict(nlong=1, nch=2, lr=P, ws=P, nb=8)):
        assert grad(**bad) == BAD
    assert "lg_edge_sqdist_grad" in _native.last_error()


def test_edge_lists_leave_room_in_32_bits():
    """Positions a few beyond the last list entry, and a list's length rounded up to chunks of 128, fit an int."""
    big, m = 1 << 62, (2 ** 31 - 1 - 128) // 2
    assert L.lg_edge_graph_workspace_bytes(4, m) > 0 and L.lg_edge_graph_workspace_bytes(4, m + 1) == 0
    assert L.lg_edge_graph(4, m + 1, P, P, P, P, P, P, P, big, None) == BAD
    assert L.lg_edge_sqdist(4, m + 1, 3, 0, P, P, 3, P, P, big, None) == BAD
    assert L.lg_edge_sqdist_grad(4, m + 1, 3, 0, P, P, P, 0, None, None, 0, None, None, P, 3, P, P, P, big, None) == BAD
