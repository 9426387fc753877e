"""Differentiable node features: embedding rows, layer norm, edge distances.

What a graph model computes before its graph operators (the features whose
distances weigh the edges) and after them (rows of eigenvectors as features),
as torch functions of CUDA tensors:

  embedding_lookup(table, ids, scale=None, padding_idx=None)
                            rows of a table by id, scaled by a number or by a
                            value per column; the table's gradient is summed
                            over the sorted ids
  layer_norm(x, weight=None, bias=None, eps=1e-5)
                            layer norm over the last dimension
  EdgeDistances(idx, n)     the edges of a graph, kept for repeated calls;
                            ``EdgeDistances(idx, n)(x)`` are the squared
                            distances of x along them
  edge_sqdist(x, idx)       the same for one call

Element types: float32, float64, float16 and bfloat16.  Arithmetic and sums
are in float32 (float64 for float64), each result is rounded once.  Sums run
in a fixed order, so equal inputs give equal bits.  Calls run on the current
stream of their tensors' device, allocate from torch and wait for nothing
(``EdgeDistances`` checks its indices when it is built, which waits once; the
rest can be captured into CUDA graphs).  The gradients are not differentiable
themselves.  There is no CPU implementation.

Squared distances are the ``x_edge_dists`` of
``gpu_eigsh.imgp.make_imgp_precision_matvec``.  That operator differentiates
only with respect to its two scalars; gradients with respect to the distances
go through the matrix values of ``gpu_eigsh.differentiable_eigsh``, or through
a matvec of torch operations given to ``gpu_eigsh.funm_torch.slq_logdet``.
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd.function import once_differentiable

from . import _native

__all__ = ["embedding_lookup", "layer_norm", "EdgeDistances", "edge_sqdist"]

_L = _native.lib
_CODES = {torch.float32: _native.LG_F32, torch.float64: _native.LG_F64, torch.float16: _native.LG_F16,
          torch.bfloat16: _native.LG_BF16}
_MAX_ROWS = 2 ** 31 - 2


def _acc(dtype: torch.dtype) -> torch.dtype:
    return torch.float64 if dtype == torch.float64 else torch.float32


# The current stream's handle: torch's own short way where this build has it
# (0.1 us; through a Stream object 2.2 us, of the 8 us that a small call takes).
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(dev: torch.device, fn, *args):
    """fn(*args, stream) on the current stream of `dev`, which becomes the
    current device for the call."""
    i = dev.index
    if torch.cuda.current_device() == i:
        rc = fn(*args, _stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _stream(i))
    if rc < 0:
        _native.check(rc)


def _once(backward):
    """once_differentiable, entered only where a graph of the backward pass is
    being made (its guards cost as much as a small launch)."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_features(name: str, t) -> int:
    if not torch.is_tensor(t) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float64, float16 or bfloat16, got {t.dtype}")
    return code


def _same_device(t, name: str, other, other_name: str):
    if t.device != other.device:
        raise ValueError(f"{name} is on {t.device}, {other_name} on {other.device}")


def _rows2d(t: torch.Tensor, dim: int):
    """t as (rows, dim) with unit stride along the row, and its row stride;
    copied only where the strides do not allow that."""
    t2 = t.reshape(-1, dim) if t.dim() != 2 else t
    if t2.stride(1) != 1 and dim > 1 or (t2.shape[0] > 1 and t2.stride(0) < dim):
        t2 = t2.contiguous()
    return t2, (t2.stride(0) if t2.shape[0] > 1 else dim)


# ---------------------------------------------------------------------------
# Embedding lookup
# ---------------------------------------------------------------------------
def _scale_args(scale):
    """(mode, device pointer, value) of lg_rows_gather / lg_rows_scatter."""
    if scale is None:
        return _native.LG_SCALE_NONE, None, 1.0
    if torch.is_tensor(scale):
        return _native.LG_SCALE_COLUMN, scale.data_ptr(), 1.0
    return _native.LG_SCALE_VALUE, None, scale


def _gather(table, ids, scale, padding, out_shape):
    """lg_rows_gather of checked arguments."""
    rows, dim = table.shape
    out = torch.empty(out_shape, dtype=table.dtype, device=table.device)
    if ids.numel():
        t, ld = _rows2d(table, dim)
        mode, sp, sv = _scale_args(scale)
        _call(table.device, _L.lg_rows_gather, rows, dim, _CODES[table.dtype], t.data_ptr(), ld, ids.numel(),
              ids.data_ptr(), ids.dtype == torch.int64, mode, sp, sv, padding is not None, padding or 0,
              out.data_ptr())
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, scale, ids, padding, out_shape):
        ctx.save_for_backward(table, ids, scale if torch.is_tensor(scale) else None)
        ctx.scale, ctx.padding = None if torch.is_tensor(scale) else scale, padding
        return _gather(table, ids, scale, padding, out_shape)

    @staticmethod
    @_once
    def backward(ctx, g):
        table, ids, column = ctx.saved_tensors
        scale = ctx.scale if column is None else column
        rows, dim = table.shape
        n, dev, code = ids.numel(), table.device, _CODES[table.dtype]
        d_table = d_scale = None
        want_scale = column is not None and ctx.needs_input_grad[1]
        make = torch.empty if n else torch.zeros
        if ctx.needs_input_grad[0]:
            d_table = make((rows, dim), dtype=table.dtype, device=dev)
        if want_scale:
            d_scale = make(dim, dtype=column.dtype, device=dev)
        if n:
            g2, ld_g = _rows2d(g, dim)
            t, ld = _rows2d(table, dim)
            mode, sp, sv = _scale_args(scale)
            nb = _L.lg_rows_scatter_workspace_bytes(rows, dim, code, n, want_scale)
            ws = torch.empty(nb, dtype=torch.uint8, device=dev)
            _call(dev, _L.lg_rows_scatter, rows, dim, code, t.data_ptr(), ld, n, ids.data_ptr(),
                  ids.dtype == torch.int64, mode, sp, sv, ctx.padding is not None, ctx.padding or 0, g2.data_ptr(),
                  ld_g, _ptr(d_table), _ptr(d_scale), ws.data_ptr(), nb)
        return d_table, d_scale, None, None, None


def embedding_lookup(table, ids, scale=None, padding_idx=None):
    """scale * table[ids]: rows of `table` (rows, dim) by `ids` (any shape, int32
    or int64), as a tensor of shape (*ids.shape, dim).

    scale : None, a number, or a (dim,) tensor, one value per column (float32,
        or float64 for a float64 table).  Gradients flow to `table` and to a
        scale tensor.
    padding_idx : an id equal to it (any integer, also outside the table) gives
        a row of zeros and takes no gradient.

    Any other id outside [0, rows) reads nothing, gives a row of NaN and takes
    no gradient (the ids stay on the device, so the call cannot raise for
    them).  The gradient is dense (rows, dim); the contributions of one id are
    added in the order of the ids.
    """
    _check_features("table", table)
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"table must be (rows, dim), got shape {tuple(table.shape)}")
    if not torch.is_tensor(ids) or not ids.is_cuda or ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("ids must be an int32 or int64 CUDA tensor")
    _same_device(ids, "ids", table, "table")
    rows, dim = table.shape
    if rows > _MAX_ROWS or ids.numel() > _MAX_ROWS or dim > 2 ** 20:
        raise ValueError("at most 2^31 - 2 rows and ids, and 2^20 columns")
    if torch.is_tensor(scale):
        if scale.dtype != _acc(table.dtype):
            raise TypeError(f"scale must be {_acc(table.dtype)} for a {table.dtype} table, got {scale.dtype}")
        if scale.shape != (dim,):
            raise ValueError(f"scale must have shape ({dim},), got {tuple(scale.shape)}")
        _same_device(scale, "scale", table, "table")
        scale = scale.contiguous()
    elif scale is not None:
        scale = float(scale)
    if padding_idx is not None:
        padding_idx = int(padding_idx)
        if not -2 ** 63 <= padding_idx < 2 ** 63:
            raise ValueError("padding_idx must fit 64 bits")
    ids = ids.contiguous()
    out_shape = (*ids.shape, dim)
    if torch.is_grad_enabled() and (table.requires_grad or (torch.is_tensor(scale) and scale.requires_grad)):
        return _Lookup.apply(table, scale, ids, padding_idx, out_shape)
    return _gather(table, ids, scale, padding_idx, out_shape)


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def _norm_forward(x, weight, bias, eps, keep):
    dim = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rows = x.numel() // dim
    mean = rstd = None
    if keep:
        mean, rstd = torch.empty((2, rows), dtype=_acc(x.dtype), device=x.device)
    if rows:
        x2, ld = _rows2d(x, dim)
        p = weight if weight is not None else bias
        _call(x.device, _L.lg_layer_norm_forward, rows, dim, _CODES[x.dtype], x2.data_ptr(), ld,
              _CODES[x.dtype if p is None else p.dtype], _ptr(weight), _ptr(bias), eps, y.data_ptr(), _ptr(mean),
              _ptr(rstd))
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_like = None if bias is None else bias.dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, g):
        x, weight, mean, rstd = ctx.saved_tensors
        dim, dev, code = x.shape[-1], x.device, _CODES[x.dtype]
        rows = x.numel() // dim
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        pdtype = weight.dtype if weight is not None else ctx.bias_like or x.dtype
        make = torch.empty if rows else torch.zeros
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dw = make(dim, dtype=pdtype, device=dev) if need_w else None
        db = make(dim, dtype=pdtype, device=dev) if need_b else None
        if rows:
            x2, ld_x = _rows2d(x, dim)
            g2, ld_g = _rows2d(g, dim)
            nb, ws = 0, None
            if need_w or need_b:
                nb = _L.lg_layer_norm_workspace_bytes(rows, dim, code)
                ws = torch.empty(nb, dtype=torch.uint8, device=dev)
            _call(dev, _L.lg_layer_norm_backward, rows, dim, code, x2.data_ptr(), ld_x, g2.data_ptr(), ld_g,
                  _CODES[pdtype], _ptr(weight), mean.data_ptr(), rstd.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db),
                  _ptr(ws), nb)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x (..., dim) over its last dimension:
    (x - mean) / sqrt(var + eps) * weight + bias, var the mean squared deviation.

    weight, bias : (dim,) tensors or None, of x's type, or float32 for a 16-bit
        x (both of the same type).  Gradients flow to x, weight and bias.
    """
    _check_features("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last dimension of at least 1, got shape {tuple(x.shape)}")
    dim = x.shape[-1]
    if x.numel() // dim > _MAX_ROWS or dim > 2 ** 24:
        raise ValueError("at most 2^31 - 2 rows and 2^24 columns")
    eps = float(eps)
    if not (0.0 <= eps < math.inf):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if not torch.is_tensor(p) or not p.is_cuda:
            raise TypeError(f"{name} must be a CUDA tensor")
        if p.dtype != x.dtype and not (p.dtype == torch.float32 and x.dtype in (torch.float16, torch.bfloat16)):
            raise TypeError(f"{name} must be {x.dtype}{'' if x.dtype == _acc(x.dtype) else ' or torch.float32'}, "
                            f"got {p.dtype}")
        if p.shape != (dim,):
            raise ValueError(f"{name} must have shape ({dim},), got {tuple(p.shape)}")
        _same_device(p, name, x, "x")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have the same type")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ---------------------------------------------------------------------------
# Edge distances
# ---------------------------------------------------------------------------
class _EdgeDist(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, graph):
        ctx.save_for_backward(x)
        ctx.graph = graph
        return graph._forward(x)

    @staticmethod
    @_once
    def backward(ctx, g):
        return ctx.graph._backward(ctx.saved_tensors[0], g), None


class EdgeDistances:
    """The edges of a graph of n vertices: idx (2, M) int64, edge e between
    vertices idx[0, e] and idx[1, e] (the edge lists of gpu_eigsh.imgp;
    repeated edges and edges from a vertex to itself are allowed).

    Called with features x (n, dim) it returns the squared distances (M,)
    |x[idx[0, e]] - x[idx[1, e]]|^2 in float32 (float64 for a float64 x), with
    gradients to x.  Building it sorts the edge ends, checks the indices (one
    wait for the device) and keeps 24 bytes an edge; any number of calls may
    use it at once, on any stream that has waited for the one it was built on.
    """

    def __init__(self, idx, n: int):
        if not torch.is_tensor(idx) or not idx.is_cuda:
            raise TypeError("idx must be a CUDA tensor")
        if idx.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"idx must be int64 or int32, got {idx.dtype}")
        if idx.dim() != 2 or idx.shape[0] != 2:
            raise ValueError(f"idx must be (2, M), got shape {tuple(idx.shape)}")
        n, m = int(n), int(idx.shape[1])
        if not 1 <= n <= _MAX_ROWS or 2 * m > _MAX_ROWS:
            raise ValueError("n must be at least 1; at most 2^31 - 2 vertices and 2^30 - 1 edges")
        self.n, self.m, self.device = n, m, idx.device
        self._long = None
        if m == 0:
            return
        dev = self.device
        self._stream = _stream(dev.index)
        idx = idx.to(torch.int64).contiguous()
        self._ends = torch.empty(2 * m, dtype=torch.int32, device=dev)
        self._rowptr = torch.empty(n + 1, dtype=torch.int32, device=dev)
        self._other, self._eid = torch.empty((2, 2 * m), dtype=torch.int32, device=dev)
        bad = torch.empty(1, dtype=torch.int32, device=dev)
        nb = _L.lg_edge_graph_workspace_bytes(n, m)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev)
        _call(dev, _L.lg_edge_graph, n, m, idx.data_ptr(), self._ends.data_ptr(), self._rowptr.data_ptr(),
              self._other.data_ptr(), self._eid.data_ptr(), bad.data_ptr(), ws.data_ptr(), nb)
        degree = self._rowptr[1:] - self._rowptr[:-1]
        found = torch.stack([bad[0], degree.max()]).tolist()
        if found[0]:
            raise ValueError("edge index out of range [0, n)")
        if found[1] > _native.LG_EDGE_CHUNK:
            self._long = self._chunks(degree)

    def _chunks(self, degree):
        """The vertices with long edge lists and the chunks of their lists."""
        c = _native.LG_EDGE_CHUNK
        row = torch.nonzero(degree > c).reshape(-1)
        count = (degree[row].long() + c - 1) // c
        first = torch.cumsum(count, 0) - count
        total = int(count.sum())
        which = torch.repeat_interleave(torch.arange(row.numel(), device=row.device), count)
        begin = self._rowptr[row].long()[which] + c * (torch.arange(total, device=row.device) - first[which])
        i32 = [t.to(torch.int32).contiguous() for t in (row, first, row[which], begin)]
        return row.numel(), total, i32

    def _use(self):
        """Makes the lists known to the current stream when it is not the one
        they were allocated on."""
        if _stream(self.device.index) != self._stream:
            cur = torch.cuda.current_stream(self.device)
            for t in (self._ends, self._rowptr, self._other, *(self._long[2] if self._long else ())):
                t.record_stream(cur)

    def _check(self, x):
        _check_features("x", x)
        if x.dim() != 2 or x.shape[0] != self.n or x.shape[1] < 1 or x.shape[1] > 2 ** 20:
            raise ValueError(f"x must be ({self.n}, dim), got shape {tuple(x.shape)}")
        if x.device != self.device:
            raise ValueError(f"x is on {x.device}, the edges on {self.device}")

    def _forward(self, x):
        dim = x.shape[1]
        out = torch.empty(self.m, dtype=_acc(x.dtype), device=self.device)
        if self.m:
            x2, ld = _rows2d(x, dim)
            self._use()
            _call(self.device, _L.lg_edge_sqdist, self.n, self.m, dim, _CODES[x.dtype], self._ends.data_ptr(),
                  x2.data_ptr(), ld, out.data_ptr())
        return out

    def _backward(self, x, g):
        dim = x.shape[1]
        if self.m == 0:
            return torch.zeros((self.n, dim), dtype=x.dtype, device=self.device)
        dx = torch.empty((self.n, dim), dtype=x.dtype, device=self.device)
        x2, ld = _rows2d(x, dim)
        g = g.contiguous()
        code = _CODES[x.dtype]
        nlong = nchunks = nb = 0
        row = first = chunk_row = chunk_first = ws = None
        if self._long is not None:
            nlong, nchunks, lists = self._long
            row, first, chunk_row, chunk_first = (t.data_ptr() for t in lists)
            nb = _L.lg_edge_sqdist_grad_workspace_bytes(nchunks, dim, code)
            ws = torch.empty(nb, dtype=torch.uint8, device=self.device)
        self._use()
        _call(self.device, _L.lg_edge_sqdist_grad, self.n, self.m, dim, code, self._rowptr.data_ptr(),
              self._other.data_ptr(), self._eid.data_ptr(), nlong, row, first, nchunks, chunk_row, chunk_first,
              x2.data_ptr(), ld, g.data_ptr(), dx.data_ptr(), _ptr(ws), nb)
        return dx

    def __call__(self, x):
        self._check(x)
        if torch.is_grad_enabled() and x.requires_grad:
            return _EdgeDist.apply(x, self)
        return self._forward(x)


def edge_sqdist(x, idx):
    """Squared distances of the rows of x (n, dim) along the edges idx (2, M);
    see EdgeDistances, which a program with a fixed graph builds once."""
    _check_features("x", x)
    if x.dim() != 2:
        raise ValueError(f"x must be (n, dim), got shape {tuple(x.shape)}")
    return EdgeDistances(idx, x.shape[0])(x)
