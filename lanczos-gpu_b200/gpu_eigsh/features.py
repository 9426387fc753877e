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
in a fixed order, so equal calls give equal bits (an order may depend on the
strides and the alignment of the inputs).  Calls run on the current
stream of their tensors' device, allocate from torch and wait for nothing
(``EdgeDistances`` checks its indices when it is built, which waits once; the
rest can be captured into CUDA graphs; as with torch's own operations, capture a
backward pass only when no eager autograd graph of the same leaves is alive).
The gradients are not differentiable themselves (a second backward pass raises),
and there are no forward-mode derivatives (NotImplementedError).  There is no
CPU implementation.

Squared distances are the ``x_edge_dists`` of
``gpu_eigsh.imgp.make_imgp_precision_matvec``.  That operator differentiates
only with respect to its two scalars; gradients with respect to the distances
go through the matrix values of ``gpu_eigsh.differentiable_eigsh``, or through
a matvec of torch operations given to ``gpu_eigsh.funm_torch.slq_logdet``.

The argument checks, allocations and autograd nodes are compiled
(csrc/torch/features.cpp -> _lib/_torch_features.so), because these calls come
many times a step on small inputs.
"""
from __future__ import annotations

import importlib.util
import json
import operator
from pathlib import Path

import torch

from . import _native  # noqa: F401  (loads liblanczos_b200.so, which the binding calls)

__all__ = ["embedding_lookup", "layer_norm", "EdgeDistances", "edge_sqdist"]


_BUILD = "build it with `python lanczos-gpu_b200/build.py`.  There is no Python fallback."


def _load(path=Path(__file__).resolve().parent / "_lib" / "_torch_features.so"):
    if not path.exists():
        raise ImportError(f"{path} is missing; {_BUILD}")
    built_for = path.with_suffix(".json")
    if built_for.exists():
        version = json.loads(built_for.read_text())["torch"]
        if version != torch.__version__:
            raise ImportError(f"{path} was built for torch {version}, this is {torch.__version__}; {_BUILD}")
    try:
        spec = importlib.util.spec_from_file_location("_torch_features", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    except ImportError as e:
        raise ImportError(f"{path} does not load ({e}); {_BUILD}") from e
    return mod


_C = _load()


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
    if padding_idx is not None:
        padding_idx = operator.index(padding_idx)
        if not -2 ** 63 <= padding_idx < 2 ** 63:
            raise ValueError("padding_idx must fit 64 bits")
    if scale is None:
        return _C.embedding_lookup(table, ids, None, 1.0, False, padding_idx)
    if isinstance(scale, torch.Tensor):
        return _C.embedding_lookup(table, ids, scale, 1.0, False, padding_idx)
    return _C.embedding_lookup(table, ids, None, float(scale), True, padding_idx)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x (..., dim) over its last dimension:
    (x - mean) / sqrt(var + eps) * weight + bias, var the mean squared deviation.

    weight, bias : (dim,) tensors or None, of x's type, or float32 for a 16-bit
        x (both of the same type).  Gradients flow to x, weight and bias.
    """
    return _C.layer_norm(x, weight, bias, eps)


class EdgeDistances:
    """The edges of a graph of n vertices: idx (2, M) int64 or int32, edge e
    between vertices idx[0, e] and idx[1, e] (the edge lists of gpu_eigsh.imgp;
    repeated edges and edges from a vertex to itself are allowed).

    Called with features x (n, dim) it returns the squared distances (M,)
    |x[idx[0, e]] - x[idx[1, e]]|^2 in float32 (float64 for a float64 x), with
    gradients to x.  Building it sorts the edge ends, checks the indices
    (ValueError; one wait for the device) and keeps 24 bytes an edge; any number
    of calls may use it at once, on any stream that has waited for the one it
    was built on.  Keep it as long as a captured CUDA graph that uses it.
    """

    def __init__(self, idx, n: int):
        self._graph = _C.edge_graph(idx, n)
        self.n, self.m = self._graph.n, self._graph.m

    def __call__(self, x):
        return _C.edge_sqdist(x, self._graph)


def edge_sqdist(x, idx):
    """Squared distances of the rows of x (n, dim) along the edges idx (2, M);
    see EdgeDistances, which a program with a fixed graph builds once."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError("x must be a CUDA tensor")
    if x.dim() != 2:
        raise ValueError(f"x must be (n, dim), got shape {tuple(x.shape)}")
    return _C.edge_sqdist(x, _C.edge_graph(idx, x.shape[0]))
