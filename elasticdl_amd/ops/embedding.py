"""Embedding lookup with scaling and pooling, and its gradient by sorted ids.

``embedding_lookup`` reads rows of a local table [rows, dim] for ids, or
pools bags of ids, with the padded-with--1 convention of the preprocessing
layers:

    out[b] = c[b] * sum over l of w[b, l] * table[ids[b, l]]

c[b] is ``scale`` over 1 (sum), n (mean) or sqrt(n) (sqrtn), with n the ids of
bag b, at least 1 (the combiners of layers/embedding.py). Its gradient sorts
the ids and sums each row's gradients in the order that the sort leaves them
in, in 32 bits: the same call gives the same bits, however often an id occurs.

``coalesce_rows`` is the same sum over (ids, rows) pairs, as unique ids in
order with their rows: what ``deduplicate_indexed_slices`` runs on a GPU.

On CUDA devices these are the kernels of csrc/embedding_kernels.hip; on the
CPU the same formulas in torch (ops/reference.py).
"""

from typing import Optional, Tuple

import torch

from elasticdl_amd.ops import reads_directly, reference, require_native

_COMBINERS = {None: -1, "sum": 0, "mean": 1, "sqrtn": 2}
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_MOST = 2 ** 31 - 4097  # positions and rows are 32-bit


def takes(table: torch.Tensor, ids: torch.Tensor,
          weights: Optional[torch.Tensor] = None) -> bool:
    """Whether ``embedding_lookup`` has these sizes and types; for callers
    that have another way."""
    given = (table, ids) if weights is None else (table, ids, weights)
    return (reads_directly(*given) and table.dtype in _DTYPES
            and ids.dtype in (torch.int64, torch.int32)
            and (weights is None or weights.dtype in _DTYPES)
            and table.shape[0] < _MOST and table.shape[1] < 2 ** 20
            and ids.numel() < _MOST)


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor,
                     weights: Optional[torch.Tensor] = None,
                     combiner: Optional[str] = None,
                     scale: float = 1.0) -> torch.Tensor:
    """Rows of ``table`` [rows, dim] for ``ids``, times ``scale``.

    Without a combiner ids have any shape, and the result is [*ids, dim];
    with "sum", "mean" or "sqrtn" ids are [bags, length] and the result is
    [bags, dim]. Ids below zero are padding: a row of zeros, or no part of
    their bag (their weights are not read). An id past the table raises
    IndexError on the CPU; on a GPU, where the ids are not read back, its
    output is NaN and it has no gradient.

    ``weights`` [bags, length] multiply each id's row; the mean's and
    sqrtn's divisor counts ids, not weights. (tf.nn.embedding_lookup_sparse
    divides by the weights' sum and the root of their squares' sum: for its
    results divide the weights by these first and take "sum".) The result has
    the table's type (float32, bfloat16 or float16), rounded once from a sum
    in 32 bits. The table's gradient is dense, in the table's type; weights
    have one too. Rows of the table may be strided; ids are fewer than
    2^31 - 4096.

    In code that is captured into a graph, take gradients with
    ``torch.autograd.grad`` (or drop eager graphs of the same leaves first):
    ``backward()`` accumulates on the stream of the eager graph's leaves,
    which ends the capture."""
    code = _COMBINERS.get(combiner)
    if code is None:
        raise ValueError(f"unknown combiner {combiner!r}")
    if table.is_cuda:
        return require_native().embedding_lookup(table, ids, weights, code,
                                                 scale)
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"table is {tuple(table.shape)}, not [rows, dim]")
    if table.dtype not in _DTYPES:
        raise TypeError("table must be float32, bfloat16 or float16, not "
                        f"{table.dtype}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32, not {ids.dtype}")
    if ids.device != table.device:
        raise ValueError(
            f"ids are on {ids.device}, and the table on {table.device}")
    if combiner is not None and ids.dim() != 2:
        raise ValueError("ids of bags must be [bags, length], not "
                         f"{tuple(ids.shape)}")
    if weights is not None:
        if combiner is None:
            raise ValueError("weights need a combiner")
        if weights.shape != ids.shape or weights.device != ids.device:
            raise ValueError("weights must have the ids' shape and device")
        if weights.dtype not in _DTYPES:
            raise TypeError("weights must be float32, bfloat16 or float16, "
                            f"not {weights.dtype}")
    return reference.embedding_lookup(table, ids, weights, combiner, scale)


def coalesce_rows(values: torch.Tensor, ids: torch.Tensor
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(summed rows [u, dim], unique ids [u] in order) of values [n, dim] and
    ids [n], any int64. GPU only, without a gradient; it reads back how many
    ids there are, so it cannot be captured into a graph."""
    if not values.is_cuda:
        raise ValueError("coalesce_rows runs on a GPU; use "
                         "deduplicate_indexed_slices")
    rows, unique = require_native().coalesce_rows(
        values.detach().contiguous(), ids.contiguous())
    return rows, unique
