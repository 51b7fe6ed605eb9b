"""Token embedding with scale, position table and vocabulary shards; gradients by sorted tokens.

``y[t] = scale * weight[ids[t]] + position_weight[position[t]]``, formed in fp32 and rounded once
into the tables' dtype, in one kernel (`csrc/kernels/embedding.hip`).  The backward adds the
gradient rows of each token's occurrences in token order and in fp32 -- the same bits on every
run -- and writes the parameters' flat-buffer gradients in place where they are bound
(`parallel/flat.py`): only the rows that occur are touched then, and no dense gradient exists
(autograd gets none for them; their post-accumulate hooks still fire).  A parameter with other hooks
takes its gradient through autograd: they see it, and may change it, before it is added.
A pass that builds a graph of its own (``create_graph``) can be differentiated again.
CPU tensors use plain torch operations, and so do calls whose launch would go unnoticed: on dual
numbers (forward-mode derivatives), inside function transforms (``torch.vmap``, ``torch.func``), under
``torch.compile``, ``torch.jit.trace`` or a dispatch mode, and of tensor classes that dispatch
operations themselves.  torch.autocast changes nothing: both tables and the result are of one type.
"""
import math

import torch

from ..backend.exceptions import SMPInvalidArgumentError
from ._ext import ext


def _rows_torch(ids, table, padding_idx, fill):
    """Rows of a table; `fill` where an id is none of its rows."""
    rows = table.shape[0]
    outside = (ids < 0) | (ids >= rows)
    if padding_idx is not None and not 0 <= padding_idx < rows:
        padding_idx = None
    y = torch.nn.functional.embedding(ids.clamp(0, rows - 1), table, padding_idx)
    return y.masked_fill(outside.unsqueeze(-1), fill)


def _embedding_torch(ids, weight, padding_idx, scale, vocab_start, position_ids, position_weight, nan_outside=False):
    """In torch's operations.  nan_outside: ids outside a whole table give NaN, as by the kernels,
    instead of torch's own error."""
    if vocab_start is not None:
        pad = None if padding_idx is None else padding_idx - vocab_start
        y = _rows_torch(ids - vocab_start, weight, pad, 0.0)
    elif nan_outside:
        y = _rows_torch(ids, weight, padding_idx, math.nan)
    else:
        y = torch.nn.functional.embedding(ids, weight, padding_idx)
    if position_weight is None:
        return y if scale == 1.0 else (y.float() * scale).to(weight.dtype)
    if position_ids is None:
        position_ids = torch.arange(ids.shape[-1], device=ids.device).expand(ids.shape)
    if nan_outside:
        p = _rows_torch(position_ids, position_weight, None, math.nan)
    else:
        p = torch.nn.functional.embedding(position_ids, position_weight)
    return (y.float() * scale + p.float()).to(weight.dtype)


MAX_TOKENS = 1 << 27
MAX_ROWS = (1 << 31) - 1
MAX_COLUMNS = 1 << 24
MAX_VECTORS = ((1 << 24) - 1) * 1024  # of 8 elements, in the output: what one launch writes
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _table_ok(rows, dim):
    return rows < MAX_ROWS and dim <= MAX_COLUMNS


def _list_ok(n, dim):
    return n <= MAX_TOKENS and n * ((dim + 7) // 8) <= MAX_VECTORS


def _check_ids(name, t, device):
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64):
        raise SMPInvalidArgumentError(f"{name} must be an int32 or int64 tensor")
    if t.device != device:
        raise SMPInvalidArgumentError(f"{name} is on {t.device}, the table on {device}")


def embedding(ids, weight, padding_idx=None, scale=1.0, vocab_start=None, position_ids=None, position_weight=None):
    """``scale * weight[ids] + position_weight[position_ids]`` -> ``[*ids.shape, dim]``.

    ``weight`` [rows, dim] fp32 / fp16 / bf16; ``ids`` int32 or int64 of any shape.
    ``padding_idx``: a token id that gets no gradient (negative: counted from the table's end).
    ``vocab_start``: the table holds the ids ``vocab_start .. vocab_start + rows - 1`` of a larger
    vocabulary; the other ids give zeros and take no gradient.  Without it an id outside the table
    is an error: IndexError on the CPU, a row of NaN on the GPU (nothing waits for the ids there).
    ``position_weight`` [positions, dim]: rows added unscaled, chosen by ``position_ids``
    (broadcast to ``ids``) or, without them, by the place in the last dimension."""
    if not torch.is_tensor(weight) or weight.dim() != 2 or weight.dtype not in _FLOATS or 0 in weight.shape:
        raise SMPInvalidArgumentError("weight must be a [rows, dim] fp32 / fp16 / bf16 tensor")
    _check_ids("ids", ids, weight.device)
    rows, dim = weight.shape
    if not _table_ok(rows, dim):
        raise SMPInvalidArgumentError(f"tables of fewer than {MAX_ROWS} rows, of at most {MAX_COLUMNS} columns, are supported")
    n = ids.numel()
    if not _list_ok(n, dim):
        raise SMPInvalidArgumentError(f"{n} tokens of {dim} in one call: at most {MAX_TOKENS} tokens and {8 * MAX_VECTORS} "
                                      f"elements are supported")
    scale = float(scale)
    if not math.isfinite(scale):
        raise SMPInvalidArgumentError(f"scale must be finite, got {scale}")
    if vocab_start is not None:
        vocab_start = int(vocab_start)
        if vocab_start < 0 or (padding_idx is not None and padding_idx < 0):
            raise SMPInvalidArgumentError("vocab_start, and padding_idx beside it, must not be negative")
    elif padding_idx is not None:
        if not -rows <= padding_idx < rows:
            raise SMPInvalidArgumentError(f"padding_idx {padding_idx} is not a row of a table of {rows}")
        padding_idx = padding_idx % rows
    if position_weight is None:
        if position_ids is not None:
            raise SMPInvalidArgumentError("position_ids need a position_weight")
    else:
        if not torch.is_tensor(position_weight) or position_weight.dim() != 2 \
                or position_weight.shape[1] != weight.shape[1] or not 0 < position_weight.shape[0] < MAX_ROWS:
            raise SMPInvalidArgumentError("position_weight must be [positions, dim] with weight's dim")
        if position_weight.dtype != weight.dtype or position_weight.device != weight.device:
            raise SMPInvalidArgumentError("position_weight must have weight's dtype and device")
        if position_ids is not None:
            _check_ids("position_ids", position_ids, weight.device)
            try:
                position_ids = position_ids.expand(ids.shape)
            except RuntimeError:
                raise SMPInvalidArgumentError(f"position_ids {tuple(position_ids.shape)} do not broadcast to "
                                              f"{tuple(ids.shape)}") from None
        elif ids.dim() == 0 or ids.shape[-1] > position_weight.shape[0]:
            raise SMPInvalidArgumentError(f"ids {tuple(ids.shape)} need position_ids: the position table has "
                                          f"{position_weight.shape[0]} rows")
    if weight.is_cuda and not torch.compiler.is_compiling():
        start = vocab_start or 0
        y = ext().embedding(weight, position_weight, ids, position_ids, scale, start, vocab_start is not None,
                            -1 if padding_idx is None else padding_idx - start,
                            getattr(weight, "_smp_fused_grad", False),
                            getattr(position_weight, "_smp_fused_grad", False))
        if y is not None:
            return y
    return _embedding_torch(ids, weight, padding_idx, scale, vocab_start, position_ids, position_weight, weight.is_cuda)


def lookup(ids, weight, padding_idx=None, vocab_start=None):
    """``embedding`` without scale and positions, for modules: tables of other types (fp64), empty
    shards, and tables or lists beyond the kernels' sizes go through plain torch operations."""
    if weight.dtype in _FLOATS and 0 not in weight.shape and _table_ok(*weight.shape) and _list_ok(ids.numel(), weight.shape[1]):
        return embedding(ids, weight, padding_idx, vocab_start=vocab_start)
    return _embedding_torch(ids, weight, padding_idx, 1.0, vocab_start, None, None)
