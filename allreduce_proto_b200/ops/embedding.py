"""Embedding lookup with scaling, and the gradient of its table.

The gradient is summed by sorted tokens: every row of the table is written once, the sum of its tokens' rows in float32,
in parts that are joined in the tokens' order.  It is the same for the same inputs, whatever ran beside it, so ranks that
hold replicas agree; and it can be added straight into a gradient bucket, where only the rows that tokens name are
touched.  Tokens outside of the table give a row of zeros and no gradient: padded places (-1), or the tokens of another
rank's part of a table that is split by rows (look up ``tokens - first_row`` and allreduce the rows)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _native
from .._native import IbcommError
from ..parallel.communicator import dtype_code


def _check(tokens: torch.Tensor, padding_idx: Optional[int], rows: int) -> int:
    if tokens.dtype not in (torch.int32, torch.int64):
        raise IbcommError(_native.NOT_SUPPORTED, f"tokens are int32 or int64, got {tokens.dtype}")
    if padding_idx is None:
        return -1
    if not 0 <= padding_idx < rows:
        raise IbcommError(_native.INVALID_ARGUMENT, f"padding_idx {padding_idx} is no row of {rows}")
    return int(padding_idx)


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None,
              out_dtype=None, grad_into: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * weight[tokens]``, of shape ``tokens.shape + (width,)`` and type ``out_dtype`` (default: the table's).

    ``tokens`` int32 or int64, ``weight`` ``(rows, width)`` float32, float16 or bfloat16; on the current stream.
    Differentiable in ``weight``, backward and once (forward-mode derivatives and ``torch.jit.trace`` are refused): its
    gradient is summed in float32 and comes in the table's type, without the row ``padding_idx``.  With ``grad_into`` (a
    tensor of the table's shape, such as its view in a gradient bucket) the backward pass adds the gradient there instead,
    and autograd has nothing to add to ``weight.grad`` (``torch.autograd.grad`` finds a gradient of zeros, or none); lookups
    that add into one tensor belong on one stream, since nothing orders their backward passes otherwise.  A table with
    tensor hooks has its gradient handed to them and added by autograd as usual where ``weight.grad`` is ``grad_into``;
    elsewhere the backward pass is refused."""
    padding = _check(tokens, padding_idx, weight.shape[0] if weight.dim() == 2 else 0)
    out_code = -1 if out_dtype is None else dtype_code(out_dtype)
    tokens = tokens.contiguous()
    if grad_into is not None:
        if grad_into.shape != weight.shape or not grad_into.is_contiguous() or grad_into.device != weight.device:
            raise IbcommError(_native.INVALID_ARGUMENT, "grad_into must be contiguous, of the table's shape and on its GPU")
        if grad_into.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise IbcommError(_native.NOT_SUPPORTED, f"no embedding of {grad_into.dtype}")
    return _native.fast().embedding(tokens, weight, out_code, float(scale), padding, grad_into)


def embedding_grad(tokens: torch.Tensor, grad: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                   num_rows: Optional[int] = None, dtype=None, accumulate: bool = False, scale: float = 1.0,
                   padding_idx: Optional[int] = None) -> torch.Tensor:
    """The gradient of :func:`embedding`'s table: row ``v`` = ``scale`` times the sum of ``grad``'s rows at the places
    where ``tokens`` is ``v``.

    ``out`` (contiguous, ``(rows, width)``) is overwritten, rows without tokens with zeros; with ``accumulate`` the sums
    are added to it and only rows that tokens name are touched (in float32 tables subnormal numbers, below 1.2e-38, are
    added as zero).  Without ``out`` a table of ``num_rows`` rows in ``dtype``
    (default: ``grad``'s) is made.  Types float32, float16, bfloat16 in any mixture; sums in float32, rounded once.  Not
    differentiable itself.  ``tokens`` and ``grad`` may come from several ranks (``all_gather`` both): with many rows that
    few tokens name, that is less to send than the table's gradient."""
    if out is None:
        if num_rows is None or num_rows < 0 or accumulate:
            raise IbcommError(_native.INVALID_ARGUMENT, "give out, or num_rows without accumulate")
        if grad.dim() < 1:
            raise IbcommError(_native.INVALID_ARGUMENT, "grad must hold a row of the table's width for every token")
        padding = _check(tokens, padding_idx, num_rows)
        out = torch.empty(num_rows, grad.shape[-1], dtype=dtype or grad.dtype, device=grad.device)
    else:
        if num_rows is not None or dtype is not None:
            raise IbcommError(_native.INVALID_ARGUMENT, "out has its own rows and type")
        padding = _check(tokens, padding_idx, out.shape[0] if out.dim() == 2 else 0)
    _native.fast().embedding_grad(tokens.contiguous(), grad.contiguous(), out, padding, float(scale), bool(accumulate))
    return out
