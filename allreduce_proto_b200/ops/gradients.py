"""The norm of a training step's gradients, and clipping: what comes between the allreduce and the optimizer.

The norm is that of all tensors taken as one vector.  CUDA tensors: one pass over the gradients for the norm, one more
where something is to be scaled; nothing is read back to the host, so the calls can be captured in a CUDA graph.  Sums are
kept in float64 and joined in a fixed order: ranks with the same gradients in tensors of the same layout (sizes, order,
addresses modulo 32 bytes, as in gradient buckets) get the same bits.  CPU tensors (float32, float64) are handled by the
host library."""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Union

import torch

from .. import _native
from .._native import GradTensor, IbcommError, check
from ..parallel.communicator import Communicator, _ptr, dtype_code

Tensors = Union[torch.Tensor, Sequence[torch.Tensor]]
_EPS = 1e-6


def _list(tensors: Tensors) -> list:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _power(norm_type: float) -> int:
    if norm_type == 2:
        return 2
    if norm_type == math.inf:
        return 0
    raise IbcommError(_native.NOT_SUPPORTED, f"norm_type is 2 or inf, got {norm_type}")


def _host_list(tensors: list, outs: list):
    items = (GradTensor * len(tensors))()
    for item, t, o in zip(items, tensors, outs):
        if not isinstance(t, torch.Tensor) or not isinstance(o, torch.Tensor):
            raise TypeError("a torch.Tensor is expected")
        if t.is_cuda or o.is_cuda:
            raise IbcommError(_native.INVALID_ARGUMENT, "the tensors must live on one kind of device")
        if o.shape != t.shape:
            raise IbcommError(_native.INVALID_ARGUMENT, "an output must match its tensor in shape and strides")
        item.in_, item.out, item.len_elements = _ptr(t), _ptr(o), t.numel()
        item.dtype_in, item.dtype_out = dtype_code(t.dtype), dtype_code(o.dtype)
    return items


def _on_host(tensors: list) -> bool:
    return bool(tensors) and isinstance(tensors[0], torch.Tensor) and not tensors[0].is_cuda


def _several(comm: Optional[Communicator]) -> bool:
    return comm is not None and comm.world_size > 1


def _host_norm(items, tensors: list, power: int, comm: Optional[Communicator]) -> torch.Tensor:
    total = C.c_double(0.0)
    check(_native.lib().ibcomm_grad_sum_host(items, len(tensors), power, C.byref(total)))
    joined = total.value
    if _several(comm):
        sums = torch.empty(comm.world_size, dtype=torch.float64)
        comm.all_gather(torch.tensor([joined], dtype=torch.float64), sums)
        joined = float(sums.sum() if power == 2 else sums.amax())
    norm = math.sqrt(joined) if power == 2 else joined
    return torch.tensor(norm, dtype=torch.float64)


def _result(norm: torch.Tensor, tensors: list) -> torch.Tensor:
    return norm if any(t.dtype == torch.float64 for t in tensors) else norm.float()


def _rank_sums(tensors: list, power: int, comm: Optional[Communicator]) -> Optional[torch.Tensor]:
    """Every rank's sum of squares (or maximum), on the GPU; None where this rank has all there is."""
    if not _several(comm):
        return None
    mine = _native.fast().grad_norm(tensors, power, None, 1)
    sums = torch.empty(comm.world_size, dtype=torch.float64, device=mine.device)
    comm.all_gather(mine, sums)
    return sums


def grad_norm(tensors: Tensors, *, norm_type: float = 2.0, comm: Optional[Communicator] = None) -> torch.Tensor:
    """The norm of all ``tensors`` taken as one vector, a tensor without dimensions on their device (float64 where one
    of them is, else float32).

    ``norm_type`` 2 or ``inf`` (the largest magnitude).  CUDA: float32, float64, float16 and bfloat16 in any mixture,
    any dense layout, on the current stream.  ``comm``: the ranks hold different parts (see
    :meth:`GradientBuckets.reduce_scatter`), and the norm is that of all parts; every rank calls.  Without tensors the
    norm is zero.  The norm is a number: nothing is differentiated through it."""
    tensors, power = _list(tensors), _power(norm_type)
    if not tensors:
        if _several(comm):
            raise IbcommError(_native.INVALID_ARGUMENT, "a rank has to bring a tensor, of no elements if it has none")
        return torch.zeros(())
    if _on_host(tensors):
        return _result(_host_norm(_host_list(tensors, tensors), tensors, power, comm), tensors)
    return _native.fast().grad_norm(tensors, power, _rank_sums(tensors, power, comm), 0)


def clip_grad_norm(tensors: Tensors, max_norm: float, *, out: Optional[Tensors] = None, norm_type: float = 2.0,
                   comm: Optional[Communicator] = None) -> torch.Tensor:
    """Scales ``tensors`` by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm they had (see :func:`grad_norm`).

    In place unless ``out`` is given: one tensor per tensor, of the same shape, into which the scaled values go, rounded
    once; float32 may go to the 16-bit types and back (the float32 gradients an optimizer wants of bfloat16 buckets).
    No memory that is written may belong to two tensors of the call.  Gradients whose norm is not finite become NaN, or
    zero where they were finite and the norm is infinite (NaN with an infinite ``max_norm``); check the returned norm to
    skip such a step.  What a tensor holds beside gradients, such as the padding of ``GradientBuckets.flat``, becomes NaN
    with them: hand over the gradients alone, or call :meth:`GradientBuckets.clip_grad_norm`."""
    tensors, power = _list(tensors), _power(norm_type)
    outs = tensors if out is None else _list(out)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise IbcommError(_native.INVALID_ARGUMENT, f"max_norm is not negative, got {max_norm}")
    if len(outs) != len(tensors):
        raise IbcommError(_native.INVALID_ARGUMENT, "one output per tensor is expected")
    if not tensors:
        return grad_norm(tensors, norm_type=norm_type, comm=comm)
    if _on_host(tensors):
        items = _host_list(tensors, outs)
        norm = _host_norm(items, tensors, power, comm)
        c = max_norm / (float(norm) + _EPS)
        check(_native.lib().ibcomm_scale_grads_host(items, len(tensors), 1.0 if c >= 1.0 else c))
        return _result(norm, tensors)
    return _native.fast().clip_grads(tensors, None if out is None else outs, power, max_norm, _rank_sums(tensors, power, comm))
