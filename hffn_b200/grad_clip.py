"""The global gradient norm over many tensors and clipping by it, without a host synchronisation
(``hffn_grad_norm`` / ``hffn_clip_grad_norm``): one launch reads every tensor, one more scales them, whatever their
number. No counterpart in the reference, whose training step has no clipping.

``HFFNTrainRuntime.clip_grad_norm`` clips the compact gradients of an HFFN stack together with a model's other
gradients; these functions take any list of float32 and bfloat16 CUDA tensors.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as native

DTYPES = {torch.float32: native.F32, torch.bfloat16: native.BF16}


def _dense(t: torch.Tensor) -> bool:
    """Whether the tensor's entries fill one stretch of memory, each once (contiguous, or a permutation of it)."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected = stride * size
    return True


def _check(tensors, what: str) -> list[torch.Tensor]:
    tensors = list(tensors)
    for t in tensors:
        if not isinstance(t, torch.Tensor) or t.dtype not in DTYPES or t.layout != torch.strided:
            raise ValueError(f"{what} must be float32 or bfloat16 tensors")
        if not t.is_cuda or t.device != tensors[0].device:
            raise ValueError(f"{what} must be on one CUDA device")
        if not _dense(t):
            raise ValueError(f"{what} must be dense in memory")
    return tensors


def _arrays(tensors):
    count = len(tensors)
    return ((ctypes.c_void_p * count)(*[t.data_ptr() for t in tensors]),
            (ctypes.c_int64 * count)(*[t.numel() for t in tensors]),
            (ctypes.c_int32 * count)(*[DTYPES[t.dtype] for t in tensors]))


def _buffers(tensors):
    """The norm (a float32 scalar) and the workspace of a call, from torch's allocator on the current stream."""
    device = tensors[0].device if tensors else torch.device("cuda", torch.cuda.current_device())
    size = int(native.lib.hffn_grad_norm_workspace(len(tensors)))
    return device, torch.empty((), device=device), torch.empty(size, dtype=torch.uint8, device=device)


def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm over every entry of ``tensors`` (float32 / bfloat16, dense, on one CUDA device): a float32 scalar on
    that device, computed in float64 and rounded once. An empty list has norm 0 (on the current device)."""
    tensors = _check(tensors, "tensors")
    device, norm, work = _buffers(tensors)
    pointers, counts, types = _arrays(tensors)
    with torch.cuda.device(device):
        native.check(native.lib.hffn_grad_norm(len(tensors), pointers, counts, types, norm.data_ptr(), work.data_ptr(),
                                               native.stream_handle(device)), "hffn_grad_norm")
    return norm


@torch.no_grad()
def clip_grad_norm(tensors, max_norm: float, out=None) -> torch.Tensor:
    """Scale every entry by ``min(1, max_norm / (norm + 1e-6))`` and return the norm before it (``grad_norm``), a
    float32 scalar on the device; the host waits for nothing.

    In place, or into ``out``: one tensor of the same shape for each (float32 or bfloat16, e.g. an optimizer's float32
    buffers for bfloat16 gradients). The scaled values are computed in float32 and rounded once to the output's type.
    With a norm that is infinite or NaN the factor is 0 or NaN, as with ``torch.nn.utils.clip_grad_norm_``.
    Refused (ValueError): tensors that share memory with one that is written, an output that overlaps another tensor's
    input, a negative ``max_norm``."""
    tensors = _check(tensors, "tensors")
    outs = tensors if out is None else _check(out, "outputs")
    if len(outs) != len(tensors) or any(o.shape != t.shape or (o is not t and o.stride() != t.stride())
                                        for o, t in zip(outs, tensors)):
        raise ValueError("out needs one tensor of the same shape and strides for each")
    if tensors and outs[0].device != tensors[0].device:
        raise ValueError("outputs must be on the tensors' device")
    device, norm, work = _buffers(tensors)
    pointers, counts, types = _arrays(tensors)
    out_pointers, _, out_types = _arrays(outs)
    with torch.cuda.device(device):
        native.check(native.lib.hffn_clip_grad_norm(len(tensors), pointers, out_pointers, counts, types, out_types,
                                                    float(max_norm), norm.data_ptr(), work.data_ptr(),
                                                    native.stream_handle(device)), "hffn_clip_grad_norm")
    torch.autograd.graph.increment_version(outs)
    return norm
