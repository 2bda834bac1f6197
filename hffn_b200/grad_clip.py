"""The global gradient norm over many tensors and clipping by it, without a host synchronisation
(``hffn_grad_norm`` / ``hffn_clip_grad_norm``): one launch reads every tensor, one more scales them, whatever their
number. No counterpart in the reference, whose training step has no clipping.

``HFFNTrainRuntime.clip_grad_norm`` clips the compact gradients of an HFFN stack together with a model's other
gradients; these functions take any list of float32 and bfloat16 CUDA tensors.
"""
from __future__ import annotations

from array import array

import torch

from . import _native as native

_CODES = {torch.float32: native.F32, torch.bfloat16: native.BF16}


def _dense(t: torch.Tensor) -> bool:
    """Whether the tensor's entries fill one stretch of memory, each once (contiguous, or a permutation of it)."""
    if t.layout != torch.strided:
        return False
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected = stride * size
    return True


class _List:
    """A checked list of tensors and the host arrays of the native calls. Written as passes of C-level calls over the
    list: a model has hundreds of gradients, and this is the host's cost of a call."""

    def __init__(self, tensors, what: str) -> None:
        tensors = self.tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        try:
            types = [_CODES[t.dtype] for t in tensors]
            devices = set(map(torch.Tensor.get_device, tensors))
            self.contiguous = list(map(torch.Tensor.is_contiguous, tensors))
            if not all(self.contiguous) and not all(c or _dense(t) for c, t in zip(self.contiguous, tensors)):
                raise ValueError(f"{what} must be dense in memory")
            self.pointers = array("Q", map(torch.Tensor.data_ptr, tensors))
            self.counts = array("q", map(torch.Tensor.numel, tensors))
        except (KeyError, TypeError, AttributeError, RuntimeError):
            raise ValueError(f"{what} must be dense float32 or bfloat16 tensors") from None
        if len(devices) > 1 or -1 in devices:
            raise ValueError(f"{what} must be on one CUDA device")
        self.types = array("i", types)
        self.device = devices.pop() if devices else torch.cuda.current_device()

    def __len__(self) -> int:
        return len(self.tensors)


def _address(a: array) -> int:
    return a.buffer_info()[0]


def _buffers(tensors: _List):
    """The norm (a float32 scalar) and the workspace of a call, from torch's allocator on the current stream."""
    device = torch.device("cuda", tensors.device)
    size = native.lib.hffn_grad_norm_workspace(len(tensors))
    return torch.empty((), device=device), torch.empty(size, dtype=torch.uint8, device=device)


def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm over every entry of ``tensors`` (one or many, float32 / bfloat16, dense, on one CUDA device): a float32
    scalar on that device, computed in float64 and rounded once. An empty list has norm 0 (on the current device). Outside
    autograd: the norm carries no derivative, whatever the tensors require."""
    tensors = _List(tensors, "tensors")
    norm, work = _buffers(tensors)
    with native.on_device(tensors.device):
        native.check(native.lib.hffn_grad_norm(len(tensors), _address(tensors.pointers), _address(tensors.counts),
                                               _address(tensors.types), norm.data_ptr(), work.data_ptr(),
                                               native.raw_stream(tensors.device)), "hffn_grad_norm")
    return norm


def clip_grad_norm(tensors, max_norm: float, out=None) -> torch.Tensor:
    """Scale every entry by ``min(1, max_norm / (norm + 1e-6))`` and return the norm before it (``grad_norm``), a
    float32 scalar on the device; the host waits for nothing.

    In place, or into ``out``: one tensor for each (float32 or bfloat16, e.g. an optimizer's float32 buffers for bfloat16
    gradients), contiguous with as many entries, or of the same shape and strides. The scaled values are computed in
    float32 and rounded once to the output's type.
    With a norm that is infinite or NaN the factor is 0 or NaN, as with ``torch.nn.utils.clip_grad_norm_`` (an infinite
    norm under an infinite ``max_norm``: NaN; for the norm alone there is ``grad_norm``).
    Refused (ValueError): tensors that share memory with one that is written, an output that overlaps another tensor's
    input, a negative ``max_norm``."""
    tensors = _List(tensors, "tensors")
    outs = tensors if out is None else _List(out, "outputs")
    if outs is not tensors:
        if len(outs) != len(tensors) or outs.counts != tensors.counts:
            raise ValueError("out needs one tensor with as many entries for each")
        if len(outs) and outs.device != tensors.device:
            raise ValueError("outputs must be on the tensors' device")
        if not all(tensors.contiguous) or not all(outs.contiguous):
            if any(not (a and b) and (t.shape != o.shape or t.stride() != o.stride()) for a, b, t, o in
                   zip(tensors.contiguous, outs.contiguous, tensors.tensors, outs.tensors)):
                raise ValueError("outputs that are not contiguous need their tensor's shape and strides")
    norm, work = _buffers(tensors)
    with native.on_device(tensors.device):
        native.check(native.lib.hffn_clip_grad_norm(
            len(tensors), _address(tensors.pointers), _address(outs.pointers), _address(tensors.counts),
            _address(tensors.types), _address(outs.types), float(max_norm), norm.data_ptr(), work.data_ptr(),
            native.raw_stream(tensors.device)), "hffn_clip_grad_norm")
    torch.autograd.graph.increment_version(outs.tensors)
    return norm
