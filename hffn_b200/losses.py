"""The loss of a language model's head: softmax cross entropy of ``hidden @ weight.T`` over a large vocabulary, computed
piece by piece without the ``[tokens, vocabulary]`` logits, with its gradients (``hffn_linear_ce_forward`` /
``hffn_linear_ce_backward``). It stands beside the training runtime's MSE loss (``HFFNTrainRuntime.step_mse``); the
reference has no loss. ``pythia.causal_lm_loss`` is the loss of a whole Pythia model through it.

Types: float32 and bfloat16 (hidden and weight alike); losses are float32, sums are held in float32 or more.
"""
from __future__ import annotations

from functools import lru_cache

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _native as native
from .runtime import DTYPES, MAX_TOKENS

REDUCTIONS = tuple(native.REDUCE_CODES)


def _check(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, reduction: str) -> None:
    if reduction not in native.REDUCE_CODES:
        raise ValueError("reduction must be 'none', 'mean' or 'sum'")
    if hidden.dtype not in DTYPES or weight.dtype != hidden.dtype:
        raise ValueError("hidden and weight must both be float32 or both bfloat16")
    if targets.dtype != torch.int64:
        raise ValueError("targets must be int64")
    if not hidden.is_cuda or weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError("hidden, weight and targets must be on one CUDA device")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] \
            or targets.shape != hidden.shape[:-1]:
        raise ValueError("expected hidden [..., d], weight [vocabulary, d] and targets [...]")
    if weight.shape[0] < 1 or weight.shape[1] < 8 or weight.shape[1] % 8:
        raise ValueError("weight needs at least one row and a width that is a multiple of 8")
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        raise ValueError("weight must be contiguous and 16-byte aligned")
    if not 1 <= targets.numel() <= MAX_TOKENS:
        raise ValueError("unsupported token count")
    if unpack_dual(hidden).tangent is not None or unpack_dual(weight).tangent is not None:
        raise ValueError("forward-mode derivatives are not supported")


@lru_cache(maxsize=256)
def _sizes(code: int, n: int, d: int, vocab: int) -> tuple[int, int, int]:
    """Bytes of the state, the forward's and the backward's workspace; ValueError for sizes the kernels do not take."""
    sizes = (native.lib.hffn_linear_ce_state_bytes(code, n, d, vocab),
             native.lib.hffn_linear_ce_forward_workspace(code, n, d, vocab),
             native.lib.hffn_linear_ce_backward_workspace(code, n, d, vocab))
    if min(sizes) < 0:
        native.check(native.HFFN_ERR_ARGUMENT, "linear cross entropy")
    return sizes


def _forward(hidden, weight, targets, ignore_index, reduction, for_backward=True):
    """The losses of hidden [N, d] (any row stride) and the state that ``_backward`` reads."""
    n, d = hidden.shape
    vocab, device, code = weight.shape[0], hidden.device, DTYPES[hidden.dtype]
    if hidden.stride(1) != 1 or (n > 1 and hidden.stride(0) < d):
        hidden = hidden.contiguous()
    targets = targets.contiguous()
    state_bytes, work_bytes, _ = _sizes(code, n, d, vocab)
    loss = torch.empty(n if reduction == "none" else (), device=device)
    if for_backward:
        state = torch.empty(state_bytes, dtype=torch.uint8, device=device)
        work = torch.empty(work_bytes, dtype=torch.uint8, device=device)
        addresses = state.data_ptr(), work.data_ptr()
    else:                                     # one buffer; the state's size is a multiple of 256
        state = torch.empty(state_bytes + work_bytes, dtype=torch.uint8, device=device)
        addresses = state.data_ptr(), state.data_ptr() + state_bytes
    with native.on_device(device.index):
        native.check(native.lib.hffn_linear_ce_forward(
            code, hidden.data_ptr(), hidden.stride(0), weight.data_ptr(), targets.data_ptr(), ignore_index,
            native.REDUCE_CODES[reduction], for_backward, loss.data_ptr(), *addresses, n, d, vocab,
            native.raw_stream(device.index)), "hffn_linear_ce_forward")
    return loss, state


def _backward(weight, state, n, reduction, grad_loss, want_hidden=True, want_weight=True):
    (vocab, d), device, code = weight.shape, weight.device, DTYPES[weight.dtype]
    grad_loss = grad_loss.float().contiguous()
    grad_hidden = torch.empty(n, d, dtype=weight.dtype, device=device) if want_hidden else None
    grad_weight = torch.empty_like(weight) if want_weight else None
    work = torch.empty(_sizes(code, n, d, vocab)[2], dtype=torch.uint8, device=device)
    with native.on_device(device.index):
        native.check(native.lib.hffn_linear_ce_backward(
            code, weight.data_ptr(), native.REDUCE_CODES[reduction], grad_loss.data_ptr(),
            grad_hidden.data_ptr() if want_hidden else None, grad_weight.data_ptr() if want_weight else None,
            state.data_ptr(), work.data_ptr(), n, d, vocab, native.raw_stream(device.index)), "hffn_linear_ce_backward")
    return grad_hidden, grad_weight


class LinearCrossEntropyFunction(torch.autograd.Function):
    """``apply(hidden [N, d], weight, targets [N], ignore_index, reduction)`` -> the losses. The forward keeps what the
    backward needs (the kept rows' hidden states and log sums); the backward recomputes the logits."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        loss, state = _forward(hidden, weight, targets, ignore_index, reduction)
        ctx.save_for_backward(weight, state)
        ctx.n, ctx.reduction = hidden.shape[0], reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        weight, state = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        return (*_backward(weight, state, ctx.n, ctx.reduction, grad_loss, wanted[0], wanted[1]), None, None, None)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits ``hidden @ weight.T`` against ``targets``, differentiable in ``hidden`` and
    ``weight``, without the logits.

    ``hidden`` [..., d] and ``weight`` [vocabulary, d]: both float32 or both bfloat16, d a multiple of 8, the weight
    contiguous; ``targets`` [...] int64. Returns float32: the token losses [...] (``reduction="none"``), their sum, or
    their mean over the tokens that are not ignored. A token whose target is ``ignore_index`` has loss 0 and gradient
    0 and takes no part in anything, whatever its hidden state holds; when every token is ignored the mean is 0 and so
    are the gradients. A target outside [0, vocabulary) that is not ``ignore_index`` makes its token's loss (and the
    sum and the mean) NaN and gives no gradient: it is found without a host synchronisation.

    Accuracy. bfloat16: products of the inputs as they are; the probabilities less the targets (``reduction="none"``: times
    the gradient of the token's loss) are held in bfloat16 (2^-8 of each) on their way into the gradients. float32: the
    operands of the products are held as two fp16 parts. In the losses a row's entries keep 22 bits down to 2^-17 of its
    largest and are held to 2^-39 of that below, whatever the other rows hold. The gradients sum over rows, and there small
    terms beside large ones keep less: an entry of ``weight`` in ``grad_hidden``, or of ``hidden`` (times its token's
    gradient, for ``reduction="none"``) in ``grad_weight``, is held to 2^-39 of that tensor's largest, and a probability to
    2^-39: a row of ``grad_weight`` whose id is nowhere more probable than 1e-9 is off by up to two thousandths of itself,
    and is 0 from about 1e-12 on. A NaN or infinity of ``hidden`` stays with its token in the losses and ``grad_hidden``,
    one of ``weight`` reaches all.

    Memory. What the backward needs is kept until then: the kept rows of ``hidden`` (in ``hidden``'s type) and, for float32
    and more than 16 tokens, the head's two parts, as many bytes as ``weight`` (scoring allocates those for the call). The
    backward works on about 256 MB of probabilities at a time.

    Arguments are checked before any launch (ValueError); an empty batch is refused. No second derivatives, and none in
    forward mode: a tensor with a tangent is refused."""
    _check(hidden, weight, targets, reduction)
    rows, flat = (hidden, targets) if hidden.dim() == 2 else (hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1))
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        loss = LinearCrossEntropyFunction.apply(rows, weight, flat, int(ignore_index), reduction)
    else:
        loss, _ = _forward(rows, weight, flat, int(ignore_index), reduction, for_backward=False)
    return loss.view(targets.shape) if reduction == "none" and hidden.dim() != 2 else loss


@torch.no_grad()
def linear_cross_entropy_gradients(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                                   grad_loss: torch.Tensor | None = None, ignore_index: int = -100,
                                   reduction: str = "mean") -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, grad_hidden, grad_weight)`` of ``linear_cross_entropy`` in one call, outside autograd (a training loop
    with gradients of its own; a step captured into a CUDA graph: torch's engine cannot capture a backward whose leaves
    still belong to a graph made on another stream, this call can be captured at any time). ``grad_loss``: the gradient
    of the loss (float32, of its shape; default 1)."""
    _check(hidden, weight, targets, reduction)
    shape = targets.shape if reduction == "none" else ()
    if grad_loss is not None and (grad_loss.shape != shape or not grad_loss.is_floating_point()
                                  or grad_loss.device != hidden.device):
        raise ValueError("grad_loss must be a floating tensor of the loss's shape on its device")
    loss, state = _forward(hidden.reshape(-1, hidden.shape[-1]), weight, targets.reshape(-1), int(ignore_index),
                           reduction)
    grad_loss = torch.ones_like(loss) if grad_loss is None else grad_loss.reshape(loss.shape)
    grad_hidden, grad_weight = _backward(weight, state, targets.numel(), reduction, grad_loss)
    return loss.view(shape), grad_hidden.view(hidden.shape), grad_weight


def device_errors(device=None) -> int:
    """The error flag of the loss's kernels on ``device`` (0: none; the code of a wait that ran out otherwise; the losses
    or gradients of the call it ran out in are NaN). Synchronises."""
    flag = native.ctypes.c_int32(0)
    with torch.cuda.device(device):
        native.check(native.lib.hffn_linear_ce_error(native.ctypes.byref(flag), 0), "hffn_linear_ce_error")
    return int(flag.value)
