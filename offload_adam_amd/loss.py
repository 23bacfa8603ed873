"""Cross entropy of a linear output layer, without its logits.

The logits of a language model are the largest tensor of its training step: 4096
tokens of the 8B model are 1 GB in bf16, 2.1 GB in the fp32 that the loss needs, and
as much again for their gradient.  ``linear_cross_entropy`` takes the hidden states
and the output layer's weight instead; HIP kernels fold each tile of logits into a
running maximum and sum while it is in registers and compute it again for the
gradients.  The reference has no counterpart: its example's model returns logits
(examples/e2e_train/train.py).
"""

import torch

from . import _lib
from .qweight import base as _qbase

_CASTABLE = (torch.float32, torch.float16, torch.bfloat16)
_REDUCTIONS = {"none": _lib.OA_LOSS_NONE, "mean": _lib.OA_LOSS_MEAN, "sum": _lib.OA_LOSS_SUM}


def _rows(t):
    """2-D operand of the kernels: unit column stride, columns and row stride multiples
    of 8 elements, 16-byte aligned.  Anything else is copied, zero-padded."""
    rows, cols = t.shape
    if cols % 8 == 0 and cols <= 1 << 20 and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, cols, cols
    stride = t.stride(0) if rows > 1 else -(-cols // 8) * 8
    if (cols % 8 == 0 and t.stride(1) == 1 and stride >= cols and stride % 8 == 0
            and stride <= 1 << 20 and t.data_ptr() % 16 == 0):
        return t, cols, stride
    padded = -(-cols // 8) * 8
    out = torch.zeros((rows, padded), dtype=t.dtype, device=t.device)
    out[:, :cols].copy_(t)
    return out, padded, padded


def _plain(weight, dtype):
    if isinstance(weight, _qbase.QWeightBase):
        return _qbase._dequantized(weight, dtype)
    return weight


def _head_args(x, w, target, ignore_index, reduction):
    x, hidden, ldx = _rows(x)
    w, _, ldw = _rows(w)
    args = [x.data_ptr(), ldx, w.data_ptr(), ldw, _lib.dtype_code(x.dtype), target.data_ptr(),
            x.shape[0], hidden, w.shape[0], ignore_index, _REDUCTIONS[reduction]]
    return args, hidden, (x, w)


def _workspace(device, tokens, hidden, vocab, backward, dx, dw):
    nbytes = _lib.load().oa_linear_ce_workspace_bytes(tokens, hidden, vocab, backward, dx, dw)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        dev, tokens = x.device, x.shape[0]
        lib = _lib.load()
        with _lib.device_guard(dev):
            w = _plain(weight, x.dtype)
            args, hidden, keep = _head_args(x, w, target, ignore_index, reduction)
            loss = torch.empty((tokens,) if reduction == "none" else (), dtype=torch.float32,
                               device=dev)
            stats = torch.empty(tokens + 1, dtype=torch.float32, device=dev)  # lse, count
            if loss.numel():
                ws = _workspace(dev, tokens, hidden, w.shape[0], 0, 0, 0)
                code = lib.oa_linear_ce_forward(
                    *args, loss.data_ptr(), stats.data_ptr(), stats.data_ptr() + 4 * tokens,
                    ws.data_ptr(), ws.numel(), _lib.current_stream_ptr())
                _lib.check(code, "oa_linear_ce_forward")
        ctx.save_for_backward(x, weight, target, stats)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @_qbase.first_derivatives_only
    def backward(ctx, saved, grad):
        x, weight, target, stats = saved
        want_dx, want_dw = ctx.needs_input_grad[:2]
        tokens, dev = x.shape[0], x.device
        if tokens == 0:
            return (torch.zeros_like(x) if want_dx else None,
                    torch.zeros(weight.shape, dtype=x.dtype, device=dev) if want_dw else None,
                    None, None, None)
        lib = _lib.load()
        with _lib.device_guard(dev):
            w = _plain(weight, x.dtype)
            args, hidden, keep = _head_args(x, w, target, ctx.ignore_index, ctx.reduction)
            vocab = w.shape[0]
            grad = grad.contiguous()
            dx = torch.empty((tokens, hidden), dtype=x.dtype, device=dev) if want_dx else None
            dw = torch.empty((vocab, hidden), dtype=x.dtype, device=dev) if want_dw else None
            ws = _workspace(dev, tokens, hidden, vocab, 1, int(want_dx), int(want_dw))
            code = lib.oa_linear_ce_backward(
                *args, stats.data_ptr(), stats.data_ptr() + 4 * tokens, grad.data_ptr(),
                dx.data_ptr() if want_dx else None, dw.data_ptr() if want_dw else None,
                ws.data_ptr(), ws.numel(), _lib.current_stream_ptr())
            _lib.check(code, "oa_linear_ce_backward")
            if hidden != x.shape[1]:  # operands were padded
                dx = dx[:, :x.shape[1]].contiguous() if want_dx else None
                dw = dw[:, :x.shape[1]].contiguous() if want_dw else None
        return dx, dw, None, None, None


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    """``F.cross_entropy(F.linear(x, weight).float(), target)`` without the logits.

    ``x``: hidden states (..., hidden), bf16 or fp16, on the GPU; ``weight``: the output
    layer's (vocab, hidden) in the same dtype, or a quantised weight of this package
    (decoded for the call); under ``torch.autocast`` both are cast to its dtype.
    ``target``: int64 of ``x``'s leading shape.  Tokens whose
    target is ``ignore_index`` take no part: their losses and gradients are 0, whatever
    their rows of ``x`` hold.  Any other target outside [0, vocab) gives NaN.

    ``reduction``: ``"mean"`` over the tokens that take part (NaN if there are none),
    ``"sum"``, or ``"none"`` (losses of ``target``'s shape).  The loss is fp32;
    logits, exponentials and sums are fp32 throughout, and only the logits' gradient is
    rounded to 16 bits, once, between the two products that use it.  (fp16 with a gradient
    per token: hidden states enter the weight's gradient scaled by a power of two, off by
    2^-17 at most for tokens whose gradient is 2^-20 of the largest or more.)  Gradients flow to
    ``x`` and ``weight``; taking second derivatives or forward-mode ones raises.  Results
    do not depend on anything but the arguments: no atomics, one order of summation.

    Works on ``x``'s device and the current stream, synchronises nothing, and may be
    captured into a graph, with the backward pass inside the same capture and no eager
    graph of the same leaves alive (torch ends the process when such a leaf's gradient
    is accumulated during a capture).
    """
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("x and weight must be tensors")
    decoded = weight.dtype
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    ignore_index = int(ignore_index)
    if not -2**63 <= ignore_index < 2**63:
        raise ValueError(f"ignore_index must be an int64, got {ignore_index}")
    low = _qbase.autocast_dtype(x)
    if low is not None:  # what F.linear casts
        if x.dtype in _CASTABLE:
            x = x.to(low)
        if weight.dtype in _CASTABLE:
            decoded = low
            if not isinstance(weight, _qbase.QWeightBase):
                weight = weight.to(low)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x must be bfloat16 or float16, got {x.dtype}")
    if decoded != x.dtype:
        raise TypeError(f"weight must have x's dtype {x.dtype}, got {weight.dtype}")
    if not isinstance(target, torch.Tensor) or target.dtype != torch.int64:
        raise TypeError("target must be an int64 tensor")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target has shape {tuple(target.shape)}, expected {tuple(x.shape[:-1])}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("weight must not be empty")
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor (no CPU path exists)")
    if weight.device != x.device or target.device != x.device:
        raise ValueError("x, weight and target must be on the same GPU")
    flat, rows = target, x
    if target.dim() != 1:
        flat, rows = target.reshape(-1), x.reshape(-1, x.shape[-1])
    loss = _LinearCrossEntropy.apply(rows, weight, flat.contiguous(), ignore_index, reduction)
    return loss.reshape(target.shape) if reduction == "none" else loss
