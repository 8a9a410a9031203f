"""Distillation from a teacher's listed logits through the student's frozen head, with
the gradient for the hidden states.

Per row, with the student's q = softmax(hidden . weight^T / temperature) and the teacher's
p on its listed tokens (``top_logits`` gives indices, logits and log-sum-exp):

    loss = KL(p || q),   mass = the student's probability of the listed tokens.

With ``teacher_lse`` p is the teacher's true probability and all unlisted tokens form one
bucket on both sides; without it p is renormalised over the list.  The student's logits
are sums in fp32 and are not rounded before the softmax.  Where a gradient is wanted it
is formed in the forward call (the upstream gradient only scales rows), so what stays
until backward is one fp32 array of the hidden states' shape; the vocabulary-sized array
lives in the call's workspace, 16 bits per logit and at most 4 GB at a time.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._spec import BRAIN, HALF, LONG, SINGLE, WIDE_FLOATS, Number, Operand, admit, refuse

MAX_K = 256
_HIDDEN = Operand(HALF, BRAIN, ndim=2, layout=None)
_WEIGHT = {dtype: Operand(dtype, ndim=2, layout=None, frozen=True) for dtype in (HALF, BRAIN)}
_INDICES = Operand(LONG, ndim=2, layout=None)
_LOGITS = Operand(*WIDE_FLOATS, ndim=2, layout=None, frozen=True)
_LSE = Operand(SINGLE, ndim=1, layout=None, frozen=True, optional=True)
_TEMPERATURE = Number()


def _operand(t, width):
    """t [rows, h] contiguous, 16-byte aligned, with zero columns up to `width`."""
    if t.shape[1] == width and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    out = torch.empty((t.shape[0], width), dtype=t.dtype, device=t.device)
    _lib.call("sb_pad_rows", t.data_ptr(), t.shape[0], t.shape[1], t.stride(0), width, out.data_ptr(),
              _lib.raw_stream(t.device))
    return out


class _HeadDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, indices, logits, teacher_lse, temperature, gradient):
        rows, width = hidden.shape
        vocab, listed = weight.shape[0], indices.shape[1]
        padded = -(-width // 8) * 8
        dev = hidden.device
        loss = hidden.new_empty(rows, dtype=SINGLE)
        mass = hidden.new_empty(rows, dtype=SINGLE)
        place = hidden.new_empty(rows, dtype=torch.int32)
        du = hidden.new_empty((rows, padded), dtype=SINGLE) if gradient else None
        if rows:
            x, w = _operand(hidden, padded), _operand(weight, padded)
            indices, logits = indices.contiguous(), logits.contiguous()
            lse = None if teacher_lse is None else teacher_lse.contiguous()
            nbytes = _lib.query("sb_distill_workspace_bytes", rows, padded, vocab, listed, int(gradient))
            scratch = hidden.new_empty(nbytes, dtype=torch.uint8)
            _lib.call("sb_distill_forward", x.data_ptr(), rows, padded, w.data_ptr(), vocab,
                      _lib.wide_dtype_code(w.dtype), indices.data_ptr(), logits.data_ptr(),
                      _lib.wide_dtype_code(logits.dtype), listed, _lib.ptr(lse), temperature, loss.data_ptr(),
                      mass.data_ptr(), _lib.ptr(du), place.data_ptr(), scratch.data_ptr(), nbytes,
                      _lib.raw_stream(dev))
        if gradient:
            ctx.save_for_backward(du, place)
        ctx.meta = (hidden.dtype, width)
        ctx.mark_non_differentiable(mass)
        ctx.set_materialize_grads(False)
        return loss, mass

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_unused):
        if grad_loss is None or not ctx.needs_input_grad[0]:
            return (None,) * 7
        du, place = ctx.saved_tensors
        dtype, width = ctx.meta
        rows, padded = du.shape
        dx = du.new_empty((rows, padded), dtype=dtype)
        if rows:
            with _lib.on_device(du.device):
                g = grad_loss.contiguous()
                _lib.call("sb_distill_backward", du.data_ptr(), place.data_ptr(), g.data_ptr(), rows, padded,
                          dx.data_ptr(), _lib.wide_dtype_code(dtype), _lib.raw_stream(du.device))
        return (dx[:, :width],) + (None,) * 6


def check_lists(indices, vocab):
    """ValueError if an index is neither -1 nor in [0, vocab), or a row lists a token twice
    (waits for the device)."""
    faults = torch.empty(2, device=indices.device, dtype=LONG)
    _lib.call("sb_distill_check", indices.data_ptr(), indices.shape[0], indices.shape[1], vocab, faults.data_ptr(),
              _lib.stream_of(indices.device))
    outside, repeats = faults.tolist()
    if outside:
        refuse("fused_linear_distillation", f"{outside} indices lie outside the vocabulary [0, {vocab})")
    if repeats:
        refuse("fused_linear_distillation", f"{repeats} indices repeat a token their row already lists")


def fused_linear_distillation(hidden, weight, indices, logits, teacher_lse=None, *, temperature=1.0,
                              validate=True):
    """(loss, mass) per row, fp32 [N], for CUDA hidden [N, H] and a frozen head weight
    [V, H] of one dtype (fp16/bf16), the teacher's listed tokens, indices [N, K] (int64,
    -1 where a row lists fewer) with logits [N, K] (fp16/bf16/fp32), and optionally its
    log-sum-exp [N] (fp32) at the same temperature.  K <= 256.  Only loss is
    differentiable, with respect to hidden; it carries no temperature^2 factor.  Rows
    without a listed token give zeros.  ``validate`` checks the indices and waits for
    the device; without it an index outside the vocabulary counts as unused and repeats
    within a row give an unspecified loss."""
    entry = "fused_linear_distillation"
    device = hidden.device if isinstance(hidden, torch.Tensor) else None
    admit(entry, device, hidden=(hidden, _HIDDEN))
    admit(entry, device, weight=(weight, _WEIGHT[hidden.dtype]), indices=(indices, _INDICES), logits=(logits, _LOGITS),
          teacher_lse=(teacher_lse, _LSE), temperature=(temperature, _TEMPERATURE))
    rows, vocab = hidden.shape[0], weight.shape[0]
    if vocab == 0 or weight.shape[1] == 0:
        refuse(entry, f"weight {tuple(weight.shape)} has an empty vocabulary or hidden size")
    if not (hidden.shape[1] == weight.shape[1] and indices.shape[0] == rows and logits.shape == indices.shape
            and (teacher_lse is None or teacher_lse.shape == (rows,))):
        refuse(entry, f"hidden {tuple(hidden.shape)}, weight {tuple(weight.shape)}, indices {tuple(indices.shape)}, "
                      f"logits {tuple(logits.shape)} and teacher_lse "
                      f"{None if teacher_lse is None else tuple(teacher_lse.shape)} do not line up")
    if not 1 <= indices.shape[1] <= MAX_K:
        refuse(entry, f"indices list {indices.shape[1]} tokens per row; between 1 and {MAX_K} are taken")
    if not temperature > 0:
        refuse(entry, f"temperature is {temperature!r}; a positive value is required")
    with _lib.on_device(device):
        if validate and rows:
            check_lists(indices.contiguous(), vocab)
        gradient = hidden.requires_grad and torch.is_grad_enabled()
        return _HeadDistillation.apply(hidden, weight, indices, logits, teacher_lse, float(temperature), gradient)
