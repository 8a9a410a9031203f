"""The k largest logits of each row and the row's log-sum-exp, in one pass: what a
teacher sends a student instead of its whole vocabulary row.

Values come in falling order, equal ones by the lower index, NaN above +inf; the
log-sum-exp is that of ``logits / temperature`` (-inf for a row of -inf, NaN for one
with a NaN).  ``fused_linear_distillation`` takes the three as they are.
"""

from __future__ import annotations

import torch

from .. import _lib
from .._spec import WIDE_FLOATS, Number, Operand, admit, refuse

MAX_K = 256
_LOGITS = Operand(*WIDE_FLOATS, ndim=2, layout=None)
_K = Number(integral=True, minimum=1)
_TEMPERATURE = Number()


def top_logits(logits, k, *, temperature=1.0):
    """(values, indices, lse) for CUDA logits [N, V] (fp16/bf16/fp32, unit column stride,
    any row stride): values [N, k] in the logits' dtype, int64 indices [N, k], fp32 lse
    [N].  1 <= k <= min(V, 256).  Nothing is differentiable."""
    entry = "top_logits"
    device = logits.device if isinstance(logits, torch.Tensor) else None
    admit(entry, device, logits=(logits, _LOGITS), k=(k, _K), temperature=(temperature, _TEMPERATURE))
    rows, vocab = logits.shape
    if k > min(vocab, MAX_K):
        refuse(entry, f"k is {k}; at most {min(vocab, MAX_K)} of {vocab} columns can be listed")
    if not temperature > 0:
        refuse(entry, f"temperature is {temperature!r}; a positive value is required")
    if vocab > 1 and logits.stride(1) != 1:
        refuse(entry, "logits has a strided last dimension; unit stride is required there")
    with _lib.on_device(device):
        values = torch.empty((rows, k), device=device, dtype=logits.dtype)
        indices = torch.empty((rows, k), device=device, dtype=torch.int64)
        lse = torch.empty(rows, device=device, dtype=torch.float32)
        if rows:
            _lib.call("sb_top_logits", logits.data_ptr(), _lib.wide_dtype_code(logits.dtype), rows, vocab,
                      logits.stride(0), int(k), float(temperature), values.data_ptr(), indices.data_ptr(),
                      lse.data_ptr(), _lib.raw_stream(device))
    return values, indices, lse
