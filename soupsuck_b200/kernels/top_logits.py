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
_CODES = {dtype: _lib.wide_dtype_code(dtype) for dtype in WIDE_FLOATS}
_launch = _lib.entry("sb_top_logits")


def top_logits(logits, k, *, temperature=1.0):
    """(values, indices, lse) for CUDA logits [N, V] (fp16/bf16/fp32, unit column stride,
    any row stride): values [N, k] in the logits' dtype, int64 indices [N, k], fp32 lse
    [N].  1 <= k <= min(V, 256).  Nothing is differentiable."""
    # One row takes 13 us on the device, and as long on the host: what is plainly right
    # is let through here, everything else meets the rules.
    plain = (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype in _CODES and logits.dim() == 2
             and type(k) is int and k >= 1 and type(temperature) is float and 0.0 < temperature < float("inf"))
    if not plain:
        _check(logits, k, temperature)
    rows, vocab = logits.shape
    stride, unit = logits.stride()
    if k > min(vocab, MAX_K):
        refuse("top_logits", f"k is {k}; at most {min(vocab, MAX_K)} of {vocab} columns can be listed")
    if unit != 1 and vocab > 1:
        refuse("top_logits", "logits has a strided last dimension; unit stride is required there")
    device = logits.device
    with _lib.on_device(device):
        values = logits.new_empty((rows, k))
        indices = logits.new_empty((rows, k), dtype=torch.int64)
        lse = logits.new_empty(rows, dtype=torch.float32)
        if rows:
            _launch(logits.data_ptr(), _CODES[logits.dtype], rows, vocab, stride, k, temperature, values.data_ptr(),
                    indices.data_ptr(), lse.data_ptr(), _lib.raw_stream(device))
    return values, indices, lse


def _check(logits, k, temperature):
    entry = "top_logits"
    device = logits.device if isinstance(logits, torch.Tensor) else None
    admit(entry, device, logits=(logits, _LOGITS), k=(k, _K), temperature=(temperature, _TEMPERATURE))
    if not temperature > 0:
        refuse(entry, f"temperature is {temperature!r}; a positive value is required")
