"""Verification of drafted tokens against the target model's probabilities, from given
random numbers (speculative sampling): the emitted tokens follow the target's
distribution whatever the draft model's is.

Draft s of a sequence is accepted while ``u_s * q_s(x_s) < p_s(x_s)``.  At the first
rejected place one token comes from the residual ``max(p - q, 0)``, after the last
draft one from the target itself, as ``argmax_v r_v / noise_v`` with noise from Exp(1)
-- a draw from ``r / sum(r)`` that needs no sum.  All of it is single fp32 operations
and maxima, so the result is exactly that of the formulas, ties to the lowest index.
"""

from __future__ import annotations

import torch

from .. import _lib
from .._spec import LONG, SINGLE, WIDE_FLOATS, Operand, admit, refuse

_PROBS = Operand(*WIDE_FLOATS, ndim=3, layout=None)
_LIKE = {dtype: Operand(dtype, ndim=3, layout=None, optional=True) for dtype in WIDE_FLOATS}
_TOKENS = Operand(LONG, ndim=2, layout=None)
_NUMBERS = Operand(SINGLE, ndim=2, layout=None)
_LENS = Operand(LONG, ndim=1, layout=None, optional=True)


_CODES = {dtype: _lib.wide_dtype_code(dtype) for dtype in WIDE_FLOATS}
_launch = _lib.entry("sb_verify_drafts")


def verify_drafts(target_probs, draft_tokens, uniforms, noise, draft_probs=None, *, draft_lens=None):
    """(accepted [B], tokens [B, S + 1]), int64, for target_probs [B, S + 1, V], drafted
    tokens [B, S] (int64), uniforms [B, S] in [0, 1), noise [B, V] > 0 (draws from Exp(1)),
    draft_probs [B, S, V] of the target's dtype (fp16/bf16/fp32) or None where the drafts
    were looked up, not sampled, and draft_lens [B] (int64) where sequences have fewer than
    S drafts.  tokens holds the accepted drafts, the token drawn behind them (-1 where the
    probabilities leave none) and -1 to its end.  A drafted token outside [0, V) is
    rejected."""
    # (Host time counts here too: what is plainly right skips the rules.)
    place = target_probs.get_device() if isinstance(target_probs, torch.Tensor) else -1
    plain = (place >= 0 and target_probs.dim() == 3 and target_probs.dtype in _CODES
             and _is(draft_tokens, LONG, 2, place) and _is(uniforms, SINGLE, 2, place) and _is(noise, SINGLE, 2, place)
             and (draft_probs is None or _is(draft_probs, target_probs.dtype, 3, place))
             and (draft_lens is None or _is(draft_lens, LONG, 1, place)))
    if not plain:
        _check(target_probs, draft_tokens, uniforms, noise, draft_probs, draft_lens)
    batch, places, vocab = target_probs.shape
    drafts = places - 1
    if not (draft_tokens.shape == (batch, drafts) == uniforms.shape and noise.shape == (batch, vocab)
            and (draft_probs is None or draft_probs.shape == (batch, drafts, vocab))
            and (draft_lens is None or draft_lens.shape == (batch,))):
        shape = lambda t: None if t is None else tuple(t.shape)  # noqa: E731
        refuse("verify_drafts", f"target_probs {shape(target_probs)}, draft_tokens {shape(draft_tokens)}, uniforms "
                                f"{shape(uniforms)}, noise {shape(noise)}, draft_probs {shape(draft_probs)} and draft_lens "
                                f"{shape(draft_lens)} do not line up")
    if vocab == 0:
        refuse("verify_drafts", f"target_probs {tuple(target_probs.shape)} has an empty vocabulary")
    t_batch, t_row, t_unit = target_probs.stride()
    n_batch, n_unit = noise.stride()
    d_batch, d_row, d_unit = (0, 0, 1) if draft_probs is None else draft_probs.stride()
    if vocab > 1 and not t_unit == n_unit == d_unit == 1:
        refuse("verify_drafts", "target_probs, noise or draft_probs has a strided last dimension; unit stride is "
                                "required there")
    device = target_probs.device
    with _lib.on_device(device):
        tokens_in, u = draft_tokens.contiguous(), uniforms.contiguous()
        lens = None if draft_lens is None else draft_lens.contiguous()
        accepted = tokens_in.new_empty(batch)
        tokens = tokens_in.new_empty((batch, places))
        if batch:
            _launch(target_probs.data_ptr(), t_batch, t_row, _lib.ptr(draft_probs), d_batch, d_row,
                    _CODES[target_probs.dtype], batch, drafts, vocab, tokens_in.data_ptr(), u.data_ptr(),
                    noise.data_ptr(), n_batch, _lib.ptr(lens), accepted.data_ptr(), tokens.data_ptr(),
                    _lib.raw_stream(device))
    return accepted, tokens


def _is(t, dtype, ndim, place):
    return isinstance(t, torch.Tensor) and t.get_device() == place and t.dtype is dtype and t.dim() == ndim


def _check(target_probs, draft_tokens, uniforms, noise, draft_probs, draft_lens):
    entry = "verify_drafts"
    device = target_probs.device if isinstance(target_probs, torch.Tensor) else None
    admit(entry, device, target_probs=(target_probs, _PROBS))
    admit(entry, device, draft_tokens=(draft_tokens, _TOKENS), uniforms=(uniforms, _NUMBERS), noise=(noise, _NUMBERS),
          draft_probs=(draft_probs, _LIKE[target_probs.dtype]), draft_lens=(draft_lens, _LENS))
