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


def _rows_unit(entry, name, t):
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        refuse(entry, f"{name} has a strided last dimension; unit stride is required there")


def verify_drafts(target_probs, draft_tokens, uniforms, noise, draft_probs=None, *, draft_lens=None):
    """(accepted [B], tokens [B, S + 1]), int64, for target_probs [B, S + 1, V], drafted
    tokens [B, S] (int64), uniforms [B, S] in [0, 1), noise [B, V] > 0 (draws from Exp(1)),
    draft_probs [B, S, V] of the target's dtype (fp16/bf16/fp32) or None where the drafts
    were looked up, not sampled, and draft_lens [B] (int64) where sequences have fewer than
    S drafts.  tokens holds the accepted drafts, the token drawn behind them (-1 where the
    probabilities leave none) and -1 to its end.  A drafted token outside [0, V) is
    rejected."""
    entry = "verify_drafts"
    device = target_probs.device if isinstance(target_probs, torch.Tensor) else None
    admit(entry, device, target_probs=(target_probs, _PROBS))
    admit(entry, device, draft_tokens=(draft_tokens, _TOKENS), uniforms=(uniforms, _NUMBERS), noise=(noise, _NUMBERS),
          draft_probs=(draft_probs, _LIKE[target_probs.dtype]), draft_lens=(draft_lens, _LENS))
    batch, places, vocab = target_probs.shape
    drafts = draft_tokens.shape[1]
    lines_up = (places == drafts + 1 and draft_tokens.shape[0] == batch
                and uniforms.shape == draft_tokens.shape and noise.shape == (batch, vocab)
                and (draft_probs is None or draft_probs.shape == (batch, drafts, vocab))
                and (draft_lens is None or draft_lens.shape == (batch,)))
    if not lines_up:
        refuse(entry, f"target_probs {tuple(target_probs.shape)}, draft_tokens {tuple(draft_tokens.shape)}, "
                      f"uniforms {tuple(uniforms.shape)}, noise {tuple(noise.shape)}, draft_probs "
                      f"{None if draft_probs is None else tuple(draft_probs.shape)} and draft_lens "
                      f"{None if draft_lens is None else tuple(draft_lens.shape)} do not line up")
    if vocab == 0:
        refuse(entry, f"target_probs {tuple(target_probs.shape)} has an empty vocabulary")
    _rows_unit(entry, "target_probs", target_probs)
    _rows_unit(entry, "noise", noise)
    if draft_probs is not None:
        _rows_unit(entry, "draft_probs", draft_probs)
    with _lib.on_device(device):
        tokens_in, u = draft_tokens.contiguous(), uniforms.contiguous()
        lens = None if draft_lens is None else draft_lens.contiguous()
        accepted = torch.empty(batch, device=device, dtype=LONG)
        tokens = torch.empty((batch, drafts + 1), device=device, dtype=LONG)
        if batch:
            q = draft_probs
            _lib.call("sb_verify_drafts", target_probs.data_ptr(), target_probs.stride(0), target_probs.stride(1),
                      _lib.ptr(q), 0 if q is None else q.stride(0), 0 if q is None else q.stride(1),
                      _lib.wide_dtype_code(target_probs.dtype), batch, drafts, vocab, tokens_in.data_ptr(),
                      u.data_ptr(), noise.data_ptr(), noise.stride(0), _lib.ptr(lens), accepted.data_ptr(),
                      tokens.data_ptr(), _lib.raw_stream(device))
    return accepted, tokens
