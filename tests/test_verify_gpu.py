"""Draft verification against the sequence-by-sequence definition: all outputs are whole
numbers and have to be equal (every decision is a single fp32 operation or a maximum)."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import distill_oracle as D
from tests.helpers import np_of

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(batch, drafts, vocab, dtype=torch.float32, seed=0, spread=2.0, near=0.6):
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn((batch, drafts + 1, vocab), device="cuda", generator=g) * spread
    q = torch.softmax(base[:, :drafts] + near * torch.randn((batch, drafts, vocab), device="cuda", generator=g), -1)
    e = torch.empty((batch, drafts, vocab), device="cuda").exponential_(generator=g).clamp_min_(1e-30)
    tokens = (q / e).argmax(-1) if drafts else torch.empty((batch, 0), device="cuda", dtype=torch.int64)
    noise = torch.empty((batch, vocab), device="cuda").exponential_(generator=g).clamp_min_(1e-30)
    return (torch.softmax(base, -1).to(dtype), tokens, torch.rand((batch, drafts), device="cuda", generator=g), noise,
            q.to(dtype))


def _check(target, tokens, uniforms, noise, draft=None, lens=None):
    from soupsuck_b200.kernels import verify_drafts
    accepted, out = verify_drafts(target, tokens, uniforms, noise, draft, draft_lens=lens)
    ra, ro = D.verify_drafts(np_of(target.float()), np_of(tokens), np_of(uniforms), np_of(noise),
                             None if draft is None else np_of(draft.float()), None if lens is None else np_of(lens))
    np.testing.assert_array_equal(np_of(accepted), ra)
    np.testing.assert_array_equal(np_of(out), ro)
    return np_of(accepted), np_of(out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,drafts,vocab", [
    (1, 1, 1), (1, 4, 151936), (3, 2, 7), (5, 7, 1000), (64, 3, 4099), (9, 40, 513), (2, 5, 32001), (300, 2, 2048),
])
def test_sampled_and_looked_up(dtype, batch, drafts, vocab):
    target, tokens, u, noise, draft = _inputs(batch, drafts, vocab, dtype, seed=vocab + batch)
    accepted, _ = _check(target, tokens, u, noise, draft)
    if batch * drafts > 60 and vocab > 100:
        assert 0 < accepted.sum() < batch * drafts
    _check(target, tokens, u, noise, None)


def test_ragged_lengths():
    target, tokens, u, noise, draft = _inputs(40, 6, 3001)
    lens = torch.arange(40, device="cuda") % 9 - 1  # -1 and 7 are cut to 0 and 6
    _check(target, tokens, u, noise, draft, lens)
    _check(target, tokens, u, noise, None, lens)


def test_no_drafts_samples_from_the_target():
    target, tokens, u, noise, _ = _inputs(6, 0, 5000)
    accepted, out = _check(target, tokens, u, noise)
    assert (accepted == 0).all() and out.shape == (6, 1) and (out >= 0).all()


def test_all_accepted_and_all_rejected():
    target, tokens, u, noise, draft = _inputs(8, 4, 999)
    accepted, out = _check(target, tokens, torch.zeros_like(u), noise, draft)
    assert (accepted == 4).all() and (out[:, 4] >= 0).all()
    gone = target.clone().scatter_(2, torch.cat([tokens, tokens[:, :1]], 1)[:, :, None], 0.0)
    accepted, _ = _check(gone, tokens, u, noise, draft)
    assert (accepted == 0).all()


def test_equal_distributions_accept_below_one():
    target, tokens, u, noise, _ = _inputs(8, 4, 777)
    accepted, _ = _check(target, tokens, u.clamp_max(0.999), noise, target[:, :4].contiguous())
    assert (accepted == 4).all()


def test_zero_residual_falls_back_to_the_target():
    """q >= p everywhere although the draft was rejected: the token comes from p itself."""
    target, tokens, u, noise, draft = _inputs(4, 2, 1500)
    accepted, out = _check(target, tokens, torch.full_like(u, 0.9999), noise, target[:, :2] * 2)
    assert (accepted == 0).all() and (out[:, 0] >= 0).all()


def test_empty_distribution_gives_minus_one():
    target, tokens, u, noise, draft = _inputs(3, 2, 600)
    target[1] = 0
    accepted, out = _check(target, tokens, u, noise, draft)
    assert accepted[1] == 0 and (out[1] == -1).all()


def test_masked_columns_ties_and_odd_values():
    target, tokens, u, noise, draft = _inputs(6, 3, 2000)
    target[:, :, ::2] = 0
    draft[:, :, ::3] = 0
    noise.fill_(0.5)  # scores tie wherever probabilities do
    target[2] = 1.0 / 2000
    _check(target, tokens, u, noise, draft)
    target[4, :, 11] = float("nan")
    draft[5, :, 13] = float("nan")
    noise[0, 17] = 1e-38
    _check(target, tokens, u, noise, draft)


def test_tokens_outside_the_vocabulary_are_rejected():
    target, tokens, u, noise, draft = _inputs(4, 3, 100)
    tokens[0, 0], tokens[1, 1], tokens[2, 2] = -1, 100, 1 << 40
    _check(target, tokens, u, noise, draft)
    _check(target, tokens, u, noise, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_operands(dtype):
    target, tokens, u, noise, draft = _inputs(6, 4, 1203, dtype)
    wide = torch.zeros((6, 5, 1300), device="cuda", dtype=dtype)
    wide[:, :, 5:1208] = target
    turned = draft.transpose(0, 1).contiguous().transpose(0, 1)
    loud = torch.ones((6, 1500), device="cuda")
    loud[:, 3:1206] = noise
    _check(wide[:, :, 5:1208], tokens.t().contiguous().t(), u.t().contiguous().t(), loud[:, 3:1206], turned)
    _check(target[:1].expand(6, -1, -1), tokens, u, noise[:1].expand(6, -1), draft)


def test_emitted_tokens_follow_the_target():
    """The first emitted token of many sequences that share one target: frequencies within five
    standard deviations of the target's probabilities, whatever the draft distribution is."""
    vocab, batch = 12, 40000
    g = torch.Generator(device="cuda").manual_seed(3)
    p = torch.softmax(torch.randn(vocab, device="cuda", generator=g), 0)
    q = torch.softmax(torch.randn(vocab, device="cuda", generator=g), 0)
    e = torch.empty((batch, 1, vocab), device="cuda").exponential_(generator=g).clamp_min_(1e-30)
    tokens = (q / e).argmax(-1)
    from soupsuck_b200.kernels import verify_drafts
    _, out = verify_drafts(p.expand(batch, 2, vocab), tokens, torch.rand((batch, 1), device="cuda", generator=g),
                           torch.empty((batch, vocab), device="cuda").exponential_(generator=g).clamp_min_(1e-30),
                           q.expand(batch, 1, vocab))
    count = torch.bincount(out[:, 0], minlength=vocab).double()
    sigma = (batch * p.double() * (1 - p.double())).sqrt()
    assert ((count - batch * p.double()).abs() <= 5 * sigma).all()


def test_empty_batch_and_refusals():
    from soupsuck_b200.kernels import verify_drafts
    target, tokens, u, noise, draft = _inputs(4, 3, 50)
    accepted, out = verify_drafts(target[:0], tokens[:0], u[:0], noise[:0])
    assert accepted.shape == (0,) and out.shape == (0, 4)
    for bad in (lambda: verify_drafts(target[:, :3], tokens, u, noise, draft),
                lambda: verify_drafts(target, tokens, u, noise, draft[:, :2]),
                lambda: verify_drafts(target, tokens, u, noise, draft.half()),
                lambda: verify_drafts(target, tokens.int(), u, noise, draft),
                lambda: verify_drafts(target, tokens, u.double(), noise, draft),
                lambda: verify_drafts(target, tokens, u, noise[:, :49], draft),
                lambda: verify_drafts(target.cpu(), tokens, u, noise, draft),
                lambda: verify_drafts(target.transpose(1, 2), tokens, u, noise, draft),
                lambda: verify_drafts(target, tokens, u, noise, draft, draft_lens=torch.zeros(3, device="cuda", dtype=torch.int64)),
                lambda: verify_drafts(target[..., :0], tokens, u, noise[:, :0])):
        with pytest.raises(ValueError, match="verify_drafts"):
            bad()
