"""Distillation through the frozen head against the definition in 64 bits.

Tolerances, from the arithmetic.  A logit is a sum in runs of 256 products whose 16 tensor-core
additions may each cut off one ulp of the run's magnitude sum, runs added to nearest: with
A = sum |h_i W_vi| / tau, |dz_v| <= d = A (16 * 2^-23 + (H / 256 + 4) 2^-24), the last 4 for the
scaling and exponents.  The loss moves by sum_v |q_v - p_v| |dz_v| <= 2 d; logarithms, exponentials
(2^-22) and the sums over the list and the tiles add at most 2^-17 (1 + loss).  mass moves by d.
The gradient's terms dz_v W_v are rounded once to the 16-bit type (u = 2^-11, bf16 2^-8), carry the
exponentials' error and d, and the result is rounded once: |error| <= spread (u + 2^-18 + 2 d) +
u |dx| + the type's smallest step; values more than 2^-28 below the row's largest are lost, at most
that much per column of W's largest element.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import distill_oracle as D
from tests.helpers import np_of

pytestmark = pytest.mark.gpu

HALF, BRAIN = torch.float16, torch.bfloat16


def _inputs(rows, hidden, vocab, k, dtype=HALF, seed=0, tail=True, temperature=1.0, answered=1.0, scale=2.0, near=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((rows, hidden), device="cuda", generator=g) * scale).to(dtype)
    w = (torch.randn((vocab, hidden), device="cuda", generator=g) / math.sqrt(hidden)).to(dtype)
    teacher = (x.float() + near * torch.randn((rows, hidden), device="cuda", generator=g)) @ w.float().t()
    logits, indices = torch.topk(teacher, min(k, vocab), dim=1)
    mixed = torch.rand(logits.shape, device="cuda", generator=g).argsort(1)
    logits, indices = logits.gather(1, mixed), indices.gather(1, mixed)
    lse = torch.logsumexp(teacher / temperature, 1) if tail else None
    if answered < 1:
        indices[torch.rand(rows, device="cuda", generator=g) >= answered] = -1
    upstream = torch.randn(rows, device="cuda", generator=g)
    return x.requires_grad_(), w, indices, logits, lse, upstream


def _check(x, w, indices, logits, lse, upstream, temperature=1.0, validate=True):
    from soupsuck_b200 import _lib
    from soupsuck_b200.kernels import fused_linear_distillation
    loss, mass = fused_linear_distillation(x, w, indices, logits, lse, temperature=temperature, validate=validate)
    assert loss.dtype == mass.dtype == torch.float32 and loss.requires_grad and not mass.requires_grad
    (dx,) = torch.autograd.grad(loss, x, upstream)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    wide = lambda t: None if t is None else np_of(t.detach().float()).astype(np.float64)
    xs, ws = wide(x), wide(w)
    rl, rm, rg, spread = D.distillation(xs, ws, np_of(indices), wide(logits), wide(lse), temperature, wide(upstream))
    hidden = xs.shape[1]
    a = (np.abs(xs) @ np.abs(ws).T).max(1) / temperature
    d = a * (16 * 2.0 ** -23 + (hidden / 256 + 4) * 2.0 ** -24)
    assert (np.abs(wide(loss) - rl) <= 2 * d + 2.0 ** -17 * (1 + np.abs(rl))).all(), np.abs(wide(loss) - rl).max()
    assert (np.abs(wide(mass) - rm) <= d + 2.0 ** -17).all(), np.abs(wide(mass) - rm).max()
    u, tiny = (2.0 ** -11, 2.0 ** -24) if x.dtype == HALF else (2.0 ** -8, 2.0 ** -133)
    lost = 2.0 ** -28 * ws.shape[0] * np.abs(ws).max() * np.abs(wide(upstream))[:, None] / temperature
    room = spread * (u + 2.0 ** -18 + 2 * d[:, None]) + u * np.abs(rg) + tiny + lost
    off = np.abs(wide(dx) - rg)
    assert (off <= room).all(), (off - room).max()
    gone = ~((np_of(indices) >= 0) & (np_of(indices) < ws.shape[0])).any(1)
    assert not wide(loss)[gone].any() and not wide(mass)[gone].any() and not wide(dx)[gone].any()
    assert _lib.take_device_error(x.device) == 0
    return loss, mass, dx


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("rows,hidden,vocab,k", [
    (1, 8, 7, 3), (1, 64, 128, 1), (3, 33, 129, 5), (5, 1536, 1000, 64), (77, 64, 4103, 200), (130, 256, 257, 256),
    (256, 320, 2048, 20), (257, 136, 5000, 33), (300, 896, 20011, 64), (600, 512, 3000, 7),
])
def test_sizes(dtype, tail, rows, hidden, vocab, k):
    _check(*_inputs(rows, hidden, vocab, k, dtype, seed=rows + vocab, tail=tail))


@pytest.mark.parametrize("temperature", [0.5, 2.0, 4.0])
@pytest.mark.parametrize("tail", [True, False])
def test_temperature(temperature, tail):
    _check(*_inputs(40, 128, 3001, 50, tail=tail, temperature=temperature), temperature=temperature)


@pytest.mark.parametrize("tail", [True, False])
def test_unanswered_rows(tail):
    args = _inputs(500, 128, 2000, 16, tail=tail, answered=0.37)
    args[5][(args[2] < 0).all(1)] = float("inf")  # never touched
    loss, mass, dx = _check(*args[:5], torch.where(torch.isinf(args[5]), 0.0, args[5]))
    from soupsuck_b200.kernels import fused_linear_distillation
    again, _ = fused_linear_distillation(*args[:5])
    assert torch.equal(torch.autograd.grad(again, args[0], args[5])[0], dx)


def test_no_row_answered_and_no_rows():
    x, w, indices, logits, lse, upstream = _inputs(9, 64, 500, 4)
    _check(x, w, torch.full_like(indices, -1), logits, lse, upstream)
    from soupsuck_b200.kernels import fused_linear_distillation
    empty = x.detach()[:0].requires_grad_()
    loss, mass = fused_linear_distillation(empty, w, indices[:0], logits[:0], lse[:0])
    loss.sum().backward()
    assert loss.shape == mass.shape == (0,) and empty.grad.shape == empty.shape


@pytest.mark.parametrize("tail", [True, False])
def test_ragged_lists_and_masked_teacher_logits(tail):
    x, w, indices, logits, lse, upstream = _inputs(64, 96, 1500, 30, tail=tail)
    place = torch.arange(30, device="cuda")
    indices[place[None, :] >= (torch.arange(64, device="cuda") % 31)[:, None]] = -1
    logits[5, ::2] = -float("inf")  # listed, but impossible for the teacher
    logits[7] = -float("inf")
    if tail:
        lse[9] = -float("inf")
        indices[9] = -1
    _check(x, w, indices, logits, lse, upstream)


@pytest.mark.parametrize("tail", [True, False])
def test_every_token_listed(tail):
    _check(*_inputs(20, 64, 100, 100, tail=tail))


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("tail", [True, False])
def test_peaked_students(dtype, tail):
    """Logits up to about 60: peaks on and off the list, tails far below the row's maximum."""
    x, w, indices, logits, lse, upstream = _inputs(96, 256, 4000, 8, dtype, tail=tail)
    with torch.no_grad():
        token = torch.arange(96, device="cuda") * 41
        x += (w[token].float() * torch.linspace(0, 55, 96, device="cuda")[:, None]).to(dtype)
        indices[::3, 0] = torch.where((indices[::3] == token[::3, None]).any(1), indices[::3, 0], token[::3])
    _check(x, w, indices, logits, lse, upstream)


def test_teacher_tail_where_the_student_has_none():
    """The student is sure of a listed token (q_rest about e^-40) while the teacher keeps a third
    of its probability off the list: the unlisted gradient is p_rest's, not q_rest's."""
    x, w, indices, logits, lse, upstream = _inputs(8, 128, 1000, 4)
    with torch.no_grad():
        x.zero_()
        x += (w[indices[:, 0]].float() * 45).to(x.dtype)
        logits[:] = torch.log(torch.tensor([0.4, 0.15, 0.1, 0.05], device="cuda"))
        lse.zero_()
    _check(x, w, indices, logits, lse, upstream)


def test_matching_student_has_almost_no_gradient():
    """Teacher and student alike: the loss is at rounding level and never below zero by more."""
    x, w, indices, logits, lse, upstream = _inputs(50, 512, 3000, 40, near=0.0)
    _check(x, w, indices, logits, lse, upstream)


def test_gradient_against_differences():
    """Central differences of the loss along random directions (fp32 loss, step 2^-6 of hidden):
    truncation below 2^-12 * third derivative (<= 4 |W u|^3), rounding 2 * the loss's tolerance /
    step, and the gradient's own."""
    x, w, indices, logits, lse, upstream = _inputs(24, 128, 900, 12, seed=3)
    from soupsuck_b200.kernels import fused_linear_distillation
    loss, _ = fused_linear_distillation(x, w, indices, logits, lse)
    (dx,) = torch.autograd.grad(loss.sum(), x)
    g = torch.Generator(device="cuda").manual_seed(9)
    for _ in range(4):
        # Steps that fp16 holds exactly: hidden rounded to 2^-6, moved by 2^-6 per coordinate.
        base = (x.detach().float() * 64).round() / 64
        u = torch.randint(0, 2, x.shape, device="cuda", generator=g).float() * 2 - 1
        up = fused_linear_distillation((base + u / 64).half(), w, indices, logits, lse)[0].double()
        down = fused_linear_distillation((base - u / 64).half(), w, indices, logits, lse)[0].double()
        here = base.half().requires_grad_()
        loss, _ = fused_linear_distillation(here, w, indices, logits, lse)
        (dx,) = torch.autograd.grad(loss.sum(), here)
        slope = (dx.double() * u.double()).sum(1)
        wu = (u.double() @ w.double().t()).abs().amax(1)
        a = (base.double().abs() @ w.double().abs().t()).amax(1)
        d = a * (16 * 2.0 ** -23 + (128 / 256 + 4) * 2.0 ** -24)
        noise = 2 * (2 * d + 2.0 ** -17 * (1 + loss.double())) * 32
        room = noise + 4 * wu ** 3 / 64 ** 2 / 6 + 2.0 ** -10 * (dx.double().abs().sum(1) + wu)
        assert (((up - down) * 32 - slope).abs() <= room).all()


def test_strides_alignment_and_list_dtypes():
    x, w, indices, logits, lse, upstream = _inputs(40, 72, 600, 10)
    wide = torch.zeros((40, 100), device="cuda", dtype=HALF)
    wide[:, 3:75] = x.detach()
    xs = wide[:, 3:75].requires_grad_()
    ws = w.t().contiguous().t()
    _check(xs, ws, indices.t().contiguous().t(), logits.t().contiguous().t(), lse.repeat_interleave(2)[::2], upstream)
    off = torch.empty(40 * 72 + 1, device="cuda", dtype=HALF)
    off[1:] = x.detach().reshape(-1)
    _check(off[1:].view(40, 72).requires_grad_(), w, indices, logits.half(), lse, upstream)
    _check(x, w, indices, logits.bfloat16(), lse, upstream)


def test_evaluation_matches_training_and_repeats():
    from soupsuck_b200.kernels import fused_linear_distillation
    x, w, indices, logits, lse, upstream = _inputs(300, 256, 9000, 32)
    first = _check(x, w, indices, logits, lse, upstream)
    second = _check(x, w, indices, logits, lse, upstream, validate=False)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.no_grad():
        loss, mass = fused_linear_distillation(x, w, indices, logits, lse)
    assert not loss.requires_grad and torch.equal(loss, first[0]) and torch.equal(mass, first[1])
    # One graph, two backward passes, on another stream than the forward's.
    loss, _ = fused_linear_distillation(x, w, indices, logits, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = torch.autograd.grad(loss, x, upstream, retain_graph=True)[0]
        b = torch.autograd.grad(loss, x, 2 * upstream)[0]
    side.synchronize()
    assert torch.equal(a, first[2]) and torch.allclose(b.float(), 2 * a.float(), rtol=2 ** -10, atol=2 ** -23)


def test_more_rows_than_one_block_holds():
    """15000 rows of 151936 tokens are worked off in two blocks (4 GB of exponentials hold 14080).  Rows
    do not depend on one another: losses equal those of two smaller calls exactly; the product's splits
    differ with the rows, so gradients may differ by their runs: 64 tensor-core additions each, one ulp
    of a magnitude sum of at most 2 max|W| apiece on either side, and one rounding to fp16."""
    from soupsuck_b200.kernels import fused_linear_distillation
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, hidden, vocab, k = 15000, 64, 151936, 4
    x = torch.randn((rows, hidden), device="cuda", generator=g).half()
    w = (torch.randn((vocab, hidden), device="cuda", generator=g) / 8).half()
    indices = torch.randint(vocab // 4, (rows, k), device="cuda", generator=g) + torch.arange(k, device="cuda") * (vocab // 4)
    logits = torch.rand((rows, k), device="cuda", generator=g) * 3
    lse = torch.logsumexp(logits, 1) + 0.3
    indices[::7] = -1

    def call(part):
        leaf = x[part].clone().requires_grad_()
        loss, mass = fused_linear_distillation(leaf, w, indices[part], logits[part], lse[part], validate=False)
        return loss.detach(), mass, torch.autograd.grad(loss.sum(), leaf)[0]

    whole, first, second = call(slice(None)), call(slice(0, 8000)), call(slice(8000, None))
    for got, a, b in zip(whole[:2], first, second):
        assert torch.equal(got, torch.cat([a, b]))
    dx, parts = whole[2].float(), torch.cat([first[2], second[2]]).float()
    assert torch.isfinite(dx).all() and not dx[::7].any()
    runs = 2 * 64 * 2.0 ** -23 * 2 * w.float().abs().max()
    assert ((dx - parts).abs() <= 2.0 ** -10 * parts.abs() + runs).all()


def test_rows_with_nan_stay_apart():
    from soupsuck_b200.kernels import fused_linear_distillation
    x, w, indices, logits, lse, upstream = _inputs(20, 64, 700, 6)
    clean, _ = fused_linear_distillation(x, w, indices, logits, lse)
    (good,) = torch.autograd.grad(clean, x, upstream)
    with torch.no_grad():
        x[3, 5] = float("nan")
        logits[8, 2] = float("nan")
    loss, mass = fused_linear_distillation(x, w, indices, logits, lse)
    (dx,) = torch.autograd.grad(loss, x, upstream)
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[[3, 8]] = True
    assert torch.isnan(loss[bad]).all() and torch.isnan(dx[bad]).any(1).all()
    assert torch.equal(loss[~bad], clean[~bad]) and torch.equal(dx[~bad], good[~bad])


def test_unchecked_indices_stay_inside():
    """Without validation: indices outside the vocabulary count as unused."""
    x, w, indices, logits, lse, upstream = _inputs(30, 64, 700, 6)
    odd = indices.clone()
    odd[::2, 1], odd[1::2, 4], odd[5] = 700, -7, 1 << 40
    plain = torch.where((odd < 0) | (odd >= 700), -1, odd)
    from soupsuck_b200.kernels import fused_linear_distillation
    a = fused_linear_distillation(x, w, odd, logits, lse, validate=False)
    b = fused_linear_distillation(x, w, plain, logits, lse)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    _check(x, w, plain, logits, lse, upstream)


def test_refusals():
    from soupsuck_b200.kernels import fused_linear_distillation as f
    x, w, indices, logits, lse, _ = _inputs(6, 64, 300, 5)
    outside, repeated = indices.clone(), indices.clone()
    outside[2, 1] = 300
    repeated[4, 3] = repeated[4, 0]
    many = torch.zeros((6, 257), device="cuda", dtype=torch.int64)
    for bad, why in ((lambda: f(x, w, outside, logits, lse), "outside"), (lambda: f(x, w, repeated, logits, lse), "repeat"),
                     (lambda: f(x, w, indices - 302, logits, lse), "outside"),
                     (lambda: f(x.float(), w, indices, logits, lse), "dtype"), (lambda: f(x, w.bfloat16(), indices, logits, lse), "dtype"),
                     (lambda: f(x, w.clone().requires_grad_(), indices, logits, lse), "frozen"),
                     (lambda: f(x, w, indices.int(), logits, lse), "dtype"), (lambda: f(x, w, indices, logits[:, :4], lse), "line up"),
                     (lambda: f(x, w, indices, logits, lse[:5]), "line up"), (lambda: f(x, w[:, :32], indices, logits, lse), "line up"),
                     (lambda: f(x, w, many, many.float(), lse), "256"), (lambda: f(x, w, indices[:, :0], logits[:, :0], lse), "256"),
                     (lambda: f(x, w[:0], indices, logits, lse), "empty"), (lambda: f(x, w, indices, logits, lse, temperature=0.0), "positive"),
                     (lambda: f(x.detach().cpu(), w, indices, logits, lse), "CUDA"), (lambda: f(x, w, indices, logits, lse.double()), "dtype")):
        with pytest.raises(ValueError, match=why):
            bad()
