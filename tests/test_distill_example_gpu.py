"""The distillation operators together: the head boundary against its definition, and the example,
a LoRA student trained on a teacher's lists that then drafts for it."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import distill_oracle as D
from tests.helpers import np_of

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "distill_draft_model.py"
    spec = importlib.util.spec_from_file_location("distill_draft_model", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_head_takes_batches_and_averages_answered_positions():
    """Teacher lists straight from top_logits.  The mean's tolerance is the largest row's (a logit's
    2^-17 at |z| < 16 twice, and 2^-17 (1 + loss))."""
    from soupsuck_b200.head import distilled_head
    from soupsuck_b200.kernels import top_logits
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((3, 7, 64), device="cuda", generator=g).half()
    w = (torch.randn((900, 64), device="cuda", generator=g) / 8).half()
    teacher = torch.randn((3, 7, 900), device="cuda", generator=g) * 2
    values, indices, lse = top_logits(teacher.view(21, 900), 10, temperature=1.5)
    values, indices, lse = values.view(3, 7, 10), indices.view(3, 7, 10).clone(), lse.view(3, 7)
    indices[:, :3] = -1
    loss, mass = distilled_head(x, w, indices, values, lse, temperature=1.5)
    rl, rm, _, _ = D.distillation(np_of(x.float()).reshape(21, 64), np_of(w.float()), np_of(indices).reshape(21, 10),
                                  np_of(values).reshape(21, 10), np_of(lse).reshape(21), 1.5)
    assert abs(loss.item() - rl.sum() / 12) <= 2.0 ** -16 + 2.0 ** -17 * (1 + rl.max())
    assert abs(mass.item() - rm.sum() / 12) <= 2.0 ** -16
    half, _ = distilled_head(x, w, indices, values, lse, temperature=1.5, num_items_in_batch=24)
    assert half.item() == pytest.approx(loss.item() / 2, rel=1e-6)
    nothing, covered = distilled_head(x, w, torch.full_like(indices, -1), values, lse, temperature=1.5)
    assert nothing.item() == 0 and covered.item() == 0


def test_distilled_student_drafts_better():
    """Training on the lists takes most of the divergence away, and the teacher then accepts more."""
    before, after, first, last = _example().run(steps=120, contexts=1024)
    assert last < 0.25 * first
    assert after > before + 0.1


def test_lists_feed_the_loss_without_conversion():
    """A student that is its own teacher: top_logits' outputs taken as they are give a loss at
    rounding level (below 2^-16) and the listed tokens' share of exp(logits - lse)."""
    from soupsuck_b200.kernels import fused_linear_distillation, top_logits
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((30, 128), device="cuda", generator=g).half()
    w = (torch.randn((2000, 128), device="cuda", generator=g) / 8).half()
    logits = x.float() @ w.float().t()
    values, indices, lse = top_logits(logits, 50)
    loss, mass = fused_linear_distillation(x, w, indices, values, lse)
    assert (loss.abs() <= 2.0 ** -16).all()
    np.testing.assert_allclose(np_of(mass), np_of((values - lse[:, None]).exp().sum(1)), rtol=2.0 ** -14)
