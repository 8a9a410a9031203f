"""The distillation operators without a GPU: their 64-bit oracle against first principles, the
refusals of tensors that are not on a device, and the C entries' checks of arguments."""

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import distill_oracle as D


@pytest.fixture(scope="module")
def lib():
    from soupsuck_b200 import _lib
    if not _lib.LIB_PATH.exists():
        from soupsuck_b200 import build
        build.build()
    return _lib.load()


def _case(seed, tail, rows=5, hidden=7, vocab=23, k=6):
    rng = np.random.default_rng(seed)
    x, w = rng.normal(size=(rows, hidden)), rng.normal(size=(vocab, hidden))
    teacher = rng.normal(size=(rows, vocab)) * 2
    indices = np.argsort(-teacher, 1)[:, :k]
    indices[1, 3:] = -1
    indices[2] = -1
    logits = np.take_along_axis(teacher, np.maximum(indices, 0), 1)
    return x, w, indices, logits, (np.log(np.exp(teacher / 1.3).sum(1)) if tail else None)


@pytest.mark.parametrize("tail", [True, False])
def test_oracle_gradient_against_differences(tail):
    """Central differences of the 64-bit loss, step 1e-5: truncation and rounding below 1e-8."""
    x, w, indices, logits, lse = _case(0, tail)
    upstream = np.arange(1.0, 6.0)
    _, _, grad, spread = D.distillation(x, w, indices, logits, lse, 1.3, upstream)
    assert (np.abs(grad) <= spread + 1e-15).all()
    for i in range(x.shape[0]):
        for j in range(x.shape[1]):
            up, down = x.copy(), x.copy()
            up[i, j] += 1e-5
            down[i, j] -= 1e-5
            slope = (D.distillation(up, w, indices, logits, lse, 1.3)[0][i]
                     - D.distillation(down, w, indices, logits, lse, 1.3)[0][i]) / 2e-5
            assert abs(slope * upstream[i] - grad[i, j]) <= 1e-7 * (1 + abs(grad[i, j]))


@pytest.mark.parametrize("tail", [True, False])
def test_oracle_divergence_of_dense_distributions(tail):
    """The loss is KL of two dense distributions: the list's own (renormalised), or the list and one
    bucket, which the teacher's and the student's other tokens share out alike."""
    x, w, indices, logits, lse = _case(1, tail)
    loss, mass, _, _ = D.distillation(x, w, indices, logits, lse, 1.3)
    z = x @ w.T / 1.3
    q = np.exp(z - z.max(1, keepdims=True))
    q /= q.sum(1, keepdims=True)
    for i in range(len(x)):
        cols = indices[i][indices[i] >= 0]
        if not len(cols):
            assert loss[i] == 0 and mass[i] == 0
            continue
        t = logits[i][indices[i] >= 0] / 1.3
        p = np.zeros(w.shape[0])
        if tail:
            p[cols] = np.exp(t - lse[i])
            others = np.setdiff1d(np.arange(w.shape[0]), cols)
            p[others] = (1 - p.sum()) * q[i, others] / q[i, others].sum()
        else:
            p[cols] = np.exp(t) / np.exp(t).sum()
        some = p > 0
        assert loss[i] == pytest.approx((p[some] * np.log(p[some] / q[i, some])).sum(), rel=1e-10, abs=1e-12)
        assert loss[i] > 0 and mass[i] == pytest.approx(q[i, cols].sum(), rel=1e-12)


def test_oracle_top_logits_order():
    z = np.array([[1.0, np.nan, 2.0, 2.0, np.inf, -np.inf], [0.0, -0.0, 0.0, -1.0, 5.0, 5.0]])
    values, indices, lse = D.top_logits(z, 4, 0.5)
    assert indices.tolist() == [[1, 4, 2, 3], [4, 5, 0, 1]]
    assert np.isnan(lse[0])
    assert lse[1] == pytest.approx(np.log(np.exp(z[1] / 0.5).sum()))


def test_oracle_verification_emits_the_target_distribution():
    """Exact over the draft: the probability that the oracle's rule emits v equals p_v (acceptance
    min(q, p) plus the residual's share), and the race draws from the residual."""
    rng = np.random.default_rng(2)
    p, q = rng.dirichlet(np.ones(6)), rng.dirichlet(np.ones(6))
    residual = np.maximum(p - q, 0)
    emitted = np.minimum(p, q) + (1 - np.minimum(p, q).sum()) * residual / residual.sum()
    np.testing.assert_allclose(emitted, p, atol=1e-12)
    batch = 20000
    tokens = rng.choice(6, size=(batch, 1), p=q)
    _, out = D.verify_drafts(np.broadcast_to(p, (batch, 2, 6)), tokens, rng.random((batch, 1)),
                             rng.exponential(size=(batch, 6)), np.broadcast_to(q, (batch, 1, 6)))
    count = np.bincount(out[:, 0], minlength=6)
    assert (np.abs(count - batch * p) <= 5 * np.sqrt(batch * p * (1 - p))).all()


def test_tensors_on_the_host_are_refused():
    from soupsuck_b200.kernels import fused_linear_distillation, top_logits, verify_drafts
    z = torch.randn(2, 8)
    with pytest.raises(ValueError, match="top_logits: logits is on cpu"):
        top_logits(z, 2)
    with pytest.raises(ValueError, match="top_logits: logits is a list"):
        top_logits([[1.0]], 1)
    with pytest.raises(ValueError, match="verify_drafts: target_probs is on cpu"):
        verify_drafts(torch.rand(1, 2, 8), torch.zeros(1, 1, dtype=torch.int64), torch.rand(1, 1), torch.rand(1, 8))
    with pytest.raises(ValueError, match="fused_linear_distillation: hidden is on cpu"):
        fused_linear_distillation(z.half(), z.half(), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))


def test_c_entries_refuse_before_any_launch(lib):
    from soupsuck_b200 import _lib
    before = lib.sb_launch_count()
    one = ctypes.c_void_p(16)
    assert lib.sb_top_logits(one, 7, 1, 8, 8, 1, 1.0, one, one, one, None) == _lib.SB_EINVAL
    assert lib.sb_top_logits(one, 0, 1, 8, 8, 9, 1.0, one, one, one, None) == _lib.SB_EINVAL
    assert b"k must be" in lib.sb_last_error()
    assert lib.sb_top_logits(one, 0, 1, 8, 8, 1, 0.0, one, one, one, None) == _lib.SB_EINVAL
    assert lib.sb_top_logits(None, 0, 1, 8, 8, 1, 1.0, one, one, one, None) == _lib.SB_EINVAL
    assert lib.sb_top_logits(None, 0, 0, 8, 8, 1, 1.0, None, None, None, None) == _lib.SB_OK
    assert lib.sb_verify_drafts(one, 8, 8, None, 0, 0, 1, 1, 1, 0, one, one, one, 8, None, one, one, None) == _lib.SB_EINVAL
    assert lib.sb_verify_drafts(one, 8, 8, None, 0, 0, 1, 1, 1, 8, None, one, one, 8, None, one, one, None) == _lib.SB_EINVAL
    forward = lambda h, dtype, k, tau, ws: lib.sb_distill_forward(  # noqa: E731
        one, 4, h, one, 100, dtype, one, one, 1, k, None, tau, one, one, None, one, ws, 0, None)
    assert forward(12, 0, 4, 1.0, one) == _lib.SB_EINVAL
    assert forward(16, 1, 4, 1.0, one) == _lib.SB_EINVAL
    assert forward(16, 0, 257, 1.0, one) == _lib.SB_EINVAL
    assert forward(16, 0, 4, -1.0, one) == _lib.SB_EINVAL
    assert forward(16, 0, 4, 1.0, one) == _lib.SB_EWORKSPACE
    assert lib.sb_distill_backward(one, one, one, 4, 12, one, 0, None) == _lib.SB_EINVAL
    assert lib.sb_distill_check(one, 4, 0, 100, one, None) == _lib.SB_EINVAL
    assert lib.sb_pad_rows(one, 4, 9, 9, 12, one, None) == _lib.SB_EINVAL
    assert lib.sb_launch_count() == before


def test_workspace_follows_the_gradient_and_has_a_ceiling(lib):
    small = lib.sb_distill_workspace_bytes(3300, 1536, 151936, 64, 0)
    train = lib.sb_distill_workspace_bytes(3300, 1536, 151936, 64, 1)
    assert 0 < small < 2 ** 28 < 3300 * 151936 * 2 < train < 2 ** 31
    # Long batches: 4 GB of exponentials, the rest grows with the rows' lists and lookups alone.
    assert lib.sb_distill_workspace_bytes(100000, 1536, 151936, 64, 1) < 7 * 2 ** 30
    assert lib.sb_distill_workspace_bytes(0, 1536, 151936, 64, 1) == 0
