"""The k largest logits and the log-sum-exp against the sorted rows in 64 bits.

Values and indices are exact.  Tolerance of the log-sum-exp: the sum's relative error is at most
that of 2^x (2^-22), of its argument (half an ulp of a number below 32 where the term counts:
2^-20 ln 2), and of a thread's and the merges' sequential additions (v / 512 + 40, half an ulp
each); the logarithm's and the product's roundings add three ulps of the result.
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import distill_oracle as D
from tests.helpers import np_of

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _check(logits, k, temperature=1.0):
    from soupsuck_b200.kernels import top_logits
    values, indices, lse = top_logits(logits, k, temperature=temperature)
    assert values.dtype == logits.dtype and indices.dtype == torch.int64 and lse.dtype == torch.float32
    wide = np_of(logits.float())
    rv, ri, rl = D.top_logits(wide, k, temperature)
    np.testing.assert_array_equal(np_of(indices), ri)
    np.testing.assert_array_equal(np_of(values.float()), rv.astype(np.float32))
    finite = np.isfinite(rl)
    got = np_of(lse).astype(np.float64)
    np.testing.assert_array_equal(got[~finite], rl[~finite])
    terms = 2.0 ** -22 + 2.0 ** -20 * np.log(2) + (logits.shape[1] / 512 + 40) * 2.0 ** -24
    room = terms + 3 * 2.0 ** -23 * np.abs(rl[finite])
    assert (np.abs(got[finite] - rl[finite]) <= room).all(), np.abs(got[finite] - rl[finite]).max()


def _normal(rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, vocab), device="cuda", generator=g) * scale).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 255, 255), (4, 256, 256), (7, 1000, 64), (1, 4097, 1),
    (2, 16391, 17), (1, 151936, 64), (37, 32001, 200), (320, 5003, 100),
])
def test_sizes(dtype, rows, vocab, k):
    _check(_normal(rows, vocab, dtype, seed=vocab), k)


@pytest.mark.parametrize("temperature", [0.25, 1.0, 3.0])
def test_temperature(temperature):
    _check(_normal(5, 20011, torch.bfloat16), 33, temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,pad", [(1, 0), (3, 5), (0, 64)])
def test_strides_and_alignment(dtype, offset, pad):
    rows, vocab = 9, 10007
    base = _normal(1, offset + rows * (vocab + pad), dtype)[0]
    _check(base[offset:].view(rows, vocab + pad)[:, :vocab], 50)


def test_row_stride_zero_and_reversed_order():
    row = _normal(1, 6001, torch.float16)
    _check(row.expand(4, -1), 20)
    both = _normal(8, 6001, torch.float32)
    _check(both[::2], 20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [300, 20000, 151936])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "zeros", "lowest", "masked", "all_masked", "few"])
def test_orders_ties_and_masks(dtype, vocab, kind):
    low = torch.finfo(dtype).min
    z = _normal(2, vocab, dtype, seed=5)
    if kind == "equal":
        z.fill_(1.5)
    elif kind in ("rising", "falling"):
        z = z.sort(dim=1, descending=kind == "falling").values
    elif kind == "zeros":
        z = torch.where(z > 0, 0.0, -0.0).to(dtype)
    elif kind == "lowest":
        z.fill_(low)
        z[1, vocab // 2:] = -1.0
    elif kind == "masked":
        z[:, : vocab - 40] = -float("inf")
    elif kind == "all_masked":
        z.fill_(-float("inf"))
    elif kind == "few":
        z.fill_(low)
        z[:, 7], z[:, vocab - 1] = 2.0, 2.0
    _check(z, 60)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(dtype):
    z = _normal(4, 9000, dtype)
    z[0, 4000] = float("inf")
    z[1, 77] = float("nan")
    z[1, 8999] = float("nan")
    z[2, :] = float("nan")
    z[3, 0] = -float("inf")
    from soupsuck_b200.kernels import top_logits
    values, indices, lse = top_logits(z, 9)
    rv, ri, rl = D.top_logits(np_of(z.float()), 9)
    np.testing.assert_array_equal(np_of(indices), ri)
    np.testing.assert_array_equal(np_of(values.float()), rv.astype(np.float32))
    assert lse[0].item() == float("inf") and torch.isnan(lse[1:3]).all() and torch.isfinite(lse[3])


def test_largest_magnitudes_of_fp32():
    z = torch.full((2, 5000), torch.finfo(torch.float32).min, device="cuda")
    z[1, 9] = torch.finfo(torch.float32).max
    from soupsuck_b200.kernels import top_logits
    values, indices, lse = top_logits(z, 3)
    assert indices.tolist() == [[0, 1, 2], [9, 0, 1]]
    assert lse.tolist() == [torch.finfo(torch.float32).min, torch.finfo(torch.float32).max]


def test_empty_and_side_stream():
    from soupsuck_b200.kernels import top_logits
    values, indices, lse = top_logits(torch.empty((0, 100), device="cuda"), 5)
    assert values.shape == (0, 5) and indices.shape == (0, 5) and lse.shape == (0,)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z = _normal(16, 40000, torch.float16)
        got = top_logits(z, 12)[1]
    side.synchronize()
    np.testing.assert_array_equal(np_of(got), D.top_logits(np_of(z.float()), 12)[1])


def test_repeat_calls_agree():
    from soupsuck_b200.kernels import top_logits
    z = _normal(50, 30000, torch.bfloat16)
    first, second = top_logits(z, 100), top_logits(z, 100)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals():
    from soupsuck_b200.kernels import top_logits
    z = _normal(4, 300, torch.float16)
    for bad in (lambda: top_logits(z, 0), lambda: top_logits(z, 257), lambda: top_logits(z[:, :9], 10),
                lambda: top_logits(z.double(), 3), lambda: top_logits(z[0], 3), lambda: top_logits(z.cpu(), 3),
                lambda: top_logits(z.t(), 3), lambda: top_logits(z, 3, temperature=0.0),
                lambda: top_logits(z, 3, temperature=-1.0), lambda: top_logits(z, 3, temperature=float("inf")),
                lambda: top_logits(z, 2.5), lambda: top_logits(z[:, :0], 1)):
        with pytest.raises(ValueError, match="top_logits"):
            bad()
