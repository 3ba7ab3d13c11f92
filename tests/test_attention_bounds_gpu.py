"""What the general bounds of the attention tests leave open: the second part
of the probabilities in the few-rows kernel, and calls of as many sequences as
the operators take."""
import math

import pytest

torch = pytest.importorskip("torch")

from pitorch_b200 import api  # noqa: E402
from serve_ref import HALF, Batch, check  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [1, 4])
def test_few_rows_keep_probabilities_beyond_the_type(ptlib, dtype, group):
    """Two keys of nearly equal weight, 1 and e = exp(-x), and values +1 and -1: (1 - e) / (1 + e) is of the size that a
    probability rounded to the type would lose. In two parts it is off by half a step of half a step: of a = 1 the bound
    is h^2 (f16: half a step of 2^-24 / 2^7 too), 2^-22 of the exponential and 40 roundings of 2^-24, the score x's
    relative 2^-17 (68 products and three scalings of 2^-24), and the result's own h."""
    kv, hd = 64, 64
    b = Batch([(1, 1)], kv, group, hd, 16, dtype)
    page = int(b.table[0, 0])
    b.kp[page, :, :2] = 0.0
    b.kp[page, :, 1, 0] = -(torch.arange(kv, device="cuda") + 1) / 64.0 * (1 / 16 if dtype == "bf16" else 1 / 128)
    b.vp[page, :, 0], b.vp[page, :, 1] = 1.0, -1.0
    b.q.zero_()
    b.q[..., 0] = 1.0
    got = b.attend(ptlib, scale=0.125)[:1].reshape(kv, group, hd)
    x = -b.kp[page, :, 1, 0].double()[:, None, None] / 8
    want = ((1 - (-x).exp()) / (1 + (-x).exp())).expand(kv, group, hd)
    h = HALF[dtype]
    assert float((x / 2).max()) < 1.1 * h and float((x / 2).min()) > h / 100   # where rounding to the type shows
    off = h * h + 2.0 ** -32 + 2.0 ** -22 + 40 * 2.0 ** -24 + x * 2.0 ** -17 + want * h + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert float(off.max()) < h / 8
    check(got, want, off)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, 60])   # the few-rows and the many-rows kernels
def test_as_many_sequences_as_the_operators_take(ptlib, dtype, max_q):
    n = api.PTC_SERVE_MAX_SEQS
    lens = [((r * 37) % 90, (1, 0, 2, 1)[r % 4]) for r in range(n)]
    b = Batch(lens, 2, 1, 128, 16, dtype, seed=3)
    want, bound = b.reference()
    got = b.attend(ptlib, max_q=max_q)
    assert int(b.err) == 0
    check(got[: b.total], want, bound)
    assert bool((got[b.total:] == 7.0).all())
    assert torch.equal(b.attend(ptlib, max_q=max_q), got)
