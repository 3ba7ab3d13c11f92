"""f16 attention where a few keys outweigh a long flat tail: 8192 keys of
e^-17.4 of the largest weight each. A probability of 2^-25 of the row's
reference rounds to nothing in f16, but 8000 of them are a quarter of a
thousandth of the row, and stand in its sum."""
import math

import pytest

torch = pytest.importorskip("torch")

from serve_ref import Batch  # noqa: E402

pytestmark = pytest.mark.gpu
GAP = 17.40625   # exact in f16: 8 * GAP / 8 in the product, e^-GAP = 2^-25.1


@pytest.mark.parametrize("new", [1, 40])   # the few-rows and the many-rows kernel
@pytest.mark.parametrize("sinks", [[0, 16, 32, 48], [4000, 4016, 4032, 4048]])
def test_a_flat_tail_keeps_its_weight(ptlib, new, sinks):
    """Heads enough that most of them stay whole in one CTA, a sink for each of the parts that share an item's keys.

    An element is 16 n w / (4 + n w) for n tail keys of weight w = e^-GAP. Its relative error: a probability is
    rounded to a step of 2^-24 relative to 2^7 times the reference, so by at most 2^-32 of the largest weight and
    2^-32 / w of itself; the result by 2^-11; n + 32 additions and the exponent 25.1 of the scores, whose 32-bit error
    of 4 steps is relative to it, by 2^-24 each. (A tail that is met before its sinks has a reference of its own.)"""
    n, hd, heads = 8192, 32, 600
    b = Batch([(n - new, new)], heads, 1, hd, 64, "f16")
    pages = b.table[0].long()
    k, v = torch.zeros(n, hd, dtype=torch.float16, device="cuda"), torch.full((n, hd), 16.0, dtype=torch.float16, device="cuda")
    k[sinks, 0], v[sinks] = GAP, 0.0
    b.kp[pages] = k.reshape(-1, 1, 64, hd).expand(-1, heads, -1, -1)
    b.vp[pages] = v.reshape(-1, 1, 64, hd).expand(-1, heads, -1, -1)
    b.q.zero_()
    b.q[..., 0] = 8.0
    got = b.attend(ptlib, scale=0.125)[: b.total].double()
    assert int(b.err) == 0
    w = math.exp(-GAP)
    tail = (torch.arange(n - new, n, device="cuda", dtype=torch.float64) + 1 - len(sinks))[:, None, None] * w
    want = 16 * tail / (len(sinks) + tail)
    off = 2.0 ** -32 / w + 2.0 ** -11 + (n + 32 + 4 * 25.2) * 2.0 ** -24
    worst = ((got - want).abs() / want).max()
    assert float(worst) <= off
