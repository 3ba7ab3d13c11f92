"""Where the sampling weights have to be exact: logits far from zero, small
temperatures, and temperatures at the low end of the type."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from serve_ref import sample_ref  # noqa: E402
from test_serve_gpu import run_sample  # noqa: E402

pytestmark = pytest.mark.gpu


def border_rules():
    """(d, t, m): steps d below the maximum, temperatures and min_p, all exact in f32, whose weight e^(d/t) is within
    3e-10 of min_p, but not within 4e-12: nine times the bound of a weight's error, 2^-42 of it and half a unit of 2^-43."""
    r = np.random.default_rng(7)
    t = (0.01 + 0.02 * r.random(200000)).astype(np.float32)
    d = -np.float32(1 / 128) * r.integers(1, 4, t.size).astype(np.float32)
    w = np.exp(d.astype(np.longdouble) / t.astype(np.longdouble))
    m = w.astype(np.float32)
    gap = np.abs(m.astype(np.longdouble) - w) / w
    pick = (w > 0.1) & (gap > 4e-12) & (gap < 3e-10)
    return d[pick], t[pick], m[pick], (w >= m.astype(np.longdouble))[pick]


@pytest.mark.parametrize("top", [0.0, 1.0, -65536.0, 65536.0 + 1.0])
def test_min_p_at_its_border_wherever_the_logits_are(ptlib, top):
    d, t, m, keeps = border_rules()
    n = len(d)
    assert n > 200 and 0.3 < keeps.mean() < 0.7
    x = torch.full((n, 8), -math.inf, device="cuda")
    x[:, 2] = top
    x[:, 5] = torch.from_numpy(d).cuda() + top
    assert torch.equal(x[:, 5].double() - top, torch.from_numpy(d).cuda().double())   # the difference is exact
    got = run_sample(ptlib, x, t.tolist(), None, None, m.tolist(), [1 - 2.0 ** -24] * n)
    assert got == [5 if k else 2 for k in keeps]


def test_an_offset_of_all_logits_changes_nothing(ptlib):
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = (torch.randn(64, 5000, generator=g, device="cuda") * 300).round() / 128
    u, t = torch.rand(64, generator=g, device="cuda").tolist(), [0.01 + 0.02 * i for i in range(64)]
    want = run_sample(ptlib, x, t, None, [0.95] * 64, None, u)
    for off in (-65536.0, 4096.0, 65536.0 - 32):
        y = x + off
        assert torch.equal(y.double() - off, x.double())
        assert run_sample(ptlib, y, t, None, [0.95] * 64, None, u) == want
