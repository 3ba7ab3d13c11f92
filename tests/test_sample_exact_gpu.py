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


def test_temperatures_at_the_low_end_of_the_type(ptlib):
    """Weights are whole units of 2^-43 of the largest, so that what is below half of one is never chosen, not for u = 0
    either, however small the distance and the temperature are."""
    rows = [(t, d) for t in (1e-38, 3e-39, 1e-40, 1e-42, 3e-44, 1.5e-45) for d in (1.5e-37, 9.9e-38, 7e-38, 5e-38, 3.3e-38, 2.1e-38, 1.3e-38)]
    x = torch.zeros(len(rows), 40, device="cuda")
    t = torch.tensor([r[0] for r in rows])
    x[:, :39] = -torch.tensor([r[1] for r in rows], device="cuda")[:, None]
    assert bool((t > 0).all()) and bool((x[:, :39] < 0).all())
    units = (x.double() / t.double().cuda()[:, None]).exp() * 2.0 ** 43
    heavy = torch.where(units < 0.5, -math.inf, x)   # what has weight
    for u in (0.0, 0.3, 0.9):
        f = float(torch.tensor(u))
        for p in (1.0, 0.9):
            got = run_sample(ptlib, x, t.tolist(), None, [p] * len(rows), None, [u] * len(rows))
            assert got == [sample_ref(heavy[i], float(t[i]), top_p=float(torch.tensor(p)), u=f) for i in range(len(rows))]
