"""pt_forward_step_sampled on its default and its quiet path: the token is the
definition's for the very logits that the step left, and a call that cannot
sample does not move the context."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from conftest import rel_err  # noqa: E402
from pitorch_b200 import api, synth  # noqa: E402
from serve_ref import sample_ref  # noqa: E402

pytestmark = pytest.mark.gpu
RULES = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.02, 40, 0.9, 0.0), (0.05, 0, 0.5, 0.1), (3.0, 1, 1.0, 0.0), (0.3, 500, 0.99, 0.01)]


def f(v):
    return float(np.float32(v))


def device_logits(ctx):
    L = ctx.L
    L.ptc_decoder_logits_dev.restype, L.ptc_decoder_logits_dev.argtypes = C.c_void_p, [C.c_void_p]
    out = np.empty(ctx.cfg.vocab_size, np.float32)
    L.ptc_d2h(L.pt_ptc_ctx(C.byref(ctx.ctx)), out.ctypes.data, L.ptc_decoder_logits_dev(ctx.ptc_decoder()), out.nbytes)
    return out


@pytest.mark.parametrize("name", ["tiny", "stories15M"])
@pytest.mark.parametrize("sync", [0, 1])
def test_the_token_is_the_definitions(ptlib, name, sync):
    ctx = api.Context(synth.make_blob(name), device=0)
    ctx.ctx.sync_logits = sync
    rng = np.random.default_rng(21)
    tok = 11
    for i in range(3 * len(RULES)):
        t, k, p, mp = RULES[i % len(RULES)]
        u = f(rng.random())
        nxt = ctx.forward_step_sampled(tok, u, t, k, p, mp)
        x = device_logits(ctx)
        assert nxt == sample_ref(torch.from_numpy(x), f(t), k, f(p), f(mp), u)
        if sync:
            assert np.array_equal(ctx.logits(), x)
        assert ctx.pos == i + 1
        tok = nxt
    ctx.close()


def test_a_vocabulary_that_cannot_be_sampled_leaves_the_context(ptlib, capfd):
    cfg = (64, 176, 1, 4, 4, api.PTC_SAMPLE_MAX_VOCAB + 1, 32)
    one, two = (api.Context(synth.make_blob(cfg), device=0) for _ in range(2))
    first = one.forward_step(5)
    assert two.forward_step(5) == first
    for _ in range(2):
        assert one.forward_step_sampled(first, 0.5) == -1
        assert "pt_forward_step_sampled" in capfd.readouterr().err
        assert one.pos == 1
    one.forward_step(first)
    two.forward_step(first)
    assert one.pos == 2
    assert rel_err(one.logits(), two.logits()) <= 1e-4   # (the decode kernels' sums have no fixed order)
    one.close()
    two.close()
