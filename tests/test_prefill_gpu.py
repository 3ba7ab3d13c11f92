"""A prompt in one pass (pt_prefill) and sampled steps against the same work
token by token and against the reference's greedy streams."""
import numpy as np
import pytest

from conftest import rel_err
from pitorch_b200 import api, synth

pytestmark = pytest.mark.gpu
TOL = 1e-4   # of the largest logit, as every decode path (test_decode_gpu.py)


def contexts(cfg):
    blob = synth.make_blob(cfg)
    return api.Context(blob, device=0), api.Context(blob, device=0)


# a multi-query model, heads of 8, and a head size that only the small kernels take
EXTRA = {"grouped": (96, 256, 3, 12, 4, 1024, 96), "odd": (120, 64, 2, 5, 1, 1000, 300)}


@pytest.mark.parametrize("name,parts", [("tiny", [1]), ("tiny", [7, 1, 30]), ("tiny", [64]), ("grouped", [17, 60]), ("odd", [299]),
                                        ("odd", [257, 3]), ("stories15M", [130, 90])])
def test_prefill_equals_token_by_token(ptlib, name, parts):
    cfg = EXTRA.get(name) or synth.CONFIGS[name]
    one, all_ = contexts(cfg)
    tokens = np.random.default_rng(sum(parts)).integers(0, cfg[5], size=sum(parts)).astype(np.int32)
    at = 0
    for n in parts:
        nxt = all_.prefill(tokens[at:at + n])
        for t in tokens[at:at + n]:
            want = one.forward_step(int(t))
        at += n
        assert all_.pos == one.pos == at
        assert rel_err(all_.logits(), one.logits()) <= TOL
        top2 = np.sort(one.logits())[-2:]
        if top2[1] - top2[0] > 2 * TOL * np.abs(one.logits()).max():
            assert nxt == want
    # and the cache it leaves serves steps
    for t in tokens[: cfg[6] - at][:3]:
        one.forward_step(int(t))
        all_.forward_step(int(t))
        assert rel_err(all_.logits(), one.logits()) <= TOL
    one.close()
    all_.close()


def test_prefill_then_decode_follows_the_reference_stream(ptlib):
    ctx = api.Context(synth.make_blob("stories15M"), device=0)
    prompt = synth.make_prompt(32000)
    want = ctx.generate_greedy(prompt, 64)   # pinned to the reference by test_decode_gpu.py
    ctx.reset_kv()
    out = [ctx.prefill(prompt)]
    while len(out) < 64 - len(prompt) + 1:
        out.append(ctx.forward_step(out[-1]))
    assert out == want[len(prompt) - 1:].tolist()
    ctx.close()


def test_prefill_refusals_leave_the_context(ptlib, capfd):
    ctx = api.Context(synth.make_blob("tiny"), device=0)
    first = ctx.forward_step(5)
    for bad in ([], [1] * 64, [1, -1], [1, 1024]):
        with pytest.raises(ValueError):
            ctx.prefill(bad)
        assert "ptc_decoder_prefill" in capfd.readouterr().err
    assert ctx.pos == 1
    ref = api.Context(synth.make_blob("tiny"), device=0)
    assert ref.forward_step(5) == first and ref.forward_step(first) == ctx.forward_step(first)
    assert np.array_equal(ref.logits(), ctx.logits()) or rel_err(ref.logits(), ctx.logits()) <= TOL
    ref.close()
    ctx.close()


@pytest.mark.parametrize("sync", [0, 1])
def test_sampled_steps(ptlib, sync):
    torch = pytest.importorskip("torch")
    from serve_ref import sample_ref
    ctx = api.Context(synth.make_blob("stories15M"), device=0)
    ctx.ctx.sync_logits = sync
    chk = api.Context(synth.make_blob("stories15M"), device=0)
    rng = np.random.default_rng(9)
    tok = 11
    f = lambda v: float(np.float32(v))  # noqa: E731
    for t, k, p, mp in ((0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.02, 40, 0.9, 0.0), (0.05, 0, 0.5, 0.1), (3.0, 1, 1.0, 0.0)):
        u = f(rng.random())
        nxt = ctx.forward_step_sampled(tok, u, t, k, p, mp)
        chk.forward_step(tok)
        got = ctx.logits() if sync else None
        x = got if sync else chk.logits()
        want = sample_ref(torch.from_numpy(x), f(t), k, f(p), f(mp), u)
        if sync or t == 0.0 or k == 1:
            assert nxt == want   # the very logits it was drawn from
        assert 0 <= nxt < 32000
        tok = nxt
    ctx.close()
    chk.close()
