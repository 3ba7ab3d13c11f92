"""Sampling on a rank whose classifier is vocab-parallel: the decoder then
holds its own rows of the logits alone, and no token may be drawn from them
before the others' were gathered. One GPU: the rank embeds, runs all layers
and keeps no other rank's keys, so its stage waits for nobody."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from conftest import rel_err  # noqa: E402
from pitorch_b200 import api, synth  # noqa: E402
from serve_ref import sample_ref  # noqa: E402

pytestmark = pytest.mark.gpu
vp = C.c_void_p


class ptc_vocab_split(C.Structure):
    _fields_ = ([(n, C.c_int) for n in ("row0", "rows", "ranks", "rank", "combine", "x_local", "embed_local")]
                + [(n, vp) for n in ("cls_rows", "rms_final", "embedding", "box")]
                + [("x_out", vp * 8), ("n_x_out", C.c_int), ("key_out", vp * 2), ("n_key_out", C.c_int), ("sent", vp)])


def declare(L):
    for name, args in (("ptc_decoder_set_links", [vp, vp, vp, vp, vp, C.c_longlong]),
                       ("ptc_decoder_set_vocab_parallel", [vp, C.POINTER(ptc_vocab_split)]),
                       ("ptc_decoder_set_input", [vp, C.c_int, vp]), ("ptc_decoder_enqueue_stage", [vp, C.c_int]),
                       ("ptc_decoder_enqueue_fetch", [vp, C.c_int])):
        getattr(L, name).argtypes, getattr(L, name).restype = args, None
    L.ptc_decoder_logits_dev.argtypes, L.ptc_decoder_logits_dev.restype = [vp], vp


def test_no_token_from_one_ranks_logits(ptlib, capfd):
    L = ptlib
    declare(L)
    cfg = synth.CONFIGS["tiny"]
    dim, V = cfg[0], cfg[5]
    whole, part = (api.Context(synth.make_blob("tiny"), device=0) for _ in range(2))
    for t in (5, 900):   # a cache, and logits of an earlier step in the buffer
        whole.forward_step(t)
        part.forward_step(t)
    c, dec = L.pt_ptc_ctx(C.byref(part.ctx)), part.ptc_decoder()

    def put(a):
        a = np.ascontiguousarray(a)
        p = L.ptc_alloc(c, a.nbytes)
        L.ptc_h2d(c, p, a.ctypes.data, a.nbytes)
        return p

    w = whole.ctx.w
    rows = lambda p, n: np.ctypeslib.as_array(p, shape=(n,))  # noqa: E731
    boxes = [L.ptc_mailbox_alloc(c, dim + 8) for _ in range(4)]
    assert all(boxes)
    L.ptc_decoder_set_links(dec, boxes[0], boxes[1], put(np.zeros(1, np.uint32)), put(np.zeros(1, np.int32)), 1000000)
    split = ptc_vocab_split(0, V // 2, 2, 0, 0, 1, 1, put(rows(w.wcls, V * dim)[: V // 2 * dim]), put(rows(w.rms_final_weight, dim)),
                            put(rows(w.token_embedding, V * dim)), boxes[2], (vp * 8)(boxes[3]), 1, (vp * 2)(), 0,
                            put(np.zeros(2, np.uint32)))
    L.ptc_decoder_set_vocab_parallel(dec, C.byref(split))
    assert 0 <= L.ptc_decoder_sample(dec, 1.0, 0, 1.0, 0.0, 0.5) < V   # the plain steps' logits are whole

    rule = (0.7, 0, 0.9, 0.0)
    for step in range(2):
        L.ptc_decoder_set_input(dec, 2 + step, put(np.array([77], np.int32)))
        L.ptc_decoder_enqueue_stage(dec, 1)
        L.ptc_sync(c)
        whole.forward_step(77)
        want = whole.logits()
        got = np.empty(V, np.float32)
        logits = L.ptc_decoder_logits_dev(dec)
        L.ptc_d2h(c, got.ctypes.data, logits, got.nbytes)
        assert rel_err(got[: V // 2], want[: V // 2]) <= 1e-4   # its own rows of this step
        capfd.readouterr()
        assert L.ptc_decoder_sample(dec, *rule, 0.5) == -1
        assert "ptc_decoder_sample" in capfd.readouterr().err
        # the other rank's rows arrive
        L.ptc_h2d(c, logits + V // 2 * 4, want[V // 2:].ctypes.data, V // 2 * 4)
        L.ptc_decoder_enqueue_fetch(dec, 1)
        L.ptc_sync(c)
        got[V // 2:] = want[V // 2:]
        f = lambda v: float(np.float32(v))  # noqa: E731
        for u in (0.03, 0.5, 0.97):
            assert L.ptc_decoder_sample(dec, *rule, u) == sample_ref(torch.from_numpy(got), f(0.7), 0, f(0.9), 0.0, f(u))
    # the split undone: plain steps again
    L.ptc_decoder_set_vocab_parallel(dec, None)
    L.ptc_decoder_set_links(dec, None, None, None, None, 0)
    part.forward_step(3)
    assert 0 <= L.ptc_decoder_sample(dec, 1.0, 0, 1.0, 0.0, 0.5) < V
    for b in boxes:
        L.ptc_mailbox_free(b)
    whole.close()
    part.close()
