"""A refused call leaves nothing behind: the CUDA error it met belongs to it
alone, and the next good call succeeds and says so."""
import contextlib
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from pitorch_b200 import api  # noqa: E402
from serve_ref import Batch, check, ints, sample_ref  # noqa: E402

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def broken_stream():
    """A stream in a capture that is already invalid (it was waited for): a launch there is refused by the runtime."""
    rt = C.CDLL("libcudart.so.12")
    s, g = C.c_void_p(), C.c_void_p()
    torch.cuda.synchronize()
    assert rt.cudaStreamCreateWithFlags(C.byref(s), 1) == 0
    assert rt.cudaStreamBeginCapture(s, 2) == 0   # relaxed: other streams go on
    assert rt.cudaStreamSynchronize(s) != 0
    rt.cudaGetLastError()
    yield s.value
    assert rt.cudaStreamEndCapture(s, C.byref(g)) != 0
    rt.cudaGetLastError()
    assert rt.cudaStreamDestroy(s) == 0
    torch.cuda.synchronize()


def calls(L):
    """Each operator on small inputs: (name, call on a stream, check of its result)."""
    b = Batch([(20, 3)], 2, 1, 32, 8, "f32")
    w = Batch([(20, 60)], 2, 1, 32, 8, "bf16")
    outs = [torch.zeros_like(x.q) for x in (b, w)]
    x, u, tok = torch.randn(1, 500, device="cuda"), torch.full((1,), 0.5, device="cuda"), ints([-5])
    samp = api.ptc_sample_args(api.PTC_F32, 1, 500, x.data_ptr(), 500, None, None, None, None, u.data_ptr(), tok.data_ptr())
    new, q = torch.randn(3, 3 * 64, device="cuda"), torch.zeros(3, 64, device="cuda")
    pos, slots = ints([0, 1, 2]), ints([0, 1, 2])
    app = api.ptc_append_args(b.cache(), 3, 2, new.data_ptr(), new.data_ptr() + 256, new.data_ptr() + 512, 192, 192, 192, pos.data_ptr(),
                              slots.data_ptr(), None, 0, q.data_ptr(), 64, b.err.data_ptr())
    past, add, free, table = ints([0]), ints([5]), ints([3]), ints([-1])
    kv, start, sl, ps, used = ints([9]), ints([9, 9]), ints([9] * 5), ints([9] * 5), ints([9])
    plan = api.ptc_pages_args(1, 8, 1, 5, 1, 9, *(t.data_ptr() for t in (past, add, free, table, kv, start, sl, ps, used)), b.err.data_ptr())
    rope = torch.zeros(16, 4, 2, device="cuda")
    args = [y.attn_args(o) for y, o in zip((b, w), outs)]

    def same(got, want):
        assert torch.equal(got, want)

    keep = (new, x, u, tok, pos, slots, past, add, free, table, kv, start, sl, ps, used)
    return [("sample", lambda s: L.ptc_sample_tokens(samp, s), lambda: same(tok, ints([sample_ref(x[0])]))),
            ("attend", lambda s: L.ptc_paged_attention(args[0], s), lambda: check(outs[0][:3], *b.reference())),
            ("attend many", lambda s: L.ptc_paged_attention(args[1], s), lambda: check(outs[1][:60], *w.reference())),
            ("pages", lambda s: L.ptc_plan_pages(plan, s), lambda: same(sl, ints([24, 25, 26, 27, 28]))),
            ("rope", lambda s: L.ptc_rope_table(rope.data_ptr(), 16, 8, s), lambda: same(rope[0, :, 0], torch.ones(4, device="cuda"))),
            ("append", lambda s: L.ptc_kv_append(app, s), lambda: same(q, new[:, :64]))], keep


def test_a_refused_call_does_not_refuse_the_next(ptlib, capfd):
    ops, keep = calls(ptlib)
    stream = torch.cuda.Stream()
    got = []
    with broken_stream() as broken:   # (nothing may wait for the device meanwhile)
        for bad, refused, _ in ops:
            for good, call, _ in ops:
                got.append((bad, refused(broken), good, call(stream.cuda_stream), call(stream.cuda_stream)))
    assert [g for g in got if (g[1], g[3], g[4]) != (-1, 0, 0)] == []
    for name, _, result in ops:
        result()
