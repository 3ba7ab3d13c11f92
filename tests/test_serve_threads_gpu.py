"""Calls of the serving operators from two host threads at once, on streams
(and workspaces) of their own, with very different sizes: a thread's call
must not depend on what the other one asks of the same kernel."""
import threading

import pytest

torch = pytest.importorskip("torch")

from pitorch_b200 import api  # noqa: E402
from serve_ref import CODE, DT, Batch, sample_ref  # noqa: E402

pytestmark = pytest.mark.gpu
CALLS = 400


def at_once(*calls):
    """Each of `calls` (a function of a stream handle) CALLS times in a thread; the numbers of refused calls."""
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    refused, start = [0] * len(calls), threading.Barrier(len(calls))

    def work(i):
        start.wait()
        for _ in range(CALLS):
            refused[i] += calls[i](streams[i].cuda_stream) != 0

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return refused


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, 60])
def test_attention_of_many_and_of_one_sequence(ptlib, dtype, max_q):
    """(4096 sequences take 16 KB more of shared memory than one; max_q 60 picks the many-rows kernels.)"""
    many = Batch([(r % 3, 1) for r in range(api.PTC_SERVE_MAX_SEQS)], 1, 1, 128, 16, dtype, seed=1)
    one = Batch([(100, 1)], 1, 1, 128, 16, dtype, seed=2)
    outs = [torch.zeros_like(b.q) for b in (many, one)]
    args = [b.attn_args(o, max_q=max_q) for b, o in zip((many, one), outs)]
    want = [b.attend(ptlib, max_q=max_q) for b in (many, one)]
    assert at_once(*(lambda s, a=a: ptlib.ptc_paged_attention(a, s) for a in args)) == [0, 0]
    for b, o, w in zip((many, one), outs, want):
        assert int(b.err) == 0
        assert torch.equal(o[: b.total], w[: b.total])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sampling_of_large_and_small_vocabularies(ptlib, dtype):
    rows = [torch.randn(1, v, device="cuda").to(DT[dtype]) for v in (262144, 40000)]   # one kernel: eight CTAs a row
    u = torch.full((1,), 0.25, device="cuda")
    toks = [torch.full((1,), -5, dtype=torch.int32, device="cuda") for _ in rows]
    args = [api.ptc_sample_args(CODE[dtype], 1, x.shape[1], x.data_ptr(), x.shape[1], None, None, None, None, u.data_ptr(), t.data_ptr())
            for x, t in zip(rows, toks)]
    assert at_once(*(lambda s, a=a: ptlib.ptc_sample_tokens(a, s) for a in args)) == [0, 0]
    assert [int(t) for t in toks] == [sample_ref(x[0], u=0.25) for x in rows]
