"""The serving operators (include/ptc_serve.h) against 64-bit plain forms:
page tables and slot maps, the rotary cache write, paged attention, sampling."""
import math
import os
import random
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from pitorch_b200 import api  # noqa: E402
from serve_ref import CODE, DT, HALF, Batch, check, ints, plan_ref, sample_ref, stream  # noqa: E402

pytestmark = pytest.mark.gpu


# ---- page tables and slot maps ------------------------------------------------

def run_plan(L, past, new, page, free, table, max_tokens=None, n_pages=1 << 20, max_pages=None):
    n = len(past)
    cols = len(table[0]) if n else 1
    total = sum(x for x in new if x > 0)
    m = total + 4 if max_tokens is None else max_tokens
    t = {"past": ints(past), "new": ints(new), "free": ints(free), "table": ints(table).reshape(n, cols)}
    out = {k: torch.full((c,), -99, dtype=torch.int32, device="cuda")
           for k, c in (("kv_len", n), ("q_start", n + 1), ("slots", m), ("positions", m), ("used", 1))}
    err = ints([0])
    a = api.ptc_pages_args(n, page, cols if max_pages is None else max_pages, m, len(free), n_pages, t["past"].data_ptr(),
                           t["new"].data_ptr(), t["free"].data_ptr(), t["table"].data_ptr(), out["kv_len"].data_ptr(),
                           out["q_start"].data_ptr(), out["slots"].data_ptr(), out["positions"].data_ptr(),
                           out["used"].data_ptr(), err.data_ptr())
    assert L.ptc_plan_pages(a, stream()) == 0
    torch.cuda.synchronize()
    return dict({k: v.tolist() for k, v in out.items()}, table=t["table"].tolist(), err=int(err))


@pytest.mark.parametrize("n,page,most_past,most_new,seed", [
    (1, 16, 0, 1, 0), (1, 1, 5, 9, 1), (3, 7, 40, 20, 2), (64, 16, 4096, 1, 3), (333, 16, 200, 70, 4),
    (513, 128, 3000, 40, 5), (1025, 3, 30, 5, 6), (4096, 16, 100, 3, 7)])
def test_plan_matches_the_definition(ptlib, n, page, most_past, most_new, seed):
    r = random.Random(seed)
    past = [r.randint(0, most_past) for _ in range(n)]
    new = [r.choice([0, 1, r.randint(0, most_new)]) for _ in range(n)]
    cols = max(-(-(p + q) // page) for p, q in zip(past, new)) + 1
    pages = list(range(sum(-(-(p + q) // page) for p, q in zip(past, new)) + 5))
    r.shuffle(pages)
    table = []
    for p in past:
        h = -(-p // page)
        table.append(pages[:h] + [-1] * (cols - h))
        del pages[:h]
    want = plan_ref(past, new, page, pages, table)
    got = run_plan(ptlib, past, new, page, pages, table)
    total = sum(new)
    assert got["err"] == 0
    assert got["table"] == want[0] and got["kv_len"] == want[1] and got["q_start"] == want[2]
    assert got["slots"] == want[3] + [-1] * 4 and got["positions"] == want[4] + [-1] * 4
    assert got["used"] == [want[5]] and got["q_start"][-1] == total


@pytest.mark.parametrize("what,bit", [("pages", api.PTC_SERVE_ERR_PAGES), ("table", api.PTC_SERVE_ERR_TABLE),
                                      ("tokens", api.PTC_SERVE_ERR_TOKENS), ("negative", api.PTC_SERVE_ERR_LENGTH),
                                      ("overflow", api.PTC_SERVE_ERR_LENGTH)])
def test_plan_that_does_not_fit_changes_nothing(ptlib, what, bit):
    past, new, page, free = [5, 0, 9], [4, 17, 3], 4, list(range(10, 40))
    table = [[1, 2] + [-1] * 4, [-1] * 6, [3, 4, 5] + [-1] * 3]
    if what == "pages":
        free = free[:5]
    if what == "table":
        new[1] = 25
    if what == "negative":
        new[2] = -1
    if what == "overflow":
        past[0], new[0] = 2 ** 31 - 2, 5
    got = run_plan(ptlib, past, new, page, free, table, max_tokens=20 if what == "tokens" else 64)
    assert got["err"] == bit
    assert got["table"] == table and got["used"] == [0]
    assert got["q_start"] == [0] * 4 and got["kv_len"] == past
    assert set(got["slots"]) == {-1} and set(got["positions"]) == {-1}


def test_plan_reports_a_bad_held_page(ptlib):
    got = run_plan(ptlib, [3, 2], [2, 2], 4, [6, 7], [[-1, -1], [9, -1]], n_pages=10)
    assert got["err"] == api.PTC_SERVE_ERR_INDEX
    assert got["slots"][:4] == [-1, 6 * 4, 38, 39] and got["positions"][:4] == [3, 4, 2, 3]


def test_plan_of_no_sequences(ptlib):
    got = run_plan(ptlib, [], [], 4, [1], [], max_tokens=3)
    assert got["err"] == 0 and got["q_start"] == [0] and got["slots"] == [-1] * 3 and got["used"] == [0]


# ---- rotary write ---------------------------------------------------------------

def append_case(L, dtype, lens, kv, group, hd, page, layout="heads", rope=True, packed=True, in_place=False):
    b = Batch(lens, kv, group, hd, page, dtype, seed=hd + page, layout=layout)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    heads, total, dt = b.heads, b.total, DT[dtype]
    row = (heads + 2 * kv) * hd
    qkv = torch.randn(total, row, generator=g, device="cuda").to(dt)
    n_pos = max(p + q for p, q in lens)
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    table = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    pos = [p + j for p, q in lens for j in range(q)]
    slots = [int(b.table[r, (p + j) // page]) * page + (p + j) % page for r, (p, q) in enumerate(lens) for j in range(q)]
    keep = qkv.clone()
    q = qkv[:, : heads * hd]
    out = q if in_place else torch.empty(total, heads * hd, dtype=dt, device="cuda")
    kb, vb = b.kp.clone(), b.vp.clone()
    positions, slots_t = ints(pos), ints(slots)
    e = qkv.element_size()
    a = api.ptc_append_args(b.cache(), total, heads, qkv.data_ptr(), qkv.data_ptr() + heads * hd * e,
                            qkv.data_ptr() + (heads + kv) * hd * e, row, row, row, positions.data_ptr(),
                            slots_t.data_ptr(), table.data_ptr() if rope else None, n_pos if rope else 0,
                            out.data_ptr(), out.stride(0), b.err.data_ptr())
    assert L.ptc_kv_append(a, stream()) == 0
    torch.cuda.synchronize()
    assert int(b.err) == 0
    x = keep.double().reshape(total, heads + 2 * kv, hd)
    turned = x.clone()
    if rope:
        cs = table.double()[torch.tensor(pos, device="cuda")][:, None]
        u, w = x[..., 0::2], x[..., 1::2]
        turned[..., 0::2] = u * cs[..., 0] - w * cs[..., 1]
        turned[..., 1::2] = u * cs[..., 1] + w * cs[..., 0]
        # two products and a sum in 32 bits, one rounding to the type
        mag = (u.abs() + w.abs()).repeat_interleave(2, -1)
        bound = mag * 3 * 2.0 ** -24 + turned.abs() * HALF[dtype] + (2.0 ** -25 if dtype == "f16" else 1e-30)
    else:
        bound = torch.full_like(x, 1e-30)
    check(out.reshape(total, heads, hd), turned[:, :heads], bound[:, :heads])
    s = torch.tensor(slots, device="cuda")
    pg, off = s // page, s % page
    check(b.kp[pg, :, off], turned[:, heads:heads + kv], bound[:, heads:heads + kv])
    assert torch.equal(b.vp[pg, :, off], keep.reshape(total, -1, hd)[:, heads + kv:])
    # nothing else of the cache changed (bits: what no sequence owns is NaN)
    kb[pg, :, off], vb[pg, :, off] = b.kp[pg, :, off], b.vp[pg, :, off]
    bits = torch.int32 if dtype == "f32" else torch.int16
    assert torch.equal(kb.contiguous().view(bits), b.kp.contiguous().view(bits))
    assert torch.equal(vb.contiguous().view(bits), b.vp.contiguous().view(bits))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,kv,group,hd,page,layout", [
    ([(0, 1)], 1, 1, 8, 1, "heads"), ([(1023, 1)] * 5, 12, 1, 64, 16, "heads"), ([(3, 130), (0, 7), (77, 0), (9, 1)], 2, 3, 48, 7, "tokens"),
    ([(50000, 3)], 5, 8, 128, 64, "heads"), ([(10, 40)], 3, 1, 120, 24, "tokens"), ([(0, 33)], 40, 1, 16, 16, "heads")])
def test_append_matches_64_bits(ptlib, dtype, lens, kv, group, hd, page, layout):
    append_case(ptlib, dtype, lens, kv, group, hd, page, layout)


def test_append_without_rotation_and_in_place(ptlib):
    append_case(ptlib, "bf16", [(4, 9), (0, 2)], 2, 2, 64, 16, rope=False)
    append_case(ptlib, "f32", [(4, 9), (0, 2)], 2, 2, 64, 16, in_place=True)


def test_append_skips_padding_and_reports_bad_rows(ptlib):
    b = Batch([(0, 6)], 2, 1, 16, 4, "f32")
    kp, vp = b.kp.clone(), b.vp.clone()
    x = torch.randn(6, 32, device="cuda")
    out = torch.full_like(x, 5.0)
    table = torch.ones(8, 8, 2, device="cuda")
    positions = ints([-1, 0, 1, 8, -3, 2])          # padding, ok, ok, past the table, negative, ok
    slots = ints([3, -1, b.n_pages * 4, 1, 2, 0])   # ignored, not stored, out of range, -, -, ok
    a = api.ptc_append_args(b.cache(), 6, 2, x.data_ptr(), x.data_ptr(), x.data_ptr(), 32, 32, 32, positions.data_ptr(),
                            slots.data_ptr(), table.data_ptr(), 8, out.data_ptr(), 32, b.err.data_ptr())
    assert ptlib.ptc_kv_append(a, stream()) == 0
    torch.cuda.synchronize()
    assert int(b.err) == api.PTC_SERVE_ERR_INDEX
    assert [bool((out[t] == 5.0).all()) for t in range(6)] == [True, False, False, True, True, False]
    assert torch.equal(b.vp[0, :, 0].reshape(-1), x[5])
    vp[0, :, 0], kp[0, :, 0] = b.vp[0, :, 0], b.kp[0, :, 0]
    assert torch.equal(vp.view(torch.int32), b.vp.view(torch.int32)) and torch.equal(kp.view(torch.int32), b.kp.view(torch.int32))


def test_rope_table_is_the_decoders(ptlib):
    n, hd = 300, 48
    t = torch.empty(n, hd // 2, 2, device="cuda")
    assert ptlib.ptc_rope_table(t.data_ptr(), n, hd, stream()) == 0
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
    want = torch.stack([ang.cos(), ang.sin()], -1)
    # the reference's polynomials: 32-bit angles (up to 300 * 2^-22) and 7th to 9th degree series (2e-4 at the quarter turn)
    assert float((t.double() - want).abs().max()) < 300 * 2.0 ** -22 + 2e-4


# ---- paged attention ---------------------------------------------------------------

RAGGED = [(0, 1), (5, 1), (130, 70), (0, 0), (17, 0), (0, 129), (511, 1), (64, 64), (1000, 33)]
ATTN = [   # lens, kv heads, group, hd, page, window
    ([(0, 1)], 1, 1, 8, 1, 0),
    ([(1023, 1)], 12, 1, 64, 16, 0),
    ([(1, 1), (16, 1), (63, 1), (64, 1), (255, 1), (3000, 1)], 2, 4, 128, 16, 0),
    ([(40000, 1)], 2, 8, 64, 64, 0),
    ([(700, 5), (3, 4), (0, 6)], 3, 3, 80, 7, 0),
    (RAGGED, 2, 1, 48, 16, 0),
    (RAGGED, 1, 4, 64, 24, 0),
    (RAGGED, 2, 3, 128, 1000, 0),
    (RAGGED, 1, 7, 96, 3, 100),
    (RAGGED, 4, 2, 16, 16, 1),
    ([(0, 700)], 1, 2, 128, 64, 0),
    ([(5000, 300)], 2, 4, 128, 128, 0),
    ([(3000, 257)], 1, 1, 64, 16, 700),
    ([(0, 1300), (10, 1)], 1, 1, 56, 32, 0),
    ([(9, 1)] * 200 + [(0, 3)] * 101, 2, 2, 32, 8, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention_matches_64_bits(ptlib, dtype, case):
    lens, kv, group, hd, page, window = ATTN[case]
    b = Batch(lens, kv, group, hd, page, dtype, seed=case, layout="tokens" if case % 3 == 2 else "heads")
    want, bound = b.reference(window)
    got = b.attend(ptlib, window)
    assert int(b.err) == 0
    assert bool((got[b.total:] == 7.0).all())   # rows behind the last sequence
    check(got[: b.total], want, bound)
    assert not bool(b.work[:4096].any())        # the flags are zero again
    assert torch.equal(b.attend(ptlib, window), got)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_result_does_not_hang_on_max_q(ptlib, dtype):
    b = Batch([(300, 40), (20, 1), (0, 5)], 2, 2, 64, 16, dtype)
    want, bound = b.reference()
    for m in (0, 1, 40, 100000):
        check(b.attend(ptlib, max_q=m)[: b.total], want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread,scale", [(30.0, None), (1e-3, None), (1.0, -0.2), (1.0, 0.0)])
def test_attention_of_peaked_flat_and_negative_scores(ptlib, dtype, spread, scale):
    b = Batch([(900, 1), (300, 150)], 2, 2, 64, 16, dtype, spread=spread)
    want, bound = b.reference(scale=scale)
    check(b.attend(ptlib, scale=scale)[: b.total], want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_without_a_position_are_zero(ptlib, dtype):
    b = Batch([(-3, 5), (-140, 140), (-2, 2), (4, 2)], 2, 2, 32, 8, dtype)   # kv_len 2, 0, 0, 6
    want, bound = b.reference()
    got = b.attend(ptlib)
    check(got[: b.total], want, bound)
    assert not bool(got[:3].any()) and not bool(got[5:147].any())
    assert int(b.err) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [6, 140])
def test_largest_window_and_longest_length(ptlib, dtype, new):
    b = Batch([(-3, new), (40, new), (20, new)], 2, 2, 32, 8, dtype)
    want, bound = b.reference()
    check(b.attend(ptlib, window=2 ** 31 - 1)[: b.total], want, bound)
    assert int(b.err) == 0
    # a length that no table holds: what the table holds is used (all of it behind the other rows' positions here)
    b.kv_len[1] = 2 ** 31 - 1
    got = b.attend(ptlib, window=0)
    assert int(b.err) & api.PTC_SERVE_ERR_LENGTH
    for r in (0, 2):
        check(got[r * new:(r + 1) * new], want[r * new:(r + 1) * new], bound[r * new:(r + 1) * new])


FIRST_CALL = """
import sys, torch
sys.path[:0] = [%r, %r]
import pitorch_b200
from pitorch_b200 import api
from serve_ref import Batch, check, stream
L = pitorch_b200.lib()
b = Batch([(300, %d), (7, %d)], 2, 2, 64, 16, %r)
out = torch.zeros_like(b.q)
args = b.attn_args(out)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    assert L.ptc_paged_attention(args, stream()) == 0
g.replay()
torch.cuda.synchronize()
check(out[: b.total], *b.reference())
"""


@pytest.mark.parametrize("dtype,new", [("f32", 1), ("f32", 60), ("bf16", 1), ("bf16", 60)])
def test_first_call_of_a_process_may_be_captured(ptlib, dtype, new):
    here = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALL % (os.path.dirname(here), here, new, new, dtype)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 150])
def test_bad_pages_and_lengths_are_left_out(ptlib, dtype, new):
    b = Batch([(100, new), (100, new), (100, new), (100, new)], 2, 2, 64, 16, dtype)
    want, bound = b.reference()
    b.table[1, 2] = b.n_pages       # positions 32..47 left out
    b.table[1, 3] = -1              # and 48..63
    b.kv_len[2] = b.cols * 16 + 5   # longer than the table row
    got = b.attend(ptlib)
    assert int(b.err) == api.PTC_SERVE_ERR_INDEX | api.PTC_SERVE_ERR_LENGTH
    for r in (0, 3):
        check(got[r * new:(r + 1) * new], want[r * new:(r + 1) * new], bound[r * new:(r + 1) * new])
    # sequence 1 as if it were without those positions
    pages = b.table[1].clamp(0, b.n_pages - 1).long()
    rows = lambda c: c[pages].double().transpose(0, 1).reshape(b.kv, -1, 64)[:, : 100 + new]  # noqa: E731
    key, val = rows(b.kp), rows(b.vp).clone()
    val[:, 32:64] = 0
    q = b.q[new:2 * new].double().reshape(new, 2, 2, 64)
    s = torch.einsum("qkgd,ktd->kgqt", q, key) / 8
    t = torch.arange(100 + new, device="cuda")
    hide = (t[None] > 100 + torch.arange(new, device="cuda")[:, None]) | ((t >= 32) & (t < 64))[None]
    o = torch.einsum("kgqt,ktd->qkgd", torch.softmax(s.masked_fill(hide, -math.inf), -1), val).reshape(new, 4, 64)
    check(got[new:2 * new], o, bound[:new].amax() * 4)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_with_inconsistent_starts(ptlib, dtype):
    b = Batch([(50, 3), (50, 3), (50, 3)], 2, 1, 32, 8, dtype)
    want, bound = b.reference()
    b.q_start.copy_(ints([0, 3, 2, b.q.shape[0] + 1]))   # falls, then passes the rows
    got = b.attend(ptlib)
    assert int(b.err) == api.PTC_SERVE_ERR_LENGTH
    check(got[:3], want[:3], bound[:3])
    assert bool((got[3:] == 7.0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_strides_and_a_contiguous_cache(ptlib, dtype):
    """q as part of a packed row, out with a longer row, K and V interleaved, one page per sequence."""
    b = Batch([(37, 3), (90, 131)], 2, 2, 64, 256, dtype)
    want, bound = b.reference()
    both = torch.empty(b.n_pages, 2, 256, 2, 64, dtype=DT[dtype], device="cuda")
    both[:, :, :, 0], both[:, :, :, 1] = b.kp, b.vp
    wide = torch.randn(b.total, 4 * 64 + 200, device="cuda").to(DT[dtype])
    wide[:, 8: 8 + 256] = b.q[: b.total].reshape(b.total, 256)
    out = torch.full((b.total, 256 + 24), 3.0, dtype=DT[dtype], device="cuda")
    a = b.attn_args(out, q=wide)
    a.q, a.n_tokens = wide.data_ptr() + 8 * wide.element_size(), b.total
    a.cache.k, a.cache.v = both.data_ptr(), both.data_ptr() + 64 * both.element_size()
    a.cache.page_stride, a.cache.head_stride, a.cache.token_stride = 2 * 256 * 128, 256 * 128, 128
    assert ptlib.ptc_paged_attention(a, stream()) == 0
    torch.cuda.synchronize()
    check(out[:, :256].reshape(b.total, 4, 64), want, bound)
    assert bool((out[:, 256:] == 3.0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 140])
def test_attention_offsets_past_32_bits(ptlib, dtype, new):
    b = Batch([(60, new)], 1, 1, 64, 128, dtype)
    want, bound = b.reference()
    far = (1 << 31) + 64   # elements between pages
    buf = {}
    for name, c in (("k", b.kp), ("v", b.vp)):
        buf[name] = torch.empty((b.n_pages - 1) * far + 128 * 64, dtype=DT[dtype], device="cuda")
        for pg in range(b.n_pages):
            buf[name][pg * far: pg * far + 128 * 64] = c[pg].reshape(-1)
    out = torch.empty_like(b.q)
    a = b.attn_args(out)
    a.cache.k, a.cache.v, a.cache.page_stride = buf["k"].data_ptr(), buf["v"].data_ptr(), far
    assert ptlib.ptc_paged_attention(a, stream()) == 0
    torch.cuda.synchronize()
    check(out[: b.total], want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_captured_and_replayed(ptlib, dtype):
    """One graph, replayed after the lengths, the table and the rows changed; two graphs with workspaces of their own."""
    lens = [(900, 1), (64, 1), (5, 1)]
    b, c = (Batch(lens, 2, 2, 64, 16, dtype, seed=s) for s in (1, 2))
    outs = [torch.zeros_like(x.q) for x in (b, c)]
    for x, o in zip((b, c), outs):   # first calls outside of the captures
        assert ptlib.ptc_paged_attention(x.attn_args(o), stream()) == 0
    graphs = []
    for x, o in zip((b, c), outs):
        g = torch.cuda.CUDAGraph()
        args = x.attn_args(o)
        with torch.cuda.graph(g):
            assert ptlib.ptc_paged_attention(args, stream()) == 0
        graphs.append(g)
    b.kv_len.copy_(ints([400, 2, 6]))
    b.lens = [(399, 1), (1, 1), (5, 1)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    for x, o in zip((b, c), outs):
        check(o[: x.total], *x.reference())


# ---- sampling ---------------------------------------------------------------------------

def run_sample(L, x, temperature=None, top_k=None, top_p=None, min_p=None, u=None, vocab=None):
    rows, vocab = x.shape[0], x.shape[1] if vocab is None else vocab
    dev = lambda v, dt: None if v is None else torch.tensor(v, dtype=dt, device="cuda")  # noqa: E731
    t = [dev(temperature, torch.float32), dev(top_k, torch.int32), dev(top_p, torch.float32), dev(min_p, torch.float32),
         dev([0.5] * rows if u is None else u, torch.float32)]
    out = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda")
    code = {v: CODE[k] for k, v in DT.items()}[x.dtype]
    a = api.ptc_sample_args(code, rows, vocab, x.data_ptr(), x.stride(0), *(None if v is None else v.data_ptr() for v in t),
                            out.data_ptr())
    assert L.ptc_sample_tokens(a, stream()) == 0
    torch.cuda.synchronize()
    assert int(out[-1]) == -5
    return out[:-1].tolist()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 1024, 4097, 32000, 50257, 131071, 262144])
def test_sampling_matches_the_definition(ptlib, dtype, vocab):
    g = torch.Generator(device="cuda")
    g.manual_seed(vocab)
    rows = 12 if vocab < 100000 else 6
    wide = torch.randn(rows, vocab + 3, generator=g, device="cuda").mul_(2.5).to(DT[dtype])
    x = wide[:, 1: 1 + vocab]   # rows at odd addresses
    if vocab > 100:
        x[2, vocab // 10:] = -math.inf
        x[3, 5] = 40.0
    r = random.Random(vocab)
    temp = [r.choice([0.0, 0.3, 0.8, 1.0, 1.7]) for _ in range(rows)]
    k = [r.choice([0, 1, 3, 40, vocab, vocab // 2 + 1]) for _ in range(rows)]
    p = [r.choice([1.0, 0.9, 0.5, 0.99, 1e-6]) for _ in range(rows)]
    mp = [r.choice([0.0, 0.0, 0.1, 1.0]) for _ in range(rows)]
    u = [r.choice([0.0, r.random(), r.random(), 1 - 2.0 ** -24]) for _ in range(rows)]
    f = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    got = run_sample(ptlib, x, temp, k, p, mp, u)
    want = [sample_ref(x[i], f(temp[i]), k[i], f(p[i]), f(mp[i]), f(u[i])) for i in range(rows)]
    assert got == want


@pytest.mark.parametrize("vocab", [3, 300, 32000, 140001])
def test_sampling_ties_go_by_index(ptlib, vocab):
    """Equal logits: the rules keep the lowest indexes, and -0 equals 0."""
    x = torch.zeros(6, vocab, device="cuda")
    x[:, ::2] = -0.0
    n = vocab // 3
    got = run_sample(ptlib, x, [1.0, 1.0, 1.0, 0.0, 1.0, 1.0], [n, 0, 0, 0, 0, 1], [1.0, 0.25, 1.0, 1.0, 0.0, 1.0],
                     [0.0, 0.0, 1.0, 0.0, 0.0, 0.0], [0.999, 0.999, 0.5, 0.9, 0.9, 0.9])
    want = [sample_ref(x[0], 1.0, n, u=float(torch.tensor(0.999))), sample_ref(x[0], 1.0, 0, 0.25, u=float(torch.tensor(0.999))),
            sample_ref(x[0], u=0.5), 0, 0, 0]
    assert got == want


def test_sampling_two_levels_of_ties(ptlib):
    x = torch.full((3, 5000), -math.log(2.0), device="cuda")
    x[:, 4990:] = 0.0   # ten of weight 1, the others of weight 1/2
    got = run_sample(ptlib, x, [1.0] * 3, [1000, 15, 0], [1.0, 1.0, 0.01], None, [0.01, 0.999, 0.99])
    assert got == [sample_ref(x[0], 1.0, 1000, u=float(torch.tensor(0.01))), 4999,
                   sample_ref(x[0], 1.0, 0, float(torch.tensor(0.01)), u=float(torch.tensor(0.99)))]


def test_sampling_infinities_and_nan(ptlib):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[nan, -inf, -inf, nan, -inf], [nan, 1.0, -inf, 1.0, nan], [inf, 3.0, inf, nan, 2.0],
                      [-inf, -inf, -3e38, -inf, -inf], [3e38, -3e38, 3e38, 0.0, nan], [-inf, nan, 5.0, 5.0, 4.0]], device="cuda")
    assert run_sample(ptlib, x, [1.0] * 6, [0, 0, 0, 0, 3, 0], [1.0, 0.9, 1.0, 1.0, 1.0, 1.0], None,
                      [0.5, 0.75, 0.75, 0.99, 0.75, 0.0]) == [-1, 3, 2, 2, 2, 2]
    assert run_sample(ptlib, x, [0.0] * 6) == [-1, 1, 0, 2, 0, 2]
    assert run_sample(ptlib, x) == [-1, 3, 2, 2, 2, 3]


def test_sampling_defaults_and_limits_of_u(ptlib):
    x = torch.randn(4, 999, device="cuda")
    want = [sample_ref(x[i], u=0.5) for i in range(4)]
    assert run_sample(ptlib, x) == want
    # u outside [0, 1) is taken as the nearest kept token
    got = run_sample(ptlib, x, [1.0] * 4, [2] * 4, None, None, [1.0, -1.0, 5.0, math.nan])
    for i, t in enumerate(got):
        two = sorted(torch.topk(x[i], 2).indices.tolist())
        assert t == two[1 if i in (0, 2) else 0]


def test_sampling_frequencies(ptlib):
    """Many draws of one row follow its weights: each count within 6 standard deviations."""
    n = 20000
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device="cuda").repeat(n, 1)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    got = torch.tensor(run_sample(ptlib, x, u=torch.rand(n, generator=g, device="cuda").tolist()))
    p = torch.softmax(x[0].double().cpu(), 0)
    c = torch.bincount(got, minlength=5).double()
    assert bool(((c - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all())


# ---- the operators together ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_steps_of_a_batch(ptlib, dtype):
    """Prompts of three requests, then single tokens: pages, append, attention and sampling as a server runs them,
    one captured step replayed; against a plain contiguous computation of the same steps."""
    L, dt = ptlib, DT[dtype]
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    n, kv, heads, hd, page, cols, n_pages, V, rows = 3, 2, 4, 32, 8, 16, 64, 512, 96
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    emb, w_qkv, w_cls = rand(V, 64).to(dt), (rand(64, (heads + 2 * kv) * hd) / 8).to(dt), (rand(heads * hd, V) / 6).to(dt)
    kc, vc = torch.full((2, n_pages, kv, page, hd), math.nan, dtype=dt, device="cuda")
    rope = torch.empty(cols * page, hd // 2, 2, device="cuda")
    assert L.ptc_rope_table(rope.data_ptr(), cols * page, hd, stream()) == 0
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    free = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    past, new, table, kv_len, q_start = i32(n), i32(n), i32(n, cols), i32(n), i32(n + 1)
    slots, positions, used, err = i32(rows), i32(rows), i32(1), i32(1)
    tokens, u, last = i32(rows), torch.zeros(n, device="cuda"), i32(n)
    x = torch.zeros(rows, (heads + 2 * kv) * hd, dtype=dt, device="cuda")
    q, o = torch.zeros(rows, heads * hd, dtype=dt, device="cuda"), torch.zeros(rows, heads * hd, dtype=dt, device="cuda")
    logits, nxt = torch.zeros(n, V, device="cuda"), i32(n)
    temp, top_p = torch.full((n,), 0.9, device="cuda"), torch.full((n,), 0.95, device="cuda")
    work = torch.zeros(api.PTC_ATTN_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    cache = api.ptc_paged_cache(kc.data_ptr(), vc.data_ptr(), CODE[dtype], n_pages, page, kv, hd, kv * page * hd, page * hd, hd)
    e, row = x.element_size(), x.shape[1]
    taken = 0

    def step(max_q, live):
        s = stream()
        f = free[taken:]
        assert L.ptc_plan_pages(api.ptc_pages_args(
            n, page, cols, rows, f.shape[0], n_pages, past.data_ptr(), new.data_ptr(), f.data_ptr(), table.data_ptr(),
            kv_len.data_ptr(), q_start.data_ptr(), slots.data_ptr(), positions.data_ptr(), used.data_ptr(), err.data_ptr()), s) == 0
        torch.matmul(emb[tokens[:live].long()], w_qkv, out=x[:live])
        p = x.data_ptr()
        assert L.ptc_kv_append(api.ptc_append_args(
            cache, rows, heads, p, p + heads * hd * e, p + (heads + kv) * hd * e, row, row, row, positions.data_ptr(),
            slots.data_ptr(), rope.data_ptr(), cols * page, q.data_ptr(), heads * hd, err.data_ptr()), s) == 0
        assert L.ptc_paged_attention(api.ptc_attn_args(
            cache, n, rows, heads, max_q, cols, 0, 1 / math.sqrt(hd), q.data_ptr(), heads * hd, o.data_ptr(), heads * hd,
            table.data_ptr(), kv_len.data_ptr(), q_start.data_ptr(), work.data_ptr(), work.numel(), err.data_ptr()), s) == 0
        last.copy_(q_start[1:] - 1)
        logits.copy_(o[last.long()].float() @ w_cls.float())
        assert L.ptc_sample_tokens(api.ptc_sample_args(
            api.PTC_F32, n, V, logits.data_ptr(), V, temp.data_ptr(), None, top_p.data_ptr(), None, u.data_ptr(), nxt.data_ptr()), s) == 0

    prompts = [list(range(3, 40)), [7], list(range(100, 150))]
    hist = [list(p) for p in prompts]
    tokens[: sum(map(len, prompts))] = ints(sum(prompts, []))
    new.copy_(ints([len(p) for p in prompts]))
    graph = None
    for it in range(12):
        u.copy_(torch.rand(n, generator=g, device="cuda"))
        if it == 0:
            step(64, sum(map(len, prompts)))
        elif graph is None:
            # a step's free list starts where the last one ended; decode steps take theirs from a fixed tail
            torch.cuda.synchronize()
            taken = int(used)
            graph = torch.cuda.CUDAGraph()
            step(1, n)
            with torch.cuda.graph(graph):
                step(1, n)
        else:
            free[taken:] = torch.roll(free[taken:], -int(used))
            graph.replay()
        torch.cuda.synchronize()
        assert int(err) == 0
        # the same step over whole contiguous sequences, in 64 bits from the stored roundings
        for r in range(n):
            h = torch.tensor(hist[r], device="cuda")
            y = (emb[h] @ w_qkv).double().reshape(len(hist[r]), -1, hd)
            cs = rope[: len(hist[r])].double()[:, None]
            t = y.clone()
            t[..., 0::2] = y[..., 0::2] * cs[..., 0] - y[..., 1::2] * cs[..., 1]
            t[..., 1::2] = y[..., 0::2] * cs[..., 1] + y[..., 1::2] * cs[..., 0]
            qq, kk, vv = t[-1, :heads], t[:, heads:heads + kv], y[:, heads + kv:]
            s = torch.einsum("kgd,tkd->kgt", qq.reshape(kv, heads // kv, hd), kk) / math.sqrt(hd)
            a = torch.einsum("kgt,tkd->kgd", torch.softmax(s, -1), vv).reshape(-1)
            got = o[int(last[r])].double()
            # q, k, v, probabilities and the result are each rounded to the type: a few half steps of the values
            # (the 32-bit products of the plain side may also round differently from row to row)
            tol = 12 * HALF[dtype] * float(vv.abs().max()) * (1 + float(s.abs().max())) + 1e-4
            assert float((got - a).abs().max()) <= tol
            assert int(nxt[r]) == sample_ref(logits[r], float(temp[r]), 0, float(top_p[r]), 0.0, float(u[r]))
            hist[r].append(int(nxt[r]))
        past.copy_(kv_len)
        new.fill_(1)
        tokens[:n] = nxt
