"""What the serving operators refuse before they touch the GPU: each bad
argument gives -1, a message that names the call, and nothing else."""
import ctypes as C

import pytest

from pitorch_b200 import api

A = 0x10000   # stands for device addresses: a refused call reads none of them


def cache(**kw):
    c = api.ptc_paged_cache(A, A, api.PTC_BF16, 4, 16, 2, 64, 2048, 1024, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def made(cls, base, kw):
    a = cls(*base)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def pages(**kw):
    return made(api.ptc_pages_args, (2, 16, 4, 8, 4, 8) + (A,) * 10, kw)


def append(**kw):
    return made(api.ptc_append_args, (cache(**kw.pop("cache", {})), 3, 4, A, A, A, 256, 128, 128, A, A, A, 9, A, 256, A), kw)


def attn(**kw):
    return made(api.ptc_attn_args, (cache(**kw.pop("cache", {})), 2, 3, 4, 1, 4, 0, 0.125, A, 256, A, 256, A, A, A, A,
                                    api.PTC_ATTN_WORKSPACE_BYTES, A), kw)


def sample(**kw):
    return made(api.ptc_sample_args, (api.PTC_F32, 2, 100, A, 100, A, A, A, A, A, A), kw)


BAD_CACHE = [dict(dtype=3), dict(dtype=-1), dict(k=None), dict(v=A + 8), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0),
             dict(head_dim=12), dict(head_dim=136), dict(head_dim=0), dict(page_stride=2044), dict(head_stride=-8),
             dict(token_stride=4), dict(n_pages=1 << 20, page_size=1 << 12)]
BAD = ([("ptc_plan_pages", pages, kw) for kw in (
        dict(n_seqs=-1), dict(n_seqs=4097), dict(page_size=0), dict(max_pages=0), dict(max_tokens=-1), dict(n_free=-1),
        dict(n_pages=0), dict(n_pages=1 << 28), dict(past_len=None), dict(new_len=None), dict(free_pages=None),
        dict(page_table=None), dict(kv_len=None), dict(q_start=None), dict(slots=None), dict(positions=None), dict(pages_used=None))]
       + [("ptc_kv_append", append, dict(cache=c)) for c in BAD_CACHE]
       + [("ptc_kv_append", append, kw) for kw in (
           dict(n_tokens=-1), dict(n_heads=0), dict(n_pos=0), dict(q=None), dict(k=A + 2), dict(v=None), dict(positions=None),
           dict(slots=None), dict(q_out=None), dict(q_out=A + 8), dict(rope=A + 4), dict(q_stride=252), dict(k_stride=120),
           dict(v_stride=132), dict(q_out_stride=248))]
       + [("ptc_paged_attention", attn, dict(cache=c)) for c in BAD_CACHE]
       + [("ptc_paged_attention", attn, kw) for kw in (
           dict(n_seqs=-1), dict(n_seqs=4097), dict(n_tokens=-1), dict(n_tokens=(1 << 28) + 1), dict(n_heads=0), dict(n_heads=3), dict(max_q=-1), dict(max_pages=0), dict(window=-1),
           dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(q=A + 8), dict(q_stride=248), dict(q_stride=257),
           dict(out=None), dict(out_stride=128), dict(page_table=None), dict(kv_len=None), dict(q_start=None), dict(workspace=None),
           dict(workspace=A + 16), dict(workspace_bytes=api.PTC_ATTN_WORKSPACE_BYTES - 1))]
       + [("ptc_sample_tokens", sample, kw) for kw in (
           dict(dtype=7), dict(rows=-1), dict(vocab=0), dict(vocab=262145, stride=262145), dict(stride=99), dict(logits=None),
           dict(logits=A + 2), dict(u=None), dict(tokens=None))])


@pytest.mark.parametrize("name,make,kw", BAD, ids=lambda v: v if isinstance(v, str) else str(v) if isinstance(v, dict) else "")
def test_refusals(ptlib, capfd, name, make, kw):
    assert getattr(ptlib, name)(make(**kw), None) == -1
    assert name in capfd.readouterr().err


@pytest.mark.parametrize("name", ["ptc_plan_pages", "ptc_kv_append", "ptc_paged_attention", "ptc_sample_tokens"])
def test_no_arguments(ptlib, name):
    assert getattr(ptlib, name)(None, None) == -1


def test_empty_calls_need_no_gpu(ptlib):
    assert ptlib.ptc_kv_append(append(n_tokens=0, q=None, k=None, v=None, q_out=None, positions=None, slots=None), None) == 0
    assert ptlib.ptc_paged_attention(attn(n_tokens=0, q=None, out=None), None) == 0
    assert ptlib.ptc_paged_attention(attn(n_seqs=0, page_table=None, kv_len=None), None) == 0
    assert ptlib.ptc_sample_tokens(sample(rows=0, logits=None, u=None, tokens=None), None) == 0


def test_rope_table_refusals(ptlib):
    for args in ((None, 4, 8), (A + 4, 4, 8), (A, 0, 8), (A, 4, 7), (A, 4, 0), (A, 1 << 30, 8)):
        assert ptlib.ptc_rope_table(*args, None) == -1


def test_struct_layouts_match_c(tmp_path):
    import os
    import subprocess
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    names = ("ptc_pages_args", "ptc_paged_cache", "ptc_append_args", "ptc_attn_args", "ptc_sample_args")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "ptc_serve.h"', "int main(void) {"]
    for n in names:
        lines.append(f'  printf("{n} %zu\\n", sizeof({n}));')
        for f, _ in getattr(api, n)._fields_:
            lines.append(f'  printf("{n}.{f} %zu\\n", offsetof({n}, {f}));')
    for k in ("PTC_ATTN_WORKSPACE_BYTES",):
        lines.append(f'  printf("{k} %zu\\n", (size_t){k});')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "\n  return 0; }\n")
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(tmp_path / "layout")], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                                         check=True).stdout.split("\n") if l)
    for n in names:
        cls = getattr(api, n)
        assert int(got[n]) == C.sizeof(cls), n
        for f, _ in cls._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(cls, f).offset, (n, f)
    assert int(got["PTC_ATTN_WORKSPACE_BYTES"]) == api.PTC_ATTN_WORKSPACE_BYTES
