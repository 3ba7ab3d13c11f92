"""Measured cases of the batched-serving operators (include/ptc_serve.h).

Four operators that one serving step runs in this order: the page tables and
slot maps of a batch of sequences (``pages``), the rotary write of new keys
and values into a paged cache (``append``), attention of the new tokens over
that cache (``attend``), and sampling of the next tokens (``sample``). With
``own`` false, ``run`` computes them in elementary torch operations; with it
true it makes the library's calls.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}   # PTC_F32, PTC_F16, PTC_BF16
ROPE_BASE = 10000.0


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # one decode step of 64 running requests: every one gets one token
        {"name": "pages decode 64", "op": "pages", "n": 64, "new": 1, "ragged": 0, "past": 4096, "page": 16, "lens": 1},
        # a step that admits chunks of many requests at once
        {"name": "pages chunks 2047", "op": "pages", "n": 2047, "new": 64, "ragged": 1, "past": 16384, "page": 16,
         "lens": 2},
        # the keys and values of 64 decoding requests, the 110M model's heads
        {"name": "append decode 64 f32", "op": "append", "n": 64, "new": 1, "ragged": 0, "past": 1023, "page": 16,
         "lens": 3, "dtype": "f32", "kv": 12, "group": 1, "hd": 64},
        # prompts of several requests, grouped heads, an odd number of tokens
        {"name": "append prompts 8191 bf16", "op": "append", "n": 7, "new": 1171, "ragged": 1, "past": 3000,
         "page": 64, "lens": 4, "dtype": "bf16", "kv": 8, "group": 4, "hd": 128},
        # one token of one request over a full 1024-position cache, the 110M model's heads: latency
        {"name": "attend token f32", "op": "attend", "n": 1, "new": 1, "ragged": 0, "past": 1023, "page": 16,
         "lens": 5, "dtype": "f32", "kv": 12, "group": 1, "hd": 64, "window": 0},
        # a decode step of 64 requests of very different lengths
        {"name": "attend decode 64 bf16", "op": "attend", "n": 64, "new": 1, "ragged": 0, "past": 8191, "page": 16,
         "lens": 6, "dtype": "bf16", "kv": 8, "group": 4, "hd": 128, "window": 0},
        # prompts of the 15M model, 256 positions at most
        {"name": "attend prompts f32", "op": "attend", "n": 9, "new": 255, "ragged": 1, "past": 1, "page": 16,
         "lens": 7, "dtype": "f32", "kv": 6, "group": 1, "hd": 48, "window": 0},
        # decoding requests and prompt chunks in one step, a sliding window
        {"name": "attend mixed f16", "op": "attend", "n": 17, "new": 301, "ragged": 1, "past": 1500, "page": 24,
         "lens": 8, "dtype": "f16", "kv": 4, "group": 4, "hd": 64, "window": 512},
        # a chunk of a long prompt behind what the cache holds already
        {"name": "attend chunk 4096 bf16", "op": "attend", "n": 1, "new": 4096, "ragged": 0, "past": 12288,
         "page": 64, "lens": 9, "dtype": "bf16", "kv": 8, "group": 4, "hd": 128, "window": 0},
        # one request's next token, the 32000-token vocabulary: latency
        {"name": "sample 1x32000 f32", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "f32", "mix": 1},
        # a decode batch with mixed settings
        {"name": "sample 64x32000 f32", "op": "sample", "rows": 64, "vocab": 32000, "dtype": "f32", "mix": 3},
        # a large batch over a large, odd vocabulary
        {"name": "sample 256x131071 bf16", "op": "sample", "rows": 256, "vocab": 131071, "dtype": "bf16", "mix": 3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "append", "attend", "attend", "sample"])
    page = rng.choice([1, 8, 16, 24, 32, 64, 128])
    base = {"op": op, "lens": rng.randrange(1 << 30), "page": page}
    if op == "pages":
        new = _log(rng, 1, 512)
        n = _log(rng, 1, min(4096, 131072 // new))
        past = _log(rng, 1, max(1, min(16384, 512 * page, (1 << 25) // n)))
        return dict(base, n=n, new=new, ragged=rng.randrange(2), past=past)
    if op == "sample":
        vocab = _log(rng, 100, 200000)
        rows = _log(rng, 1, min(512, 33000000 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
                "mix": rng.randrange(4), "lens": base["lens"]}
    base.update(dtype=rng.choice(["f32", "bf16", "f16"]), kv=rng.randint(1, 12), group=rng.choice([1, 1, 2, 3, 4, 6, 8]),
                hd=rng.choice([32, 48, 64, 80, 96, 128]))
    width = base["kv"] * base["group"] * base["hd"]
    if op == "append":
        new = _log(rng, 1, 4096)
        n = _log(rng, 1, max(1, min(256, 8192 // new, (1 << 26) // (new * width))))
        return dict(base, n=n, new=new, ragged=rng.randrange(2), past=_log(rng, 1, 4096))
    new = rng.choice([1, _log(rng, 2, 16), _log(rng, 16, 2048)])
    while True:  # the plain form's padded scores and gathered keys have to fit, and the work stays under the largest
        n, past = _log(rng, 1, 256), _log(rng, 1, 16384)
        if (n * base["kv"] * base["group"] * new * (past + new) <= 4e8 and n * base["kv"] * (past + new) * base["hd"] <= 2.5e8):
            break
        new = max(1, new // 2)
    return dict(base, n=n, new=new, ragged=rng.randrange(2), past=past, window=rng.choice([0, 0, 0, _log(rng, 8, 2048)]))


def _lens(case):
    """(past, new) of each sequence: at most ``past`` and ``new``, the first sequence at both. A ragged batch has
    single tokens, chunks, and a few sequences with nothing new or nothing cached."""
    r = random.Random(case["lens"])
    past, new = [], []
    for i in range(case["n"]):
        past.append(case["past"] if i == 0 else r.randint(0, case["past"]))
        if case["ragged"] and i > 0:
            q = r.choice([1, r.randint(1, case["new"]), r.randint(1, case["new"])])
            if r.random() < 0.05:
                q = 0
            if r.random() < 0.1:
                past[-1] = 0
            new.append(q)
        else:
            new.append(case["new"])
    return past, new


def _pages_needed(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["op"] == "sample":
        e = 4 if case["dtype"] == "f32" else 2
        # each logit read once, one subtraction, one exponential and one addition
        return {"bytes": case["rows"] * (case["vocab"] * e + 24), "flops": 3 * case["rows"] * case["vocab"]}
    past, new = _lens(case)
    total = sum(new)
    if case["op"] == "pages":
        fresh = sum(_pages_needed(p + q, case["page"]) - _pages_needed(p, case["page"]) for p, q in zip(past, new))
        # lengths in; lengths, starts, new table entries, slots and positions out
        return {"bytes": 4 * (4 * case["n"] + 1 + 2 * fresh + 2 * total), "flops": 2 * total}
    e = 4 if case["dtype"] == "f32" else 2
    kv, group, hd = case["kv"], case["group"], case["hd"]
    if case["op"] == "append":
        rot = total * kv * (group + 1) * hd   # rotated values
        # queries, keys and values in and out once, the table rows of the positions, slots and positions
        return {"bytes": 2 * e * total * kv * (group + 2) * hd + total * (4 * hd + 8), "flops": 3 * rot}
    w = case["window"]
    pairs = cached = 0
    for p, q in zip(past, new):
        if q:
            lo = max(0, p + 1 - w) if w else 0
            cached += p + q - lo
            if w:
                pairs += sum(min(p + j + 1, w) for j in range(q))
            else:
                pairs += q * p + q * (q + 1) // 2
    return {"bytes": e * hd * (2 * cached * kv + 2 * total * kv * group), "flops": 4 * pairs * kv * group * hd}


# ---- what a program has in hand before the call -------------------------------

def _ints(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _layout(case, seed):
    """A batch's lengths and a page table over shuffled pages, as a server has them."""
    past, new = _lens(case)
    page, n = case["page"], case["n"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    need = _ints([_pages_needed(p + q, page) for p, q in zip(past, new)])
    cols = max(1, int(need.max()))
    n_pages = int(need.sum()) + 3
    free = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(cols, device="cuda")
    held = col[None, :] < need[:, None]
    table = torch.where(held, free[(first[:, None] + col[None, :]).clamp(max=n_pages - 1)], -1).to(torch.int32)
    past_t, new_t = _ints(past), _ints(new)
    q_start = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    q_start[1:] = torch.cumsum(new_t, 0)
    return past_t, new_t, table.contiguous(), q_start, n_pages, free, g


def _tokens(past, q_start, total):
    """The sequence and the position of each new token."""
    t = torch.arange(total, device="cuda")
    seq = torch.searchsorted(q_start[1:].contiguous(), t.to(torch.int32), right=True)
    return seq, past[seq] + t - q_start[seq]


def prepare(case, seed):
    s = {"case": case, "op": case["op"]}
    if case["op"] == "sample":
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rows, vocab, mix = case["rows"], case["vocab"], case["mix"]
        x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
        # some rows peaked, as after training, and in every fourth row most of the vocabulary masked
        peak = torch.randint(0, vocab, (rows, 4), generator=g, device="cuda")
        x.scatter_add_(1, peak, 8 * torch.rand(rows, 4, generator=g, device="cuda"))
        hidden = (torch.arange(rows, device="cuda") % 4 == 3)[:, None] & (torch.rand(rows, vocab, generator=g, device="cuda") < 0.9)
        s["logits"] = x.masked_fill_(hidden, -math.inf).to(DT[case["dtype"]])
        r = torch.arange(rows, device="cuda")
        full = lambda v: torch.full((rows,), v, device="cuda")  # noqa: E731
        temp = torch.tensor([0.8, 1.0, 0.0, 1.3, 0.6], device="cuda")
        s["temperature"] = temp[r % 5].contiguous() if rows > 1 else full(0.8)
        s["top_k"] = (torch.tensor([0, 40, 0, 200, 1], device="cuda", dtype=torch.int32)[r % 5] if mix & 2
                      else torch.zeros(rows, device="cuda", dtype=torch.int32)).contiguous()
        s["top_p"] = (torch.tensor([0.9, 0.95, 1.0, 0.5], device="cuda")[r % 4] if mix & 1 else full(1.0)).contiguous()
        s["min_p"] = (torch.tensor([0.0, 0.05, 0.0], device="cuda")[r % 3] if mix & 2 else full(0.0)).contiguous()
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        return s
    past, new, table, q_start, n_pages, free, g = _layout(case, seed)
    n, page, total = case["n"], case["page"], int(q_start[-1])
    s.update(past=past, new=new, q_start=q_start, kv_len=past + new, n=n, page=page, total=total, n_pages=n_pages,
             err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if case["op"] == "pages":
        # the table holds the cached tokens' pages; the others of the permutation are free
        held = (past + page - 1) // page
        col = torch.arange(table.shape[1], device="cuda")
        mine = col[None, :] < held[:, None]
        taken = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
        taken[table[mine].long()] = True
        s["free"] = free[~taken[free.long()]].contiguous()
        s["table"] = torch.where(mine, table, -1).to(torch.int32).contiguous()
        s["max_tokens"] = total + 5
        i32 = lambda k: torch.empty(k, dtype=torch.int32, device="cuda")  # noqa: E731
        s["out"] = [i32(n), i32(n + 1), i32(total + 5), i32(total + 5), i32(1)]
        return s
    dt, kv, group, hd = DT[case["dtype"]], case["kv"], case["group"], case["hd"]
    s.update(table=table, kv=kv, heads=kv * group, hd=hd, dtype=case["dtype"])
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(dt)  # noqa: E731
    s["k_cache"], s["v_cache"] = rand(n_pages, kv, page, hd), rand(n_pages, kv, page, hd)
    if case["op"] == "append":
        seq, pos = _tokens(past, q_start, total)
        s["positions"] = pos.to(torch.int32)
        s["slots"] = (table[seq, pos // page] * page + pos % page).to(torch.int32)
        s["qkv"] = rand(total, (kv * group + 2 * kv) * hd)
        s["n_pos"] = int(case["past"] + case["new"])
        inv = ROPE_BASE ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        ang = torch.arange(s["n_pos"], device="cuda", dtype=torch.float64)[:, None] * inv
        s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        s["q_out"] = torch.empty(total, kv * group, hd, dtype=dt, device="cuda")
        return s
    s["window"] = case["window"]
    s["max_q"] = case["new"]
    s["max_kv"] = case["past"] + case["new"]
    s["q"] = rand(total, kv * group, hd)
    s["out"] = torch.empty_like(s["q"])
    s["workspace"] = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    return s


# ---- plain forms ----------------------------------------------------------------

def _plain_pages(s):
    past, new, page, free = s["past"], s["new"], s["page"], s["free"]
    kv_len = past + new
    held = (past + page - 1) // page
    need = (kv_len + page - 1) // page - held
    first = torch.cumsum(need, 0) - need
    q_start = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    col = torch.arange(s["table"].shape[1], device="cuda")
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    at = (first[:, None] + col - held[:, None]).clamp(0, free.shape[0] - 1 if free.shape[0] else 0)
    table = torch.where(fresh, free[at], s["table"])
    t = torch.arange(s["max_tokens"], device="cuda")
    seq = torch.searchsorted(q_start[1:].contiguous(), t, right=True).clamp(max=s["n"] - 1)
    live = t < q_start[-1]
    pos = past[seq] + t - q_start[seq]
    slot = table[seq, (pos // page).clamp(0, table.shape[1] - 1)] * page + pos % page
    i32 = torch.int32
    return {"table": table, "kv_len": kv_len, "q_start": q_start.to(i32), "slots": torch.where(live, slot, -1).to(i32),
            "positions": torch.where(live, pos, -1).to(i32), "used": need.sum().to(i32).reshape(1)}


def _plain_append(s):
    total, heads, kv, hd, page = s["total"], s["heads"], s["kv"], s["hd"], s["page"]
    q, k, v = s["qkv"].split([heads * hd, kv * hd, kv * hd], 1)
    cs = s["rope"][s["positions"].long()]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]

    def rot(x, n):
        a, b = x.float().reshape(total, n, hd // 2, 2).unbind(-1)
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(total, n, hd).to(x.dtype)
    page_no, off = (s["slots"] // page).long(), (s["slots"] % page).long()
    s["k_cache"][page_no, :, off] = rot(k, kv)
    s["v_cache"][page_no, :, off] = v.reshape(total, kv, hd)
    return {"q": rot(q, heads), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    n, heads, kv, hd, page = s["n"], s["heads"], s["kv"], s["hd"], s["page"]
    max_q, max_kv, q_start = s["max_q"], s["max_kv"], s["q_start"].long()
    cols = -(-max_kv // page)
    table = s["table"][:, :cols].clamp(min=0).long()
    gather = lambda c: c[table].float().transpose(1, 2).reshape(n, kv, -1, hd)  # noqa: E731
    key, val = gather(s["k_cache"]), gather(s["v_cache"])
    j = torch.arange(max_q, device="cuda")
    live = j < s["new"][:, None]
    at = (q_start[:-1, None] + j).clamp(max=max(0, s["total"] - 1))
    q = s["q"][at].float().reshape(n, max_q, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)
    score = torch.matmul(q, key.transpose(2, 3)).mul_(1 / math.sqrt(hd)).reshape(n, kv, heads // kv, max_q, -1)
    t = torch.arange(key.shape[2], device="cuda")
    pos = s["past"][:, None] + j
    seen = t <= pos[..., None]
    if s["window"]:
        seen &= t > pos[..., None] - s["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.reshape(n, kv, -1, key.shape[2]), val).reshape(n, kv, heads // kv, max_q, hd)
    out = out.div_(total.clamp_(min=1e-37)).permute(0, 3, 1, 2, 4).reshape(n, max_q, heads, hd)
    return out[live].to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    vocab = x.shape[1]
    top = x.amax(1, keepdim=True)
    t = s["temperature"].double()[:, None]
    w = torch.where(x == top, 1.0, ((x - top) / t.clamp(min=1e-30)).exp())
    w = torch.where(x == -math.inf, 0.0, w)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = s["top_k"][:, None]
    rank = torch.arange(vocab, device="cuda")
    ws = torch.where((k <= 0) | (rank < k), ws, 0.0)
    before = torch.cumsum(ws, 1) - ws
    p = s["top_p"].double()[:, None]
    keep = (p >= 1) | (before < p * ws.sum(1, keepdim=True)) | (rank == 0)
    ws = torch.where(keep & (ws >= s["min_p"].double()[:, None]), ws, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, ws)
    cdf = torch.cumsum(w, 1)
    tok = (cdf <= s["u"].double()[:, None] * cdf[:, -1:]).sum(1)
    greedy = s["temperature"] == 0
    tok = torch.where(greedy, order[:, 0], tok.clamp(max=vocab - 1))
    return torch.where(top[:, 0] == -math.inf, -1, tok).to(torch.int32)


# ---- the framework's calls --------------------------------------------------------

def _stream():
    return torch.cuda.current_stream().cuda_stream


def _cache(api, s):
    page, hd = s["page"], s["hd"]
    return api.ptc_paged_cache(s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), CODE[s["dtype"]], s["n_pages"], page,
                               s["kv"], hd, s["kv"] * page * hd, page * hd, hd)


def _own_pages(s):
    from pitorch_b200 import api, lib
    kv_len, q_start, slots, positions, used = s["out"]
    a = api.ptc_pages_args(s["n"], s["page"], s["table"].shape[1], s["max_tokens"], s["free"].shape[0], s["n_pages"],
                           s["past"].data_ptr(), s["new"].data_ptr(), s["free"].data_ptr(), s["table"].data_ptr(),
                           kv_len.data_ptr(), q_start.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                           used.data_ptr(), s["err"].data_ptr())
    if lib().ptc_plan_pages(a, _stream()):
        raise RuntimeError("ptc_plan_pages refused the call")
    return {"table": s["table"], "kv_len": kv_len, "q_start": q_start, "slots": slots, "positions": positions, "used": used}


def _own_append(s):
    from pitorch_b200 import api, lib
    heads, kv, hd, qkv = s["heads"], s["kv"], s["hd"], s["qkv"]
    row, p, e = (heads + 2 * kv) * hd, qkv.data_ptr(), qkv.element_size()
    a = api.ptc_append_args(_cache(api, s), s["total"], heads, p, p + heads * hd * e, p + (heads + kv) * hd * e, row,
                            row, row, s["positions"].data_ptr(), s["slots"].data_ptr(), s["rope"].data_ptr(),
                            s["n_pos"], s["q_out"].data_ptr(), heads * hd, s["err"].data_ptr())
    if lib().ptc_kv_append(a, _stream()):
        raise RuntimeError("ptc_kv_append refused the call")
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attend(s):
    from pitorch_b200 import api, lib
    w = s["workspace"]
    a = api.ptc_attn_args(_cache(api, s), s["n"], s["total"], s["heads"], s["max_q"], s["table"].shape[1], s["window"],
                          1 / math.sqrt(s["hd"]), s["q"].data_ptr(), s["heads"] * s["hd"], s["out"].data_ptr(),
                          s["heads"] * s["hd"], s["table"].data_ptr(), s["kv_len"].data_ptr(), s["q_start"].data_ptr(),
                          w.data_ptr(), w.numel(), s["err"].data_ptr())
    if lib().ptc_paged_attention(a, _stream()):
        raise RuntimeError("ptc_paged_attention refused the call")
    return s["out"]


def _own_sample(s):
    from pitorch_b200 import api, lib
    x = s["logits"]
    a = api.ptc_sample_args(CODE[s["case"]["dtype"]], x.shape[0], x.shape[1], x.data_ptr(), x.shape[1],
                            s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(),
                            s["min_p"].data_ptr(), s["u"].data_ptr(), s["tokens"].data_ptr())
    if lib().ptc_sample_tokens(a, _stream()):
        raise RuntimeError("ptc_sample_tokens refused the call")
    return s["tokens"]


def run(s):
    if own:
        return {"pages": _own_pages, "append": _own_append, "attend": _own_attend, "sample": _own_sample}[s["op"]](s)
    return {"pages": _plain_pages, "append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["op"]](s)


# ---- the definitions in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("pages", "sample"):
        return None   # whole numbers: compared for equality
    heads, kv, hd, page = s["heads"], s["kv"], s["hd"], s["page"]
    past, new = _lens(case)
    if case["op"] == "append":
        x = s["qkv"].double().reshape(s["total"], heads + 2 * kv, hd)
        c = torch.complex(s["rope"][..., 0].double(), s["rope"][..., 1].double())[s["positions"].long()][:, None]
        turned = torch.view_as_real(torch.view_as_complex(x[:, : heads + kv].reshape(s["total"], heads + kv, hd // 2, 2).contiguous()) * c)
        turned = turned.reshape(s["total"], heads + kv, hd)
        caches = []
        for c0, rows in ((s["k_cache"], turned[:, heads:]), (s["v_cache"], x[:, heads + kv:])):
            flat = c0.double().permute(0, 2, 1, 3).reshape(-1, kv, hd)
            flat[s["slots"].long()] = rows
            caches.append(flat.reshape(-1, page, kv, hd).permute(0, 2, 1, 3).contiguous())
        return {"q": turned[:, :heads].contiguous(), "k_cache": caches[0], "v_cache": caches[1]}
    out = torch.zeros(s["total"], heads, hd, dtype=torch.float64, device="cuda")
    start = 0
    for i, (p, q) in enumerate(zip(past, new)):
        if q == 0:
            continue
        pages = s["table"][i, : -(-(p + q) // page)].long()
        rows = lambda c: c[pages].double().transpose(0, 1).reshape(kv, -1, hd)[:, : p + q]  # noqa: E731
        key, val = rows(s["k_cache"]), rows(s["v_cache"])
        pos = p + torch.arange(q, device="cuda")[:, None]
        t = torch.arange(p + q, device="cuda")[None]
        hide = t > pos
        if s["window"]:
            hide = hide | (t <= pos - s["window"])
        for h in range(heads):
            a = s["q"][start:start + q, h].double() @ key[h * kv // heads].T / math.sqrt(hd)
            a = torch.softmax(a.masked_fill(hide, -math.inf), -1)
            out[start:start + q, h] = a @ val[h * kv // heads]
        start += q
    return out
