"""Plain 64-bit forms of the serving operators and small batches to run them
on (torch tensors; the GPU holds both sides)."""
import math

import torch

from pitorch_b200 import api

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": api.PTC_F32, "f16": api.PTC_F16, "bf16": api.PTC_BF16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


class Batch:
    """Sequences (past, new) over a paged cache with shuffled pages; what no
    sequence owns (free pages, the tail of a last page) is NaN and inf."""

    def __init__(self, lens, kv, group, hd, page, dtype, seed=0, layout="heads", spread=1.0, spare_rows=3):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.lens, self.kv, self.heads, self.hd, self.page, self.dtype = lens, kv, kv * group, hd, page, dtype
        dt = DT[dtype]
        need = [max(0, -(-(p + q) // page)) for p, q in lens]
        self.n_pages = sum(need) + 2
        self.cols = max(need + [1])
        perm = torch.randperm(self.n_pages, generator=g, device="cuda").tolist()
        table, at = [], 0
        for k in need:
            table.append(perm[at:at + k] + [-7] * (self.cols - k))
            at += k
        self.table = ints(table).reshape(len(lens), self.cols)
        self.kv_len = ints([p + q for p, q in lens])
        q_start = [0]
        for _, q in lens:
            q_start.append(q_start[-1] + q)
        self.total = q_start[-1]
        self.q_start = ints(q_start)
        shape = (self.n_pages, kv, page, hd) if layout == "heads" else (self.n_pages, page, kv, hd)
        self.k = torch.randn(shape, generator=g, device="cuda").to(dt)
        self.v = torch.randn(shape, generator=g, device="cuda").to(dt)
        self.strides = ((kv * page * hd, page * hd, hd) if layout == "heads" else (page * kv * hd, hd, kv * hd))
        # as [n_pages, kv, page, hd] views
        self.kp = self.k if layout == "heads" else self.k.transpose(1, 2)
        self.vp = self.v if layout == "heads" else self.v.transpose(1, 2)
        owned = torch.zeros(self.n_pages, page, dtype=torch.bool, device="cuda")
        for r, (p, q) in enumerate(lens):
            for c in range(need[r]):
                owned[table[r][c], : min(page, p + q - c * page)] = True
        bad = (~owned)[:, None, :, None].expand(-1, kv, -1, hd)
        self.kp.masked_fill_(bad, math.inf)
        self.vp.masked_fill_(bad, math.nan)
        self.q = (torch.randn(self.total + spare_rows, self.heads, hd, generator=g, device="cuda") * spread).to(dt)
        self.err = ints([0])
        self.work = torch.zeros(api.PTC_ATTN_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    def cache(self):
        return api.ptc_paged_cache(self.k.data_ptr(), self.v.data_ptr(), CODE[self.dtype], self.n_pages, self.page,
                                   self.kv, self.hd, *self.strides)

    def attn_args(self, out, window=0, scale=None, q=None, max_q=None):
        q = self.q if q is None else q
        return api.ptc_attn_args(self.cache(), len(self.lens), q.shape[0], self.heads,
                                 max([n for _, n in self.lens] + [0]) if max_q is None else max_q, self.cols, window,
                                 1 / math.sqrt(self.hd) if scale is None else scale, q.data_ptr(), q.stride(0),
                                 out.data_ptr(), out.stride(0), self.table.data_ptr(), self.kv_len.data_ptr(),
                                 self.q_start.data_ptr(), self.work.data_ptr(), self.work.numel(), self.err.data_ptr())

    def attend(self, L, window=0, scale=None, max_q=None):
        out = torch.full_like(self.q, 7.0)
        assert L.ptc_paged_attention(self.attn_args(out, window, scale, max_q=max_q), stream()) == 0
        torch.cuda.synchronize()
        return out

    def rows(self, c, r):
        p, q = self.lens[r]
        n = p + q
        if n <= 0:
            return torch.zeros(self.kv, 0, self.hd, dtype=torch.float64, device="cuda")
        pages = self.table[r, : -(-n // self.page)].long()
        return c[pages].double().transpose(0, 1).reshape(self.kv, -1, self.hd)[:, :n]

    def reference(self, window=0, scale=None):
        """(out, bound): attention in 64 bits and how far the kernels may be off, element by element.

        With A = sum_t p_t |v_t| an element's error is at most
          A * (2 ds + h + (n + 32) 2^-24) + |out| * half a step of the type,
        ds the absolute error of a score: a product of hd terms in 32 bits whose
        factors may be held as three bfloat16 parts (2^-22 of sum |q k|), its
        scaling and the subtraction of the maximum (2^-22 of the largest |score|);
        h the rounding of the probabilities to the type (0 for f32); n additions;
        f16 probabilities below 2^-14 have steps of 2^-24."""
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        out = torch.zeros(self.total, self.heads, self.hd, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        h, at, group = HALF[self.dtype], 0, self.heads // self.kv
        for r, (p, n) in enumerate(self.lens):
            if n <= 0:
                continue
            key, val = self.rows(self.kp, r), self.rows(self.vp, r)
            q = self.q[at:at + n].double().reshape(n, self.kv, group, self.hd).permute(1, 2, 0, 3)
            s = torch.einsum("kgqd,ktd->kgqt", q, key) * scale
            sa = torch.einsum("kgqd,ktd->kgqt", q.abs(), key.abs()) * abs(scale)
            pos = p + torch.arange(n, device="cuda")[:, None]
            t = torch.arange(key.shape[1], device="cuda")[None]
            hide = t > pos
            if window:
                hide = hide | (t <= pos - window)
            top = s.masked_fill(hide, -math.inf).amax(-1, keepdim=True) if key.shape[1] else s.new_full(s.shape[:3] + (1,), -math.inf)
            w = (s - top.clamp(min=-1e300)).exp().masked_fill(hide, 0.0)
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            o, a = torch.einsum("kgqt,ktd->kgqd", w, val), torch.einsum("kgqt,ktd->kgqd", w, val.abs())
            sa = sa.masked_fill(hide, 0.0).amax(-1, keepdim=True) if key.shape[1] else top.new_zeros(top.shape)
            ds = sa * ((self.hd + 4) * 2.0 ** -24 + 2.0 ** -22) + sa * 2.0 ** -22
            keys = float(key.shape[1])
            b = a * (2 * ds + (0 if self.dtype == "f32" else h) + (keys + 32) * 2.0 ** -24) + o.abs() * h
            if self.dtype == "f16":
                b = b + keys * 2.0 ** -25 * (val.abs().amax() if key.shape[1] else 0.0) + 2.0 ** -25
            out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, self.heads, self.hd)
            bound[at:at + n] = b.permute(2, 0, 1, 3).reshape(n, self.heads, self.hd)
            at += n
        return out, bound + 1e-30


def check(got, want, bound):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(),
                           float(((got.double() - want).abs() / bound).nan_to_num(1e9).max()))


def plan_ref(past, new, page, free, table):
    """Page tables and slot maps by the definition, in plain Python."""
    table = [list(r) for r in table]
    used, q_start, kv_len, slots, positions = 0, [0], [], [], []
    for r, (p, n) in enumerate(zip(past, new)):
        held, need = -(-p // page), -(-(p + n) // page)
        for c in range(held, need):
            table[r][c] = free[used]
            used += 1
        for j in range(n):
            positions.append(p + j)
            slots.append(table[r][(p + j) // page] * page + (p + j) % page)
        q_start.append(q_start[-1] + n)
        kv_len.append(p + n)
    return table, kv_len, q_start, slots, positions, used


def sample_ref(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5):
    """One row's token by the definition, in 64 bits (x: 1-D tensor)."""
    x = x.double().cpu()
    x = torch.where(x.isnan(), -math.inf, x)
    top = float(x.max())
    if top == -math.inf:
        return -1
    if not temperature > 0:
        return int((x == top).nonzero()[0])
    w = torch.where(x == top, 1.0, ((x - top) / temperature).exp())
    w = torch.where(x == -math.inf, 0.0, w)
    order = torch.sort(x, descending=True, stable=True).indices
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        m = w[order]
        before = torch.cumsum(m, 0) - m
        keep = before < top_p * m.sum()
        keep[0] = True
        order = order[keep]
    kept = torch.zeros_like(w)
    kept[order] = torch.where(w[order] >= min_p, w[order], 0.0)
    cdf = torch.cumsum(kept, 0)
    return int((cdf <= u * float(cdf[-1])).sum())
