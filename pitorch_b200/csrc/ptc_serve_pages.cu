// ptc_serve_pages.cu -- page tables and slot maps of a batch, and the rotary
// write of new keys and values into the paged cache (include/ptc_serve.h).
#include <limits.h>

#include "ptc_internal.h"
#include "ptc_serve.cuh"

namespace ptc {

const char *check_cache(const ptc_paged_cache &c) {
    if (!dtype_ok(c.dtype)) return "the cache's type is none of PTC_F32, PTC_F16, PTC_BF16";
    if (!c.k || !c.v || !aligned16(c.k) || !aligned16(c.v)) return "the cache's k and v have to be 16-byte aligned";
    if (c.n_pages < 1 || c.page_size < 1 || c.n_kv_heads < 1) return "the cache has no pages, tokens or heads";
    if ((long long)c.n_pages * c.page_size > INT_MAX) return "n_pages * page_size passes 2^31";
    if (c.head_dim < 8 || c.head_dim > 128 || c.head_dim % 8) return "head_dim has to be a multiple of 8, 8 to 128";
    const long long u = 16 / dtype_bytes(c.dtype);
    if (c.page_stride < 0 || c.head_stride < 0 || c.token_stride < 0 || c.page_stride % u || c.head_stride % u ||
        c.token_stride % u)
        return "the cache's strides have to be multiples of 16 bytes";
    return nullptr;
}

// ---------------------------------------------------------------------------
// Page tables and slot maps: two exclusive scans over the sequences (new
// tokens and new pages), then one search per token and per new page.
//
// One kernel. Every CTA scans all sequences itself (at most 4096, from L2) --
// 1 us of the 3.5 (64 sequences) or 6.4 us (2047 with 43,000 new tokens) that a
// call takes on the GPU, against a second launch or a grid barrier -- so each also knows whether the step fits before
// it writes anything. A table entry is read only where cached tokens lie and
// written only behind them, so no CTA reads what another writes.
// ---------------------------------------------------------------------------
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_MAX_TOKENS = 1 << 30;   // a row and a grid's step behind it fit 32 bits

__device__ __forceinline__ int pages_of(int tokens, int page) { return (int)(((unsigned)tokens + page - 1) / (unsigned)page); }

// Last r with start[r] <= i (start rises from 0; empty sequences share a start).
__device__ __forceinline__ int seq_of(const int *start, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) k_plan_pages(ptc_pages_args a) {
    extern __shared__ int plan_smem[];
    int *tok0 = plan_smem;                 // [n + 1] first row of each sequence
    int *page0 = plan_smem + a.n_seqs + 1;   // [n + 1] first new page of each sequence
    __shared__ long long wt[PLAN_THREADS / 32], wp[PLAN_THREADS / 32];
    __shared__ int bad_all;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n_seqs, P = a.page_size;
    if (tid == 0) bad_all = 0;
    __syncthreads();

    // Thread i owns `per` consecutive sequences. The sums are 64-bit until
    // they are known to fit.
    const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS, r0 = min(n, tid * per), r1 = min(n, r0 + per);
    long long st = 0, sp = 0;
    int bad = 0;
    for (int r = r0; r < r1; r++) {
        const int past = a.past_len[r], add = a.new_len[r];
        if (past < 0 || add < 0 || (long long)past + add > INT_MAX) {
            bad |= PTC_SERVE_ERR_LENGTH;
            continue;
        }
        const int held = pages_of(past, P), all = pages_of(past + add, P);
        if (all > a.max_pages) bad |= PTC_SERVE_ERR_TABLE;
        st += add;
        sp += all - held;
    }
    long long it = st, ip = sp;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, it, o), y = __shfl_up_sync(0xffffffffu, ip, o);
        if (lane >= o) it += x, ip += y;
    }
    if (lane == 31) wt[warp] = it, wp[warp] = ip;
    if (bad) atomicOr(&bad_all, bad);
    __syncthreads();
    long long bt = 0, bp = 0, total_t = 0, total_p = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; w++) {
        if (w == warp) bt = total_t, bp = total_p;
        total_t += wt[w];
        total_p += wp[w];
    }
    bad = bad_all;
    if (total_t > a.max_tokens) bad |= PTC_SERVE_ERR_TOKENS;
    if (total_p > a.n_free) bad |= PTC_SERVE_ERR_PAGES;

    const int step = gridDim.x * PLAN_THREADS, first = blockIdx.x * PLAN_THREADS + tid;
    if (bad) {   // the same decision in every CTA
        for (int t = first; t < a.max_tokens; t += step) a.slots[t] = a.positions[t] = -1;
        for (int r = first; r <= n; r += step) {
            a.q_start[r] = 0;
            if (r < n) a.kv_len[r] = a.past_len[r];
        }
        if (first == 0) {
            *a.pages_used = 0;
            serve_err(a.err, bad);
        }
        return;
    }
    int at_t = (int)(bt + it - st), at_p = (int)(bp + ip - sp);
    for (int r = r0; r < r1; r++) {
        const int past = a.past_len[r], add = a.new_len[r];
        tok0[r] = at_t;
        page0[r] = at_p;
        at_t += add;
        at_p += pages_of(past + add, P) - pages_of(past, P);
    }
    if (tid == 0) tok0[n] = (int)total_t, page0[n] = (int)total_p;
    __syncthreads();

    const int total = (int)total_t, fresh = (int)total_p;
    bool outside = false;
    for (int t = first; t < a.max_tokens; t += step) {
        int slot = -1, pos = -1;
        if (t < total) {
            const int r = seq_of(tok0, n, t), past = a.past_len[r], held = pages_of(past, P);
            pos = past + t - tok0[r];
            const int col = pos / P;
            const int page = col < held ? a.page_table[(size_t)r * a.max_pages + col] : a.free_pages[page0[r] + col - held];
            if ((unsigned)page < (unsigned)a.n_pages) slot = page * P + pos % P;
            else outside = true;
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
    for (int g = first; g < fresh; g += step) {
        const int r = seq_of(page0, n, g);
        a.page_table[(size_t)r * a.max_pages + pages_of(a.past_len[r], P) + g - page0[r]] = a.free_pages[g];
    }
    for (int r = first; r <= n; r += step) {
        a.q_start[r] = tok0[r];
        if (r < n) a.kv_len[r] = a.past_len[r] + a.new_len[r];
    }
    if (first == 0) *a.pages_used = fresh;
    if (outside) serve_err(a.err, PTC_SERVE_ERR_INDEX);
}

// ---------------------------------------------------------------------------
// Rotary write. Bound by memory: every element of q, k and v is read and
// written once. A thread keeps one 16-byte column of the head dimension, with
// its (cos, sin) pairs in registers, and walks over the row's heads (q, then
// k, then v), so the table is read once per row and column, not per head.
// Measured: 4362 tokens of 32 + 8 + 8 heads of 128 in bf16: 21 us for 109 MB, 5.1
// TB/s (0.78 of a measured copy); 64 tokens of 12 + 12 + 12 heads of 64 in f32:
// 2.5 us, which is a launch and one memory round trip.
// ---------------------------------------------------------------------------
constexpr int AP_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(AP_THREADS) k_kv_append(ptc_append_args a, int cols, int lanes) {
    constexpr int N = Vec16<T>::N;
    const int col = threadIdx.x % cols, lane = threadIdx.x / cols;
    if (lane >= lanes) return;
    const ptc_paged_cache &c = a.cache;
    const int t = blockIdx.x, hd = c.head_dim, nh = a.n_heads, nkv = c.n_kv_heads;
    const int pos = a.positions[t], slot = a.slots[t];
    bool store = slot >= 0 && slot < c.n_pages * c.page_size;
    bool live = pos >= 0 && (!a.rope || pos < a.n_pos);
    if (threadIdx.x == 0 && ((!live && pos != -1) || (!store && slot != -1))) serve_err(a.err, PTC_SERVE_ERR_INDEX);
    if (!live) return;
    float cs[N], sn[N];   // the pairs' factors, one per element pair
    if (a.rope) {
        const float2 *row = (const float2 *)a.rope + (size_t)pos * (hd / 2) + col * (N / 2);
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const float2 f = row[i];
            cs[i] = f.x;
            sn[i] = f.y;
        }
    }
    const long long cell = store ? (long long)(slot / c.page_size) * c.page_stride + (long long)(slot % c.page_size) * c.token_stride : 0;
    const int heads = store ? nh + 2 * nkv : nh;
    for (int h = lane; h < heads; h += lanes) {
        const T *src;
        T *dst;
        if (h < nh) {
            src = (const T *)a.q + t * a.q_stride + (long long)h * hd;
            dst = (T *)a.q_out + t * a.q_out_stride + (long long)h * hd;
        } else if (h < nh + nkv) {
            src = (const T *)a.k + t * a.k_stride + (long long)(h - nh) * hd;
            dst = (T *)c.k + cell + (h - nh) * c.head_stride;
        } else {
            src = (const T *)a.v + t * a.v_stride + (long long)(h - nh - nkv) * hd;
            dst = (T *)c.v + cell + (h - nh - nkv) * c.head_stride;
        }
        Vec16<T> x = *(const Vec16<T> *)(src + col * N);
        if (a.rope && h < nh + nkv) {
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                const float u = Elem<T>::up(x.e[2 * i]), w = Elem<T>::up(x.e[2 * i + 1]);
                x.e[2 * i] = Elem<T>::down(u * cs[i] - w * sn[i]);
                x.e[2 * i + 1] = Elem<T>::down(u * sn[i] + w * cs[i]);
            }
        }
        *(Vec16<T> *)(dst + col * N) = x;
    }
}

}  // namespace ptc

extern "C" int ptc_plan_pages(const ptc_pages_args *p, void *stream) {
    if (!p) SERVE_REFUSE("no arguments");
    const ptc_pages_args a = *p;
    if (a.n_seqs < 0 || a.n_seqs > PTC_SERVE_MAX_SEQS) SERVE_REFUSE("n_seqs %d is outside 0..%d", a.n_seqs, PTC_SERVE_MAX_SEQS);
    if (a.page_size < 1 || a.max_pages < 1 || a.max_tokens < 0 || a.max_tokens > ptc::PLAN_MAX_TOKENS || a.n_free < 0 || a.n_pages < 1)
        SERVE_REFUSE("bad size (page_size %d, max_pages %d, max_tokens %d, n_free %d, n_pages %d)", a.page_size,
                     a.max_pages, a.max_tokens, a.n_free, a.n_pages);
    if ((long long)a.n_pages * a.page_size > INT_MAX) SERVE_REFUSE("n_pages * page_size passes 2^31");
    if (!a.q_start || !a.pages_used || (a.n_seqs && (!a.past_len || !a.new_len || !a.page_table || !a.kv_len)) ||
        (a.max_tokens && (!a.slots || !a.positions)) || (a.n_free && !a.free_pages))
        SERVE_REFUSE("a required pointer is NULL");
    cudaStream_t s = (cudaStream_t)stream;
    ptc::MemoryDevice on(a.q_start);
    SERVE_CUDA(on.error());
    int n_sm = 0;
    SERVE_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, on.device()));
    const size_t smem = (size_t)2 * (a.n_seqs + 1) * sizeof(int);
    static_assert(2 * (PTC_SERVE_MAX_SEQS + 1) * sizeof(int) <= 48 * 1024 - 512, "what a kernel has without asking");
    const int want = (a.max_tokens + ptc::PLAN_THREADS - 1) / ptc::PLAN_THREADS;
    SERVE_CUDA(ptc::launch_kernel(ptc::k_plan_pages, want < 1 ? 1 : want < n_sm ? want : n_sm, ptc::PLAN_THREADS, smem, s, a));
    return 0;
}

extern "C" int ptc_rope_table(float *table, int n_pos, int head_dim, void *stream) {
    if (!table || ((uintptr_t)table & 7) || n_pos < 1 || head_dim < 2 || head_dim % 2 || (long long)n_pos * (head_dim / 2) > (1 << 30))
        SERVE_REFUSE("bad table (n_pos %d, head_dim %d)", n_pos, head_dim);
    cudaStream_t s = (cudaStream_t)stream;
    ptc::MemoryDevice on(table);
    SERVE_CUDA(on.error());
    SERVE_CUDA(ptc::launch_rope_table((float2 *)table, n_pos, head_dim, s));
    return 0;
}

extern "C" int ptc_kv_append(const ptc_append_args *p, void *stream) {
    if (!p) SERVE_REFUSE("no arguments");
    const ptc_append_args a = *p;
    if (const char *why = ptc::check_cache(a.cache)) SERVE_REFUSE("%s", why);
    if (a.n_tokens < 0 || a.n_heads < 1 || (a.rope && a.n_pos < 1))
        SERVE_REFUSE("bad size (n_tokens %d, n_heads %d, n_pos %d)", a.n_tokens, a.n_heads, a.n_pos);
    if (a.n_tokens == 0) return 0;
    const long long u = 16 / ptc::dtype_bytes(a.cache.dtype), hd = a.cache.head_dim;
    if (!a.q || !a.k || !a.v || !a.q_out || !a.positions || !a.slots) SERVE_REFUSE("a required pointer is NULL");
    if (!ptc::aligned16(a.q) || !ptc::aligned16(a.k) || !ptc::aligned16(a.v) || !ptc::aligned16(a.q_out) ||
        ((uintptr_t)a.rope & 7))
        SERVE_REFUSE("q, k, v and q_out have to be 16-byte aligned, rope 8-byte aligned");
    if (a.q_stride % u || a.k_stride % u || a.v_stride % u || a.q_out_stride % u || a.q_stride < a.n_heads * hd ||
        a.q_out_stride < a.n_heads * hd || a.k_stride < a.cache.n_kv_heads * hd || a.v_stride < a.cache.n_kv_heads * hd)
        SERVE_REFUSE("row strides have to be multiples of 16 bytes and hold a row");
    cudaStream_t s = (cudaStream_t)stream;
    ptc::MemoryDevice on(a.q_out);
    SERVE_CUDA(on.error());
    const int cols = (int)(hd / u), lanes = ptc::AP_THREADS / cols;
    const auto kernel = a.cache.dtype == PTC_F32   ? ptc::k_kv_append<float>
                        : a.cache.dtype == PTC_F16 ? ptc::k_kv_append<__half>
                                                   : ptc::k_kv_append<__nv_bfloat16>;
    SERVE_CUDA(ptc::launch_kernel(kernel, a.n_tokens, ptc::AP_THREADS, 0, s, a, cols, lanes));
    return 0;
}
