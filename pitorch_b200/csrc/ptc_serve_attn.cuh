// ptc_serve_attn.cuh -- how paged attention is cut into work (shared by its
// kernels).
//
// An item is (sequence, K/V head, row tile): the query heads of one K/V head
// are packed as rows, row i = token group.div(i), head i % group, and a tile has
// a fixed number of them, so a key that is read serves them all. An item's
// work is counted in units of a fixed number of keys, and the units of all
// items, laid end to end, are cut into one equal range per CTA. So one long
// sequence among short ones, or one sequence alone, loads the whole GPU
// evenly, whatever the lengths are, and these are only known on the device.
//
// A CTA that has part of an item writes its running maximum, sum and
// unnormalised output to the workspace. The last one to arrive at the item's
// counter adds the parts in their order (the result does not depend on who is
// last), writes the rows and sets the counter back to zero. Only a CTA's
// first and last item can be partial, so two slots per CTA are enough: slot
// 2c holds a part that began before CTA c, slot 2c + 1 one that begins in it.
#pragma once

#include "ptc_serve.cuh"

namespace ptc {

constexpr int ATTN_MAX_SEQS = PTC_SERVE_MAX_SEQS;
// Dynamic shared memory of a kernel behind `bytes` of its own: the sequences' first units (attn_prefix).
constexpr int attn_smem(int bytes, int n_seqs) { return bytes + (n_seqs + 1) * (int)sizeof(int); }
constexpr int ATTN_MAX_KEYS = 1 << 30;  // positions and rows stay below it, so that sums with a tile or a window fit
constexpr int ATTN_FLAG_BYTES = 4096;   // counters at the front of the workspace, one per CTA
constexpr float LOG2E = 1.4426950408889634f;

// Query heads of a K/V head, and division by their number: by a multiplication
// with floor(2^32 / n) + 1, which is at most one too high below 2^31.
struct Group {
    int n;
    unsigned magic;
    explicit Group(int heads) : n(heads), magic(heads > 1 ? (unsigned)((1ull << 32) / heads) + 1 : 0) {}
    __device__ __forceinline__ int div(int i) const {
        if (n == 1) return i;
        const int q = (int)__umulhi((unsigned)i, magic);
        return q * n > i ? q - 1 : q;
    }
};

// One sequence as the kernels use it; bad lengths give no rows.
struct AttnSeq {
    int q0;     // first row of q and out
    int n;      // rows (tokens)
    int pos0;   // position of the first one (may be negative)
    int cap;    // cached positions that the page table can hold
    int bad;
};

__device__ __forceinline__ AttnSeq attn_seq(const ptc_attn_args &a, int r) {
    AttnSeq s;
    s.q0 = a.q_start[r];
    const int q1 = a.q_start[r + 1], kv = a.kv_len[r];
    const long long room = min((long long)a.max_pages * a.cache.page_size, (long long)ATTN_MAX_KEYS);
    s.n = q1 - s.q0;
    s.bad = 0;
    s.pos0 = kv - s.n;
    s.cap = kv;
    if (s.q0 < 0 || q1 < s.q0 || q1 > a.n_tokens || kv < 0) s.bad = PTC_SERVE_ERR_LENGTH, s.n = 0;
    else if (kv > room) s.bad = PTC_SERVE_ERR_LENGTH, s.cap = (int)room;
    return s;
}

// The keys [lo, hi) that rows [i0, i1) of a sequence see (i = token * group.n + head).
__device__ __forceinline__ void attn_keys(const AttnSeq &s, Group group, int window, int i0, int i1, int &lo, int &hi) {
    hi = min(s.pos0 + group.div(i1 - 1) + 1, s.cap);
    lo = window > 0 ? max(0, s.pos0 + group.div(i0) - window + 1) : 0;
}

// Units of row tile m of a sequence: one at least, so that rows that see nothing are written.
template <int ROWS, int KEYS>
__device__ __forceinline__ int attn_units(const AttnSeq &s, Group group, int window, int m) {
    int lo, hi;
    attn_keys(s, group, window, m * ROWS, min(s.n * group.n, (m + 1) * ROWS), lo, hi);
    return hi > lo ? (hi + KEYS - 1) / KEYS - lo / KEYS : 1;
}

// pre[r] = units of one K/V head of the sequences before r, by all THREADS
// threads of the CTA; pre[n_seqs] is the total. scratch: THREADS / 32 ints. A
// total past 2^31 / heads leaves nothing to do (LENGTH).
template <int ROWS, int KEYS, int THREADS>
__device__ void attn_prefix(const ptc_attn_args &a, Group group, int *pre, long long *scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n_seqs;
    const int per = (n + THREADS - 1) / THREADS, r0 = min(n, tid * per);
    long long sum = 0;
    int bad = 0;
    for (int k = 0; k < per; k++) {
        const int r = r0 + k;
        const bool mine = r < n;
        AttnSeq s = {0, 0, 0, 0, 0};
        if (mine) s = attn_seq(a, r);
        bad |= s.bad;
        const long long rows = (long long)s.n * group.n;
        const int tiles = (int)((rows + ROWS - 1) / ROWS);
        long long u = 0;
        if (tiles <= 8)
            for (int m = 0; m < tiles; m++) u += attn_units<ROWS, KEYS>(s, group, a.window, m);
        // a long chunk's tiles are counted by the whole warp
        unsigned many = __ballot_sync(0xffffffffu, tiles > 8);
        while (many) {
            const int src = __ffs(many) - 1;
            many &= many - 1;
            AttnSeq b;
            b.n = __shfl_sync(0xffffffffu, s.n, src);
            b.pos0 = __shfl_sync(0xffffffffu, s.pos0, src);
            b.cap = __shfl_sync(0xffffffffu, s.cap, src);
            const int all = __shfl_sync(0xffffffffu, tiles, src);
            long long v = 0;
            for (int m = lane; m < all; m += 32) v += attn_units<ROWS, KEYS>(b, group, a.window, m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == src) u = v;
        }
        if (mine) pre[r] = (int)min(u, (long long)INT32_MAX);
        sum += u;
    }
    if (bad && blockIdx.x == 0) serve_err(a.err, bad);
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w == warp) before = total;
        total += scratch[w];
    }
    if (total > INT32_MAX / a.cache.n_kv_heads) {
        if (tid == 0 && blockIdx.x == 0) serve_err(a.err, PTC_SERVE_ERR_LENGTH);
        total = before = sum = inc = 0;
        for (int k = 0; k < per; k++)
            if (r0 + k < n) pre[r0 + k] = 0;
    }
    int at = (int)(before + inc - sum);
    for (int k = 0; k < per; k++)
        if (r0 + k < n) {
            const int u = pre[r0 + k];
            pre[r0 + k] = at;
            at += u;
        }
    if (tid == 0) pre[n] = (int)total;
    __syncthreads();
}

// One item and the part of it that a CTA has.
struct AttnItem {
    AttnSeq s;
    int r, head;        // sequence, K/V head
    int i0, i1;         // its rows
    int lo, hi;         // the keys they see
    int first, units;   // its first unit among all, and how many it has
};

// The item that holds unit u. All threads of a CTA get the same.
template <int ROWS, int KEYS>
__device__ AttnItem attn_find(const ptc_attn_args &a, Group group, const int *pre, int u) {
    AttnItem it;
    const int heads = a.cache.n_kv_heads;
    int lo = 0, hi = a.n_seqs;   // last r with pre[r] * heads <= u (sequences without units share their start)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] * heads <= u) lo = mid;
        else hi = mid;
    }
    it.r = lo;
    const int per = pre[lo + 1] - pre[lo], in = u - pre[lo] * heads;
    it.head = in / per;
    it.s = attn_seq(a, lo);
    int rest = in - it.head * per, m = 0, n;
    for (;; m++) {
        n = attn_units<ROWS, KEYS>(it.s, group, a.window, m);
        if (rest < n) break;
        rest -= n;
    }
    it.i0 = m * ROWS;
    it.i1 = min(it.s.n * group.n, (m + 1) * ROWS);
    attn_keys(it.s, group, a.window, it.i0, it.i1, it.lo, it.hi);
    it.first = u - rest;
    it.units = n;
    return it;
}

// CTA c of C has units [first(c), first(c + 1)) of `total`; owner(u) is the one that has unit u.
__device__ __forceinline__ int attn_first(int c, int C, int total) { return (int)((long long)c * total / C); }
__device__ __forceinline__ int attn_owner(int u, int C, int total) { return (int)((((long long)u + 1) * C - 1) / total); }

// Element t of a sequence: its offset in the cache without the head's share, or -1.
__device__ __forceinline__ long long attn_cell(const ptc_attn_args &a, int page, int off) {
    return (unsigned)page < (unsigned)a.cache.n_pages ? page * a.cache.page_stride + off * a.cache.token_stride : -1;
}

__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
    const __half2 v = __floats2half2_rn(x, y);
    return *(const uint32_t *)&v;
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *(const uint32_t *)&v;
}

// Probabilities are 2^(score - reference + lift), for the product with V, the
// sum and the outputs alike. f16 has no value between 0 and 2^-24, so that a
// long tail of small ones would vanish from the product while it stands in the
// sum; with a reference that is at most 2^8 too low (the kernels' rise), 2^7
// more keep them below 2^15, inside its range, and the tail seven bits longer.
template <typename T>
struct Lift {
    static constexpr float BY = 0.f;
};
template <>
struct Lift<__half> {
    static constexpr float BY = 7.f;
};

// 2^x by the special function unit (relative error 2^-22; 2^-inf is 0).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cp_async16_or_zero(unsigned dst, const void *src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Adds up an item's parts, which CTAs c0 to c1 left in their slots (MT rows of
// HDP outputs, MT maxima, MT sums), and writes its rows: weights first, a warp
// per row and a lane per part, then the weighted sums, with the parts shared
// out where there are few rows. All THREADS threads; smem: MT floats a part
// and 4 a thread or 4 outputs, whichever is more.
template <typename T, int HDP, int MT, int SLOT, int THREADS>
__device__ void attn_merge(const ptc_attn_args &a, const AttnItem &it, Group group, float *slots, int c0, int c1, float *smem) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rows = it.i1 - it.i0, hd = a.cache.head_dim, parts = c1 - c0 + 1;
    float *wgt = smem, *red = smem + (MT * parts + 3) / 4 * 4;
    auto part = [&](int p) { return slots + (long long)(2 * (c0 + p) + (p == 0)) * SLOT; };
    for (int r = warp; r < rows; r += THREADS / 32) {
        float top = -INFINITY, sum = 0.f;
        for (int p = lane; p < parts; p += 32) top = fmaxf(top, __ldcg(part(p) + MT * HDP + r));
        top = warp_max(top);
        const float ref = top == -INFINITY ? 0.f : top;
        for (int p = lane; p < parts; p += 32) {
            const float f = exp2f(__ldcg(part(p) + MT * HDP + r) - ref);
            wgt[r * parts + p] = f;
            sum += f * __ldcg(part(p) + MT * HDP + MT + r);
        }
        sum = warp_sum(sum);
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        for (int p = lane; p < parts; p += 32) wgt[r * parts + p] *= inv;
    }
    __syncthreads();
    const int cols = rows * (HDP / 4), shares = max(1, THREADS / cols);
    for (int i = tid; i < cols * shares; i += THREADS) {
        const int share = i / cols, x = i % cols, r = x / (HDP / 4), d = x % (HDP / 4) * 4;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int p = share; p < parts; p += shares) {
            const float f = wgt[r * parts + p];
            const float4 v = __ldcg((const float4 *)(part(p) + r * HDP + d));
            acc.x += f * v.x;
            acc.y += f * v.y;
            acc.z += f * v.z;
            acc.w += f * v.w;
        }
        *(float4 *)(red + i * 4) = acc;
    }
    __syncthreads();
    for (int x = tid; x < cols; x += THREADS) {
        const int r = x / (HDP / 4), d = x % (HDP / 4) * 4;
        if (d >= hd) continue;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int share = 0; share < shares; share++) {
            const float4 v = *(const float4 *)(red + (share * cols + x) * 4);
            acc.x += v.x;
            acc.y += v.y;
            acc.z += v.z;
            acc.w += v.w;
        }
        const int row = it.i0 + r, tok = group.div(row);
        T *dst = (T *)a.out + (it.s.q0 + tok) * a.out_stride + (long long)(it.head * group.n + row - tok * group.n) * hd + d;
        dst[0] = Elem<T>::down(acc.x);
        dst[1] = Elem<T>::down(acc.y);
        dst[2] = Elem<T>::down(acc.z);
        dst[3] = Elem<T>::down(acc.w);
    }
}

// The kernel for many rows (ptc_serve_attn_wide.cu): 16-bit types, scale > 0.
cudaError_t launch_attn_wide(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s);
// The one for many rows of f32 (ptc_serve_attn_f32.cu).
cudaError_t launch_attn_f32(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s);

}  // namespace ptc
