// ptc_serve_attn.cu -- attention of new tokens over a paged KV cache
// (include/ptc_serve.h): the kernel for few rows per K/V head.
#include "ptc_serve_attn.cuh"

namespace ptc {

// ---------------------------------------------------------------------------
// Few rows (single tokens, short chunks): bound by reading the cache once.
//
// The four warps of a CTA work on their own 16 keys of each 64-key unit and
// never wait for each other before the item ends: each keeps a running
// maximum, sum and output of the item's rows, and fills its own ring of
// shared-memory stages with 16-byte asynchronous copies, the page numbers one
// stage further ahead in registers. 16-bit types go through
// mma.sync.m16n8k16 (a tile has 16 rows, of which a single token fills
// `group`; the tensor pipe is busy for a quarter of the time that the copies
// take, so the unused rows cost little), f32 through fused multiply-adds on MT rows. Rows of a
// stage are padded by 16 bytes, which keeps ldmatrix and the 128-bit reads
// free of bank conflicts for every head size. Measured: 64 sequences of up to
// 8192 positions, 32 heads in groups of 4, 128 elements of bf16: 197 to 209 us for
// 1.08 GB of keys and values, 5.2 to 5.5 TB/s (0.79 to 0.83 of a measured copy;
// the second product of the probabilities takes 5% of it).
// 64 f32 tokens over up to 1024 positions of 12 heads of 64: 64 us for 211 MB. One f32 token over 1024 positions
// of 12 heads of 64: 8.9 us, of which the reads are 1: two searches of the work
// table, the page lookup, one read, a counter and the sum of 16 parts follow
// one another.
// ---------------------------------------------------------------------------
constexpr int NA_WARPS = 4;
constexpr int NA_THREADS = NA_WARPS * 32;
constexpr int NA_KEYS = 16;                   // keys of a warp's stage
constexpr int NA_UNIT = NA_WARPS * NA_KEYS;   // keys of a unit
constexpr int NA_STAGES = 3;
// A row's reference for its probabilities is raised only when a score passes it
// by this (sums and outputs are relative to the same value, and stay below 2^8
// times the keys' number).
constexpr float NA_RISE = 8.f;
constexpr int NA_MAX_CTAS = 444;               // three per SM: the parts that one item can have

template <typename T, int HDP, int MT>
struct NarrowShape {
    static constexpr int ROW = HDP * (int)sizeof(T) + 16;   // bytes of a key in a stage
    static constexpr int CH = HDP * (int)sizeof(T) / 16;    // 16-byte chunks of it
    static constexpr int STAGE = 2 * NA_KEYS * ROW;         // K, then V
    static constexpr int WARP = NA_STAGES * STAGE;
    // floats of a workspace slot: output, maxima, sums; whole 16 bytes, for the vector accesses to the next slot
    static constexpr int SLOT = (MT * (HDP + 2) + 3) / 4 * 4;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], unsigned at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], unsigned at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A warp's rows of an item on tensor cores: lane l has rows l / 4 and l / 4 + 8.
template <typename T, int HDP, int MT>
struct NarrowRows {
    static_assert(MT == 16, "an m16n8k16 tile has 16 rows");
    uint32_t q[HDP / 16][4];
    float o[HDP / 8][4];
    float m[2], l[2];
    int lo[2], hi[2];

    __device__ void begin(const ptc_attn_args &a, const AttnItem &it, Group group, const float *) {
        const int lane = threadIdx.x & 31, hd = a.cache.head_dim;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = it.i0 + lane / 4 + 8 * h, tok = group.div(i);
            const bool real = i < it.i1;
            const T *src = (const T *)a.q + (it.s.q0 + (real ? tok : 0)) * a.q_stride +
                           (long long)(it.head * group.n + (real ? i - tok * group.n : 0)) * hd;
#pragma unroll
            for (int k = 0; k < HDP / 16; k++)
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int d = k * 16 + b * 8 + (lane & 3) * 2;
                    q[k][h + 2 * b] = real && d < hd ? *(const uint32_t *)(src + d) : 0;
                }
            const int pos = it.s.pos0 + tok;
            hi[h] = real ? min(pos + 1, it.s.cap) : 0;
            lo[h] = a.window > 0 ? pos - a.window + 1 : 0;
            m[h] = -INFINITY;
            l[h] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < HDP / 8; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][e] = 0.f;
    }

    // 16 keys from `key` on, in the stage at `at`; bit k of `there`: key k is in the cache
    __device__ void step(unsigned at, const char *, int key, unsigned there, float scale, const float *, float *) {
        using S = NarrowShape<T, HDP, MT>;
        const int lane = threadIdx.x & 31;
        float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, s2[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};   // two chains of products
        const unsigned kat = at + ((lane & 7) + ((lane >> 4) << 3)) * S::ROW + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int k = 0; k < HDP / 16; k++) {
            uint32_t b[4];
            ldmatrix4(b, kat + k * 32);
            mma16816(k & 1 ? s2[0] : s[0], q[k], b[0], b[1], T());
            mma16816(k & 1 ? s2[1] : s[1], q[k], b[2], b[3], T());
        }
#pragma unroll
        for (int x = 0; x < 8; x++) s[x >> 2][x & 3] += s2[x >> 2][x & 3];
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int c = n * 8 + (lane & 3) * 2 + e, t = key + c;
                    const bool see = t < hi[h] && t >= lo[h] && (there >> c & 1);
                    float &v = s[n][2 * h + e];
                    v = see ? v * scale : -INFINITY;
                    top[h] = fmaxf(top[h], v);
                }
        if (__any_sync(0xffffffffu, top[0] > m[0] + NA_RISE || top[1] > m[1] + NA_RISE)) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float t = fmaxf(top[h], m[h]);
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                const float f = t == -INFINITY ? 0.f : exp2f(m[h] - t);
                m[h] = t;
                l[h] *= f;
#pragma unroll
                for (int n = 0; n < HDP / 8; n++) o[n][2 * h] *= f, o[n][2 * h + 1] *= f;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float ref = m[h] == -INFINITY ? 0.f : m[h] - Lift<T>::BY;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float &v = s[n][2 * h + e];
                    v = exp2_fast(v - ref);
                    l[h] += v;
                }
        }
        // The product with V wants probabilities of V's type: rounded, and what the rounding left, as a second product
        // (rounded alone they would add as large an error as the result's own rounding).
        uint32_t p[4], rest[4];
#pragma unroll
        for (int x = 0; x < 4; x++) {
            float &u = s[x >> 1][2 * (x & 1)], &w = s[x >> 1][2 * (x & 1) + 1];
            p[x] = pack2(u, w, T());
            const T *r = (const T *)&p[x];
            rest[x] = pack2(u - Elem<T>::up(r[0]), w - Elem<T>::up(r[1]), T());
        }
        const unsigned vat = at + NA_KEYS * S::ROW + (lane & 15) * S::ROW + (lane >> 4) * 16;
#pragma unroll
        for (int n = 0; n < HDP / 16; n += 2) {   // two at a time: the second products follow the first at a distance
            uint32_t b[2][4];
            ldmatrix4t(b[0], vat + n * 32);
            ldmatrix4t(b[1], vat + n * 32 + 32);
#pragma unroll
            for (int x = 0; x < 4; x++) mma16816(o[2 * n + x], p, b[x >> 1][2 * (x & 1)], b[x >> 1][2 * (x & 1) + 1], T());
#pragma unroll
            for (int x = 0; x < 4; x++) mma16816(o[2 * n + x], rest, b[x >> 1][2 * (x & 1)], b[x >> 1][2 * (x & 1) + 1], T());
        }
    }

    // this warp's maximum, sum and output of each row into shared memory
    __device__ void end(float *mw, float *lw, float *ow) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float sum = l[h];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = lane / 4 + 8 * h;
            if ((lane & 3) == 0) mw[row] = m[h], lw[row] = sum;
#pragma unroll
            for (int n = 0; n < HDP / 8; n++)
                *(float2 *)(ow + row * HDP + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
    }
};

// The same in 32-bit arithmetic. Scores: lane l has key l % 16 and every
// other 16-byte chunk of its row (l / 16 picks which); outputs: elements
// l, l + 32, ... of every row.
template <int HDP, int MT>
struct NarrowRows<float, HDP, MT> {
    static constexpr int E = HDP / 32;
    float o[MT][E], m[MT], l[MT];

    __device__ void begin(const ptc_attn_args &, const AttnItem &, Group, const float *) {
#pragma unroll
        for (int r = 0; r < MT; r++) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) o[r][e] = 0.f;
        }
    }

    // qs: [MT][HDP] rows, then [MT] first and [MT] end of the keys each sees (as ints)
    __device__ void step(unsigned, const char *stage, int key, unsigned there, float scale, const float *qs, float *ps) {
        using S = NarrowShape<float, HDP, MT>;
        const int lane = threadIdx.x & 31, k = lane & 15, half = lane >> 4;
        const int *lo = (const int *)(qs + MT * HDP), *hi = lo + MT;
        float s[MT];
#pragma unroll
        for (int r = 0; r < MT; r++) s[r] = 0.f;
        const char *row = stage + k * S::ROW;
#pragma unroll
        for (int c = 0; c < S::CH; c += 2) {
            const float4 x = *(const float4 *)(row + (c + half) * 16);
#pragma unroll
            for (int r = 0; r < MT; r++) s[r] = dot4(x, *(const float4 *)(qs + r * HDP + (c + half) * 4), s[r]);
        }
        const int t = key + k;
        bool rise = false;
#pragma unroll
        for (int r = 0; r < MT; r++) {
            s[r] += __shfl_xor_sync(0xffffffffu, s[r], 16);
            s[r] = t < hi[r] && t >= lo[r] && (there >> k & 1) ? s[r] * scale : -INFINITY;
            rise |= s[r] > m[r] + NA_RISE;
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int r = 0; r < MT; r++) {
                float top = fmaxf(s[r], m[r]);
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float f = top == -INFINITY ? 0.f : exp2f(m[r] - top);
                m[r] = top;
                l[r] *= f;
#pragma unroll
                for (int e = 0; e < E; e++) o[r][e] *= f;
            }
        }
#pragma unroll
        for (int r = 0; r < MT; r++) {
            const float p = exp2_fast(s[r] - (m[r] == -INFINITY ? 0.f : m[r]));
            l[r] += p;   // of this lane's keys
            if (half == 0) ps[r * NA_KEYS + k] = p;
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NA_KEYS; j += 4) {
            float v[4][E];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < E; e++) v[i][e] = *(const float *)(stage + (NA_KEYS + j + i) * S::ROW + (lane + 32 * e) * 4);
#pragma unroll
            for (int r = 0; r < MT; r++) {
                const float4 p = *(const float4 *)(ps + r * NA_KEYS + j);
#pragma unroll
                for (int e = 0; e < E; e++)
                    o[r][e] = fmaf(p.w, v[3][e], fmaf(p.z, v[2][e], fmaf(p.y, v[1][e], fmaf(p.x, v[0][e], o[r][e]))));
            }
        }
        __syncwarp();
    }

    __device__ void end(float *mw, float *lw, float *ow) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < MT; r++) {
            float sum = l[r];
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) mw[r] = m[r], lw[r] = sum;
#pragma unroll
            for (int e = 0; e < E; e++) ow[r * HDP + lane + 32 * e] = o[r][e];
        }
    }
};

template <typename T, int HDP, int MT>
__global__ void __launch_bounds__(NA_THREADS) k_attn_narrow(ptc_attn_args a, Group group) {
    using S = NarrowShape<T, HDP, MT>;
    constexpr int SLOT = S::SLOT;
    extern __shared__ __align__(16) char na_smem[];
    __shared__ long long scratch[NA_WARPS];
    __shared__ __align__(16) float qs[sizeof(T) == 4 ? MT * (HDP + 2) : 4];
    __shared__ __align__(16) float ps[NA_WARPS][sizeof(T) == 4 ? MT * NA_KEYS : 4];
    __shared__ float mw[NA_WARPS][MT], lw[NA_WARPS][MT];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = a.cache.head_dim, heads = a.cache.n_kv_heads;
    char *ring = na_smem + warp * S::WARP;
    int *pre = (int *)(na_smem + NA_WARPS * S::WARP);
    unsigned *flags = (unsigned *)a.workspace;
    float *slots = (float *)((char *)a.workspace + ATTN_FLAG_BYTES);

    attn_prefix<MT, NA_UNIT, NA_THREADS>(a, group, pre, scratch);
    const int total = pre[a.n_seqs] * heads, C = min((int)gridDim.x, total), c = blockIdx.x;
    if (c >= C) return;
    const int u1 = attn_first(c + 1, C, total);
    const float scale = a.scale * LOG2E;

    for (int u = attn_first(c, C, total); u < u1;) {
        const AttnItem it = attn_find<MT, NA_UNIT>(a, group, pre, u);
        const int seg0 = u - it.first, seg1 = min(it.units, seg0 + u1 - u), rows = it.i1 - it.i0;
        // This warp's keys: 16 of every unit. Lanes 0..15 look up a key each.
        const int n = seg1 - seg0, key0 = (it.lo / NA_UNIT + seg0) * NA_UNIT + warp * NA_KEYS;
        const int *table = a.page_table + (long long)it.r * a.max_pages;
        const long long base = it.head * a.cache.head_stride;
        auto look = [&](int j) {   // the page number of this lane's key of unit j
            const int t = key0 + j * NA_UNIT + (lane & 15);
            return j < n && t < it.hi && t >= it.lo ? table[t / a.cache.page_size] : 0;
        };
        auto fill = [&](int j, int page) {   // unit j into its stage; which of its keys are there
            const int t = key0 + j * NA_UNIT + (lane & 15);
            long long cell = -1;
            if (j < n && t < it.hi && t >= it.lo) {
                cell = attn_cell(a, page, t % a.cache.page_size);
                if (cell < 0) serve_err(a.err, PTC_SERVE_ERR_INDEX);
            }
            const unsigned there = __ballot_sync(0xffffffffu, cell >= 0) & 0xffffu;
            if (j < n) {
                const unsigned at = smem_u32(ring + (j % NA_STAGES) * S::STAGE);
                const long long cell0 = __shfl_sync(0xffffffffu, cell, 0);
                if (32 % S::CH == 0 && __all_sync(0xffffffffu, cell >= 0 && cell == cell0 + (lane & 15) * a.cache.token_stride)) {
                    // all there and one after the other, as in a page: no lane has to ask another for its key
                    constexpr int EACH = 32 / (S::CH <= 32 ? S::CH : 32);   // keys of a step
                    const int k0 = lane / S::CH, ch = lane % S::CH, e = ch * (16 / (int)sizeof(T));
                    const bool real = e < hd;
                    const long long off = cell0 + base + k0 * a.cache.token_stride + (real ? e : 0), step = EACH * a.cache.token_stride;
                    const T *k = (const T *)a.cache.k + off, *v = (const T *)a.cache.v + off;
                    const unsigned to = at + k0 * S::ROW + ch * 16;
#pragma unroll
                    for (int i = 0; i < NA_KEYS / EACH; i++, k += step, v += step) {
                        cp_async16_or_zero(to + i * EACH * S::ROW, k, real);
                        cp_async16_or_zero(to + (NA_KEYS + i * EACH) * S::ROW, v, real);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < NA_KEYS * S::CH / 32; i++) {
                        const int x = i * 32 + lane, k = x / S::CH, ch = x % S::CH;
                        const long long from = __shfl_sync(0xffffffffu, cell, k);
                        const int e = ch * (16 / (int)sizeof(T));
                        const bool real = from >= 0 && e < hd;
                        const long long off = real ? from + base + e : 0;
                        cp_async16_or_zero(at + k * S::ROW + ch * 16, (const T *)a.cache.k + off, real);
                        cp_async16_or_zero(at + (NA_KEYS + k) * S::ROW + ch * 16, (const T *)a.cache.v + off, real);
                    }
                }
            }
            cp_async_commit();
            return there;
        };
        unsigned there[NA_STAGES];
        int pages[NA_STAGES];
#pragma unroll
        for (int j = 0; j < NA_STAGES; j++) pages[j] = look(j);
#pragma unroll
        for (int j = 0; j < NA_STAGES - 1; j++) there[j] = fill(j, pages[j]);
        int page = pages[NA_STAGES - 1];
        // the queries, while the first keys are on their way
        if constexpr (sizeof(T) == 4) {
            int *lim = (int *)(qs + MT * HDP);
            for (int i = tid; i < MT * HDP; i += NA_THREADS) {
                const int r = i / HDP, d = i % HDP, row = it.i0 + r, tok = group.div(row);
                qs[i] = r < rows && d < hd ? Elem<T>::up(((const T *)a.q)[(it.s.q0 + tok) * a.q_stride +
                                                                         (long long)(it.head * group.n + row - tok * group.n) * hd + d])
                                           : 0.f;
            }
            if (tid < MT) {
                const int pos = it.s.pos0 + group.div(it.i0 + tid);
                lim[tid] = a.window > 0 ? pos - a.window + 1 : 0;
                lim[MT + tid] = tid < rows ? min(pos + 1, it.s.cap) : 0;
            }
            __syncthreads();
        }
        NarrowRows<T, HDP, MT> st;
        st.begin(a, it, group, qs);
        for (int j = 0; j < n; j++) {
            cp_async_wait<NA_STAGES - 2>();
            __syncwarp();
            const unsigned have = there[0];
#pragma unroll
            for (int i = 0; i + 2 < NA_STAGES; i++) there[i] = there[i + 1];
            there[NA_STAGES - 2] = fill(j + NA_STAGES - 1, page);
            page = look(j + NA_STAGES);
            const char *stage = ring + (j % NA_STAGES) * S::STAGE;
            st.step(smem_u32(stage), stage, key0 + j * NA_UNIT, have, scale, qs, ps[warp]);
            __syncwarp();
        }
        cp_async_wait<0>();
        __syncthreads();   // the stages are free: the warps' outputs go there
        float *ow = (float *)na_smem;
        st.end(mw[warp], lw[warp], ow + warp * MT * HDP);
        __syncthreads();

        const bool whole = seg1 - seg0 == it.units;
        float *slot = slots + (long long)(2 * c + (seg0 == 0)) * SLOT;
        for (int i = tid; i < rows * (HDP / 4); i += NA_THREADS) {
            const int r = i / (HDP / 4), d = i % (HDP / 4) * 4;
            if (d >= hd) continue;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < NA_WARPS; w++) top = fmaxf(top, mw[w][r]);
            const float ref = top == -INFINITY ? 0.f : top;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NA_WARPS; w++) {
                const float f = exp2f(mw[w][r] - ref);
                const float4 x = *(const float4 *)(ow + (w * MT + r) * HDP + d);
                sum += f * lw[w][r];
                acc.x += f * x.x;
                acc.y += f * x.y;
                acc.z += f * x.z;
                acc.w += f * x.w;
            }
            if (whole) {
                const float inv = sum > 0.f ? 1.f / sum : 0.f;
                const int row = it.i0 + r, tok = group.div(row);
                T *dst = (T *)a.out + (it.s.q0 + tok) * a.out_stride + (long long)(it.head * group.n + row - tok * group.n) * hd + d;
                dst[0] = Elem<T>::down(acc.x * inv);
                dst[1] = Elem<T>::down(acc.y * inv);
                dst[2] = Elem<T>::down(acc.z * inv);
                dst[3] = Elem<T>::down(acc.w * inv);
            } else {
                *(float4 *)(slot + r * HDP + d) = acc;
                if (d == 0) slot[MT * HDP + r] = top, slot[MT * HDP + MT + r] = sum;
            }
        }
        if (!whole) {
            const int c0 = attn_owner(it.first, C, total), c1 = attn_owner(it.first + it.units - 1, C, total);
            __syncthreads();
            if (tid == 0) {
                last = atom_add_acq_rel(&flags[c0], 1u) == (unsigned)(c1 - c0);
            }
            __syncthreads();
            if (last) {
                attn_merge<T, HDP, MT, SLOT, NA_THREADS>(a, it, group, slots, c0, c1, ow);
                if (tid == 0) flags[c0] = 0;
            }
        }
        __syncthreads();   // the next item fills the stages again
        u += seg1 - seg0;
    }
}

template <typename T, int HDP, int MT>
static cudaError_t launch_narrow(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s) {
    auto kernel = k_attn_narrow<T, HDP, MT>;
    constexpr int ring = NA_WARPS * NarrowShape<T, HDP, MT>::WARP;
    const int smem = attn_smem(ring, a.n_seqs);
    static_assert(NA_WARPS * MT * HDP * 4 <= NA_WARPS * NarrowShape<T, HDP, MT>::WARP, "the outputs fit the stages");
    // (and so do a merge's weights and sums: MT a part, of at most the CTAs, and 4 floats a thread or an output)
    static_assert((MT * NA_MAX_CTAS + 3) * 4 + 4 * (NA_THREADS > MT * HDP / 4 ? NA_THREADS : MT * HDP / 4) * 4 <=
                      NA_WARPS * NarrowShape<T, HDP, MT>::WARP, "a merge fits the stages");
    cudaError_t e = allow_smem(kernel, attn_smem(ring, ATTN_MAX_SEQS));
    int per = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, NA_THREADS, smem);
    if (e != cudaSuccess) return e;
    if (per < 1) return cudaErrorInvalidConfiguration;
    int grid = per * n_sm;
    const long long fit = (long long)(PTC_ATTN_WORKSPACE_BYTES - ATTN_FLAG_BYTES) / (2 * NarrowShape<T, HDP, MT>::SLOT * sizeof(float));
    if (grid > fit) grid = (int)fit;
    if (grid > NA_MAX_CTAS) grid = NA_MAX_CTAS;
    static_assert(NA_MAX_CTAS <= ATTN_FLAG_BYTES / 4, "a counter per CTA");
    return launch_kernel(kernel, grid, NA_THREADS, smem, s, a, group);
}

template <typename T, int MT>
static cudaError_t launch_narrow_hd(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s) {
    const int hd = a.cache.head_dim;
    if (hd <= 32) return launch_narrow<T, 32, MT>(a, group, n_sm, s);
    if (hd <= 64) return launch_narrow<T, 64, MT>(a, group, n_sm, s);
    if (hd <= 96) return launch_narrow<T, 96, MT>(a, group, n_sm, s);
    return launch_narrow<T, 128, MT>(a, group, n_sm, s);
}

}  // namespace ptc

extern "C" int ptc_paged_attention(const ptc_attn_args *p, void *stream) {
    if (!p) SERVE_REFUSE("no arguments");
    ptc_attn_args a = *p;
    if (const char *why = ptc::check_cache(a.cache)) SERVE_REFUSE("%s", why);
    if (a.n_seqs < 0 || a.n_tokens < 0 || a.max_pages < 1 || a.max_q < 0 || a.window < 0)
        SERVE_REFUSE("bad size (n_seqs %d, n_tokens %d, max_q %d, max_pages %d, window %d)", a.n_seqs, a.n_tokens, a.max_q,
                     a.max_pages, a.window);
    if (a.n_seqs > ptc::ATTN_MAX_SEQS) SERVE_REFUSE("n_seqs %d passes %d", a.n_seqs, ptc::ATTN_MAX_SEQS);
    if (a.n_heads < 1 || a.n_heads % a.cache.n_kv_heads)
        SERVE_REFUSE("n_heads %d is no multiple of n_kv_heads %d", a.n_heads, a.cache.n_kv_heads);
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) SERVE_REFUSE("scale is not finite");
    if ((long long)a.n_tokens * a.n_heads > ptc::ATTN_MAX_KEYS) SERVE_REFUSE("n_tokens * n_heads passes 2^30");
    if (a.n_seqs == 0 || a.n_tokens == 0) return 0;
    if (a.window >= ptc::ATTN_MAX_KEYS) a.window = 0;   // it hides nothing
    const long long u = 16 / ptc::dtype_bytes(a.cache.dtype), hd = a.cache.head_dim;
    if (!a.q || !a.out || !a.page_table || !a.kv_len || !a.q_start || !a.workspace) SERVE_REFUSE("a required pointer is NULL");
    if (!ptc::aligned16(a.q) || !ptc::aligned16(a.out) || a.q_stride % u || a.out_stride % u ||
        a.q_stride < a.n_heads * hd || a.out_stride < a.n_heads * hd)
        SERVE_REFUSE("q and out have to be 16-byte aligned, their strides multiples of 16 bytes that hold a row");
    if (((uintptr_t)a.workspace & 255) || a.workspace_bytes < PTC_ATTN_WORKSPACE_BYTES)
        SERVE_REFUSE("the workspace needs %zu bytes at a 256-byte boundary", PTC_ATTN_WORKSPACE_BYTES);
    cudaStream_t s = (cudaStream_t)stream;
    ptc::MemoryDevice on(a.out);
    SERVE_CUDA(on.error());
    int n_sm = 0;
    SERVE_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, on.device()));
    const ptc::Group group(a.n_heads / a.cache.n_kv_heads);
    const long long most = (long long)(a.max_q < 1 ? 1 : a.max_q) * group.n;   // rows of a K/V head
    // The kernel by the rows of the longest sequence: few rows are bound by reading the keys, which the few-rows kernel
    // does with less to start, many by the products. Measured in a graph at 8 K/V heads, few-rows against many-rows
    // kernel, us, for 16 sequences of about 1000 positions (64 of 250; 4 of 8000):
    //   bf16, heads of 128  16 rows 29, 46 (37, 62; 46, 57)  32 rows 40, 46 (58, 61; 61, 58)  48 rows 52, 45 (79, 61; 77, 59)
    //   f16, heads of 64    32 rows 27, 37 (37, 51; 39, 44)  48 rows 35, 38 (47, 50; 49, 44)  64 rows 42, 39 (58, 52; 54, 42)
    //   f32, heads of 64    16 rows 46, 71 (65, 92)  24 rows 67, 84 (84, 93)  32 rows 92, 94 (114, 96)
    //   f32, heads of 128   16 rows 96, 137 (137, 173)  24 rows 146, 154 (192, 177)  32 rows 207, 166 (260, 180)
    if (a.cache.dtype == PTC_F32) {
        // rows in registers: as many as the longest sequence fills, up to 8
        if (most > 24) SERVE_CUDA(ptc::launch_attn_f32(a, group, n_sm, s));
        else if (most <= 1) SERVE_CUDA((ptc::launch_narrow_hd<float, 1>(a, group, n_sm, s)));
        else if (most <= 4) SERVE_CUDA((ptc::launch_narrow_hd<float, 4>(a, group, n_sm, s)));
        else SERVE_CUDA((ptc::launch_narrow_hd<float, 8>(a, group, n_sm, s)));
    } else if (most > 32 && a.scale > 0.f) {
        SERVE_CUDA(ptc::launch_attn_wide(a, group, n_sm, s));
    } else if (a.cache.dtype == PTC_F16) {
        SERVE_CUDA((ptc::launch_narrow_hd<__half, 16>(a, group, n_sm, s)));
    } else {
        SERVE_CUDA((ptc::launch_narrow_hd<__nv_bfloat16, 16>(a, group, n_sm, s)));
    }
    return 0;
}
