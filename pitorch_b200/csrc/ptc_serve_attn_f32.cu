// ptc_serve_attn_f32.cu -- attention of new tokens over a paged KV cache
// (include/ptc_serve.h): the kernel for many rows per K/V head in f32.
//
// Bound by fused multiply-adds (the tensor cores have no f32 product; three
// bf16 parts of each factor would take six products and three times the
// shared memory, which the queries of a tile alone would fill). A CTA has 64
// rows and 64 keys at a time; a thread 4 x 4 scores and 4 rows of outputs, so
// that a 128-bit read of shared memory feeds 8 multiply-adds a lane. The
// sixteen threads of a row are one half-warp, which keeps the row's maximum,
// sum and probabilities among themselves; the keys of the next unit are on
// their way meanwhile. Measured: 2048 tokens behind up to 2048, 16 heads of 128:
// 36 TFLOP/s, half of what the multiply-add units can do; nine prompts of up to
// 255 tokens, 6 heads of 48: 26 us, bound by the chain of one item's steps.
#include "ptc_serve_attn.cuh"

namespace ptc {

constexpr int FA_ROWS = 64, FA_KEYS = 64, FA_THREADS = 256;
constexpr int FA_MAX_CTAS = 296;   // the parts that one item can have

template <int HDP>
struct F32Shape {
    static constexpr int ROW = HDP + 4;              // floats of a row: 16 bytes more, so that 8 rows lie in 8 bank groups
    static constexpr int TILE = FA_KEYS * ROW;
    static constexpr int P_ROW = FA_KEYS + 4;
    static constexpr int FLOATS = 5 * TILE + FA_ROWS * P_ROW;   // queries, two stages of K and V, probabilities
    static constexpr int SLOT = FA_ROWS * (HDP + 2);
};

template <int HDP>
__global__ void __launch_bounds__(FA_THREADS) k_attn_f32(ptc_attn_args a, Group group) {
    using S = F32Shape<HDP>;
    constexpr int E = HDP / 32;   // pairs of outputs of a thread and row
    extern __shared__ __align__(16) float fa_smem[];
    __shared__ long long scratch[FA_THREADS / 32];
    __shared__ long long cells[3][FA_KEYS];   // where the keys of three units lie (-1: nowhere)
    __shared__ int last;
    float *const qs = fa_smem, *const kv = qs + S::TILE, *const ps = kv + 4 * S::TILE;
    int *pre = (int *)(fa_smem + S::FLOATS);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, hd = a.cache.head_dim, heads = a.cache.n_kv_heads;
    unsigned *flags = (unsigned *)a.workspace;
    float *slots = (float *)((char *)a.workspace + ATTN_FLAG_BYTES);

    attn_prefix<FA_ROWS, FA_KEYS, FA_THREADS>(a, group, pre, scratch);
    const int total = pre[a.n_seqs] * heads, C = min((int)gridDim.x, total), c = blockIdx.x;
    if (c >= C) return;
    const int u1 = attn_first(c + 1, C, total);
    const float scale = a.scale * LOG2E;

    for (int u = attn_first(c, C, total); u < u1;) {
        const AttnItem it = attn_find<FA_ROWS, FA_KEYS>(a, group, pre, u);
        const int seg0 = u - it.first, n = min(it.units - seg0, u1 - u), rows = it.i1 - it.i0;
        const int first = (it.lo / FA_KEYS + seg0) * FA_KEYS;
        const int *table = a.page_table + (long long)it.r * a.max_pages;
        const long long base = it.head * a.cache.head_stride;
        auto look = [&](int j) {   // the cells of unit j, by the first threads
            const int t = first + j * FA_KEYS + tid;
            if (tid >= FA_KEYS || j >= n) return;
            long long cell = -1;
            if (t < it.hi && t >= it.lo) {
                const int page = t / a.cache.page_size;
                cell = attn_cell(a, table[page], t - page * a.cache.page_size);
                if (cell < 0) serve_err(a.err, PTC_SERVE_ERR_INDEX);
            }
            cells[j % 3][tid] = cell;
        };
        auto fill = [&](int j) {   // unit j into its stage
            if (j < n) {
                float *k = kv + (j & 1) * 2 * S::TILE, *v = k + S::TILE;
                for (int x = tid; x < FA_KEYS * (HDP / 4); x += FA_THREADS) {
                    const int key = x / (HDP / 4), d = x % (HDP / 4) * 4;
                    const long long cell = cells[j % 3][key];
                    const bool real = cell >= 0 && d < hd;
                    const long long off = real ? cell + base + d : 0;
                    cp_async16_or_zero(smem_u32(k + key * S::ROW + d), (const float *)a.cache.k + off, real);
                    cp_async16_or_zero(smem_u32(v + key * S::ROW + d), (const float *)a.cache.v + off, real);
                }
            }
            cp_async_commit();
        };
        look(0);
        look(1);
        __syncthreads();
        for (int x = tid; x < FA_ROWS * (HDP / 4); x += FA_THREADS) {
            const int r = x / (HDP / 4), d = x % (HDP / 4) * 4, row = it.i0 + r, tok = group.div(row);
            const bool real = r < rows && d < hd;
            const long long off = real ? (it.s.q0 + tok) * a.q_stride + (long long)(it.head * group.n + row - tok * group.n) * hd + d : 0;
            cp_async16_or_zero(smem_u32(qs + r * S::ROW + d), (const float *)a.q + off, real);
        }
        fill(0);
        float o[4][E][2], m[4], l[4];
        int lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = ty * 4 + i, pos = it.s.pos0 + group.div(it.i0 + r);
            hi[i] = r < rows ? min(pos + 1, it.s.cap) : 0;
            lo[i] = a.window > 0 ? pos - a.window + 1 : 0;
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) o[i][e][0] = o[i][e][1] = 0.f;
        }
        for (int j = 0; j < n; j++) {
            cp_async_wait<0>();
            __syncthreads();   // unit j is there, and nobody reads the other stage any more
            fill(j + 1);
            look(j + 2);
            const float *k = kv + (j & 1) * 2 * S::TILE, *v = k + S::TILE;
            const long long *cell = cells[j % 3];
            float s[4][4];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int b = 0; b < 4; b++) s[i][b] = 0.f;
#pragma unroll 4
            for (int d = 0; d < hd; d += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = *(const float4 *)(qs + (ty * 4 + i) * S::ROW + d);
#pragma unroll
                for (int b = 0; b < 4; b++) y[b] = *(const float4 *)(k + (tx + 16 * b) * S::ROW + d);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int b = 0; b < 4; b++) s[i][b] = dot4(x[i], y[b], s[i][b]);
            }
            bool there[4];
#pragma unroll
            for (int b = 0; b < 4; b++) there[b] = cell[tx + 16 * b] >= 0;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float top = m[i];
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const int t = first + j * FA_KEYS + tx + 16 * b;
                    s[i][b] = there[b] && t < hi[i] && t >= lo[i] ? s[i][b] * scale : -INFINITY;
                    top = fmaxf(top, s[i][b]);
                }
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float ref = top == -INFINITY ? 0.f : top, f = exp2f(m[i] - ref);
                m[i] = top;
                l[i] *= f;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const float p = exp2_fast(s[i][b] - ref);
                    l[i] += p;
                    ps[(ty * 4 + i) * S::P_ROW + tx + 16 * b] = p;
                }
#pragma unroll
                for (int e = 0; e < E; e++) o[i][e][0] *= f, o[i][e][1] *= f;
            }
            __syncwarp();
#pragma unroll 2
            for (int t = 0; t < FA_KEYS; t += 4) {
                float4 p[4];
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] = *(const float4 *)(ps + (ty * 4 + i) * S::P_ROW + t);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    float2 y[4];
#pragma unroll
                    for (int b = 0; b < 4; b++) y[b] = *(const float2 *)(v + (t + b) * S::ROW + 32 * e + 2 * tx);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        o[i][e][0] = fmaf(p[i].w, y[3].x, fmaf(p[i].z, y[2].x, fmaf(p[i].y, y[1].x, fmaf(p[i].x, y[0].x, o[i][e][0]))));
                        o[i][e][1] = fmaf(p[i].w, y[3].y, fmaf(p[i].z, y[2].y, fmaf(p[i].y, y[1].y, fmaf(p[i].x, y[0].y, o[i][e][1]))));
                    }
                }
            }
            __syncwarp();
        }
        cp_async_wait<0>();

        const bool whole = n == it.units;
        float *slot = slots + (long long)(2 * c + (seg0 == 0)) * S::SLOT;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = ty * 4 + i, row = it.i0 + r, tok = group.div(row);
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
            if (r >= rows) continue;
            const float inv = l[i] > 0.f ? 1.f / l[i] : 0.f;
            float *dst = whole ? (float *)a.out + (it.s.q0 + tok) * a.out_stride + (long long)(it.head * group.n + row - tok * group.n) * hd : slot + r * HDP;
#pragma unroll
            for (int e = 0; e < E; e++)
                if (32 * e + 2 * tx < hd) *(float2 *)(dst + 32 * e + 2 * tx) = whole ? make_float2(o[i][e][0] * inv, o[i][e][1] * inv) : make_float2(o[i][e][0], o[i][e][1]);
            if (!whole && tx == 0) slot[FA_ROWS * HDP + r] = m[i], slot[FA_ROWS * (HDP + 1) + r] = l[i];
        }
        if (!whole) {
            const int c0 = attn_owner(it.first, C, total), c1 = attn_owner(it.first + it.units - 1, C, total);
            __syncthreads();
            if (tid == 0) last = atom_add_acq_rel(&flags[c0], 1u) == (unsigned)(c1 - c0);
            __syncthreads();
            if (last) {
                attn_merge<float, HDP, FA_ROWS, S::SLOT, FA_THREADS>(a, it, group, slots, c0, c1, fa_smem);
                if (tid == 0) flags[c0] = 0;
            }
        }
        __syncthreads();   // the next item fills the tiles again
        u += n;
    }
}

template <int HDP>
static cudaError_t launch(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s) {
    using S = F32Shape<HDP>;
    static_assert(FA_ROWS * FA_MAX_CTAS + 3 + FA_ROWS * HDP <= S::FLOATS, "a merge fits the tiles");
    static_assert(FA_MAX_CTAS * 2 * (long long)S::SLOT * 4 + ATTN_FLAG_BYTES <= (long long)PTC_ATTN_WORKSPACE_BYTES, "two slots for each CTA");
    auto kernel = k_attn_f32<HDP>;
    const int smem = attn_smem(S::FLOATS * 4, a.n_seqs);
    cudaError_t e = allow_smem(kernel, attn_smem(S::FLOATS * 4, ATTN_MAX_SEQS));
    int per = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, FA_THREADS, smem);
    if (e != cudaSuccess) return e;
    if (per < 1) return cudaErrorInvalidConfiguration;
    const int grid = per * n_sm < FA_MAX_CTAS ? per * n_sm : FA_MAX_CTAS;
    return launch_kernel(kernel, grid, FA_THREADS, smem, s, a, group);
}

cudaError_t launch_attn_f32(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s) {
    return a.cache.head_dim <= 64 ? launch<64>(a, group, n_sm, s) : launch<128>(a, group, n_sm, s);
}

}  // namespace ptc
