// ptc_serve_attn_wide.cu -- attention of new tokens over a paged KV cache
// (include/ptc_serve.h): the kernel for many rows per K/V head, 16-bit types.
//
// One CTA per SM on tcgen05 tensor cores. An item has 256 rows, as two tiles
// of 128 that share every K/V tile of 128 keys. A row tile's keys are taken in
// halves of 64, so that the scores of one half are made while the other half's
// become probabilities: the softmax takes as long as the products, and neither
// may wait for the other. (With 128 keys at a time, which tensor memory holds
// once beside the outputs, a row tile's softmax and products alternate.)
//
//   warps 0-3, 4-7  softmax of tile 0 and 1, a thread per row: scores from
//                   tensor memory, running maximum and sum, probabilities back
//                   to tensor memory as the A operand of the second product
//   warp 8          one lane issues the products: S = Q K^T (128 x 64 per tile and
//                   half) and O += P V, in an order in which each S follows the
//                   product that read the P in the same place
//   warps 9-10      Q and K tiles into shared memory, warp 11 V tiles, in the
//                   128-byte swizzle that the tensor cores read: by TMA, a box
//                   for each run of tokens that lie in one page (8 to 64); by
//                   16-byte asynchronous copies where a run ends behind the last
//                   position, and where page sizes are no multiple of 8
// Measured: 4096 tokens behind 12288 cached ones, 32 heads in groups of 4, 128
// elements of bf16: 0.96 to 1.05 ms from box to box and run to run, 1005 to 914
// TFLOP/s (0.61 to 0.55 of the measured bf16 product);
// the products alone take 0.72 ms and the softmax alone 0.68 ms. Exponentials
// as polynomials on the multiply-add units were slower (1.03 ms with an eighth
// of them, 1.06 with a quarter), and so were two copies of the softmax loop,
// one per half (1.46 ms: they do not stay in the instruction cache).
// Twelve warps are three to a scheduler, which leaves a thread 168 registers;
// a thirteenth would leave 128.
//
// Tensor memory: S0 | S1 | O0 | O1; the P of a half takes the place of its
// S. The running maximum is replaced, and O rescaled, only when it rises by
// more than 2^8 (probabilities and sums are relative to the same value, so
// nothing is lost: they stay below 2^8 and 2^8 times the keys).
#include <cuda.h>
#include <limits.h>
#include <string.h>

#include <type_traits>

#include "ptc_serve_attn.cuh"

namespace ptc {

constexpr int WA_ROWS = 256, WA_TILE = 128, WA_KEYS = 128, WA_HALF = 64;
constexpr int WA_THREADS = 12 * 32;
constexpr int WA_K_WARPS = 2, WA_V_WARPS = 1;   // that load
constexpr float WA_RISE = 8.f;
// Tensor memory, all 512 columns of it (so it begins at column 0).
constexpr unsigned TM_S = 0, TM_O = 2 * WA_KEYS;
constexpr int TM_COLS = 512;

// ---- tcgen05 ------------------------------------------------------------------

__device__ __forceinline__ void tm_alloc(unsigned *where, int cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(where)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_free(unsigned at, int cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    unsigned yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ void tc_mma_ss(unsigned d, uint64_t a, uint64_t b, unsigned idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
        "r"(idesc), "r"((int)add)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(unsigned d, unsigned a, uint64_t b, unsigned idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b),
        "r"(idesc), "r"((int)add)
        : "memory");
}
// Columns of this warp's 32 lanes. Loaded values may be used after tm_wait_ld on
// them (the registers pass through it, so that no use moves before it).
__device__ __forceinline__ void tm_ld16(uint32_t (&r)[16], unsigned at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void tm_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_st16(unsigned at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, "
                 "%9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                   "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t (&r)[32], unsigned at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
                   "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
                   "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
}
__device__ __forceinline__ void tm_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                   "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                   "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two 32-bit operations in one instruction: (a, b) = (x, y) * s + t, (a, b) += (x, y).
__device__ __forceinline__ void fma_pair(float &a, float &b, float x, float y, float s, float t) {
    asm("{\n .reg .b64 u, v, w;\n mov.b64 u, {%2, %3};\n mov.b64 v, {%4, %4};\n mov.b64 w, {%5, %5};\n fma.rn.f32x2 u, u, v, w;\n"
        " mov.b64 {%0, %1}, u;\n}"
        : "=f"(a), "=f"(b)
        : "f"(x), "f"(y), "f"(s), "f"(t));
}
__device__ __forceinline__ void add_pair(float &a, float &b, float x, float y) {
    asm("{\n .reg .b64 u, v;\n mov.b64 u, {%0, %1};\n mov.b64 v, {%2, %3};\n add.rn.f32x2 u, u, v;\n mov.b64 {%0, %1}, u;\n}"
        : "+f"(a), "+f"(b)
        : "f"(x), "f"(y));
}

// Shared-memory operand in the 128-byte swizzle: 16-bit elements in blocks of
// 64 columns (128 bytes a row), 8 rows an atom of 1024 bytes.
//   along K (rows are M or N): atoms `1024` apart
//   along M/N (rows are K, V as it lies in memory): blocks of 64 `lbo` apart,
//   groups of 8 rows 1024 apart
__device__ __forceinline__ uint64_t operand(unsigned at, unsigned lbo) {
    return (uint64_t)((at >> 4) & 0x3fff) | (uint64_t)((lbo >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: f32 accumulator, 16-bit A and B, 128 rows; b_mn: B's columns are contiguous.
template <typename T>
__device__ __forceinline__ unsigned instruction(int n, bool b_mn) {
    const unsigned f = Elem<T>::TYPE == PTC_BF16 ? 1 : 0;
    return 1u << 4 | f << 7 | f << 10 | (unsigned)b_mn << 16 | (unsigned)(n >> 3) << 17 | (unsigned)(WA_TILE >> 4) << 24;
}

// ---- the kernel -----------------------------------------------------------------

struct WideBars {
    uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t s_full[2][2], p_full[2][2];   // by row tile and half of the keys
    uint64_t o_done[2], o_full[2], done;   // a product into a tile's O; an item's last one; all products
};

struct WideShared {
    WideBars bar;
    unsigned bad[4][4];   // keys of a K tile whose page is out of range
    unsigned tmem;
    int gave_up;
    int last;
    float weight[8][WA_ROWS];   // of a merge
    long long scratch[WA_THREADS / 32];
};

template <int HDP>
struct WideShape {
    static constexpr int Q = WA_ROWS * HDP * 2, KV = WA_KEYS * HDP * 2;
    static constexpr int BYTES = Q + 4 * KV;                // Q, two K, two V
    static constexpr int SLOT = WA_ROWS * (HDP + 2);        // floats of a workspace slot
};

// A wait that gives up (and makes every later one give up at once): the
// loading warps then stop, as the stage may still be written or read, the
// others run to their end, and the kernel waits for its own copies and
// products, frees its tensor memory and reports it. (What only a failed or a
// last wait needs is kept out of the loops' code: 1049 us for the long chunk
// against 1065 with it in them.)
struct Waiter {
    volatile int *gave_up;
    int *err;
    __device__ void operator()(uint64_t *bar, unsigned parity) const {
        for (int it = 0; it < 1 << 22; it++) {
            if (mbar_try_wait(bar, parity)) return;
            if ((it & 63) == 63 && *gave_up) return;
        }
        failed();
    }
    // For what is on its way into shared or tensor memory when a role ends,
    // which may not outlive the CTA: whether or not another wait gave up.
    __device__ __noinline__ void landed(uint64_t *bar, unsigned parity) const {
        if (!mbar_wait_bounded(bar, parity, nullptr, 0)) failed();
    }
    __device__ __noinline__ void failed() const {
        *gave_up = 1;
        serve_err(err, PTC_SERVE_ERR_WAIT);
    }
};

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// One group's loads: the previous one is handed over (its barrier arrived at,
// after a fence towards the tensor cores' reads) when the next is under way.
struct Handover {
    uint64_t *pending = nullptr;
    template <int LEFT>
    __device__ void done() {
        if (!pending) return;
        asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
        fence_proxy_async_smem();
        mbar_arrive(pending);
        pending = nullptr;
    }
    __device__ void issued(uint64_t *bar) {
        cp_async_commit();
        done<1>();
        pending = bar;
    }
};

// Where 16-byte chunk `ch` of row `row` lies in a tile of `rows` rows.
__device__ __forceinline__ unsigned swizzled(int rows, int row, int ch) {
    return (unsigned)((ch >> 3) * rows * 128 + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
}

// The cache as TMA sees it: (element, token of the page, head, page) with
// boxes of 64 elements and `run` tokens; run 0: it cannot be read that way.
struct WideMaps {
    CUtensorMap k, v;
    int run;
};

__device__ __forceinline__ void tma_box(unsigned dst, const CUtensorMap *map, int x, int token, int head, int page, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(token), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

// The loading warps of one kind (K with Q, or V): WARPS of them, of which this
// is the w-th. A lane looks up the cells of every 32nd key of its warp's share.
template <typename T, int HDP, int WARPS, bool KEYS>
__device__ void load_tiles(const ptc_attn_args &a, const CUtensorMap *map, int run, Group group, const int *pre, int u0, int u1, WideShared &sh, unsigned q_at, unsigned at, int w,
                           const Waiter &wait) {
    using S = WideShape<HDP>;
    constexpr int CH = HDP / 8, SHARE = WA_KEYS / WARPS, LOOKS = SHARE / 32;
    const int lane = threadIdx.x & 31, hd = a.cache.head_dim;
    const T *from = (const T *)(KEYS ? a.cache.k : a.cache.v);
    uint64_t *full = KEYS ? sh.bar.k_full : sh.bar.v_full, *empty = KEYS ? sh.bar.k_empty : sh.bar.v_empty;
    Handover over;
    int n = 0, items = 0;   // tiles and items so far
    auto stopped = [&] { return __any_sync(0xffffffffu, *wait.gave_up); };
    for (int u = u0; u < u1; items++) {
        const AttnItem it = attn_find<WA_ROWS, WA_KEYS>(a, group, pre, u);
        const int seg0 = u - it.first, tiles = min(it.units - seg0, u1 - u);
        const int *table = a.page_table + (long long)it.r * a.max_pages;
        const long long head = it.head * a.cache.head_stride;
        // a lane's run of tokens of a tile: its page, looked up one tile ahead
        const int key = w * SHARE + lane * run;
        const bool runs = run && lane * run < SHARE;
        auto look = [&](int j) {
            const int t = (it.lo / WA_KEYS + seg0 + j) * WA_KEYS + key;
            return runs && j < tiles && t < it.hi && t + run > it.lo ? table[t / a.cache.page_size] : -1;
        };
        int page = look(0);
        if (KEYS) {
            over.done<0>();   // the last S of the item before needs its K tile
            if (items > 0) wait(&sh.bar.q_empty, (items - 1) & 1);
            if (stopped()) goto end;
            // a lane has one chunk of every RATE-th row
            constexpr int RATE = WARPS * 32 / CH;
            const int ch = (w * 32 + lane) % CH;
#pragma unroll 4
            for (int row = (w * 32 + lane) / CH; row < WA_ROWS; row += RATE) {
                const int i = it.i0 + row, tok = group.div(i);
                const bool real = i < it.i1 && ch * 8 < hd;
                const long long off = real ? (it.s.q0 + tok) * a.q_stride + (long long)(it.head * group.n + i - tok * group.n) * hd + ch * 8 : 0;
                cp_async16_or_zero(q_at + (row >> 7) * (S::Q / 2) + swizzled(WA_TILE, row & 127, ch), (const T *)a.q + off, real);
            }
            over.issued(&sh.bar.q_full);
        }
        for (int j = 0; j < tiles; j++, n++) {
            const int s = n & 1, first = (it.lo / WA_KEYS + seg0 + j) * WA_KEYS, mine = page;
            const unsigned stage = at + s * S::KV;
            page = look(j + 1);
            if (run && first >= it.lo && first + WA_KEYS <= it.hi && __all_sync(0xffffffffu, !runs || (unsigned)mine < (unsigned)a.cache.n_pages)) {
                // a whole tile
                if (KEYS && lane < LOOKS) sh.bad[n & 3][w * LOOKS + lane] = 0;
                if (n >= 2) wait(&empty[s], ((n >> 1) - 1) & 1);
                if (stopped()) goto end;
                if (lane == 0) mbar_expect_tx(&full[s], SHARE * HDP * 2);
                else mbar_arrive(&full[s]);
                if (runs)
#pragma unroll
                    for (int b = 0; b < HDP / 64; b++)
                        tma_box(stage + b * WA_KEYS * 128 + key * 128, map, b * 64, (first + key) % a.cache.page_size, it.head, mine, &full[s]);
                over.done<0>();
                continue;
            }
            if (run) {
                // Whole runs by TMA, from the first that is seen on. A run that ends behind the last position is
                // copied with zeros there, as what lies there may be anything, and V's other runs become zeros
                // (the scores of K's are masked, whatever the stage holds).
                const int t = first + key;
                const bool seen = runs && t < it.hi && t + run > it.lo, there = (unsigned)mine < (unsigned)a.cache.n_pages;
                const bool whole = seen && there && t + run <= it.hi;
                if (KEYS) {
                    if (lane < LOOKS) sh.bad[n & 3][w * LOOKS + lane] = 0;
                    __syncwarp();
                }
                if (seen && !there) {
                    serve_err(a.err, PTC_SERVE_ERR_INDEX);
                    if (KEYS)
                        for (int b = 0; b < run; b += 32) atomicOr(&sh.bad[n & 3][(key + b) >> 5], (run < 32 ? (1u << run) - 1 : ~0u) << (key & 31));
                }
                const int edge = __ffs(__ballot_sync(0xffffffffu, seen && there && !whole)) - 1;   // the lane of a run that ends inside
                const unsigned boxes = __popc(__ballot_sync(0xffffffffu, whole));
                if (n >= 2) {
                    if (!__all_sync(0xffffffffu, mbar_try_wait(&empty[s], ((n >> 1) - 1) & 1))) over.done<0>();
                    wait(&empty[s], ((n >> 1) - 1) & 1);
                }
                if (stopped()) goto end;
                if (!KEYS) {
                    unsigned none = __ballot_sync(0xffffffffu, runs && !(seen && there));
                    if (none) {
                        for (; none; none &= none - 1)
                            for (int x = lane; x < run * CH; x += 32) {
                                const int k = (__ffs(none) - 1) * run + x / CH;
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(stage + swizzled(WA_KEYS, k, x % CH)), "r"(0) : "memory");
                            }
                        fence_proxy_async_smem();
                    }
                }
                if (lane == 0) asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[s])), "r"(boxes * run * HDP * 2) : "memory");
                __syncwarp();
                if (whole)
#pragma unroll
                    for (int b = 0; b < HDP / 64; b++)
                        tma_box(stage + b * WA_KEYS * 128 + key * 128, map, b * 64, t % a.cache.page_size, it.head, mine, &full[s]);
                if (edge >= 0) {
                    const int p = __shfl_sync(0xffffffffu, mine, edge), k0 = w * SHARE + edge * run, te = first + k0;
                    const long long cell = attn_cell(a, p, te % a.cache.page_size);
#pragma unroll 4
                    for (int x = lane; x < run * CH; x += 32) {
                        const int k = x / CH, ch = x % CH;
                        const bool real = te + k < it.hi && ch * 8 < hd;
                        cp_async16_or_zero(stage + swizzled(WA_KEYS, k0 + k, ch), from + (real ? cell + k * a.cache.token_stride + head + ch * 8 : 0), real);
                    }
                    over.issued(&full[s]);
                } else {
                    over.done<0>();
                    mbar_arrive(&full[s]);
                }
                continue;
            }
            const int t0 = first + w * SHARE + lane;
            long long cell[LOOKS];
#pragma unroll
            for (int g = 0; g < LOOKS; g++) {
                const int t = t0 + g * 32;
                const bool want = t < it.hi && t >= it.lo;
                cell[g] = -1;
                if (want) {
                    const int page = t / a.cache.page_size;
                    cell[g] = attn_cell(a, table[page], t - page * a.cache.page_size);
                    if (cell[g] < 0) serve_err(a.err, PTC_SERVE_ERR_INDEX);
                }
                const unsigned bad = __ballot_sync(0xffffffffu, want && cell[g] < 0);
                if (KEYS && lane == 0) sh.bad[n & 3][w * LOOKS + g] = bad;
            }
            if (n >= 2 && !__all_sync(0xffffffffu, mbar_try_wait(&empty[s], ((n >> 1) - 1) & 1))) {
                over.done<0>();   // the stage is still read: meanwhile hand over what has landed
                wait(&empty[s], ((n >> 1) - 1) & 1);
            }
            if (stopped()) goto end;
#pragma unroll
            for (int g = 0; g < LOOKS; g++)
#pragma unroll 4
                for (int i = 0; i < CH; i++) {
                    const int x = i * 32 + lane, k = x / CH, ch = x % CH;
                    const long long c = __shfl_sync(0xffffffffu, cell[g], k);
                    const bool real = c >= 0 && ch * 8 < hd;
                    cp_async16_or_zero(stage + swizzled(WA_KEYS, w * SHARE + g * 32 + k, ch), from + (real ? c + head + ch * 8 : 0), real);
                }
            over.issued(&full[s]);
        }
        u += tiles;
    }
end:
    over.done<0>();
    for (int k = max(0, n - 2); k < n; k++) wait.landed(&full[k & 1], (k >> 1) & 1);
}

template <typename T, int HDP>
__global__ void __launch_bounds__(WA_THREADS, 1) k_attn_wide(ptc_attn_args a, const __grid_constant__ WideMaps maps, Group group) {
    using S = WideShape<HDP>;
    extern __shared__ char wa_raw[];
    __shared__ WideShared sh;
    char *wa_smem = wa_raw + (-smem_u32(wa_raw) & 1023);   // the swizzle is by address: whole atoms
    const int tid = threadIdx.x, warp = tid >> 5, heads = a.cache.n_kv_heads, hd = a.cache.head_dim;
    const unsigned q_at = smem_u32(wa_smem), k_at = q_at + S::Q, v_at = k_at + 2 * S::KV;
    int *pre = (int *)(wa_smem + S::BYTES);
    unsigned *flags = (unsigned *)a.workspace;
    float *slots = (float *)((char *)a.workspace + ATTN_FLAG_BYTES);

    attn_prefix<WA_ROWS, WA_KEYS, WA_THREADS>(a, group, pre, sh.scratch);
    const int total = pre[a.n_seqs] * heads, C = min((int)gridDim.x, total), c = blockIdx.x;
    if (c >= C) return;
    const int u0 = attn_first(c, C, total), u1 = attn_first(c + 1, C, total);

    if (tid == 0) {
        WideBars &b = sh.bar;
        mbar_init(&b.q_full, WA_K_WARPS * 32);
        mbar_init(&b.q_empty, 1);
        mbar_init(&b.done, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&b.k_full[i], WA_K_WARPS * 32);
            mbar_init(&b.v_full[i], WA_V_WARPS * 32);
            mbar_init(&b.k_empty[i], 1);
            mbar_init(&b.v_empty[i], 1);
            for (int h = 0; h < 2; h++) {
                mbar_init(&b.s_full[i][h], 1);
                mbar_init(&b.p_full[i][h], WA_TILE);
            }
            mbar_init(&b.o_done[i], 1);
            mbar_init(&b.o_full[i], 1);
        }
        sh.gave_up = 0;
        mbar_init_fence();
    }
    if (warp == 8) tm_alloc(&sh.tmem, TM_COLS);
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const Waiter wait = {&sh.gave_up, a.err};

    if (warp >= 9 + WA_K_WARPS) {
        load_tiles<T, HDP, WA_V_WARPS, false>(a, &maps.v, maps.run, group, pre, u0, u1, sh, q_at, v_at, warp - 9 - WA_K_WARPS, wait);
    } else if (warp >= 9) {
        load_tiles<T, HDP, WA_K_WARPS, true>(a, &maps.k, maps.run, group, pre, u0, u1, sh, q_at, k_at, warp - 9, wait);
    } else if (warp == 8) {
        // ---- products ----
        // The warp stays together and one elected lane issues. Every operand is
        // known before the loop (shared memory at its place, all of the tensor
        // memory, the two stages as two copies of the code), so none has to be
        // brought into the uniform registers that the instruction reads.
        constexpr int IN_BLOCK = 4;   // steps of 16 columns in a swizzled block
        const unsigned id_s = instruction<T>(WA_HALF, false), id_o = instruction<T>(HDP, true);
        typedef std::integral_constant<int, 0> Zero;
        typedef std::integral_constant<int, 1> One;
        auto scores = [&](auto t_, auto h_, auto s_) {   // S_t = Q_t K^T of half h of the keys
            constexpr int t = t_.value, h = h_.value, s = s_.value;
#pragma unroll
            for (int k = 0; k < HDP / 16; k++) {
                const unsigned off = (k / IN_BLOCK) * WA_TILE * 128 + (k % IN_BLOCK) * 32;
                tc_mma_ss(TM_S + t * WA_KEYS + h * WA_HALF, operand(q_at + t * (S::Q / 2) + off, 16),
                          operand(k_at + s * S::KV + h * WA_HALF * 128 + off, 16), id_s, k > 0);
            }
            tc_commit(&sh.bar.s_full[t][h]);
        };
        auto values = [&](auto t_, auto h_, auto s_, bool add) {   // O_t += P_t V of half h of the keys, 16 a step
            constexpr int t = t_.value, h = h_.value, s = s_.value;
#pragma unroll
            for (int k = 0; k < WA_HALF / 16; k++)
                tc_mma_ts(TM_O + t * HDP, TM_S + t * WA_KEYS + h * WA_HALF + k * 8, operand(v_at + s * S::KV + (h * WA_HALF + k * 16) * 128, WA_KEYS * 128),
                          id_o, add || h > 0 || k > 0);
            tc_commit(&sh.bar.o_done[t]);
        };
        int n = 0, items = 0, phase[2] = {0, 0};   // K/V tiles, items, K/V tiles of each row tile
        // the products of one K/V tile, stage s, and the scores of the next
        auto step = [&](auto s_, bool both, bool add, bool more, bool done) {
            constexpr int s = s_.value;
            wait(&sh.bar.v_full[s], (n >> 1) & 1);
            if (more) wait(&sh.bar.k_full[1 - s], ((n + 1) >> 1) & 1);
            auto part = [&](auto t_, auto h_) {
                constexpr int t = t_.value, h = h_.value;
                wait(&sh.bar.p_full[t][h], phase[t] & 1);
                tc_after_sync();
                if (elect_one()) {
                    values(t_, h_, s_, add);
                    if (more) scores(t_, h_, std::integral_constant<int, 1 - s>());
                    else if (h == 1) tc_commit(&sh.bar.o_full[t]);
                }
            };
            part(Zero(), Zero());
            if (both) part(One(), Zero());
            part(Zero(), One());
            if (both) part(One(), One());
            phase[0]++;
            phase[1] += both;
            if (elect_one()) {
                tc_commit(&sh.bar.v_empty[s]);
                if (more) tc_commit(&sh.bar.k_empty[1 - s]);
                if (done) tc_commit(&sh.bar.q_empty);
            }
        };
        auto first = [&](auto s_, bool both, bool done) {
            constexpr int s = s_.value;
            if (elect_one()) {
                scores(Zero(), Zero(), s_);
                if (both) scores(One(), Zero(), s_);
                scores(Zero(), One(), s_);
                if (both) scores(One(), One(), s_);
                tc_commit(&sh.bar.k_empty[s]);
                if (done) tc_commit(&sh.bar.q_empty);
            }
        };
        for (int u = u0; u < u1; items++) {
            const AttnItem it = attn_find<WA_ROWS, WA_KEYS>(a, group, pre, u);
            const int tiles = min(it.units - (u - it.first), u1 - u);
            const bool both = it.i1 - it.i0 > WA_TILE;
            wait(&sh.bar.q_full, items & 1);
            wait(&sh.bar.k_full[n & 1], (n >> 1) & 1);
            tc_after_sync();
            if (n & 1) first(One(), both, tiles == 1);
            else first(Zero(), both, tiles == 1);
            for (int j = 0; j < tiles; j++, n++) {
                if (n & 1) step(One(), both, j > 0, j + 1 < tiles, j + 2 == tiles);
                else step(Zero(), both, j > 0, j + 1 < tiles, j + 2 == tiles);
            }
            u += tiles;
        }
        // (every product has been waited for, unless a wait has given up)
        if (elect_one()) tc_commit(&sh.bar.done);
        wait.landed(&sh.bar.done, 0);
        __syncwarp();
    } else {
        // ---- softmax ----
        const int t = warp >> 2, row = tid & 127;
        const unsigned lanes = (unsigned)(warp & 3) << 21;   // this warp's 32 lanes of tensor memory
        const unsigned s_tm = TM_S + t * WA_KEYS + lanes, o_tm = TM_O + t * HDP + lanes;
        const float scale = a.scale * LOG2E;
        int n = 0, sc = 0, oc = 0, ic = 0;   // K/V tiles; those of this row tile, products into its O, its items
        for (int u = u0; u < u1;) {
            const AttnItem it = attn_find<WA_ROWS, WA_KEYS>(a, group, pre, u);
            const int seg0 = u - it.first, tiles = min(it.units - seg0, u1 - u), rows = it.i1 - it.i0;
            const bool active = t * WA_TILE < rows;   // of the tile, the same for its four warps
            const int i = it.i0 + t * WA_TILE + row, tok = group.div(i);
            const bool real = i < it.i1;
            // rows that are not there see everything: their zeros need no masking
            const int pos = it.s.pos0 + tok, hi = real ? min(pos + 1, it.s.cap) : INT_MAX, lo = real && a.window > 0 ? pos - a.window + 1 : 0;
            float m = -INFINITY, l = 0.f;   // the reference of the probabilities, and their sum
            if (active) {
                for (int j = 0; j < tiles; j++, sc++) {
#pragma unroll 1   // (one copy: two do not stay in the instruction cache)
                    for (int h = 0; h < 2; h++) {
                        const int key0 = (it.lo / WA_KEYS + seg0 + j) * WA_KEYS + h * WA_HALF;
                        wait(&sh.bar.s_full[t][h], sc & 1);
                        __syncwarp();   // (the accesses to tensor memory are the warp's)
                        tc_after_sync();
                        uint32_t x[2][32];
                        tm_ld32(x[0], s_tm + h * WA_HALF);
                        tm_ld32(x[1], s_tm + h * WA_HALF + 32);
                        const unsigned *bad = &sh.bad[(n + j) & 3][2 * h];
                        const bool mask = (bad[0] | bad[1]) != 0 || __any_sync(0xffffffffu, key0 + WA_HALF > hi || key0 < lo);
                        float top = -INFINITY;
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            tm_wait_ld(x[q]);
                            if (mask) {   // what this row does not see: a bit per key
                                const int from = max(0, lo - key0 - q * 32), to = hi - key0 - q * 32;
                                unsigned see = to >= 32 ? ~0u : to > 0 ? (1u << to) - 1 : 0;
                                see &= from >= 32 ? 0 : ~0u << from;
                                see &= ~bad[q];
#pragma unroll
                                for (int k = 0; k < 32; k++)
                                    if (!(see >> k & 1)) x[q][k] = __float_as_uint(-INFINITY);
                            }
                            float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                m0 = fmaxf(m0, fmaxf(__uint_as_float(x[q][k]), __uint_as_float(x[q][k + 1])));
                                m1 = fmaxf(m1, fmaxf(__uint_as_float(x[q][k + 2]), __uint_as_float(x[q][k + 3])));
                            }
                            top = fmaxf(top, fmaxf(m0, m1));
                        }
                        top *= scale;
                        const bool rise = top > m + WA_RISE;
                        if (j == 0 && h == 0) {
                            m = top;
                        } else if (__any_sync(0xffffffffu, rise)) {
                            // (all products but the last one into this O were done when these scores were)
                            wait(&sh.bar.o_done[t], (oc - 1) & 1);
                            __syncwarp();
                            tc_after_sync();
                            const float f = rise ? exp2f(m - top) : 1.f;
                            if (rise) m = top;
                            l *= f;
#pragma unroll 1
                            for (int d = 0; d < HDP; d += 16) {
                                uint32_t o[16];
                                tm_ld16(o, o_tm + d);
                                tm_wait_ld(o);
#pragma unroll
                                for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                                tm_st16(o_tm + d, o);
                            }
                        }
                        const float ref = m == -INFINITY ? 0.f : m - Lift<T>::BY;
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            // rounded to the type for the product with V (their sum is not). What the rounding
                            // leaves is not multiplied too, as the few-rows kernel does: that product would add half
                            // of the products' time, and the output's own rounding is of the same size (error
                            // of the long chunk against 64 bits 0.0023, of the output's rounding alone 0.0017).
                            uint32_t p[16];
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                float e[4];
#pragma unroll
                                for (int i = 0; i < 4; i += 2) {
                                    fma_pair(e[i], e[i + 1], __uint_as_float(x[q][k + i]), __uint_as_float(x[q][k + i + 1]), scale, -ref);
                                    e[i] = exp2_fast(e[i]);
                                    e[i + 1] = exp2_fast(e[i + 1]);
                                    add_pair(sum[i], sum[i + 1], e[i], e[i + 1]);
                                }
                                p[k / 2] = pack2(e[0], e[1], T());
                                p[k / 2 + 1] = pack2(e[2], e[3], T());
                            }
                            tm_st16(s_tm + h * WA_HALF + q * 16, p);
                        }
                        tm_wait_st();
                        tc_before_sync();
                        mbar_arrive(&sh.bar.p_full[t][h]);
                        oc++;
                        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    }
                }
                wait(&sh.bar.o_full[t], ic++ & 1);
                __syncwarp();
                tc_after_sync();
            }
            n += tiles;
            const bool whole = tiles == it.units;
            float *slot = slots + (long long)(2 * c + (seg0 == 0)) * S::SLOT;
            if (active) {
                const float inv = l > 0.f ? 1.f / l : 0.f;
                T *dst = (T *)a.out + (it.s.q0 + tok) * a.out_stride + (long long)(it.head * group.n + i - tok * group.n) * hd;
                float *part = slot + (t * WA_TILE + row) * HDP;
#pragma unroll 1
                for (int d = 0; d < HDP; d += 32) {
                    uint32_t x[32];
                    tm_ld32(x, o_tm + d);
                    tm_wait_ld(x);
                    if (real) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            if (d + k < hd && whole) {
                                uint4 v;
                                v.x = pack2(__uint_as_float(x[k]) * inv, __uint_as_float(x[k + 1]) * inv, T());
                                v.y = pack2(__uint_as_float(x[k + 2]) * inv, __uint_as_float(x[k + 3]) * inv, T());
                                v.z = pack2(__uint_as_float(x[k + 4]) * inv, __uint_as_float(x[k + 5]) * inv, T());
                                v.w = pack2(__uint_as_float(x[k + 6]) * inv, __uint_as_float(x[k + 7]) * inv, T());
                                *(uint4 *)(dst + d + k) = v;
                            } else if (d + k < hd) {
                                *(uint4 *)(part + d + k) = make_uint4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                                *(uint4 *)(part + d + k + 4) = make_uint4(x[k + 4], x[k + 5], x[k + 6], x[k + 7]);
                            }
                        }
                    }
                    __syncwarp();
                }
                if (!whole && real) {
                    slot[WA_ROWS * HDP + t * WA_TILE + row] = m;
                    slot[WA_ROWS * (HDP + 1) + t * WA_TILE + row] = l;
                }
                tc_before_sync();
            }
            if (!whole) {
                const int c0 = attn_owner(it.first, C, total), c1 = attn_owner(it.first + it.units - 1, C, total);
                bar_sync(1, WA_ROWS);
                if (tid == 0) {
                    sh.last = atom_add_acq_rel(&flags[c0], 1u) == (unsigned)(c1 - c0);
                }
                bar_sync(1, WA_ROWS);
                if (sh.last) {
                    // Weights of up to 8 parts at a time, a thread per row, then the weighted sums: thread x has
                    // 8 outputs of 8 rows at once, so that the loads of a part are under way together.
                    float top = -INFINITY, sum = 0.f;
                    auto part = [&](int p) { return slots + (long long)(2 * p + (p == c0)) * S::SLOT; };
                    if (tid < rows) {
#pragma unroll 4
                        for (int p = c0; p <= c1; p++) top = fmaxf(top, __ldcg(part(p) + WA_ROWS * HDP + tid));
                        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
                        for (int p = c0; p <= c1; p++) sum += exp2f(__ldcg(part(p) + WA_ROWS * HDP + tid) - ref) * __ldcg(part(p) + WA_ROWS * (HDP + 1) + tid);
                    }
                    const float norm = (sum > 0.f ? 1.f / sum : 0.f), ref = top == -INFINITY ? 0.f : top;
#pragma unroll 1
                    for (int x0 = 0; x0 < rows * (HDP / 8); x0 += 8 * WA_ROWS) {
                        float acc[8][8];
#pragma unroll
                        for (int k = 0; k < 8; k++)
#pragma unroll
                            for (int e = 0; e < 8; e++) acc[k][e] = 0.f;
#pragma unroll 1
                        for (int p0 = c0; p0 <= c1; p0 += 8) {
                            bar_sync(1, WA_ROWS);
#pragma unroll 4
                            for (int p = p0; p <= min(c1, p0 + 7); p++)
                                sh.weight[p - p0][tid] = tid < rows ? exp2f(__ldcg(part(p) + WA_ROWS * HDP + tid) - ref) * norm : 0.f;
                            bar_sync(1, WA_ROWS);
#pragma unroll 1
                            for (int p = p0; p <= min(c1, p0 + 7); p++)
#pragma unroll
                                for (int k = 0; k < 8; k++) {
                                    const int x = x0 + k * WA_ROWS + tid, r = x / (HDP / 8);
                                    if (r >= rows) continue;
                                    const float4 *from = (const float4 *)(part(p) + r * HDP + x % (HDP / 8) * 8);
                                    const float f = sh.weight[p - p0][r];
                                    const float4 v = __ldcg(from), w = __ldcg(from + 1);
                                    acc[k][0] += f * v.x;
                                    acc[k][1] += f * v.y;
                                    acc[k][2] += f * v.z;
                                    acc[k][3] += f * v.w;
                                    acc[k][4] += f * w.x;
                                    acc[k][5] += f * w.y;
                                    acc[k][6] += f * w.z;
                                    acc[k][7] += f * w.w;
                                }
                        }
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const int x = x0 + k * WA_ROWS + tid, r = x / (HDP / 8), d = x % (HDP / 8) * 8;
                            if (r >= rows || d >= hd) continue;
                            const int i2 = it.i0 + r, tk = group.div(i2);
                            uint4 v;
                            v.x = pack2(acc[k][0], acc[k][1], T());
                            v.y = pack2(acc[k][2], acc[k][3], T());
                            v.z = pack2(acc[k][4], acc[k][5], T());
                            v.w = pack2(acc[k][6], acc[k][7], T());
                            *(uint4 *)((T *)a.out + (it.s.q0 + tk) * a.out_stride + (long long)(it.head * group.n + i2 - tk * group.n) * hd + d) = v;
                        }
                    }
                    if (tid == 0) flags[c0] = 0;
                }
                bar_sync(1, WA_ROWS);   // before `last` is written again
            }
            u += tiles;
        }
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    if (warp == 8) tm_free(TM_S, TM_COLS);
}

// The driver's encoder of tensor maps, looked up once (NULL: there is none).
static decltype(&cuTensorMapEncodeTiled) tensor_map_encoder() {
    static void *found;   // written once, with the same value by whoever comes first
    void *fn = __atomic_load_n(&found, __ATOMIC_ACQUIRE);
    if (!fn) {
        cudaDriverEntryPointQueryResult how;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how) != cudaSuccess ||
            how != cudaDriverEntryPointSuccess || !fn) {
            cudaGetLastError();
            return nullptr;
        }
        __atomic_store_n(&found, fn, __ATOMIC_RELEASE);
    }
    return (decltype(&cuTensorMapEncodeTiled))fn;
}

// The tensor maps of a cache. Where a page's tokens do not come in runs of 8, or
// the driver does not take the strides, run stays 0 and the copies serve.
static WideMaps wide_maps(const ptc_paged_cache &c) {
    WideMaps m;
    memset(&m, 0, sizeof(m));
    int run = 64;
    while (c.page_size % run) run /= 2;
    if (run < 8) return m;
    const auto encode = tensor_map_encoder();
    if (!encode) return m;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.n_kv_heads, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.token_stride * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)run, 1, 1}, step[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = c.dtype == PTC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = 0; i < 2; i++)
        if (encode(i ? &m.v : &m.k, type, 4, i ? c.v : c.k, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return m;
    m.run = run;
    return m;
}

template <typename T, int HDP>
static cudaError_t launch_wide(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s) {
    using S = WideShape<HDP>;
    static_assert(2 * 148 * (long long)S::SLOT * 4 + ATTN_FLAG_BYTES <= (long long)PTC_ATTN_WORKSPACE_BYTES, "two slots for each SM");
    auto kernel = k_attn_wide<T, HDP>;
    const int smem = attn_smem(1024 + S::BYTES, a.n_seqs);
    const cudaError_t e = allow_smem(kernel, attn_smem(1024 + S::BYTES, ATTN_MAX_SEQS));
    if (e != cudaSuccess) return e;
    const long long fit = (long long)(PTC_ATTN_WORKSPACE_BYTES - ATTN_FLAG_BYTES) / (2 * S::SLOT * (int)sizeof(float));
    return launch_kernel(kernel, (unsigned)(n_sm < fit ? n_sm : fit), WA_THREADS, smem, s, a, wide_maps(a.cache), group);
}

cudaError_t launch_attn_wide(const ptc_attn_args &a, Group group, int n_sm, cudaStream_t s) {
    const bool small = a.cache.head_dim <= 64;
    if (a.cache.dtype == PTC_F16) return small ? launch_wide<__half, 64>(a, group, n_sm, s) : launch_wide<__half, 128>(a, group, n_sm, s);
    return small ? launch_wide<__nv_bfloat16, 64>(a, group, n_sm, s) : launch_wide<__nv_bfloat16, 128>(a, group, n_sm, s);
}

}  // namespace ptc
