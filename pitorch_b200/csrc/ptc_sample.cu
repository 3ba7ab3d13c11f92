// ptc_sample.cu -- sampling of the next tokens on the GPU (include/ptc_serve.h).
//
// A cluster of 1 to 8 CTAs per row; each holds its slice of the logits in
// shared memory, so the row is read from memory once. Nothing is sorted: the
// kept tokens are those at or above one threshold in the order (value, lowest
// index first), which is found by counting.
//
// Few kept (top_k up to 512): each thread's maximum is known from the load,
// and the bin in which k of these maxima lie is low enough to hold the k
// largest of all, and little more. One comparison per logit collects them (a
// few hundred) in one CTA, which ranks them against each other for all the
// rules.
//
// Otherwise:
//  1. a histogram of the logits by their distance from the maximum (4096 bins
//     of equal width down to where a weight is zero), added up through
//     distributed shared memory. The bin that holds the k-th largest is
//     collected and its members ranked: the threshold of top_k;
//  2. top_p: a bin's mass lies between its count times its lowest and highest
//     weight, 0.8% apart, so the counts alone bracket the bins in which the
//     mass can reach top_p times the total. The mass before the bracket is
//     summed exactly; inside it, the ranking of its members, after a second
//     histogram of exact masses (1024 bins) where they are many, finds the
//     last one kept;
//  3. min_p is a comparison with the weight, and the token is found from the
//     kept sums of the CTAs, of their warps and of one warp's elements.
// Where a bin has too many members to be ranked (equal logits by the
// thousand), the threshold is bisected instead.
//
// Weights are integers in units of 2^-43 of the largest, so every sum is
// exact, the order of the atomics has no effect, and the same row gives the
// same token in any batch. They are computed in 64-bit arithmetic (2^y by a
// table of 32 and a polynomial of degree 5, relative error below 2^-45): the
// running sum of 10^5 weights has to be exact to far better than the weight
// of one token, which 32-bit exponentials do not give.
#include <cooperative_groups.h>
#include <limits.h>

#include "ptc_serve.cuh"

namespace ptc {
namespace cg = cooperative_groups;

constexpr int SP_THREADS = 512;
constexpr int SP_WARPS = SP_THREADS / 32;
constexpr int SP_BINS = 4096;     // of the first histogram; the last one holds what has no weight
constexpr int SP_BINS2 = 1024;    // of the second
constexpr int SP_LIST = 1024;     // members that are ranked
constexpr int SP_FEW = 512;       // ... without a second histogram
constexpr int SP_SLICE = 16384;   // logits of a CTA, while 8 of them hold the row
constexpr float SP_RANGE = 44.f;  // weights below 2^-44 are zero
typedef unsigned long long u64;
// values that the CTAs of a row tell each other, a slot each
enum { IN_BEST, IN_FEW, IN_MASS, IN_COUNT, IN_OVER, IN_LIST, IN_BRACKET, IN_RANGE, IN_BEFORE, IN_MASS2, IN_SEG2, IN_OVER2, IN_LIST2, IN_KEPT, IN_STEP, SP_SLOTS = IN_STEP + 2 };
constexpr double SP_ONE = 8796093022208.0;   // 2^43

struct alignas(16) SampleShared {
    unsigned hist[SP_BINS];
    // the second histogram (sums of the weights' low, middle and high 15 bits),
    // or a list of all CTAs' members with their weights
    union {
        unsigned mass[3][SP_BINS2];
        struct {
            u64 key[SP_LIST], w[SP_LIST];
        } all;
    };
    u64 list[SP_LIST];   // this CTA's members
    double table[32];    // 2^(j/32)
    u64 in[SP_SLOTS][8];   // what each CTA of the cluster pushed here, by value and rank
    u64 part[SP_WARPS], part2[SP_WARPS];
    u64 border[2], found, lo, hi;
    unsigned n_list, n_few;
};

__device__ __forceinline__ float key_value(u64 key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// The order of the rules: larger value first, then lower index; -0 equals 0.
__device__ __forceinline__ u64 order_key(float v, int i) { return argmax_key(v + 0.0f, i); }

// A float that is no infinity as a double, by its bits (the conversion
// instruction has a quarter of the rate); subnormals become 0.
__device__ __forceinline__ double widen(float x) {
    const uint32_t u = __float_as_uint(x), m = u & 0x7fffffffu;
    return m < 0x00800000u ? 0.0 : __hiloint2double((int)((u & 0x80000000u) | ((m >> 3) + 0x38000000u)), (int)(u << 29));
}

// How a row's logits become bins and weights.
struct Weigh {
    float top, scale;   // bins per unit of distance
    double c, topc;     // log2(e) / temperature, and times the maximum
    const double *table;

    // Distance from the maximum in bins; NaN for an infinite maximum itself.
    __device__ float place(float x) const { return (top - x) * scale; }
    __device__ static bool heavy(float f) { return !(f >= (float)(SP_BINS - 1)); }   // has weight
    __device__ static int bin(float f) { return heavy(f) ? (int)f : SP_BINS - 1; }
    // 2^y for y = (x - top) log2(e) / temperature: y = n/32 + r, 2^(n/32) from
    // the table and the exponent, 2^r by its series (ln 2)^i / i!
    __device__ u64 weight(float x) const {
        if (!heavy(place(x))) return 0;
        if (x == top) return 1ull << 43;
        const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the rounded integer
        const double y = fma(widen(x), c, -topc), t = fma(y, 32.0, magic);
        const int n = __double2loint(t);
        const double r = fma(t - magic, -1.0 / 32.0, y);
        double p = 1.3333558146428443e-3;
        p = fma(p, r, 9.618129107628477e-3);
        p = fma(p, r, 5.550410866482158e-2);
        p = fma(p, r, 2.402265069591007e-1);
        p = fma(p, r, 6.931471805599453e-1);
        p = fma(p, r, 1.0) * table[n & 31];
        p = __hiloint2double(__double2hiint(p) + (((n >> 5) + 43) << 20), __double2loint(p));
        return (u64)__double_as_longlong(p + 4503599627370496.0) & ((1ull << 52) - 1);
    }
};

// The threshold: kept are the logits above `v`, and those equal to it up to index `i`.
struct Floor {
    float v;
    int i;
    __device__ bool keeps(float x, int at) const { return x > v || (x == v && at <= i); }
    __device__ static Floor of(u64 key) { return {key_value(key), argmax_key_index(key)}; }
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_top(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The CTA's sum of v, in every thread.
__device__ __forceinline__ u64 block_add(u64 v, u64 *part) {
    v = warp_add(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < SP_WARPS; w++) t += part[w];
    return t;
}

// The sum of v over the threads before this one, and over all.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V *part, V &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    V before = inc - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < SP_WARPS; w++) {
        if (w < warp) before += part[w];
        total += part[w];
    }
    return before;
}

template <typename T, int CL>
struct SampleRow {
    static constexpr int N = Vec16<T>::N;
    SampleShared &sh;
    cg::cluster_group &cl;
    const Vec16<T> *x;   // this CTA's slice in shared memory, -inf before and behind it
    int vecs, first;     // its vectors, and the index of the first one's first element
    int rank;
    Weigh wt;
    int turn;         // which of the two IN_STEP slots the next sum takes: the other CTAs may still read the last one

    // f(value, index) for this thread's share of the slice
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
        for (int v = threadIdx.x; v < vecs; v += SP_THREADS) {
            const Vec16<T> e = x[v];
#pragma unroll
            for (int k = 0; k < N; k++) f(Elem<T>::up(e.e[k]), first + v * N + k);
        }
    }

    // v into every CTA's slot; there after the next barrier of the cluster.
    // Stores overlap with the barrier, where loads after it would add a round
    // trip each.
    __device__ void push(int slot, u64 v) {
        if (threadIdx.x < CL) *cl.map_shared_rank(&sh.in[slot][rank], threadIdx.x) = v;
    }
    __device__ u64 pushed(int slot) const {
        u64 t = 0;
#pragma unroll
        for (int q = 0; q < CL; q++) t += sh.in[slot][q];
        return t;
    }
    __device__ u64 pushed_before(int slot) const {
        u64 t = 0;
#pragma unroll
        for (int q = 0; q < CL; q++)
            if (q < rank) t += sh.in[slot][q];
        return t;
    }

    // The counts of PER bins from bin0 on, over the cluster.
    template <int PER>
    __device__ void gather(unsigned *hist, int bin0, int (&cnt)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; i++) cnt[i] = 0;
#pragma unroll
        for (int q = 0; q < CL; q++) {
            const unsigned *h = cl.map_shared_rank(hist, (rank + q) % CL) + bin0;   // not all from the same CTA at once
#pragma unroll
            for (int i = 0; i < PER; i++) cnt[i] += h[i];
        }
    }

    // Sum over the cluster of f(value, key), a barrier of the cluster in it.
    template <typename F>
    __device__ u64 sum(F f) {
        u64 s = 0;
        each([&](float v, int i) { s += f(v, order_key(v, i)); });
        const int slot = IN_STEP + turn;
        turn ^= 1;
        push(slot, block_add(s, sh.part));
        cl.sync();
        return pushed(slot);
    }

    // The k-th largest key, by bisection.
    __device__ u64 bisect_count(u64 k, u64 top) {
        u64 lo = 0, hi = top;   // the largest key with at least k at or above it
        while (lo < hi) {
            const u64 mid = lo + (hi - lo + 1) / 2;
            if (sum([&](float, u64 e) { return (u64)(e >= mid); }) >= k) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
    // The lowest key at or above `floor` with less than `want` above it.
    __device__ u64 bisect_mass(double want, u64 floor, u64 top) {
        u64 lo = floor, hi = top;
        while (lo < hi) {
            const u64 mid = lo + (hi - lo) / 2;
            const u64 m = sum([&](float v, u64 e) { return e > mid ? wt.weight(v) : 0; });
            if ((double)m < want) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    }

    // Collects the keys of what `in` picks and sums `add` over the rest of the row;
    // one barrier of the cluster. Every CTA then has all of them in sh.all.key
    // (their number is returned; more than SP_LIST: nothing to use). The two
    // calls of a row use a list each, as the other CTAs may still read the
    // first when the second begins; the second's takes the place of the first
    // histogram, which everyone has read by then.
    template <typename In, typename Add>
    __device__ int collect(In in, Add add, u64 &total, int slot, int second) {
        static_assert(sizeof(sh.hist) >= sizeof(sh.list), "the second list fits");
        u64 *list = second ? (u64 *)sh.hist : sh.list;
        if (threadIdx.x == 0) sh.n_list = 0;
        __syncthreads();
        u64 s = 0;
        each([&](float v, int i) {
            const float f = wt.place(v);
            if (in(v, i, f)) {
                const unsigned at = atomicAdd(&sh.n_list, 1u);
                if (at < SP_LIST) list[at] = order_key(v, i);
            } else {
                s += add(v, i, f);
            }
        });
        s = block_add(s, sh.part);
        push(slot, s);
        push(slot + 1, min(sh.n_list, (unsigned)SP_LIST + 1));
        cl.sync();
        total = pushed(slot);
        const int m = (int)pushed(slot + 1);
        if (m <= SP_LIST) {
            for (int i = threadIdx.x; i < m; i += SP_THREADS) {
                int q = 0, at = i;   // member i is the at-th of CTA q
#pragma unroll
                for (int k = 0; k < CL - 1; k++) {
                    const int c = (int)sh.in[slot + 1][k];
                    if (q == k && at >= c) at -= c, q++;
                }
                sh.all.key[i] = cl.map_shared_rank(list, q)[at];
            }
            __syncthreads();
        }
        return m;
    }
};

// The running sum that the token has to exceed.
__device__ __forceinline__ u64 sample_goal(float u, u64 total) {
    const double t = (double)u * (double)total;
    const u64 goal = t > 0 ? (t < (double)total ? (u64)t : total - 1) : 0;
    return min(goal, total - 1);
}

// All the rules on m collected logits, among them the k largest: each is
// ranked against the others, by one CTA.
__device__ void few_tokens(const ptc_sample_args &a, SampleShared &sh, const Weigh &wt, int row, int m, int k, float p, u64 least, float u) {
    constexpr int EACH = SP_LIST / SP_THREADS;
    const int tid = threadIdx.x;
    u64 key[EACH], w[EACH], before[EACH], kept = 0;
    int above[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int i = tid + e * SP_THREADS;
        key[e] = i < m ? sh.list[i] : 0;
        w[e] = i < m ? wt.weight(key_value(key[e])) : 0;
        if (i < m) sh.all.key[i] = key[e], sh.all.w[i] = w[e];
        before[e] = above[e] = 0;
    }
    __syncthreads();
    for (int j = 0; j < m; j++) {   // members and mass before each
        const u64 kj = sh.all.key[j], wj = sh.all.w[j];
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (e * SP_THREADS < m && kj > key[e]) above[e]++, before[e] += wj;
    }
    u64 mass = 0;
#pragma unroll
    for (int e = 0; e < EACH; e++)
        if (tid + e * SP_THREADS < m && above[e] < k) mass += w[e];
    const double want = (double)p * (double)block_add(mass, sh.part);
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int i = tid + e * SP_THREADS;
        if (i >= m) break;
        const bool keep = above[e] < k && (above[e] == 0 || p > 1.0f || (double)before[e] < want) && w[e] >= least;
        w[e] = keep ? w[e] : 0;
        kept += w[e];
        sh.list[i] = (u64)argmax_key_index(key[e]) << 44 | w[e];   // a weight has at most 44 bits, an index 18
    }
    const u64 total = block_add(kept, sh.part), goal = sample_goal(u, total);
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int i = tid + e * SP_THREADS;
        if (i >= m || !w[e]) continue;
        const u64 mine = sh.list[i];
        u64 run = 0;   // the kept weights at lower indexes
        for (int j = 0; j < m; j++) {
            const u64 o = sh.list[j];
            run += o < mine ? o & ((1ull << 44) - 1) : 0;
        }
        if (goal >= run && goal < run + w[e]) a.tokens[row] = (int)(mine >> 44);
    }
}

template <typename T, int CL>
__global__ void __launch_bounds__(SP_THREADS, 2) k_sample(ptc_sample_args a, int slice) {
    extern __shared__ __align__(16) char sp_smem[];
    SampleShared &sh = *(SampleShared *)sp_smem;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), row = blockIdx.x / CL;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = min(a.vocab, rank * slice), n = min(slice, a.vocab - first);
    cl.barrier_arrive();   // this CTA runs: the others may write to its shared memory

    // The slice into shared memory, at the same offset from a 16-byte boundary
    // as in memory; NaN becomes -inf.
    const T *src = (const T *)a.logits + row * a.stride + first;
    constexpr int N = Vec16<T>::N;
    const int shift = (int)(((uintptr_t)src & 15) / sizeof(T)), vecs = (n + shift + N - 1) / N;
    Vec16<T> *x = (Vec16<T> *)(sp_smem + sizeof(SampleShared));
    float most = -INFINITY;   // of this thread
#pragma unroll 4
    for (int v = tid; v < vecs; v += SP_THREADS) {
        const int i0 = v * N - shift;
        Vec16<T> e;
        if (i0 >= 0 && i0 + N <= n) {
            e = *(const Vec16<T> *)(src + i0);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) e.e[k] = i0 + k >= 0 && i0 + k < n ? src[i0 + k] : Elem<T>::down(-INFINITY);
        }
        bool odd = false;
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float f = Elem<T>::up(e.e[k]);
            odd |= f != f;
            most = fmaxf(most, f);   // of a NaN and a number, the number
        }
        if (odd)
#pragma unroll
            for (int k = 0; k < N; k++)
                if (Elem<T>::up(e.e[k]) != Elem<T>::up(e.e[k])) e.e[k] = Elem<T>::down(-INFINITY);
        x[v] = e;
    }
    for (int i = tid; i < SP_BINS / 4; i += SP_THREADS) ((uint4 *)sh.hist)[i] = make_uint4(0, 0, 0, 0);
    if (tid < 32) sh.table[tid] = exp2((double)tid / 32.0);
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const int want_k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
    SampleRow<T, CL> R = {sh, cl, x, vecs, first - shift, rank, {}, 0};
    float top = warp_max(most);
    if (lane == 0) sh.part[warp] = __float_as_uint(top);
    if (tid == 0) sh.lo = sh.hi = sh.border[1] = ~0ull, sh.n_few = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SP_WARPS; w++) top = fmaxf(top, __uint_as_float((unsigned)sh.part[w]));
    cl.barrier_wait();
    R.push(IN_BEST, __float_as_uint(top));
    cl.sync();
#pragma unroll
    for (int q = 0; q < CL; q++) top = fmaxf(top, __uint_as_float((unsigned)sh.in[IN_BEST][q]));
    top += 0.0f;
    if (top == -INFINITY) {
        if (tid == 0 && rank == 0) a.tokens[row] = -1;
        return;
    }
    if (!(temp > 0.0f) || want_k == 1) {   // the first maximum
        int at = INT_MAX;
        if (most == top) R.each([&](float v, int i) { at = v == top ? min(at, i) : at; });
        at = __reduce_min_sync(0xffffffffu, at);
        __syncthreads();
        if (lane == 0) sh.part[warp] = at;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SP_WARPS; w++) at = min(at, (int)sh.part[w]);
        R.push(IN_MASS, at);
        cl.sync();
#pragma unroll
        for (int q = 0; q < CL; q++) at = min(at, (int)sh.in[IN_MASS][q]);
        if (tid == 0 && rank == 0) a.tokens[row] = at;
        return;
    }
    const double c = 1.4426950408889634 / (double)temp;
    const Weigh wt = {top, fmaxf((float)((SP_BINS - 1) / SP_RANGE * c), 1e-30f), c, (double)top * c, sh.table};
    R.wt = wt;
    const bool by_k = want_k > 0 && want_k < a.vocab, by_p = p < 1.0f;
    const double least_w = ceil((mp < 1.0f ? (double)mp : mp >= 1.0f ? 1.0 : 0.0) * SP_ONE);
    const u64 least = least_w > 0 ? (u64)least_w : 0;   // min_p as a weight
    const u64 best = order_key(top, 0);   // at or above every key
    Floor floor = {-INFINITY, INT_MAX};

    if (by_k && want_k <= SP_FEW) {
        // The bin in which k of the threads' maxima lie: at least k logits are in it or before it.
        const int mb = Weigh::bin(wt.place(most));
        if (mb < SP_BINS - 1) atomicAdd(&sh.hist[mb], 1u);
        cl.sync();
        constexpr int PER = SP_BINS / CL / SP_THREADS;
        const int bin0 = (rank * SP_THREADS + tid) * PER;
        int cnt[PER], mine = 0, own;
        R.template gather<PER>(sh.hist, bin0, cnt);
#pragma unroll
        for (int i = 0; i < PER; i++) mine += cnt[i];
        int before = block_scan(mine, (int *)sh.part, own);
        R.push(IN_FEW, own);
        cl.sync();
        before += (int)R.pushed_before(IN_FEW);
        const bool found = (int)R.pushed(IN_FEW) >= want_k;
        if (found) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (before < want_k && before + cnt[i] >= want_k)
                    for (int q = 0; q < CL; q++) *cl.map_shared_rank(&sh.border[0], q) = (u64)(bin0 + i);
                before += cnt[i];
            }
            for (int i = tid; i < SP_BINS / 4; i += SP_THREADS) ((uint4 *)sh.hist)[i] = make_uint4(0, 0, 0, 0);
            cl.sync();
            const float edge = (float)((int)sh.border[0] + 1);
            unsigned *count = cl.map_shared_rank(&sh.n_few, 0);
            u64 *list = cl.map_shared_rank(sh.list, 0);
            if (!(wt.place(most) >= edge))
                R.each([&](float v, int i) {
                    if (!(wt.place(v) >= edge)) {
                        const unsigned at = atomicAdd(count, 1u);
                        if (at < SP_LIST) list[at] = order_key(v, i);
                    }
                });
            cl.sync();
            const unsigned m = *count;
            if (m <= SP_LIST) {
                if (rank > 0) return;
                few_tokens(a, sh, wt, row, (int)m, want_k, by_p ? p : 2.0f, least, u);
                cl.sync();   // not before the others have read the count and left
                return;
            }
        } else {
            for (int i = tid; i < SP_BINS / 4; i += SP_THREADS) ((uint4 *)sh.hist)[i] = make_uint4(0, 0, 0, 0);
            cl.sync();
        }
    }
    if (by_k || by_p) {
        // counts of the bins; with top_p alone, the mass of the row
        u64 mass = 0;
        R.each([&](float v, int) {
            const float f = wt.place(v);
            if (Weigh::heavy(f)) {
                atomicAdd(&sh.hist[(int)f], 1u);
                if (!by_k) mass += wt.weight(v);
            }
        });
        R.push(IN_MASS, block_add(mass, sh.part));
        cl.sync();
        u64 total = R.pushed(IN_MASS);
        // each CTA adds up its share of the bins, PER to a thread
        constexpr int PER = SP_BINS / CL / SP_THREADS;
        const int bin0 = (rank * SP_THREADS + tid) * PER;
        int cnt[PER], mine = 0;
        R.template gather<PER>(sh.hist, bin0, cnt);
#pragma unroll
        for (int i = 0; i < PER; i++) mine += cnt[i];
        if (by_k) {
            int own;
            int before = block_scan(mine, (int *)sh.part, own);
            R.push(IN_COUNT, own);
            cl.sync();
            before += (int)R.pushed_before(IN_COUNT);
            if ((int)R.pushed(IN_COUNT) >= want_k) {   // else all that has weight is among the k largest
#pragma unroll
                for (int i = 0; i < PER; i++) {   // the bin in which the count reaches k, to every CTA
                    if (before < want_k && before + cnt[i] >= want_k)
                        for (int q = 0; q < CL; q++)
                            *cl.map_shared_rank(&sh.border[0], q) = (u64)(bin0 + i) << 40 | (u64)before << 20 | (u64)cnt[i];
                    before += cnt[i];
                }
                cl.sync();
                const int bk = (int)(sh.border[0] >> 40), in_bin = (int)(sh.border[0] & 0xfffff);
                const int rest = want_k - (int)(sh.border[0] >> 20 & 0xfffff);   // of the bin's members
                u64 over = 0;
                if (in_bin <= SP_LIST) {
                    const int m = R.collect([&](float, int, float f) { return Weigh::bin(f) == bk; },
                                            [&](float v, int, float f) { return by_p && Weigh::bin(f) < bk ? wt.weight(v) : 0; }, over, IN_OVER, 0);
                    for (int i = tid; i < m; i += SP_THREADS) {
                        const u64 e = sh.all.key[i];
                        int above = 0;
#pragma unroll 4
                        for (int j = 0; j < m; j++) above += sh.all.key[j] > e;
                        if (above == rest - 1) sh.found = e;
                    }
                    __syncthreads();
                    floor = Floor::of(sh.found);
                    if (by_p) {
                        u64 w = 0;
                        for (int i = tid; i < m; i += SP_THREADS)
                            if (sh.all.key[i] >= sh.found) w += wt.weight(key_value(sh.all.key[i]));
                        total = over + block_add(w, sh.part);
                    }
                } else {
                    const u64 cut = R.bisect_count(want_k, best);
                    floor = Floor::of(cut);
                    if (by_p) total = R.sum([&](float v, u64 e) { return e >= cut ? wt.weight(v) : 0; });
                }
                // the counts that are left for top_p
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    if (bin0 + i == bk) cnt[i] = rest;
                    if (bin0 + i > bk) cnt[i] = 0;
                }
            } else if (by_p) {
                total = R.sum([&](float v, u64) { return wt.weight(v); });
            }
        }
        if (by_p) {
            const double want = (double)p * (double)total;
            u64 kept;   // the lowest key that is kept; the largest one always is
            if (want > 0) {
                // bracket from the counts: bins whose mass can hold the border
                const float q = SP_RANGE / (SP_BINS - 1), goal = (float)(want / SP_ONE);
                float low = 0.f, high = 0.f, lows[PER], highs[PER];
                mine = 0;
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const float b = (float)(bin0 + i);
                    low += lows[i] = cnt[i] * exp2f(-(b + 1.01f) * q);
                    high += highs[i] = cnt[i] * exp2f(-(b - 0.01f) * q);
                    mine += cnt[i];
                }
                float own_l, own_h;
                int own;
                float bl = block_scan(low, (float *)sh.part, own_l), bh = block_scan(high, (float *)sh.part2, own_h);
                int before = block_scan(mine, (int *)sh.part, own);
                R.push(IN_BRACKET, (u64)__float_as_uint(own_l) << 32 | __float_as_uint(own_h));
                R.push(IN_BEFORE, own);
                cl.sync();
#pragma unroll
                for (int r = 0; r < CL; r++)
                    if (r < rank) bl += __uint_as_float((unsigned)(sh.in[IN_BRACKET][r] >> 32)), bh += __uint_as_float((unsigned)sh.in[IN_BRACKET][r]);
                before += (int)R.pushed_before(IN_BEFORE);
                // first bin that may reach the goal, with the count before it; first that must, with the count through it
                u64 lo = ~0ull, hi = ~0ull;
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    bl += lows[i];
                    bh += highs[i];
                    if (lo == ~0ull && bh * 1.0001f >= goal) lo = (u64)(bin0 + i) << 20 | (u64)before;
                    before += cnt[i];
                    if (hi == ~0ull && bl * 0.9999f >= goal) hi = (u64)(bin0 + i) << 20 | (u64)before;
                }
                const unsigned los = __ballot_sync(0xffffffffu, lo != ~0ull), his = __ballot_sync(0xffffffffu, hi != ~0ull);
                if (los && lane == __ffs(los) - 1) atomicMin(&sh.lo, lo);
                if (his && lane == __ffs(his) - 1) atomicMin(&sh.hi, hi);
                __syncthreads();
                R.push(IN_RANGE, (sh.lo & 0xffffffffull) << 32 | (sh.hi & 0xffffffffull));
                cl.sync();
                unsigned range_lo = ~0u, range_hi = ~0u;
#pragma unroll
                for (int r = 0; r < CL; r++) {
                    range_lo = min(range_lo, (unsigned)(sh.in[IN_RANGE][r] >> 32));
                    range_hi = min(range_hi, (unsigned)sh.in[IN_RANGE][r]);
                }
                const int all = (int)R.pushed(IN_BEFORE);
                if (range_hi == ~0u) range_hi = (unsigned)(SP_BINS - 2) << 20 | (unsigned)all;
                if (range_lo == ~0u) range_lo = (unsigned)(SP_BINS - 2) << 20 | (unsigned)all;
                const int b_lo = (int)(range_lo >> 20), b_hi = max(b_lo, (int)(range_hi >> 20));
                const int in_range = (int)(range_hi & 0xfffff) - (int)(range_lo & 0xfffff);
                u64 over = 0;
                int g_lo = 0, g_hi = SP_BINS2;   // the second histogram's bins that are collected
                const float g_scale = (float)SP_BINS2 / (float)(b_hi - b_lo + 1);
                auto sub = [&](float f) { return min(SP_BINS2 - 1, (int)((f - (float)b_lo) * g_scale)); };   // NaN: 0
                const float f_lo = (float)b_lo, f_hi = (float)(b_hi + 1);
                // place() of an infinite maximum is NaN, which belongs to bin 0
                auto above = [&](float f) { return b_lo > 0 && !(f >= f_lo); };
                auto inside = [&](float f) { return !(f >= f_hi) && !above(f); };
                if (in_range > SP_FEW) {
                    for (int i = tid; i < 3 * SP_BINS2; i += SP_THREADS) ((unsigned *)sh.mass)[i] = 0;
                    __syncthreads();
                    u64 s = 0;
                    R.each([&](float v, int i) {
                        const float f = wt.place(v);
                        if (f >= f_hi || !floor.keeps(v, i)) return;
                        const u64 w = wt.weight(v);
                        if (above(f)) {
                            s += w;
                        } else {   // 15 bits at a time: the sums of 2^15 of them stay below 2^30
                            const int g = sub(f);
                            atomicAdd(&sh.mass[0][g], (unsigned)(w & 0x7fff));
                            atomicAdd(&sh.mass[1][g], (unsigned)(w >> 15 & 0x7fff));
                            atomicAdd(&sh.mass[2][g], (unsigned)(w >> 30));
                        }
                    });
                    R.push(IN_MASS2, block_add(s, sh.part));
                    cl.sync();
                    const u64 sure = R.pushed(IN_MASS2);
                    constexpr int SEG2 = SP_BINS2 / CL, PER2 = SEG2 > SP_THREADS ? SEG2 / SP_THREADS : 1;
                    const int g0 = rank * SEG2 + tid * PER2;
                    u64 m[PER2], sum = 0, own_m;
#pragma unroll
                    for (int i = 0; i < PER2; i++) m[i] = 0;
                    if (tid * PER2 < SEG2) {
#pragma unroll
                        for (int r = 0; r < CL; r++) {
                            const unsigned *h = cl.map_shared_rank((unsigned *)sh.mass, (rank + r) % CL) + g0;
#pragma unroll
                            for (int i = 0; i < PER2; i++) m[i] += h[i] + ((u64)h[SP_BINS2 + i] << 15) + ((u64)h[2 * SP_BINS2 + i] << 30);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < PER2; i++) sum += m[i];
                    u64 at = block_scan(sum, sh.part, own_m);
                    R.push(IN_SEG2, own_m);
                    cl.sync();
                    at += sure + R.pushed_before(IN_SEG2);
#pragma unroll
                    for (int i = 0; i < PER2; i++) {   // the bin in which the mass reaches the goal, to every CTA
                        if ((double)at < want && (double)(at + m[i]) >= want)
                            for (int r = 0; r < CL; r++) *cl.map_shared_rank(&sh.border[1], r) = (u64)(g0 + i);
                        at += m[i];
                    }
                    cl.sync();
                    g_lo = sh.border[1] == ~0ull ? -1 : (int)sh.border[1];
                    g_hi = g_lo + 1;
                }
                // rank what is left by mass: e is kept while less than the goal is above it
                int m = SP_LIST + 1;
                if (g_lo >= 0)
                    m = R.collect([&](float v, int i, float f) { return inside(f) && sub(f) >= g_lo && sub(f) < g_hi && floor.keeps(v, i); },
                                  [&](float v, int i, float f) {
                                      return (above(f) || (inside(f) && sub(f) < g_lo)) && floor.keeps(v, i) ? wt.weight(v) : 0;
                                  }, over, IN_OVER2, by_k);
                bool done = false;
                if (m <= SP_LIST) {
                    for (int i = tid; i < m; i += SP_THREADS) sh.all.w[i] = wt.weight(key_value(sh.all.key[i]));
                    if (tid == 0) sh.found = ~0ull;
                    __syncthreads();
                    for (int i = tid; i < m; i += SP_THREADS) {
                        const u64 e = sh.all.key[i];
                        u64 more = over;
#pragma unroll 4
                        for (int j = 0; j < m; j++) more += sh.all.key[j] > e ? sh.all.w[j] : 0;
                        if ((double)more < want) atomicMin(&sh.found, e);
                    }
                    __syncthreads();
                    done = sh.found != ~0ull;
                    if (done) kept = sh.found;
                }
                if (!done) kept = R.bisect_mass(want, order_key(floor.v, floor.i), best);
            } else {
                kept = R.bisect_count(1, best);
            }
            floor = Floor::of(kept);
        }
    }

    // The kept weights in index order: a warp has a run of the slice's vectors.
    auto kept_weight = [&](float v, int i) -> u64 {
        if (!floor.keeps(v, i)) return 0;
        const u64 w = wt.weight(v);
        return w < least ? 0 : w;
    };
    auto kept_vector = [&](int v) -> u64 {
        const Vec16<T> e = x[v];
        u64 t = 0;
#pragma unroll
        for (int k = 0; k < N; k++) t += kept_weight(Elem<T>::up(e.e[k]), R.first + v * N + k);
        return t;
    };
    const int run = (vecs + SP_THREADS - 1) / SP_THREADS * 32;
    u64 s = 0;
    for (int v = warp * run + lane; v < min(vecs, (warp + 1) * run); v += 32) s += kept_vector(v);
    s = warp_add(s);
    __syncthreads();
    if (lane == 0) sh.part[warp] = s;
    __syncthreads();
    u64 own = 0;
#pragma unroll
    for (int w = 0; w < SP_WARPS; w++) own += sh.part[w];
    R.push(IN_KEPT, own);
    cl.sync();   // the last access to another CTA is before it, so each may leave from here on
    const u64 before = R.pushed_before(IN_KEPT), total = R.pushed(IN_KEPT);
    u64 goal = sample_goal(u, total);
    if (goal < before || goal >= before + own) return;
    goal -= before;
    u64 at = 0;
    int w0 = 0;   // the warp's run that holds it
    for (; w0 < SP_WARPS - 1 && at + sh.part[w0] <= goal; w0++) at += sh.part[w0];
    const int r0 = w0 * run, r1 = min(vecs, r0 + run);
    const int piece = (r1 - r0 + SP_THREADS - 1) / SP_THREADS * 32;   // and of that, a piece per warp
    const int p0 = r0 + warp * piece, p1 = min(r1, p0 + piece);
    s = 0;
    for (int v = p0 + lane; v < p1; v += 32) s += kept_vector(v);
    s = warp_add(s);
    if (lane == 0) sh.part2[warp] = s;
    __syncthreads();
    for (int w = 0; w < warp; w++) at += sh.part2[w];
    if (goal < at || goal >= at + s) return;
    for (int v0 = p0; v0 < p1; v0 += 32) {
        const int v = v0 + lane;
        const u64 w = v < p1 ? kept_vector(v) : 0;
        u64 inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (goal >= at + inc - w && goal < at + inc) {   // this lane's vector holds it
            u64 c0 = at + inc - w;
            const Vec16<T> e = x[v];
#pragma unroll
            for (int k = 0; k < N; k++) {
                const int i = R.first + v * N + k;
                const u64 wk = kept_weight(Elem<T>::up(e.e[k]), i);
                if (goal >= c0 && goal < c0 + wk) a.tokens[row] = i;
                c0 += wk;
            }
        }
        at += __shfl_sync(0xffffffffu, inc, 31);
    }
}

// CTAs per row: as many as give the batch one CTA for every place on the GPU
// (two per SM), so that a few rows are spread and many are not, but enough
// that a slice fits. Measured at 32000 logits: TODO.
static int sample_cluster(int rows, int vocab, int n_sm) {
    int c = 1;
    while (c < 8 && ((long long)rows * c * 2 <= 2 * n_sm || vocab > c * SP_SLICE)) c *= 2;
    return c;
}

template <typename T, int CL>
static cudaError_t launch_sample_cl(const ptc_sample_args &a, cudaStream_t s) {
    const int slice = (a.vocab + CL - 1) / CL;
    const size_t smem = sizeof(SampleShared) + ((size_t)slice * sizeof(T) + 47) / 16 * 16;   // with the odd ends
    cudaError_t e = cudaFuncSetAttribute(k_sample<T, CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * CL));
    cfg.blockDim = dim3(SP_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CL;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_sample<T, CL>, a, slice);
}

template <typename T>
static cudaError_t launch_sample(const ptc_sample_args &a, int n_sm, cudaStream_t s) {
    switch (sample_cluster(a.rows, a.vocab, n_sm)) {
    case 1: return launch_sample_cl<T, 1>(a, s);
    case 2: return launch_sample_cl<T, 2>(a, s);
    case 4: return launch_sample_cl<T, 4>(a, s);
    default: return launch_sample_cl<T, 8>(a, s);
    }
}

}  // namespace ptc

extern "C" int ptc_sample_tokens(const ptc_sample_args *p, void *stream) {
    if (!p) SERVE_REFUSE("no arguments");
    const ptc_sample_args a = *p;
    if (!ptc::dtype_ok(a.dtype)) SERVE_REFUSE("the logits' type is none of PTC_F32, PTC_F16, PTC_BF16");
    if (a.rows < 0 || a.rows > (1 << 24) || a.vocab < 1 || a.vocab > PTC_SAMPLE_MAX_VOCAB || a.stride < a.vocab)
        SERVE_REFUSE("bad size (rows %d, vocab %d of at most %d, stride %lld)", a.rows, a.vocab, PTC_SAMPLE_MAX_VOCAB, a.stride);
    if (a.rows == 0) return 0;
    if (!a.logits || !a.u || !a.tokens) SERVE_REFUSE("a required pointer is NULL");
    if ((uintptr_t)a.logits % ptc::dtype_bytes(a.dtype)) SERVE_REFUSE("the logits are not aligned to their type");
    cudaStream_t s = (cudaStream_t)stream;
    ptc::MemoryDevice on(a.tokens);
    SERVE_CUDA(on.error());
    int n_sm = 0;
    SERVE_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, on.device()));
    if (a.dtype == PTC_F32) SERVE_CUDA(ptc::launch_sample<float>(a, n_sm, s));
    else if (a.dtype == PTC_F16) SERVE_CUDA(ptc::launch_sample<__half>(a, n_sm, s));
    else SERVE_CUDA(ptc::launch_sample<__nv_bfloat16>(a, n_sm, s));
    return 0;
}
