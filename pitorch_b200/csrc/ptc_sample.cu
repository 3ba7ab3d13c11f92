// ptc_sample.cu -- sampling of the next tokens on the GPU (include/ptc_serve.h).
//
// A cluster of 1 to 8 CTAs per row; each holds its slice of the logits in
// shared memory, so the row is read from memory once. Nothing is sorted: the
// kept tokens are those at or above one threshold in the order (value, lowest
// index first), which is found by counting.
//
// Few kept (top_k up to 400): the load leaves the maxima of 512 groups of the
// row. The bin of equal width in which k of them lie bounds the k largest
// logits from below, and one comparison per logit collects what is above it
// (about 512 ln(512 / (512 - k)) of logits in random order) in one CTA, which
// ranks them against each other for all the rules.
//
// Otherwise:
//  1. top_k: a histogram of the logits by their distance from the maximum
//     (2048 bins of equal width down to the lowest logit that has weight),
//     added up through distributed shared memory. The bin that holds the k-th
//     largest is collected and its members ranked: the threshold;
//  2. top_p: the same with exact masses in place of counts (three sums of 15
//     bits each, as shared memory adds 32 bits at a time). The bin in which
//     the mass reaches top_p times the total is collected, and ranking its
//     members finds the last one kept;
//  3. min_p is a comparison with the weight, and the token is found from the
//     kept sums of the CTAs, of their warps and of one warp's elements.
// Where a bin has too many members to be ranked (equal logits by the
// thousand), the threshold is bisected instead.
//
// Weights are integers in units of 2^-43 of the largest, so every sum is
// exact, the order of the atomics has no effect, and the same row gives the
// same token in any batch. They are computed in 64-bit arithmetic (2^y by a
// table of 256 and a polynomial of degree 3, relative error below 2^-42 wherever
// the logits lie): the
// running sum of 10^5 weights has to be exact to far better than the weight
// of one token, which 32-bit exponentials do not give.
//
// Measured on the GPU: one row of 32000 f32 logits with top_p 13.8 us, with
// top_k 40 10.3 us, bound by a cluster's barriers (0.7 us each, six with top_p)
// and the two passes of 64-bit weights; 64 rows with mixed rules 24 us; 256 rows
// of 131071 bf16 logits 125 us against 10 us for one read of them: the rows with
// top_p alone take 33 us each, half of that in 64-bit arithmetic.
#include <cooperative_groups.h>
#include <limits.h>

#include "ptc_serve.cuh"

namespace ptc {
namespace cg = cooperative_groups;

constexpr int SP_THREADS = 512;
constexpr int SP_WARPS = SP_THREADS / 32;
constexpr int SP_BINS = 2048;
constexpr int SP_LIST = 1024;     // members that are ranked
constexpr int SP_FEW = 400;       // top_k up to here by the groups' maxima
constexpr int SP_GROUPS = 512;
constexpr int SP_SLICE = 16384;   // logits of a CTA, while 8 of them hold the row
constexpr float SP_RANGE = 44.f;  // weights below 2^-44 are zero
typedef unsigned long long u64;
// values that the CTAs of a row tell each other, a slot each
enum { IN_BEST, IN_FIRST, IN_COUNT, IN_LIST, IN_MASS, IN_LIST2, IN_KEPT, IN_STEP, SP_SLOTS = IN_STEP + 2 };
constexpr double SP_ONE = 8796093022208.0;   // 2^43

struct alignas(16) SampleShared {
    union {
        unsigned hist[3][SP_BINS];   // counts in the first, or the low, middle and high 15 bits of masses
        struct {
            u64 key[SP_LIST], w[SP_LIST];
        } all;               // the members of all CTAs, with their weights (nobody reads the histogram any more)
    };
    u64 list[SP_LIST];       // this CTA's
    float most[SP_GROUPS];   // maxima of the row's groups
    double table[256];   // 2^(j/256)
    u64 in[SP_SLOTS][8];   // what each CTA of the cluster pushed here, by value and rank
    u64 part[SP_WARPS], part2[SP_WARPS];
    u64 border[2], found;
    unsigned n_list, n_few;
    int edge;
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
    float top, most;    // the maximum, and the distance from it at which weights become zero
    float scale;        // bins per unit of distance
    double c, at;       // 256 log2(e) / temperature, and the maximum
    const double *table;

    // (the distance of an infinite maximum from itself is NaN: heavy, in bin 0)
    __device__ bool heavy(float x) const { return !(top - x >= most); }
    __device__ int bin(float x) const { return min(SP_BINS - 1, (int)((top - x) * scale)); }
    // 2^(y/256) for y = (x - top) c, n + r with |r| <= 1/2: 2^(n/256) from the
    // table and the exponent, 2^(r/256) by its series (ln 2 / 256)^i / i!, to
    // 2^-42. The difference comes first: it has an error of 2^-53 of itself, and
    // none for logits of like size, wherever they are; a product with a logit of
    // 10^5, or for a temperature of 0.01, would have one of the product.
    __device__ u64 weight(float x) const {
        if (!heavy(x)) return 0;
        if (x == top) return 1ull << 43;
        const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the rounded integer
        const double diff = widen(x) - at, t = fma(diff, c, magic);
        const int n = __double2loint(t);
        const double r = fma(diff, c, magic - t);
        constexpr double ln = 0.6931471805599453 / 256.0;
        double p = ln * ln * ln / 6.0;
        p = fma(p, r, ln * ln / 2.0);
        p = fma(p, r, ln);
        p = fma(p, r, 1.0) * table[n & 255];
        p = __hiloint2double(__double2hiint(p) + (((n >> 8) + 43) << 20), __double2loint(p));
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

    // A CTA adds up its share of the bins over the cluster, PER to a thread
    // (where there are fewer bins than threads, the last threads have none).
    static constexpr int SHARE = SP_BINS / CL, PER = SHARE > SP_THREADS ? SHARE / SP_THREADS : 1;
    __device__ int bin0() const { return rank * SHARE + threadIdx.x * PER; }
    template <int PARTS>
    __device__ void gather(u64 (&sum)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; i++) sum[i] = 0;
        if (threadIdx.x * PER >= SHARE) return;
#pragma unroll
        for (int q = 0; q < CL; q++) {
            const unsigned *h = cl.map_shared_rank(&sh.hist[0][0], (rank + q) % CL) + bin0();   // not all from the same CTA at once
#pragma unroll
            for (int i = 0; i < PER; i++)
#pragma unroll
                for (int k = 0; k < PARTS; k++) sum[i] += (u64)h[k * SP_BINS + i] << (15 * k);
        }
    }
    // The bin in which the running sum of the gathered ones reaches `want`, and
    // the sum before it, into every CTA's sh.border (false: it stays below);
    // `total` is the sum of all. Two barriers of the cluster.
    template <typename V>
    __device__ bool cross(const u64 (&sum)[PER], double share, V want, u64 &total, int slot) {
        u64 mine = 0, own;
#pragma unroll
        for (int i = 0; i < PER; i++) mine += sum[i];
        u64 before = block_scan(mine, sh.part, own);
        push(slot, own);
        cl.sync();
        before += pushed_before(slot);
        total = pushed(slot);
        const double goal = share > 0 ? share * (double)total : (double)want;
        if ((double)total < goal) return false;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if ((double)before < goal && (double)(before + sum[i]) >= goal)
                for (int q = 0; q < CL; q++) {
                    u64 *to = cl.map_shared_rank(sh.border, q);
                    to[0] = (u64)(bin0() + i);
                    to[1] = before;
                }
            before += sum[i];
        }
        cl.sync();
        return true;
    }
    __device__ void clear(int parts) {
        for (int i = threadIdx.x; i < parts * SP_BINS / 4; i += SP_THREADS) ((uint4 *)&sh.hist[0][0])[i] = make_uint4(0, 0, 0, 0);
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

    // Collects the keys of what `in` picks; one barrier of the cluster. Every
    // CTA then has all of them in sh.all.key (their number is returned; more
    // than SP_LIST: nothing to use). The two calls of a row have a barrier of
    // the cluster between them, after which nobody reads the first list.
    template <typename In>
    __device__ int collect(In in, int slot) {
        if (threadIdx.x == 0) sh.n_list = 0;
        __syncthreads();
        each([&](float v, int i) {
            if (in(v, i)) {
                const unsigned at = atomicAdd(&sh.n_list, 1u);
                if (at < SP_LIST) sh.list[at] = order_key(v, i);
            }
        });
        __syncthreads();
        push(slot, min(sh.n_list, (unsigned)SP_LIST + 1));
        cl.sync();
        const int m = (int)pushed(slot);
        if (m <= SP_LIST) {
            for (int i = threadIdx.x; i < m; i += SP_THREADS) {
                int q = 0, at = i;   // member i is the at-th of CTA q
#pragma unroll
                for (int k = 0; k < CL - 1; k++) {
                    const int c = (int)sh.in[slot][k];
                    if (q == k && at >= c) at -= c, q++;
                }
                sh.all.key[i] = cl.map_shared_rank(sh.list, q)[at];
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

// All the rules on m collected logits, among them the k largest, by one CTA:
// each is ranked against the others (its comparisons shared by as many threads
// as there are), the weights are summed in the order of the ranks, and those
// that are kept, at most k, ranked by index for the running sum.
__device__ void few_tokens(const ptc_sample_args &a, SampleShared &sh, const Weigh &wt, int row, int m, int k, float p, u64 least, float u) {
    const int tid = threadIdx.x;
    const int fit = SP_THREADS / m, lanes = fit >= 32 ? 32 : fit >= 16 ? 16 : fit >= 8 ? 8 : fit >= 4 ? 4 : fit >= 2 ? 2 : 1;
    const int per = SP_THREADS / lanes, lane = tid % lanes;
    if (tid == 0) sh.n_list = 0;
    for (int i0 = 0; i0 < m; i0 += per) {
        const int i = i0 + tid / lanes;
        const u64 e = i < m ? sh.list[i] : ~0ull;
        int rank = 0;
#pragma unroll 4
        for (int j = lane; j < m; j += lanes) rank += sh.list[j] > e;
        for (int d = 1; d < lanes; d *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, d);
        if (i < m && lane == 0) sh.all.key[rank] = e;
    }
    __syncthreads();
    // in descending order, two to a thread: the weights and the sum before each
    const int n = min(m, k);
    u64 w[2], sum, before;
#pragma unroll
    for (int e = 0; e < 2; e++) w[e] = 2 * tid + e < n ? wt.weight(key_value(sh.all.key[2 * tid + e])) : 0;
    before = block_scan(w[0] + w[1], sh.part, sum);
    const double want = (double)p * (double)sum;
    u64 kept = 0;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int i = 2 * tid + e;
        if (i < n && (i == 0 || p > 1.0f || (double)before < want) && w[e] >= least && w[e]) {
            kept += w[e];
            // a weight has at most 44 bits, an index 18
            sh.all.w[atomicAdd(&sh.n_list, 1u)] = (u64)argmax_key_index(sh.all.key[i]) << 44 | w[e];
        }
        before += w[e];
    }
    const u64 total = block_add(kept, sh.part), goal = sample_goal(u, total), weights = (1ull << 44) - 1;
    const int q = (int)sh.n_list;
    for (int i = tid; i < q; i += SP_THREADS) {
        const u64 mine = sh.all.w[i];
        u64 run = 0;   // the kept weights at lower indexes
#pragma unroll 4
        for (int j = 0; j < q; j++) {
            const u64 o = sh.all.w[j];
            run += o < mine ? o & weights : 0;
        }
        if (goal >= run && goal < run + (mine & weights)) a.tokens[row] = (int)(mine >> 44);
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
    float most = -INFINITY, lowest = INFINITY;   // of this thread; -inf left out of the second
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
            lowest = fminf(lowest, f == -INFINITY ? INFINITY : f);
        }
        if (odd)
#pragma unroll
            for (int k = 0; k < N; k++)
                if (Elem<T>::up(e.e[k]) != Elem<T>::up(e.e[k])) e.e[k] = Elem<T>::down(-INFINITY);
        x[v] = e;
    }
    if (tid < 256) sh.table[tid] = exp2((double)tid / 256.0);
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const int want_k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
    SampleRow<T, CL> R = {sh, cl, x, vecs, first - shift, rank, {}, 0};
    R.clear(3);
    float top = warp_max(most);
    lowest = -warp_max(-lowest);
    if (lane == 0) sh.part[warp] = (u64)__float_as_uint(lowest) << 32 | __float_as_uint(top);
    if (tid == 0) sh.n_few = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SP_WARPS; w++) {
        top = fmaxf(top, __uint_as_float((unsigned)sh.part[w]));
        lowest = fminf(lowest, __uint_as_float((unsigned)(sh.part[w] >> 32)));
    }
    const bool by_k = want_k > 0 && want_k < a.vocab, few = by_k && want_k <= SP_FEW, by_p = p < 1.0f;
    float group = most;   // the maximum of CL neighbouring threads: 512 / CL groups of this CTA
#pragma unroll
    for (int d = 1; d < CL; d *= 2) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, d));
    cl.barrier_wait();
    R.push(IN_BEST, (u64)__float_as_uint(lowest) << 32 | __float_as_uint(top));
    if (few)   // each of the CL threads tells one CTA
        cl.map_shared_rank(sh.most, tid % CL)[rank * (SP_GROUPS / CL) + tid / CL] = group;
    cl.sync();
#pragma unroll
    for (int q = 0; q < CL; q++) {
        top = fmaxf(top, __uint_as_float((unsigned)sh.in[IN_BEST][q]));
        lowest = fminf(lowest, __uint_as_float((unsigned)(sh.in[IN_BEST][q] >> 32)));
    }
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
        R.push(IN_FIRST, at);
        cl.sync();
#pragma unroll
        for (int q = 0; q < CL; q++) at = min(at, (int)sh.in[IN_FIRST][q]);
        if (tid == 0 && rank == 0) a.tokens[row] = at;
        return;
    }
    const double c = 1.4426950408889634 / (double)temp;   // a logit's distance in powers of two
    // bins down to the lowest logit or to where weights end, whichever is nearer
    // (above 0 for every temperature)
    const float reach = (float)(SP_RANGE / c), spread = fminf(top - lowest, reach);
    const Weigh wt = {top, reach, spread > 0.f ? fminf((SP_BINS - 1) / spread, 1e30f) : 1e30f, 256.0 * c, (double)top, sh.table};
    R.wt = wt;
    const double least_w = ceil((mp < 1.0f ? (double)mp : mp >= 1.0f ? 1.0 : 0.0) * SP_ONE);
    const u64 least = least_w > 0 ? (u64)least_w : 0;   // min_p as a weight
    const u64 best = order_key(top, 0);   // at or above every key
    Floor floor = {-INFINITY, INT_MAX};

    u64 sums[SampleRow<T, CL>::PER], total;

    if (few) {
        // the bin in which k of the groups' maxima lie: every CTA counts them for itself
        const float mine = sh.most[tid];
        if (wt.heavy(mine)) atomicAdd(&sh.hist[0][wt.bin(mine)], 1u);
        if (tid == 0) sh.edge = -1;
        __syncthreads();
        constexpr int EACH = SP_BINS / SP_THREADS;
        const uint4 h = ((const uint4 *)sh.hist[0])[tid];
        static_assert(EACH == 4, "a vector of bins per thread");
        const int cnt[EACH] = {(int)h.x, (int)h.y, (int)h.z, (int)h.w};
        int all, before = block_scan(cnt[0] + cnt[1] + cnt[2] + cnt[3], (int *)sh.part, all);
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            if (before < want_k && before + cnt[i] >= want_k) sh.edge = tid * EACH + i;
            before += cnt[i];
        }
        ((uint4 *)sh.hist[0])[tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int edge = sh.edge;
        unsigned *count = cl.map_shared_rank(&sh.n_few, 0);
        if (edge >= 0) {
            u64 *list = cl.map_shared_rank(sh.list, 0);
            if (wt.bin(most) <= edge)
                R.each([&](float v, int i) {
                    if (wt.bin(v) <= edge) {
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
        }
    }
    if (by_k) {
        R.each([&](float v, int) {
            if (wt.heavy(v)) atomicAdd(&sh.hist[0][wt.bin(v)], 1u);
        });
        cl.sync();
        R.template gather<1>(sums);
        if (R.cross(sums, 0.0, want_k, total, IN_COUNT)) {   // else all that has weight is among the k largest
            const int bk = (int)sh.border[0], rest = want_k - (int)sh.border[1];   // of the bin's members
            const int m = R.collect([&](float v, int) { return wt.heavy(v) && wt.bin(v) == bk; }, IN_LIST);
            if (m <= SP_LIST) {
                for (int i = tid; i < m; i += SP_THREADS) {
                    const u64 e = sh.all.key[i];
                    int above = 0;
#pragma unroll 4
                    for (int j = 0; j < m; j++) above += sh.all.key[j] > e;
                    if (above == rest - 1) sh.found = e;
                }
                __syncthreads();
                floor = Floor::of(sh.found);
            } else {
                floor = Floor::of(R.bisect_count(want_k, best));
            }
        }
        __syncthreads();
        R.clear(3);
        __syncthreads();
    }
    if (by_p && p > 0.0f) {
        R.each([&](float v, int i) {
            if (!wt.heavy(v) || !floor.keeps(v, i)) return;
            const u64 w = wt.weight(v);   // 15 bits at a time: the sums of 2^15 of them stay below 2^30
            const int b = wt.bin(v);
            atomicAdd(&sh.hist[0][b], (unsigned)(w & 0x7fff));
            if (w >> 15) atomicAdd(&sh.hist[1][b], (unsigned)(w >> 15 & 0x7fff));
            if (w >> 30) atomicAdd(&sh.hist[2][b], (unsigned)(w >> 30));
        });
        cl.sync();
        R.template gather<3>(sums);
        R.cross(sums, (double)p, 0, total, IN_MASS);
        const int bp = (int)sh.border[0];
        const u64 over = sh.border[1];
        const double want = (double)p * (double)total;
        const int m = R.collect([&](float v, int i) { return wt.heavy(v) && wt.bin(v) == bp && floor.keeps(v, i); }, IN_LIST2);
        if (m <= SP_LIST) {
            // ranked by mass: a member is kept while less than the goal is before it
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
            floor = Floor::of(sh.found);
        } else {
            floor = Floor::of(R.bisect_mass(want, order_key(floor.v, floor.i), best));
        }
    } else if (by_p) {
        floor = Floor::of(R.bisect_count(1, best));   // the largest alone
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
    const u64 before = R.pushed_before(IN_KEPT);
    total = R.pushed(IN_KEPT);
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

// CTAs per row: as many as leave each at least 2000 logits (four a thread) and
// the batch at most two CTAs per SM, so that few rows are spread and many are
// not, but enough that a slice fits. Measured with mixed rules in us, by 1, 2,
// 4 and 8 CTAs per row: 16 rows of 8000 logits 18.5, 14.5, 12.5, 16.5; 256 of
// them 23, 26, 36, 65; of 32000 logits 1 row -, 22.6, 16.9, 13.8; 64 rows -, 28,
// 24, 26; 256 rows -, 45, 52, 69.
static int sample_cluster(int rows, int vocab, int n_sm) {
    int c = 1;
    while (c < 8 && (((long long)rows * c * 2 <= 2 * n_sm && vocab >= 2 * c * 2000) || vocab > c * SP_SLICE)) c *= 2;
    return c;
}

// Shared memory of a CTA with a slice of n logits (and the odd ends of its vectors).
template <typename T>
static constexpr int sample_smem(int n) {
    return (int)(sizeof(SampleShared) + ((size_t)n * sizeof(T) + 47) / 16 * 16);
}

template <typename T, int CL>
static cudaError_t launch_sample_cl(const ptc_sample_args &a, cudaStream_t s) {
    const int slice = (a.vocab + CL - 1) / CL, smem = sample_smem<T>(slice);
    cudaError_t e = allow_smem(k_sample<T, CL>, sample_smem<T>(CL < 8 ? SP_SLICE : PTC_SAMPLE_MAX_VOCAB / CL));
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
