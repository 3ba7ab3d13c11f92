// ptc_sample.cu -- sampling of the next tokens on the GPU (include/ptc_serve.h).
#include "ptc_serve.cuh"

namespace ptc {

constexpr int SM_THREADS = 1024;

// A logit as the rules see it: NaN counts as -inf, and -0 as 0, so that equal
// values have equal keys.
template <typename T>
__device__ __forceinline__ float logit(T v) {
    const float x = Elem<T>::up(v);
    return x != x ? -INFINITY : x + 0.0f;
}

// Weights are held as integers in units of 2^-43 of the largest one: their
// sums are exact in any order, and 2^18 of them stay below 2^61.
__device__ __forceinline__ unsigned long long weight(float x, float top, double rt) {
    if (x == top) return 1ull << 43;
    if (x == -INFINITY) return 0;
    return (unsigned long long)__double2ll_rn(exp(((double)x - (double)top) * rt) * 8796093022208.0);
}

__device__ unsigned long long block_sum(unsigned long long v, unsigned long long *sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    unsigned long long t = 0;
    for (int w = 0; w < SM_THREADS / 32; w++) t += sh[w];
    return t;
}

// One CTA per row: the thresholds by bisection over the ordered keys.
template <typename T>
__global__ void __launch_bounds__(SM_THREADS) k_sample(ptc_sample_args a) {
    __shared__ unsigned long long sh[SM_THREADS / 32];
    const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    const T *x = (const T *)a.logits + row * a.stride;
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temp > 0.0f);

    unsigned long long best = 0;
    for (int i = tid; i < V; i += SM_THREADS) best = max(best, argmax_key(logit(x[i]), i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((tid & 31) == 0) sh[tid >> 5] = best;
    __syncthreads();
    for (int w = 0; w < SM_THREADS / 32; w++) best = max(best, sh[w]);
    const uint32_t top_key = (uint32_t)(best >> 32);
    const int first = argmax_key_index(best);
    const float top = logit(x[first]);
    if (top == -INFINITY || greedy) {
        if (tid == 0) a.tokens[row] = top == -INFINITY ? -1 : first;
        return;
    }
    const double rt = 1.0 / (double)temp;

    // top_k: the largest key with at least k keys at or above it
    const int k = a.top_k ? a.top_k[row] : 0;
    uint32_t cut = 0;
    unsigned long long ties = V;   // how many of the elements equal to `cut` are kept
    if (k > 0 && k < V) {
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t c = cut | (1u << bit);
            unsigned long long n = 0;
            for (int i = tid; i < V; i += SM_THREADS) n += float_key(logit(x[i])) >= c;
            if (block_sum(n, sh) >= (unsigned long long)k) cut = c;
        }
        unsigned long long above = 0;
        for (int i = tid; i < V; i += SM_THREADS) above += float_key(logit(x[i])) > cut;
        ties = k - block_sum(above, sh);
    }
    // mass above a key, and of the kept elements that equal `cut`
    auto mass_above = [&](uint32_t key) {
        unsigned long long m = 0;
        for (int i = tid; i < V; i += SM_THREADS) {
            const float v = logit(x[i]);
            if (float_key(v) > key) m += weight(v, top, rt);
        }
        return block_sum(m, sh);
    };
    auto key_value = [](uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key); };
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) {
        unsigned long long total = mass_above(cut);
        unsigned long long equal = 0;
        for (int i = tid; i < V; i += SM_THREADS) equal += float_key(logit(x[i])) == cut;
        equal = min(block_sum(equal, sh), ties);
        if (equal) total += equal * weight(key_value(cut), top, rt);
        const double want = (double)p * (double)total;
        uint32_t lo = cut, hi = top_key;   // the lowest key with less than `want` above it
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if ((double)mass_above(mid) < want) hi = mid;
            else lo = mid + 1;
        }
        const unsigned long long above = mass_above(lo), w = weight(key_value(lo), top, rt);
        if (lo > cut) {
            unsigned long long n = 0;
            for (int i = tid; i < V; i += SM_THREADS) n += float_key(logit(x[i])) == lo;
            ties = block_sum(n, sh);
        }
        // of the equal ones, those with less than `want` before them (one at least where it is the maximum)
        unsigned long long j = 0;
        while (j < ties && (double)(above + j * w) < want && w) j++;
        if (w) ties = j;
        if (lo == top_key && ties == 0) ties = 1;
        cut = lo;
    }
    const float mp = a.min_p ? a.min_p[row] : 0.0f;
    // rank among the equal ones and running mass, in index order
    unsigned long long done_ties = 0;
    unsigned long long total = 0;
    for (int pass = 0; pass < 2; pass++) {
        unsigned long long run = 0, want = 0;
        if (pass) {
            const float u = a.u[row];
            const double r = floor((double)u * (double)total);
            want = r > 0 ? (unsigned long long)r : 0;
            if (want >= total) want = total - 1;
        }
        done_ties = 0;
        __shared__ int found;
        if (tid == 0) found = -1;
        __syncthreads();
        for (int base = 0; base < V; base += SM_THREADS) {
            const int i = base + tid;
            const float v = i < V ? logit(x[i]) : -INFINITY;
            const uint32_t key = float_key(v);
            const bool tie = i < V && key == cut;
            // exclusive rank of this tie in the chunk
            const unsigned mask = __ballot_sync(0xffffffffu, tie);
            __syncthreads();
            if ((tid & 31) == 0) sh[tid >> 5] = __popc(mask);
            __syncthreads();
            unsigned long long before = 0, all = 0;
            for (int w = 0; w < SM_THREADS / 32; w++) {
                if (w == (tid >> 5)) before = all;
                all += sh[w];
            }
            const unsigned long long rank = done_ties + before + __popc(mask & ((1u << (tid & 31)) - 1));
            done_ties += all;
            unsigned long long w = 0;
            if (i < V && (key > cut || (tie && rank < ties))) {
                w = weight(v, top, rt);
                if ((double)w < (double)mp * 8796093022208.0) w = 0;
            }
            unsigned long long inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
                if ((tid & 31) >= o) inc += y;
            }
            __syncthreads();
            if ((tid & 31) == 31) sh[tid >> 5] = inc;
            __syncthreads();
            unsigned long long pre = 0, sum = 0;
            for (int q = 0; q < SM_THREADS / 32; q++) {
                if (q == (tid >> 5)) pre = sum;
                sum += sh[q];
            }
            const unsigned long long c1 = run + pre + inc, c0 = c1 - w;
            if (pass && w && c0 <= want && want < c1) found = i;
            run += sum;
        }
        if (!pass) total = run;
        __syncthreads();
        if (pass && tid == 0) a.tokens[row] = found;
    }
}

}  // namespace ptc

extern "C" int ptc_sample_tokens(const ptc_sample_args *p, void *stream) {
    if (!p) SERVE_REFUSE("no arguments");
    const ptc_sample_args a = *p;
    if (!ptc::dtype_ok(a.dtype)) SERVE_REFUSE("the logits' type is none of PTC_F32, PTC_F16, PTC_BF16");
    if (a.rows < 0 || a.vocab < 1 || a.vocab > PTC_SAMPLE_MAX_VOCAB || a.stride < a.vocab)
        SERVE_REFUSE("bad size (rows %d, vocab %d of at most %d, stride %lld)", a.rows, a.vocab, PTC_SAMPLE_MAX_VOCAB, a.stride);
    if (a.rows == 0) return 0;
    if (!a.logits || !a.u || !a.tokens) SERVE_REFUSE("a required pointer is NULL");
    if ((uintptr_t)a.logits % ptc::dtype_bytes(a.dtype)) SERVE_REFUSE("the logits are not aligned to their type");
    cudaStream_t s = (cudaStream_t)stream;
    ptc::MemoryDevice on(a.tokens);
    SERVE_CUDA(on.error());
    if (a.dtype == PTC_F32) ptc::k_sample<float><<<a.rows, ptc::SM_THREADS, 0, s>>>(a);
    else if (a.dtype == PTC_F16) ptc::k_sample<__half><<<a.rows, ptc::SM_THREADS, 0, s>>>(a);
    else ptc::k_sample<__nv_bfloat16><<<a.rows, ptc::SM_THREADS, 0, s>>>(a);
    SERVE_CUDA(cudaGetLastError());
    return 0;
}
