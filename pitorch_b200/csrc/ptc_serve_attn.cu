// ptc_serve_attn.cu -- attention of new tokens over a paged KV cache
// (include/ptc_serve.h).
#include "ptc_serve.cuh"

namespace ptc {

constexpr int PA_WARPS = 8;

// One warp per (row, head), a pass over the keys with the running maximum and
// sum. Lane l holds 4 elements of the head dimension.
template <typename T>
__global__ void __launch_bounds__(PA_WARPS * 32) k_paged_attn(ptc_attn_args a) {
    const ptc_paged_cache &c = a.cache;
    const int lane = threadIdx.x & 31, hd = c.head_dim;
    const int r = blockIdx.x, head = blockIdx.y, kvh = head / (a.n_heads / c.n_kv_heads);
    const int q0 = a.q_start[r], q1 = a.q_start[r + 1], kv = a.kv_len[r];
    if (q0 < 0 || q1 < q0 || q1 > a.n_tokens || kv < 0) {
        if (threadIdx.x == 0) serve_err(a.err, PTC_SERVE_ERR_LENGTH);
        return;
    }
  for (int row = q0 + (threadIdx.x >> 5); row < q1; row += PA_WARPS) {
    const int pos = kv - (q1 - q0) + row - q0;
    const bool on = lane * 4 < hd;
    float q[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0}, m = -INFINITY, sum = 0.f;
    if (on)
        for (int i = 0; i < 4; i++) q[i] = Elem<T>::up(((const T *)a.q)[row * a.q_stride + (long long)head * hd + lane * 4 + i]) * a.scale;
    int end = pos + 1;
    if (end > (long long)a.max_pages * c.page_size) {
        if (lane == 0) serve_err(a.err, PTC_SERVE_ERR_LENGTH);
        end = min((long long)end, (long long)a.max_pages * c.page_size);
    }
    int t = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    for (; t < end; t++) {
        const int page = a.page_table[(long long)r * a.max_pages + t / c.page_size];
        if ((unsigned)page >= (unsigned)c.n_pages) {
            if (lane == 0) serve_err(a.err, PTC_SERVE_ERR_INDEX);
            continue;
        }
        const long long at = page * c.page_stride + kvh * c.head_stride + (t % c.page_size) * c.token_stride + lane * 4;
        float s = 0.f;
        if (on)
            for (int i = 0; i < 4; i++) s += q[i] * Elem<T>::up(((const T *)c.k)[at + i]);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - mn), p = expf(s - mn);
        sum = sum * f + p;
        m = mn;
        if (on)
            for (int i = 0; i < 4; i++) o[i] = o[i] * f + p * Elem<T>::up(((const T *)c.v)[at + i]);
    }
    if (on)
        for (int i = 0; i < 4; i++) ((T *)a.out)[row * a.out_stride + (long long)head * hd + lane * 4 + i] = Elem<T>::down(sum > 0.f ? o[i] / sum : 0.f);
  }
}

}  // namespace ptc

extern "C" int ptc_paged_attention(const ptc_attn_args *p, void *stream) {
    if (!p) SERVE_REFUSE("no arguments");
    const ptc_attn_args a = *p;
    if (const char *why = ptc::check_cache(a.cache)) SERVE_REFUSE("%s", why);
    if (a.n_seqs < 0 || a.n_tokens < 0 || a.max_pages < 1 || a.max_q < 0 || a.window < 0)
        SERVE_REFUSE("bad size (n_seqs %d, n_tokens %d, max_q %d, max_pages %d, window %d)", a.n_seqs, a.n_tokens, a.max_q,
                     a.max_pages, a.window);
    if (a.n_heads < 1 || a.n_heads % a.cache.n_kv_heads)
        SERVE_REFUSE("n_heads %d is no multiple of n_kv_heads %d", a.n_heads, a.cache.n_kv_heads);
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) SERVE_REFUSE("scale is not finite");
    if (a.n_seqs == 0 || a.n_tokens == 0) return 0;
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
    const dim3 grid(a.n_seqs, a.n_heads);
    if (a.cache.dtype == PTC_F32) ptc::k_paged_attn<float><<<grid, ptc::PA_WARPS * 32, 0, s>>>(a);
    else if (a.cache.dtype == PTC_F16) ptc::k_paged_attn<__half><<<grid, ptc::PA_WARPS * 32, 0, s>>>(a);
    else ptc::k_paged_attn<__nv_bfloat16><<<grid, ptc::PA_WARPS * 32, 0, s>>>(a);
    SERVE_CUDA(cudaGetLastError());
    return 0;
}
