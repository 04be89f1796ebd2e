// paged_attn.cu -- attention of a batch's new tokens over a paged KV cache:
//   o = sum_s p_s v_s / sum_s p_s,  p_s = exp(scale q k_s - max),  s over the visible slots.
#include "paged.cuh"

namespace cuq {

namespace {

// One warp per (token, query head); lanes hold HD / 32 dims, one slot at a time.
template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(128) attn_paged_simple(PagedArgs a, PagedQuery q, TQ *out, size_t out_stride,
                                                         float *lse) {
    constexpr int E = HD / 32;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t head = blockIdx.y, b = blockIdx.z, kvh = head / q.group;
    uint32_t first;
    const uint32_t nq = a.tokens(b, first);
    const uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= nq || i >= a.max_q) return;
    const uint32_t tok = first + i, n = a.len(b);
    const int pos = (int)n - (int)nq + (int)i;
    uint32_t lo, hi;
    q.range(pos, n, lo, hi);
    const TQ *qr = reinterpret_cast<const TQ *>(q.q) + (size_t)tok * q.q_stride + (size_t)head * HD + lane * E;
    float qv[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) qv[e] = (float)qr[e] * q.scale, acc[e] = 0.f;
    for (uint32_t s = lo; s < hi; s++) {
        const int pg = a.page(b, s >> a.page_shift);
        if (pg < 0) continue;
        const size_t at = a.row<HD>(pg, kvh, s) + lane * E;
        const TC *kr = reinterpret_cast<const TC *>(a.k) + at, *vr = reinterpret_cast<const TC *>(a.v) + at;
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) d += qv[e] * (float)kr[e];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(~0u, d, o);
        const float mn = fmaxf(m, d), c = __expf(m - mn), w = __expf(d - mn);
        l = l * c + w;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = acc[e] * c + w * (float)vr[e];
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    TQ *o = out + (size_t)tok * out_stride + (size_t)head * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = (TQ)(acc[e] * inv);
    if (lse && lane == 0) lse[(size_t)tok * q.heads + head] = l > 0.f ? m + logf(l) : -INFINITY;
}

template <typename TQ, typename TC>
int launch_simple(const AttnPagedCall &c, cudaStream_t s) {
    const dim3 grid((c.a.max_q + 3) / 4, c.q.heads, c.a.n_seqs);
    if (c.hd == 64)
        attn_paged_simple<TQ, TC, 64><<<grid, 128, 0, s>>>(c.a, c.q, (TQ *)c.out, c.out_stride, c.lse);
    else
        attn_paged_simple<TQ, TC, 128><<<grid, 128, 0, s>>>(c.a, c.q, (TQ *)c.out, c.out_stride, c.lse);
    CUQ_CUDA_TRY(cudaGetLastError());
    return CUQ_OK;
}

}  // namespace

size_t attention_paged_workspace(const AttnPagedCall &, int) { return 0; }

int launch_attention_paged(const AttnPagedCall &c, int, cudaStream_t s) {
    if (c.type == CUQ_F32) return launch_simple<float, __half>(c, s);
    if (c.type == CUQ_F16) return launch_simple<__half, __half>(c, s);
    return launch_simple<__nv_bfloat16, __nv_bfloat16>(c, s);
}

}  // namespace cuq
