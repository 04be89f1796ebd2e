// paged_mass.cu -- the attention weight that each cached slot gathers:
//   mass[b][kv head][s] = decay mass + sum over queries and heads of exp(scale q k_s - lse).
#include "paged.cuh"

namespace cuq {

namespace {

// One warp per slot; lanes hold HD / 32 dims, one query at a time.
template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(128) mass_simple(PagedArgs a, PagedQuery q, float *mass, size_t mass_stride,
                                                   const float *lse, uint32_t last_q, float decay) {
    constexpr int E = HD / 32;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t kvh = blockIdx.y, b = blockIdx.z;
    const uint32_t n = a.len(b), s = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (s >= n) return;
    uint32_t first;
    const uint32_t nq = a.tokens(b, first);
    const uint32_t i1 = min(nq, a.max_q), i0 = (last_q && nq > last_q) ? nq - last_q : 0;
    const int pg = a.page(b, s >> a.page_shift);
    float sum = 0.f;
    if (pg >= 0) {
        const TC *kr = reinterpret_cast<const TC *>(a.k) + a.row<HD>(pg, kvh, s) + lane * E;
        float kv[E];
#pragma unroll
        for (int e = 0; e < E; e++) kv[e] = (float)kr[e];
        for (uint32_t i = i0; i < i1; i++) {
            uint32_t lo, hi;
            q.range((int)n - (int)nq + (int)i, n, lo, hi);
            if (s < lo || s >= hi) continue;
            for (uint32_t g = 0; g < q.group; g++) {
                const uint32_t tok = first + i, head = kvh * q.group + g;
                const TQ *qr = reinterpret_cast<const TQ *>(q.q) + (size_t)tok * q.q_stride + (size_t)head * HD +
                               lane * E;
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) d += (float)qr[e] * kv[e];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(~0u, d, o);
                sum += __expf(d * q.scale - lse[(size_t)tok * q.heads + head]);
            }
        }
    }
    if (lane == 0) {
        float *m = mass + ((size_t)b * a.kv_heads + kvh) * mass_stride + s;
        *m = decay == 0.f ? sum : decay * *m + sum;
    }
}

template <typename TQ, typename TC>
int launch_simple(const MassPagedCall &c, cudaStream_t s) {
    const dim3 grid((c.a.max_kv + 3) / 4, c.a.kv_heads, c.a.n_seqs);
    if (c.hd == 64)
        mass_simple<TQ, TC, 64><<<grid, 128, 0, s>>>(c.a, c.q, c.mass, c.mass_stride, c.lse, c.last_q, c.decay);
    else
        mass_simple<TQ, TC, 128><<<grid, 128, 0, s>>>(c.a, c.q, c.mass, c.mass_stride, c.lse, c.last_q, c.decay);
    CUQ_CUDA_TRY(cudaGetLastError());
    return CUQ_OK;
}

}  // namespace

int launch_attention_mass(const MassPagedCall &c, int, cudaStream_t s) {
    if (c.type == CUQ_F32) return launch_simple<float, __half>(c, s);
    if (c.type == CUQ_F16) return launch_simple<__half, __half>(c, s);
    return launch_simple<__nv_bfloat16, __nv_bfloat16>(c, s);
}

}  // namespace cuq
