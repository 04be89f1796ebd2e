// paged.cuh -- what the paged-cache kernels share: the device view of a cache
// and a batch (include/cuq.h, cuq_paged_kv / cuq_batch), typed loads and stores.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"

namespace cuq {

// Every kernel of these ops is launched as a programmatic dependent of what the
// stream holds before it, and waits (griddepcontrol.wait) in every thread before it
// reads anything that may come from there: the order is the stream's, and a launch
// costs 1 to 2 us less than one that waits for the stream to run dry.  That an earlier
// grid has waited is not enough for a later one that it let start: only its own wait
// makes what was written before visible to it.  (Reading the batch before the wait
// gained 0.5 us in the merge and 0.3 in the eviction's move, and starting the few-row
// kernel beside the many-row one 8 us of 31 in a mixed batch.)  A kernel may thus be
// resident while its inputs are still written (the selection's list and the move that
// reads it), so all of them are read by plain loads: the read-only path (ld.global.nc)
// asks for data that does not change while the kernel lives.

// SM count of the current device, asked for once per device.
int paged_sm_count();
// Let `kernel` use `bytes` of dynamic shared memory, set once per device (`done`
// holds a bit for each of the first 64; others are set every time).
template <typename K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Shared memory of the cluster's CTA `rank`, and the barrier over all of its CTAs.
__device__ __forceinline__ uint32_t peer_smem(const void *p, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(at)
                 : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ float peer_load(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The cache and the batch as a kernel sees them.  Every length and page id that
// comes from device memory is cut or checked here, so no kernel reads past a
// pool, a table or a token tensor whatever the arrays hold.
struct PagedArgs {
    void *k, *v;
    uint64_t page_stride;            // elements
    uint32_t n_pages, page_size, page_shift, kv_heads;
    const int32_t *q_start, *kv_len, *pages;
    uint32_t n_seqs, n_tok, pages_stride, max_q, max_kv;  // max_kv: already cut to the table's slots

    __device__ __forceinline__ uint32_t len(uint32_t b) const {
        const int n = kv_len[b];
        return n <= 0 ? 0u : min((uint32_t)n, max_kv);
    }
    // first token row of sequence b and its token count (at most n_tok rows in all)
    __device__ __forceinline__ uint32_t tokens(uint32_t b, uint32_t &first) const {
        const int a = q_start[b], e = q_start[b + 1];
        first = a <= 0 ? 0u : min((uint32_t)a, n_tok);
        const uint32_t end = e <= 0 ? 0u : min((uint32_t)e, n_tok);
        return end > first ? end - first : 0u;
    }
    // the sequence of token row `tok`, by a whole warp: how many sequences end at or before
    // it (q_start ascends), 32 probes at a time; n_seqs for a row of no sequence
    __device__ __forceinline__ uint32_t sequence_of(int tok) const {
        const uint32_t lane = threadIdx.x & 31;
        uint32_t lo = 0, size = n_seqs;
        while (size) {
            const uint32_t step = (size + 31) / 32, end = lo + size, last = lo + (lane + 1) * step - 1;
            lo += step * __popc(__ballot_sync(~0u, last < end && q_start[last + 1] <= tok));
            size = lo < end ? min(step - 1, end - lo) : 0;
        }
        return min(lo, n_seqs);
    }
    __device__ __forceinline__ int page(uint32_t b, uint32_t col) const {
        const int id = pages[(size_t)b * pages_stride + col];
        return (id >= 0 && (uint32_t)id < n_pages) ? id : -1;
    }
    // element offset of row `slot` of KV head h inside a pool; the page id is valid
    template <int HD>
    __device__ __forceinline__ size_t row(int page_id, uint32_t h, uint32_t slot) const {
        return (size_t)page_id * page_stride + ((size_t)h * page_size + (slot & (page_size - 1))) * HD;
    }
};

// q, lse and the mask of the attention ops.
struct PagedQuery {
    const void *q;
    size_t q_stride;
    uint32_t heads, group, group_inv;  // group_inv: ceil(2^32 / group)
    float scale;
    int causal;
    uint32_t window;

    // x / group for x below 2^16 + group (so that x * group stays below 2^32)
    __device__ __forceinline__ uint32_t div_group(uint32_t x) const { return group == 1 ? x : __umulhi(x, group_inv); }

    // the slots [lo, hi) that the query at slot `pos` of a cache of n slots sees
    __device__ __forceinline__ void range(int pos, uint32_t n, uint32_t &lo, uint32_t &hi) const {
        lo = 0;
        hi = n;
        if (pos < 0) {
            hi = 0;
            return;
        }
        if (causal) {
            hi = min(n, (uint32_t)pos + 1);
            if (window && (uint32_t)pos + 1 > window) lo = (uint32_t)pos + 1 - window;
        }
    }
};

template <typename T>
struct Pair;  // two 16-bit values in one register
template <>
struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&u));
    }
};
template <>
struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
    }
};

// eight values of any of the three types, as fp32: one 16-byte vector, or two of fp32
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 (&u)[sizeof(T) == 4 ? 2 : 1], float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(u[0].x), v[1] = __uint_as_float(u[0].y), v[2] = __uint_as_float(u[0].z);
        v[3] = __uint_as_float(u[0].w), v[4] = __uint_as_float(u[1].x), v[5] = __uint_as_float(u[1].y);
        v[6] = __uint_as_float(u[1].z), v[7] = __uint_as_float(u[1].w);
    } else {
        const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = Pair<T>::unpack(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(Pair<T>::pack(v[0], v[1]), Pair<T>::pack(v[2], v[3]),
                                               Pair<T>::pack(v[4], v[5]), Pair<T>::pack(v[6], v[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float *p, const float (&v)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// ------------------------------------------------------------ attention ----
//
// A sequence's rows are its (new token, query head of the group) pairs, token
// major.  Sequences of up to ATTN_FEW rows per KV head go to the mma.sync kernel
// (paged_attn.cu), whose tile is 16 rows and whose time is the cache's bytes;
// larger ones to the tcgen05 kernel (paged_attn_tc.cu), 2 x 128 rows.  Both may
// split the slots: parts, out normalised and the log2 of the sum of exponentials,
// go to the workspace and are joined by the merge kernel.
constexpr uint32_t ATTN_FEW = 16;

struct AttnPagedCall {
    PagedArgs a;
    PagedQuery q;
    void *out;
    size_t out_stride;
    float *lse;
    int type, cache_type;
    uint32_t hd;
    void *workspace;
};

// How a call is split; a function of the call's host-side sizes alone.
struct AttnPlan {
    bool few, many;        // which kernels run
    uint32_t few_ctas;     // of the mma.sync kernel; its warps share the blocks out evenly
    uint32_t few_rows;     // rows of a part
    uint32_t few_cluster;  // CTAs that take one (sequence, KV head) between them and join its parts; 0: runs and a merge
    uint32_t many_splits;
    uint32_t many_tiles;   // bound of the 256-row tiles of all sequences
    // whether a sequence of `tokens` attended tokens is the mma.sync kernel's
    __device__ __forceinline__ bool is_few(uint32_t tokens, uint32_t group) const {
        return few && tokens * group <= ATTN_FEW;
    }
};
AttnPlan attention_paged_plan(const AttnPagedCall &c, int sm_count);
size_t attention_paged_workspace(const AttnPagedCall &c, int sm_count);
int launch_attention_paged(const AttnPagedCall &c, int sm_count, cudaStream_t s);

// What both kernels get beside the cache and the queries.
struct AttnOut {
    void *out;
    size_t out_stride;
    float *lse;
    // parts: normalised outputs [part][rows][hd] and log2 sums [part][rows]; rows are
    // few_rows of the few, [n_tok][heads] of the many
    float *few_o, *few_lse, *many_o, *many_lse;
    uint32_t *few_units;  // [n_seqs + 1]: units of the few's sequences before each (per KV head)
    AttnPlan plan;
};
int launch_attention_many(const AttnPagedCall &c, const AttnOut &o, cudaStream_t s);
// bounded waits that gave up on this device so far (waits for the stream)
int attention_many_gave_up(cudaStream_t s, unsigned int *n);
int attention_few_gave_up(cudaStream_t s, unsigned int *n);
int launch_wait_probe(uint32_t limit_us, cudaStream_t s);

struct MassPagedCall {
    PagedArgs a;
    PagedQuery q;
    float *mass;
    size_t mass_stride;
    const float *lse;
    int type, cache_type;
    uint32_t hd, last_q;
    float decay;
};
int launch_attention_mass(const MassPagedCall &c, int sm_count, cudaStream_t s);
int attention_mass_gave_up(cudaStream_t s, unsigned int *n);

}  // namespace cuq
