// paged.cu -- serving from a paged KV cache: the checks behind the cuq_* entry
// points, rotary positions with the append, and the eviction.  The attention
// over the cache is in paged_attn.cu, the gathered attention weight in
// paged_mass.cu.
#include <cmath>
#include <limits>
#include <map>
#include <mutex>
#include <new>
#include <type_traits>
#include <utility>

#include "paged.cuh"

namespace cuq {

int sm_count_current();

int paged_sm_count() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return sm_count_current();
    int n = known[dev].load(std::memory_order_relaxed);
    if (!n) {
        n = sm_count_current();
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

constexpr int ROPE_MAX_PAIRS = 64;

// Angle per position of each pair, as a fraction of a turn in units of 2^-64.
// pos * turns then wraps by itself: the product modulo 2^64 is the angle's
// fractional turn.  The frequencies are worked out with 64-bit significands (x87's),
// a few of whose steps, for at most 0.16 turns a position, and the rounding to 2^-64
// are at most 2^-63: |pos| 2^-63 turns in all (2^-32 at pos = 2^31).
struct RopeTable {
    uint64_t turns[ROPE_MAX_PAIRS];
    float mul;  // factor on cosine and sine
    uint32_t rot;
    int adjacent;
};
}  // namespace cuq

struct cuq_rope_plan {
    cuq::RopeTable t;
};

namespace cuq {
namespace {

// ------------------------------------------------- rotary + append ----
//
// Bound by HBM for prompts (every value is read and written once) and by
// latency for a few tokens.  A CTA takes T tokens: a warp each finds its
// sequence, slot and page, the threads work out the T * rot/2 cosines and sines,
// one each, into shared memory, and then walk the rows (token, head) in units:
// the 16 values that hold 8 whole pairs, two 16-byte vectors at j and j + rot/2,
// or 16 values in a row.  4096 tokens (32 heads, 8 KV heads, head_dim 128, fp16, 101 MB)
// take 21.2 us, 4.75 TB/s, 74 % of a copy's rate (from fp32 34.8 us, 5.3 TB/s); more loads
// in flight a thread cost occupancy and made it slower (31 us).
struct RopeArgs {
    PagedArgs a;
    const int32_t *positions;
    void *q_out;
    size_t q_out_stride;
    const void *q, *k, *v;
    size_t q_stride, kv_stride;
    uint32_t heads;
};

__device__ __forceinline__ void store_as(int type, void *base, size_t at, const float (&v)[8]) {
    if (type == CUQ_F32)
        store8(reinterpret_cast<float *>(base) + at, v);
    else if (type == CUQ_F16)
        store8(reinterpret_cast<__half *>(base) + at, v);
    else
        store8(reinterpret_cast<__nv_bfloat16 *>(base) + at, v);
}

template <typename T>
__device__ constexpr int in_type_of() {
    return sizeof(T) == 4 ? CUQ_F32 : std::is_same<T, __half>::value ? CUQ_F16 : CUQ_BF16;
}

constexpr int ROPE_THREADS = 256;

template <typename TI, int HD, int T>
__global__ void __launch_bounds__(ROPE_THREADS) rope_append_kernel(RopeArgs p, RopeTable tab, int out_type,
                                                                    int cache_type) {
    __shared__ __align__(16) float cs[T][4][ROPE_MAX_PAIRS / 8][2][2];
    __shared__ int s_pos[T], s_slot[T], s_page[T];
    __shared__ int s_seq[T];
    constexpr uint32_t UNITS = HD / 16, STEP = ROPE_THREADS / UNITS;
    const uint32_t tok0 = blockIdx.x * T, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t half = tab.rot / 2, u = threadIdx.x % UNITS, rows = p.heads + 2 * p.a.kv_heads;
    griddep_wait();
    // row r (q heads, k heads, v heads) of a token
    auto source = [&](uint32_t tok, uint32_t r) -> const TI * {
        if (r < p.heads) return reinterpret_cast<const TI *>(p.q) + (size_t)tok * p.q_stride + (size_t)r * HD;
        const bool is_v = r >= p.heads + p.a.kv_heads;
        return reinterpret_cast<const TI *>(is_v ? p.v : p.k) + (size_t)tok * p.kv_stride +
               (size_t)(r - p.heads - (is_v ? p.a.kv_heads : 0)) * HD;
    };
    // into L2 while the tokens are found: 4096 tokens 23.1 us instead of 24.6 (a few tokens gain nothing by it)
    constexpr uint32_t LINES = T > 1 ? HD * sizeof(TI) / 128 : 0;
    for (uint32_t i = threadIdx.x; i < T * rows * LINES; i += ROPE_THREADS) {
        const uint32_t row = i / max(1u, LINES), t = row / rows;
        if (tok0 + t < p.a.n_tok)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(source(tok0 + t, row - t * rows) + (i % max(1u, LINES)) * (128 / sizeof(TI))));
    }
    if (warp < T) {
        const int tok = (int)(tok0 + warp);
        const int given = p.positions && tok < (int)p.a.n_tok ? p.positions[tok] : 0;
        const uint32_t n = p.a.sequence_of(tok);
        if (lane == 0) {
            int seq = -1, slot = -1, page = -1;
            if (n < p.a.n_seqs && tok < (int)p.a.n_tok) {
                uint32_t first;
                const uint32_t nq = p.a.tokens(n, first);
                const int len = (int)p.a.len(n);
                if ((uint32_t)tok >= first && (uint32_t)tok < first + nq) {
                    seq = (int)n;
                    slot = len - (int)nq + (tok - (int)first);
                    if (slot >= 0) page = p.a.page(n, (uint32_t)slot >> p.a.page_shift);
                }
            }
            s_seq[warp] = seq;
            s_slot[warp] = slot;
            s_page[warp] = page;
            s_pos[warp] = p.positions ? given : slot;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < T * half; i += ROPE_THREADS) {
        const uint32_t t = i / half, j = i % half;
        const int64_t turn = (int64_t)((uint64_t)(int64_t)s_pos[t] * tab.turns[j]);
        // the top 32 bits are the turn in [-1/2, 1/2); as an fp32 it is off by at most
        // 2^-26 turns (9.4e-8 radians, the fp32 rounding of any angle up to pi)
        const float x = (float)(int32_t)(turn >> 32) * 0x1p-31f;  // in units of pi
        float si, co;
        sincospif(x, &si, &co);
        // pairs 2 m, 2 m + 1 of unit j / 8 at [m][unit]: neighbouring units read without bank conflicts
        cs[t][(j % 8) / 2][j / 8][0][j & 1] = co * tab.mul;
        cs[t][(j % 8) / 2][j / 8][1][j & 1] = si * tab.mul;
    }
    __syncthreads();
    const bool rot_unit = u < tab.rot / 16;
    uint32_t t = 0, r = threadIdx.x / UNITS;
    for (;; r += STEP) {
        while (r >= rows) {
            r -= rows;
            t++;
        }
        if (t >= (uint32_t)T) break;
        const uint32_t tok = tok0 + t;
        const bool is_q = r < p.heads, is_v = r >= p.heads + p.a.kv_heads, turn = rot_unit && !is_v;
        if (s_seq[t] < 0 || (!is_q && s_page[t] < 0)) continue;
        const bool apart = turn && !tab.adjacent;
        const uint32_t e0 = apart ? 8 * u : 16 * u, e1 = apart ? half + 8 * u : 16 * u + 8;
        const TI *src = source(tok, r);
        void *to;
        size_t at;
        if (is_q) {
            to = p.q_out;
            at = (size_t)tok * p.q_out_stride + (size_t)r * HD;
        } else {
            const uint32_t h = r - p.heads - (is_v ? p.a.kv_heads : 0);
            to = is_v ? p.a.v : p.a.k;
            at = p.a.row<HD>(s_page[t], h, (uint32_t)s_slot[t]);
        }
        constexpr int W = sizeof(TI) == 4 ? 2 : 1;  // vectors of 8 values
        uint4 ra[W], rb[W];
#pragma unroll
        for (int w = 0; w < W; w++) {
            ra[w] = *(reinterpret_cast<const uint4 *>(src + e0) + w);
            rb[w] = *(reinterpret_cast<const uint4 *>(src + e1) + w);
        }
        const int type = is_q ? out_type : cache_type;
        if (!turn && type == in_type_of<TI>()) {  // as it is
#pragma unroll
            for (int w = 0; w < W; w++) {
                *(reinterpret_cast<uint4 *>(reinterpret_cast<TI *>(to) + at + e0) + w) = ra[w];
                *(reinterpret_cast<uint4 *>(reinterpret_cast<TI *>(to) + at + e1) + w) = rb[w];
            }
            continue;
        }
        float a[8], b[8];
        unpack8<TI>(ra, a);
        unpack8<TI>(rb, b);
        if (turn && !tab.adjacent) {
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const float4 c = *reinterpret_cast<const float4 *>(cs[t][m][u]);  // co, co, si, si
                float x = a[2 * m], y = b[2 * m];
                a[2 * m] = x * c.x - y * c.z;
                b[2 * m] = x * c.z + y * c.x;
                x = a[2 * m + 1], y = b[2 * m + 1];
                a[2 * m + 1] = x * c.y - y * c.w;
                b[2 * m + 1] = x * c.w + y * c.y;
            }
        } else if (turn) {
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const float4 c = *reinterpret_cast<const float4 *>(cs[t][m][u]);
                float *v = m < 2 ? a + 4 * m : b + 4 * (m - 2);  // pairs 2 m, 2 m + 1
                float x = v[0], y = v[1];
                v[0] = x * c.x - y * c.z;
                v[1] = x * c.z + y * c.x;
                x = v[2], y = v[3];
                v[2] = x * c.y - y * c.w;
                v[3] = x * c.w + y * c.y;
            }
        }
        store_as(type, to, at + e0, a);
        store_as(type, to, at + e1, b);
    }
}

template <typename TI>
int launch_rope_append(const RopeArgs &p, const RopeTable &t, int out_type, int cache_type, uint32_t hd,
                       cudaStream_t s) {
    // two tokens a CTA once there are CTAs enough.  16, 512, 1024, 2048, 4096 and 8192
    // tokens (32 heads, 8 KV heads, head_dim 128, fp16, in a graph) take 3.4, 4.3, 7.3, 14.0,
    // 24.5 and 44.5 us with one each, 4.4, 4.9, 6.8, 14.1, 21.3 and 35.1 with two; four each
    // made 4096 tokens 2 us slower
    const bool many = p.a.n_tok >= 1024;
    const uint32_t grid = many ? (p.a.n_tok + 1) / 2 : p.a.n_tok;
    auto launch = [&](auto kernel) {
        return launch_maybe_pdl(kernel, dim3(grid), dim3(ROPE_THREADS), 0, s, true, p, t, out_type, cache_type);
    };
    CUQ_CUDA_TRY(hd == 64 ? (many ? launch(rope_append_kernel<TI, 64, 2>) : launch(rope_append_kernel<TI, 64, 1>))
                          : (many ? launch(rope_append_kernel<TI, 128, 2>) : launch(rope_append_kernel<TI, 128, 1>)));
    return CUQ_OK;
}

// ------------------------------------------------------- eviction ----
//
// Radix selection, bound by latency: a cluster of CTAs takes one (sequence, KV head),
// each a contiguous slice of its slots.  Masses become 32-bit keys in their order
// (NaN lowest), eight a thread, kept in registers where the slice fits.
// Up to three histogram passes (11, 11, 10 bits) find the key of the last slot kept and
// how many of its equals are kept, and end at a bin that is kept whole: every CTA
// counts its own slice, adds the bins it hit into every CTA's sums through distributed
// shared memory, and works the digit out for itself.  Then the slices' counts are exchanged and the kept slots written at
// their prefix sums.  Histogram atomics count whole numbers, so their order does not
// matter.  At most five cluster barriers; with rank 0 finding the digits it was ten.
// 4096 slots take one CTA about 8.5 us, 32768 a cluster of eight 12 us, mostly barriers
// and latencies; always in three passes it was 9 and 13.
constexpr int SEL_THREADS = 512, SEL_BINS = 2048, SEL_PER = 8;
constexpr uint32_t SEL_TILE = SEL_THREADS * SEL_PER;

__device__ __forceinline__ uint32_t mass_key(float m) {
    if (m != m) return 0u;
    const uint32_t u = __float_as_uint(m + 0.f);  // -0 becomes +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct EvictArgs {
    PagedArgs a;
    const float *mass;
    size_t mass_stride;
    uint32_t keep, sink, recent;
    int32_t *kept, *new_len;
    float *mass_out;
    size_t mass_out_stride;
};

__device__ __forceinline__ void peer_add(uint32_t at, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void peer_store(uint32_t at, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(EvictArgs p) {
    __shared__ __align__(16) uint32_t hist[SEL_BINS];     // this slice's counts
    __shared__ __align__(16) uint32_t sums[3][SEL_BINS];  // the cluster's, one set a pass
    __shared__ uint32_t s_digit, s_need, s_whole, s_above[8], s_equal[8], warp_a[SEL_THREADS / 32];
    __shared__ uint2 s_run[SEL_PER * SEL_THREADS / 32];  // kept for sure and equal, by warps of slots
    uint32_t rank, ranks;
    griddep_wait();
    griddep_launch();  // the move may take its place; it waits for this grid's end
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const uint32_t x = blockIdx.x / ranks, b = x / p.a.kv_heads, h = x % p.a.kv_heads;
    const uint32_t n = p.a.len(b), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *mass = p.mass + ((size_t)b * p.a.kv_heads + h) * p.mass_stride;
    int32_t *kept = p.kept + ((size_t)b * p.a.kv_heads + h) * p.keep;
    if (h == 0 && rank == 0 && tid == 0) p.new_len[b] = (int32_t)min(n, p.keep);
    if (n <= p.keep) {  // the same for the whole cluster
        for (uint32_t i = rank * SEL_THREADS + tid; i < p.keep; i += ranks * SEL_THREADS)
            kept[i] = i < n ? (int32_t)i : -1;
        return;
    }
    auto sync = [&]() {
        if (ranks > 1)
            cluster_sync();
        else
            __syncthreads();
    };
    // the slots in between, of which `need` are kept, and this CTA's slice of all slots
    const uint32_t lo = p.sink, hi = n - p.recent;
    const uint32_t per = (n + ranks - 1) / ranks, i0 = min(n, rank * per), i1 = min(n, i0 + per);
    const bool resident = per <= SEL_TILE;
    uint32_t key[SEL_PER];
    auto load = [&](uint32_t t0) {  // the thread's keys of the tile at t0; 0 past the slice
#pragma unroll
        for (int e = 0; e < SEL_PER; e++) {
            const uint32_t i = t0 + e * SEL_THREADS + tid;
            key[e] = i < i1 ? mass_key(mass[i]) : 0u;
        }
    };
    if (resident) load(i0);
    for (uint32_t i = tid; i < SEL_BINS; i += SEL_THREADS) hist[i] = sums[0][i] = sums[1][i] = sums[2][i] = 0;
    sync();  // the sums are clear everywhere
    uint32_t need = p.keep - p.sink - p.recent, prefix = 0;
    uint32_t edge = 0xFFFFFFFFu;  // no float has this key: nothing in between is kept
    constexpr int SHIFT[3] = {21, 10, 0}, BITS[3] = {11, 11, 10};
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        if (need == 0) break;  // nothing in between is kept
        const int shift = SHIFT[pass], bits = BITS[pass], bins = 1 << bits;
        for (uint32_t t0 = i0; t0 < i1; t0 += SEL_TILE) {
            if (!resident) load(t0);
            const uint32_t first = t0 + tid;
#pragma unroll
            for (int e = 0; e < SEL_PER; e++) {
                const uint32_t i = first + e * SEL_THREADS;
                if (i >= lo && i < hi && i < i1 && (pass == 0 || (key[e] >> (shift + bits)) == prefix))
                    atomicAdd(&hist[(key[e] >> shift) & (bins - 1)], 1u);
            }
        }
        __syncthreads();
        if (ranks > 1) {
            for (uint32_t i = tid; i < (uint32_t)bins; i += SEL_THREADS) {
                const uint32_t v = hist[i];
                hist[i] = 0;
                if (v)
                    for (uint32_t r = 0; r < ranks; r++) peer_add(peer_smem(&sums[pass][i], r), v);
            }
            cluster_sync();
        }
        // the bin, from the top, in which the need-th key lies
        uint32_t *c = ranks > 1 ? sums[pass] : hist;
        constexpr int PER = SEL_BINS / SEL_THREADS;  // thread t: bins [bins - PER (t + 1), bins - PER t), from the top
        static_assert(PER == 4, "a vector of bins a thread");
        const int bin0 = bins - (int)((tid + 1) * PER);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (bin0 >= 0) {
            v = *reinterpret_cast<const uint4 *>(c + bin0);
            *reinterpret_cast<uint4 *>(c + bin0) = make_uint4(0, 0, 0, 0);
        }
        const uint32_t own = v.x + v.y + v.z + v.w;
        uint32_t incl = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t up = __shfl_up_sync(~0u, incl, d);
            if (lane >= (uint32_t)d) incl += up;
        }
        if (lane == 31) warp_a[warp] = incl;
        __syncthreads();
        const uint32_t wv = lane < SEL_THREADS / 32 ? warp_a[lane] : 0;
        uint32_t above = incl - own + __reduce_add_sync(~0u, lane < warp ? wv : 0u);
        const uint32_t down[4] = {v.w, v.z, v.y, v.x};
#pragma unroll
        for (int e = 0; e < PER; e++) {
            if (above < need && above + down[e] >= need) {  // one thread only (need > 0)
                s_digit = (uint32_t)(bin0 + PER - 1 - e);
                s_need = need - above;
                s_whole = above + down[e] == need;
            }
            above += down[e];
        }
        __syncthreads();
        edge = prefix = (prefix << bits) | s_digit;
        need = s_need;
        if (s_whole) {  // the bin is kept to its last key; it is not the lowest, since some slot goes
            edge = (prefix << shift) - 1;
            need = 0;
            break;
        }
    }
    // kept: keys above `edge`, and the first `need` equal to it
    // a tile's slots that are kept for sure and those equal to the edge, a bit a slot
    // (this thread's), and the counts of them before each 32 slots of the tile (s_run)
    auto kinds = [&](uint32_t t0, uint32_t &above, uint32_t &equal, uint32_t &na, uint32_t &ne) {
        above = equal = 0;
        __syncthreads();  // s_run may still be read
#pragma unroll
        for (int e = 0; e < SEL_PER; e++) {
            const uint32_t i = t0 + e * SEL_THREADS + tid;
            const bool in = i < i1, forced = i < lo || i >= hi;
            const bool u = in && (forced || key[e] > edge), v = in && !forced && key[e] == edge;
            above |= (uint32_t)u << e;
            equal |= (uint32_t)v << e;
            const uint32_t bu = __ballot_sync(~0u, u), bv = __ballot_sync(~0u, v);
            if (lane == 0) s_run[e * (SEL_THREADS / 32) + warp] = make_uint2(__popc(bu), __popc(bv));
        }
        __syncthreads();
        constexpr int RUNS = SEL_PER * SEL_THREADS / 32, EACH = RUNS / 32;  // a warp scans them, each in turn
        uint2 r[EACH];
        uint32_t su = 0, sv = 0;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            r[e] = s_run[lane * EACH + e];
            su += r[e].x;
            sv += r[e].y;
        }
        uint32_t iu = su, iv = sv;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t uu = __shfl_up_sync(~0u, iu, d), uv = __shfl_up_sync(~0u, iv, d);
            if (lane >= (uint32_t)d) iu += uu, iv += uv;
        }
        na = __shfl_sync(~0u, iu, 31);
        ne = __shfl_sync(~0u, iv, 31);
        __syncthreads();
        if (warp == 0) {
            iu -= su;
            iv -= sv;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                s_run[lane * EACH + e] = make_uint2(iu, iv);
                iu += r[e].x;
                iv += r[e].y;
            }
        }
        __syncthreads();
    };
    uint32_t ca = 0, ce = 0, above = 0, equal = 0;
    for (uint32_t t0 = i0; t0 < i1; t0 += SEL_TILE) {
        uint32_t na, ne;
        if (!resident) load(t0);
        kinds(t0, above, equal, na, ne);
        ca += na;
        ce += ne;
    }
    if (tid < ranks) {  // to rank tid
        peer_store(peer_smem(&s_above[rank], tid), ca);
        peer_store(peer_smem(&s_equal[rank], tid), ce);
    }
    sync();
    uint32_t base_a = 0, base_e = 0;
    for (uint32_t r = 0; r < rank; r++) base_a += s_above[r], base_e += s_equal[r];
    for (uint32_t t0 = i0; t0 < i1; t0 += SEL_TILE) {
        uint32_t na = 0, ne = 0;
        if (!resident) {
            load(t0);
            kinds(t0, above, equal, na, ne);
        }
#pragma unroll
        for (int e = 0; e < SEL_PER; e++) {
            const uint32_t u = (above >> e) & 1u, v = (equal >> e) & 1u, low = (1u << lane) - 1u;
            const uint32_t bu = __ballot_sync(~0u, u), bv = __ballot_sync(~0u, v);
            const uint2 run = s_run[e * (SEL_THREADS / 32) + warp];
            const uint32_t at_e = base_e + run.y + __popc(bv & low);
            if (u || (v && at_e < need)) {
                const uint32_t at = base_a + run.x + __popc(bu & low) + min(at_e, need);
                if (at < p.keep) kept[at] = (int32_t)(t0 + e * SEL_THREADS + tid);
            }
        }
        base_a += na;
        base_e += ne;
    }
}

// Compaction, in place: a cluster of CTAs takes one (sequence, KV head, pool), and one
// CTA more per (sequence, KV head) moves the mass.  New slot j takes old slot
// kept[j] >= j, in order: a chunk of MOVE_ROWS rows a CTA is read whole, by cp.async
// into shared memory, before any CTA of the cluster writes it, and no later chunk reads
// what an earlier one wrote.  Whole rows, because each instruction costs a cycle for
// every line that it touches: with 32-byte slices of all rows a CTA, which needs no
// cluster, the move of 16 sequences (4001 of up to 32768 slots) took 24.3 us instead of 19.8.
constexpr int MOVE_THREADS = 256, MOVE_ROWS = 192;

template <int HD>
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(EvictArgs p) {
    constexpr uint32_t LANES = HD * 2 / 16, STEP = MOVE_THREADS / LANES, PER = MOVE_ROWS / STEP;  // lanes a row
    extern __shared__ __align__(16) uint8_t stage[];
    __shared__ int64_t s_from[MOVE_ROWS], s_to[MOVE_ROWS];  // offsets of a chunk's rows; -1: does not move
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    uint32_t x = blockIdx.x / ranks;
    const uint32_t part = x % 3;  // K, V, mass
    x /= 3;
    const uint32_t h = x % p.a.kv_heads, b = x / p.a.kv_heads;
    griddep_wait();
    const uint32_t n = p.a.len(b);
    const int32_t *kept = p.kept + ((size_t)b * p.a.kv_heads + h) * p.keep;
    if (part == 2) {
        if (!p.mass_out) return;
        const float *src = p.mass + ((size_t)b * p.a.kv_heads + h) * p.mass_stride;
        float *dst = p.mass_out + ((size_t)b * p.a.kv_heads + h) * p.mass_out_stride;
        const uint32_t live = min(n, p.keep);
        constexpr uint32_t V = 16;
        for (uint32_t c = 0; c < live && rank == 0; c += MOVE_THREADS * V) {
            float v[V];
#pragma unroll
            for (uint32_t i = 0; i < V; i++) {
                const uint32_t j = c + i * MOVE_THREADS + threadIdx.x;
                v[i] = j < live ? src[kept[j]] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < V; i++) {
                const uint32_t j = c + i * MOVE_THREADS + threadIdx.x;
                if (j < live) dst[j] = v[i];
            }
            __syncthreads();
        }
        // (in place, slots past `live` may still have to be read)
        if (ranks > 1) cluster_sync();
        for (uint32_t i = live + rank * MOVE_THREADS + threadIdx.x; i < n; i += ranks * MOVE_THREADS) dst[i] = 0.f;
        return;
    }
    if (n <= p.keep) return;  // every slot stays where it is: the same for the whole cluster
    uint8_t *pool = reinterpret_cast<uint8_t *>(part ? p.a.v : p.a.k);
    auto place = [&](uint32_t slot) -> int64_t {  // offset of its row, below 0 on a hole
        const int pg = p.a.page(b, slot >> p.a.page_shift);
        return pg < 0 ? -1 : (int64_t)(p.a.row<HD>(pg, h, slot) * 2);
    };
    const uint32_t r0 = threadIdx.x / LANES, off = (threadIdx.x % LANES) * 16;
    int64_t from_next, to_next;  // this thread's row of the next chunk, looked up while a chunk is read
    auto look = [&](uint32_t c) {
        const uint32_t j = c + rank * MOVE_ROWS + threadIdx.x;
        from_next = to_next = -1;
        if (threadIdx.x >= MOVE_ROWS || j >= p.keep) return;
        const uint32_t src = (uint32_t)kept[j];
        if (src == j || src >= n) return;
        to_next = place(j);
        from_next = to_next < 0 ? -1 : place(src);
    };
    look(0);
    for (uint32_t c = 0; c < p.keep; c += ranks * MOVE_ROWS) {
        if (threadIdx.x < MOVE_ROWS) {
            s_from[threadIdx.x] = from_next;
            s_to[threadIdx.x] = to_next;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t r = i * STEP + r0;
            const int64_t from = s_from[r];
            if (from >= 0)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(stage + r * (HD * 2) + off)),
                             "l"(pool + from + off)
                             : "memory");
        }
        look(c + ranks * MOVE_ROWS);
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (ranks > 1)  // the chunk is read by every thread of the cluster
            cluster_sync();
        else
            __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t r = i * STEP + r0;
            if (s_from[r] >= 0)
                *reinterpret_cast<uint4 *>(pool + s_to[r] + off) =
                    *reinterpret_cast<const uint4 *>(stage + r * (HD * 2) + off);
        }
        __syncthreads();  // the offsets and the stage may be written again
    }
}

// slots of one CTA's slice, beyond which another joins its cluster: 32768 slots of 32
// (sequence, KV head)s took 131, 95, 65 and 43 us with 1, 2, 4 and 8 CTAs each, 4096
// slots of 8 of them 14.4 us with one and 16.4 with two or more
constexpr uint32_t SEL_SLICE = 4096;

int launch_evict(const EvictArgs &p, uint32_t hd, int sm_count, cudaStream_t s) {
    const uint32_t rows = p.a.n_seqs * p.a.kv_heads;
    uint32_t ranks = 1;
    while (ranks < 8 && (uint64_t)ranks * SEL_SLICE < p.a.max_kv && (uint64_t)rows * ranks * 2 <= 4u * sm_count) ranks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * ranks);
    cfg.blockDim = dim3(SEL_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = ranks;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    CUQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_select_kernel, p));
    if (p.a.max_kv <= p.keep && !p.mass_out) return CUQ_OK;  // nothing can move
    // as many CTAs a cluster as have rows to move, so that most calls take one or two rounds
    uint32_t movers = 1;
    while (movers < 8 && movers * MOVE_ROWS < p.keep) movers *= 2;
    const int bytes = MOVE_ROWS * (int)hd * 2;
    static std::atomic<uint64_t> allowed64, allowed128;
    CUQ_CUDA_TRY(hd == 64 ? allow_smem(evict_move_kernel<64>, bytes, allowed64)
                          : allow_smem(evict_move_kernel<128>, bytes, allowed128));
    attrs[0].val.clusterDim.x = movers;
    cfg.gridDim = dim3(rows * 3 * movers);
    cfg.blockDim = dim3(MOVE_THREADS);
    cfg.dynamicSmemBytes = (size_t)bytes;
    CUQ_CUDA_TRY(hd == 64 ? cudaLaunchKernelEx(&cfg, evict_move_kernel<64>, p)
                          : cudaLaunchKernelEx(&cfg, evict_move_kernel<128>, p));
    return CUQ_OK;
}

// ----------------------------------------------------- argument checks ----

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

int check_paged(const char *who, const cuq_paged_kv *kv, const cuq_batch *b, bool queries, PagedArgs &a) {
    CUQ_CHECK_ARG(kv && b, "%s: null descriptor", who);
    if (kv->type != CUQ_F16 && kv->type != CUQ_BF16) {
        set_error("%s: unsupported cache type %d (F16 or BF16)", who, kv->type);
        return CUQ_EUNSUPPORTED;
    }
    if (kv->head_dim != 64 && kv->head_dim != 128) {
        set_error("%s: unsupported head_dim %u (64 or 128)", who, kv->head_dim);
        return CUQ_EUNSUPPORTED;
    }
    const uint32_t ps = kv->page_size;
    if (ps < 16 || ps > 256 || (ps & (ps - 1))) {
        set_error("%s: unsupported page_size %u (a power of two, 16 to 256)", who, ps);
        return CUQ_EUNSUPPORTED;
    }
    CUQ_CHECK_ARG(kv->k && kv->v && aligned16(kv->k) && aligned16(kv->v), "%s: pools must be 16-byte aligned", who);
    CUQ_CHECK_ARG(kv->kv_heads > 0 && kv->kv_heads <= 65535 && kv->n_pages > 0 && kv->n_pages <= 0x7FFFFFFFu,
                  "%s: bad pool (%u pages, %u KV heads)", who, kv->n_pages, kv->kv_heads);
    const uint64_t dense = (uint64_t)kv->kv_heads * ps * kv->head_dim;
    const uint64_t stride = kv->page_stride ? kv->page_stride : dense;
    CUQ_CHECK_ARG(stride >= dense && stride % 8 == 0 && stride < (1ull << 38),
                  "%s: page_stride %llu (at least %llu, a multiple of 8)", who, (unsigned long long)stride,
                  (unsigned long long)dense);
    CUQ_CHECK_ARG(b->n_seqs <= 65535, "%s: %u sequences (at most 65535)", who, b->n_seqs);
    CUQ_CHECK_ARG(b->n_tok <= 0x3FFFFFFFu && b->max_kv <= 0x3FFFFFFFu && b->max_q <= 0x3FFFFFFFu &&
                      b->pages_stride <= 0x3FFFFFFFu,
                  "%s: batch sizes past 2^30", who);
    CUQ_CHECK_ARG((uint64_t)b->n_seqs * kv->kv_heads <= (1u << 24), "%s: %u sequences of %u KV heads pass 2^24", who,
                  b->n_seqs, kv->kv_heads);
    if (b->n_seqs) {
        CUQ_CHECK_ARG(b->kv_len && b->pages && aligned4(b->kv_len) && aligned4(b->pages),
                      "%s: kv_len and pages must be given", who);
        CUQ_CHECK_ARG(!queries || (b->q_start && aligned4(b->q_start)), "%s: q_start must be given", who);
    }
    a.k = kv->k;
    a.v = kv->v;
    a.page_stride = stride;
    a.n_pages = kv->n_pages;
    a.page_size = ps;
    a.page_shift = (uint32_t)__builtin_ctz(ps);
    a.kv_heads = kv->kv_heads;
    a.q_start = b->q_start;
    a.kv_len = b->kv_len;
    a.pages = b->pages;
    a.n_seqs = b->n_seqs;
    a.n_tok = b->n_tok;
    a.pages_stride = b->pages_stride;
    a.max_q = b->max_q < b->n_tok ? b->max_q : b->n_tok;
    const uint64_t slots = (uint64_t)b->pages_stride * ps;
    a.max_kv = slots < b->max_kv ? (uint32_t)slots : b->max_kv;
    CUQ_CHECK_ARG((uint64_t)b->n_seqs * kv->kv_heads * ((a.max_kv + 15) / 16) <= 0x7FFFFFFFu,
                  "%s: %u sequences of %u KV heads and %u slots pass 2^31 blocks of 16", who, b->n_seqs, kv->kv_heads,
                  a.max_kv);
    return CUQ_OK;
}

int check_heads(const char *who, const cuq_paged_kv *kv, uint32_t heads) {
    CUQ_CHECK_ARG(heads > 0 && heads <= 32768 && heads % kv->kv_heads == 0,
                  "%s: heads (%u) must be a positive multiple of kv_heads (%u)", who, heads, kv->kv_heads);
    return CUQ_OK;
}

int check_query(const char *who, const cuq_paged_kv *kv, uint32_t n_tok, const void *q, size_t q_stride, int type,
                uint32_t heads, float scale, int causal, uint32_t window, PagedQuery &out) {
    int rc = check_heads(who, kv, heads);
    if (rc) return rc;
    if (!(type == kv->type || (type == CUQ_F32 && kv->type == CUQ_F16))) {
        set_error("%s: unsupported type %d over a cache of type %d (the cache's own, or F32 over F16)", who, type,
                  kv->type);
        return CUQ_EUNSUPPORTED;
    }
    CUQ_CHECK_ARG(q && aligned16(q), "%s: q must be 16-byte aligned", who);
    CUQ_CHECK_ARG(q_stride % 8 == 0 && q_stride >= (size_t)heads * kv->head_dim,
                  "%s: q_stride %zu (a multiple of 8, at least %zu)", who, q_stride, (size_t)heads * kv->head_dim);
    CUQ_CHECK_ARG(std::isfinite(scale), "%s: scale must be finite", who);
    CUQ_CHECK_ARG((uint64_t)n_tok * heads <= 0x7FFFFFFFu, "%s: %u tokens of %u heads pass 2^31 rows", who, n_tok, heads);
    CUQ_CHECK_ARG(causal || window == 0, "%s: a window needs a causal mask", who);
    out.q = q;
    out.q_stride = q_stride;
    out.heads = heads;
    out.group = heads / kv->kv_heads;
    out.group_inv = (uint32_t)((0x100000000ull + out.group - 1) / out.group);
    out.scale = scale;
    out.causal = causal ? 1 : 0;
    out.window = window < (1u << 30) ? window : (1u << 30) - 1;  // slots are below 2^30
    return CUQ_OK;
}

// Whether a caller that polls this stream has not been told of all `count` give-ups of
// the device; it has been then.  False when out of memory.
bool told_of_give_ups(int dev, cudaStream_t s, unsigned int count, bool &news) {
    static std::mutex mu;
    static std::map<std::pair<int, cudaStream_t>, unsigned int> told;  // none: 0
    std::lock_guard<std::mutex> lock(mu);
    try {
        unsigned int &last = told[{dev, s}];
        if (count < last) last = 0;  // the device was reset
        news = count != last;
        last = count;
    } catch (const std::bad_alloc &) {
        return false;
    }
    return true;
}

}  // namespace
}  // namespace cuq

using namespace cuq;

extern "C" {

cuq_rope_plan *cuq_rope_plan_create(const cuq_rope_params *p) {
    auto bad = [](const char *what) -> cuq_rope_plan * {
        set_error("cuq_rope_plan_create: %s", what);
        return nullptr;
    };
    if (!p) return bad("null argument");
    if (p->rot_dim == 0 || p->rot_dim % 16 || p->rot_dim > 2 * ROPE_MAX_PAIRS)
        return bad("rot_dim must be a multiple of 16, 16 to 128");
    if (!(p->theta > 1.0f) || !std::isfinite(p->theta)) return bad("theta must be above 1");
    if (p->scaling < CUQ_ROPE_NONE || p->scaling > CUQ_ROPE_YARN) return bad("unknown scaling");
    if (p->scaling != CUQ_ROPE_NONE && !(p->factor >= 1.0f && std::isfinite(p->factor)))
        return bad("factor must be at least 1");
    if (p->scaling == CUQ_ROPE_LLAMA3 &&
        !(p->orig_ctx > 0 && p->low_freq > 0 && p->high_freq > p->low_freq && std::isfinite(p->high_freq)))
        return bad("LLAMA3 needs orig_ctx and 0 < low_freq < high_freq");
    if (p->scaling == CUQ_ROPE_YARN &&
        !(p->orig_ctx > 0 && p->beta_slow > 0 && p->beta_fast >= p->beta_slow && std::isfinite(p->beta_fast) &&
          p->attn_factor >= 0 && std::isfinite(p->attn_factor)))
        return bad("YARN needs orig_ctx, 0 < beta_slow <= beta_fast and attn_factor >= 0");
    cuq_rope_plan *plan = new (std::nothrow) cuq_rope_plan();
    if (!plan) return bad("out of memory");
    static_assert(std::numeric_limits<long double>::digits >= 64, "the table's error counts on 64-bit significands");
    const long double two_pi = 6.283185307179586476925286766559005768L;
    const uint32_t half = p->rot_dim / 2;
    double low = 0, high = 1;
    if (p->scaling == CUQ_ROPE_YARN) {
        auto at = [&](double turns) {  // the pair index at which orig_ctx holds that many turns
            return p->rot_dim * std::log((double)p->orig_ctx / (turns * (double)two_pi)) / (2 * std::log((double)p->theta));
        };
        low = std::fmax(0.0, std::floor(at(p->beta_fast)));
        high = std::fmin((double)p->rot_dim - 1, std::ceil(at(p->beta_slow)));
    }
    plan->t.mul = 1.f;
    for (uint32_t j = 0; j < half; j++) {
        long double f = std::pow((long double)p->theta, -2.0L * j / p->rot_dim);
        if (p->scaling == CUQ_ROPE_LINEAR) {
            f /= p->factor;
        } else if (p->scaling == CUQ_ROPE_LLAMA3) {
            long double s = (p->orig_ctx * f / two_pi - p->low_freq) / ((long double)p->high_freq - p->low_freq);
            s = std::fmin(1.0L, std::fmax(0.0L, s));
            f = (1 - s) * f / p->factor + s * f;
        } else if (p->scaling == CUQ_ROPE_YARN) {
            const long double r = std::fmin(1.0L, std::fmax(0.0L, (j - low) / std::fmax(high - low, 0.001L)));
            f = f / p->factor * r + f * (1 - r);
        }
        plan->t.turns[j] = (uint64_t)std::llrint(std::ldexp(f / two_pi, 64));  // f <= 1: below 2^62
    }
    for (uint32_t j = half; j < (uint32_t)ROPE_MAX_PAIRS; j++) plan->t.turns[j] = 0;
    if (p->scaling == CUQ_ROPE_YARN)
        plan->t.mul = p->attn_factor > 0 ? p->attn_factor : (float)(0.1 * std::log((double)p->factor) + 1.0);
    plan->t.rot = p->rot_dim;
    plan->t.adjacent = p->adjacent ? 1 : 0;
    return plan;
}

void cuq_rope_plan_free(cuq_rope_plan *p) { delete p; }

int cuq_rope_append(const cuq_rope_plan *rope, const cuq_paged_kv *kv, const cuq_batch *batch,
                    const int32_t *positions, void *q_out, size_t q_out_stride, int out_type, const void *q,
                    size_t q_stride, const void *k, const void *v, size_t kv_stride, int in_type, uint32_t heads,
                    void *stream) {
    const char *who = "cuq_rope_append";
    RopeArgs p;
    CUQ_CHECK_ARG(rope, "%s: null plan", who);
    int rc = check_paged(who, kv, batch, true, p.a);
    if (rc == CUQ_OK) rc = check_heads(who, kv, heads);
    if (rc) return rc;
    CUQ_CHECK_ARG(rope->t.rot <= kv->head_dim, "%s: rot_dim %u exceeds head_dim %u", who, rope->t.rot, kv->head_dim);
    if (in_type != CUQ_F32 && in_type != CUQ_F16 && in_type != CUQ_BF16) {
        set_error("%s: unsupported type %d (F32, F16 or BF16)", who, in_type);
        return CUQ_EUNSUPPORTED;
    }
    if (out_type != in_type && out_type != kv->type) {
        set_error("%s: unsupported output type %d (the input's or the cache's)", who, out_type);
        return CUQ_EUNSUPPORTED;
    }
    CUQ_CHECK_ARG(q && k && v && q_out && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out),
                  "%s: q, k, v and q_out must be 16-byte aligned", who);
    CUQ_CHECK_ARG(positions == nullptr || aligned4(positions), "%s: positions must be 4-byte aligned", who);
    const size_t qd = (size_t)heads * kv->head_dim, kd = (size_t)kv->kv_heads * kv->head_dim;
    CUQ_CHECK_ARG(q_stride % 8 == 0 && q_stride >= qd && q_out_stride % 8 == 0 && q_out_stride >= qd &&
                      kv_stride % 8 == 0 && kv_stride >= kd,
                  "%s: strides must be multiples of 8, at least %zu (q) and %zu (k, v)", who, qd, kd);
    CUQ_CHECK_ARG(q_out != q || (out_type == in_type && q_out_stride == q_stride),
                  "%s: q_out may be q only with its type and stride", who);
    if (batch->n_tok == 0 || batch->n_seqs == 0) return CUQ_OK;
    p.positions = positions;
    p.q_out = q_out;
    p.q_out_stride = q_out_stride;
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.kv_stride = kv_stride;
    p.heads = heads;
    cudaStream_t s = (cudaStream_t)stream;
    if (in_type == CUQ_F32)
        return launch_rope_append<float>(p, rope->t, out_type, kv->type, kv->head_dim, s);
    if (in_type == CUQ_F16)
        return launch_rope_append<__half>(p, rope->t, out_type, kv->type, kv->head_dim, s);
    return launch_rope_append<__nv_bfloat16>(p, rope->t, out_type, kv->type, kv->head_dim, s);
}

size_t cuq_attention_paged_workspace(const cuq_paged_kv *kv, const cuq_batch *batch, uint32_t heads, int type) {
    AttnPagedCall c{};
    if (check_paged("cuq_attention_paged_workspace", kv, batch, false, c.a) != CUQ_OK) return 0;
    if (check_heads("cuq_attention_paged_workspace", kv, heads) != CUQ_OK) return 0;
    c.q.heads = heads;
    c.q.group = heads / kv->kv_heads;
    c.type = type;
    c.cache_type = kv->type;
    c.hd = kv->head_dim;
    return attention_paged_workspace(c, paged_sm_count());
}

int cuq_attention_paged(const cuq_paged_kv *kv, const cuq_batch *batch, void *out, size_t out_stride, const void *q,
                        size_t q_stride, int type, float *lse, uint32_t heads, float scale, int causal,
                        uint32_t window, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "cuq_attention_paged";
    AttnPagedCall c{};
    int rc = check_paged(who, kv, batch, true, c.a);
    if (rc == CUQ_OK) rc = check_query(who, kv, batch->n_tok, q, q_stride, type, heads, scale, causal, window, c.q);
    if (rc) return rc;
    CUQ_CHECK_ARG(out && aligned16(out) && out != q, "%s: out must be 16-byte aligned and not q", who);
    CUQ_CHECK_ARG(out_stride % 8 == 0 && out_stride >= (size_t)heads * kv->head_dim,
                  "%s: out_stride %zu (a multiple of 8, at least %zu)", who, out_stride,
                  (size_t)heads * kv->head_dim);
    CUQ_CHECK_ARG(lse == nullptr || aligned4(lse), "%s: lse must be 4-byte aligned", who);
    c.out = out;
    c.out_stride = out_stride;
    c.lse = lse;
    c.type = type;
    c.cache_type = kv->type;
    c.hd = kv->head_dim;
    c.workspace = workspace;
    const int sms = paged_sm_count();
    const size_t need = attention_paged_workspace(c, sms);
    CUQ_CHECK_ARG(workspace_bytes >= need && (need == 0 || workspace),
                  "%s: workspace of %zu bytes, %zu needed (cuq_attention_paged_workspace)", who, workspace_bytes, need);
    CUQ_CHECK_ARG(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
                  "%s: workspace must be 256-byte aligned", who);
    if (batch->n_tok == 0 || batch->n_seqs == 0 || c.a.max_q == 0) return CUQ_OK;
    return launch_attention_paged(c, sms, (cudaStream_t)stream);
}

int cuq_attention_mass(const cuq_paged_kv *kv, const cuq_batch *batch, float *mass, size_t mass_stride,
                       const void *q, size_t q_stride, int type, const float *lse, uint32_t heads, float scale,
                       int causal, uint32_t window, uint32_t last_q, float decay, void *stream) {
    const char *who = "cuq_attention_mass";
    MassPagedCall c{};
    int rc = check_paged(who, kv, batch, true, c.a);
    if (rc == CUQ_OK) rc = check_query(who, kv, batch->n_tok, q, q_stride, type, heads, scale, causal, window, c.q);
    if (rc) return rc;
    CUQ_CHECK_ARG(mass && lse && aligned4(mass) && aligned4(lse), "%s: mass and lse must be given", who);
    CUQ_CHECK_ARG(mass_stride >= c.a.max_kv, "%s: mass_stride %zu is below max_kv %u", who, mass_stride, c.a.max_kv);
    CUQ_CHECK_ARG(std::isfinite(decay), "%s: decay must be finite", who);
    if (batch->n_seqs == 0 || c.a.max_kv == 0) return CUQ_OK;
    c.mass = mass;
    c.mass_stride = mass_stride;
    c.lse = lse;
    c.type = type;
    c.cache_type = kv->type;
    c.hd = kv->head_dim;
    c.last_q = last_q;
    c.decay = decay;
    return launch_attention_mass(c, paged_sm_count(), (cudaStream_t)stream);
}

int cuq_kv_evict(const cuq_paged_kv *kv, const cuq_batch *batch, const float *mass, size_t mass_stride,
                 uint32_t keep, uint32_t sink, uint32_t recent, int32_t *kept, int32_t *new_len, float *mass_out,
                 size_t mass_out_stride, void *stream) {
    const char *who = "cuq_kv_evict";
    EvictArgs p;
    int rc = check_paged(who, kv, batch, false, p.a);
    if (rc) return rc;
    CUQ_CHECK_ARG(keep > 0 && keep <= 0x3FFFFFFFu && (uint64_t)sink + recent <= keep,
                  "%s: keep %u with sink %u and recent %u (sink + recent <= keep)", who, keep, sink, recent);
    CUQ_CHECK_ARG(mass && kept && new_len && aligned4(mass) && aligned4(kept) && aligned4(new_len),
                  "%s: mass, kept and new_len must be given", who);
    CUQ_CHECK_ARG(new_len != batch->kv_len, "%s: new_len must not be the batch's kv_len", who);
    CUQ_CHECK_ARG(mass_stride >= p.a.max_kv, "%s: mass_stride %zu is below max_kv %u", who, mass_stride, p.a.max_kv);
    CUQ_CHECK_ARG(mass_out == nullptr || (aligned4(mass_out) && mass_out_stride >= p.a.max_kv),
                  "%s: mass_out_stride %zu is below max_kv %u", who, mass_out_stride, p.a.max_kv);
    CUQ_CHECK_ARG(mass_out != mass || mass_out_stride == mass_stride, "%s: mass in place needs its own stride", who);
    if (batch->n_seqs == 0) return CUQ_OK;
    p.mass = mass;
    p.mass_stride = mass_stride;
    p.keep = keep;
    p.sink = sink;
    p.recent = recent;
    p.kept = kept;
    p.new_len = new_len;
    p.mass_out = mass_out;
    p.mass_out_stride = mass_out_stride;
    return launch_evict(p, kv->head_dim, paged_sm_count(), (cudaStream_t)stream);
}

int cuq_paged_status(void *stream) {
    const cudaStream_t s = (cudaStream_t)stream;
    int dev = 0;
    CUQ_CUDA_TRY(cudaGetDevice(&dev));
    CUQ_CUDA_TRY(cudaStreamSynchronize(s));
    unsigned int few = 0, many = 0, mass = 0;
    int rc = attention_few_gave_up(s, &few);
    if (rc == CUQ_OK) rc = attention_many_gave_up(s, &many);
    if (rc == CUQ_OK) rc = attention_mass_gave_up(s, &mass);
    if (rc) return rc;
    bool news = false;
    if (!told_of_give_ups(dev, s, few + many + mass, news)) {
        set_error("cuq_paged_status: out of memory");
        return CUQ_ENOMEM;
    }
    if (!news) return CUQ_OK;
    set_error("a wait inside a paged-cache kernel gave up");
    return CUQ_ETIMEOUT;
}

int cuq_paged_wait_probe(uint32_t limit_us, void *stream) {
    CUQ_CHECK_ARG(limit_us > 0 && limit_us <= 1000000u, "cuq_paged_wait_probe: limit of %u us (1 to 1000000)", limit_us);
    return launch_wait_probe(limit_us, (cudaStream_t)stream);
}

}  // extern "C"
