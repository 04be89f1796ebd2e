// paged_attn.cu -- attention of a batch's new tokens over a paged KV cache:
//   o = sum_s p_s v_s / sum_s p_s,  p_s = exp(scale q k_s - max),  s over the visible slots.
// This file: how a call is split, the kernel for sequences of few rows (decode
// steps, short drafts) and the merge of split results.  paged_attn_tc.cu has the
// kernel for many rows.
#include "paged_tc.cuh"

namespace cuq {

using namespace ptc;

namespace {

__device__ int g_timeout;  // a bounded wait of this file's kernels gave up

// ------------------------------------------------------------ few rows ----
//
// Bound by HBM: each K and V row is read once for all the rows of its group.  A
// CTA of 4 warps takes one KV head of one sequence and `few_chunk` slots; every
// warp walks its own 16-slot blocks (w, w + 4, ...) with its own ring of FEW_ST
// stages, so nothing but the final join synchronises the warps.  A stage is the
// block's K and V rows as TMA boxes of 64 dims in the 128-byte swizzle, which
// ldmatrix then reads without bank conflicts.  Two CTAs fit an SM: 8 warps x up to
// FEW_ST blocks of 4 KB or 8 KB in flight.  Scores and outputs run on
// mma.sync.m16n8k16 (16 rows x 16 slots, fp32 accumulate); fp32 queries are two
// fp16 operands, hi and lo, and so are their probabilities.
constexpr int FEW_WARPS = 4, FEW_ST = 3, FEW_KEYS = 16;

template <int HD>
struct FewGeo {
    static constexpr int ROWS = FEW_KEYS * HD * 2;                       // K (or V) bytes of a stage
    static constexpr int RING = FEW_WARPS * FEW_ST * 2 * ROWS;
    static constexpr int Q = 16 * HD * 2;                                // one 16-row query operand
    static constexpr int SMEM = 1024 + RING + 2 * Q;
};

template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(FEW_WARPS * 32) attn_few_kernel(PagedArgs a, PagedQuery q, AttnOut o,
                                                                   const __grid_constant__ CUtensorMap mk,
                                                                   const __grid_constant__ CUtensorMap mv) {
    using G = FewGeo<HD>;
    constexpr bool SPLIT = std::is_same<TQ, float>::value;
    constexpr int CB = HD / 64;  // 64-dim column blocks
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[FEW_WARPS][FEW_ST];
    __shared__ int abort_flag;
    __shared__ float s_m[FEW_WARPS][16], s_l[FEW_WARPS][16];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t kvh = blockIdx.x, split = blockIdx.y, b = blockIdx.z;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t first;
    const uint32_t nq = a.tokens(b, first), n = a.len(b);
    const uint32_t tq = min(nq, a.max_q);  // tokens attended
    const uint32_t rows = tq * q.group;
    if (tq == 0 || !o.plan.is_few(tq, q.group)) return;
    const int pos0 = (int)n - (int)nq;
    // the slots any row sees, and this CTA's part of them
    uint32_t lo0, hi0, lo1, hi1;
    q.range(max(pos0, 0), n, lo0, hi0);
    q.range(pos0 + (int)tq - 1, n, lo1, hi1);
    const uint32_t chunk = o.plan.few_chunk, c0 = lo0 / chunk;  // chunks are counted from slot 0
    const uint32_t begin = max(lo0, (c0 + split) * chunk), end = min(hi1, (c0 + split + 1) * chunk);
    const bool direct = o.plan.few_splits == 1;
    if (begin >= end && !direct) return;  // the merge counts the live parts the same way
    const uint32_t blk0 = begin / FEW_KEYS, nblk = begin < end ? (end + FEW_KEYS - 1) / FEW_KEYS - blk0 : 0;

    if (tid == 0) {
        abort_flag = 0;
        for (int w = 0; w < FEW_WARPS; w++)
            for (int s = 0; s < FEW_ST; s++) mbar_init(&full[w][s], 1);
        mbar_init_fence();
    }
    __syncthreads();

    uint8_t *ring = smem + warp * (FEW_ST * 2 * G::ROWS);
    // page ids of this warp's blocks, one per lane, 32 blocks at a time
    auto page_of = [&](uint32_t i) -> int {
        const uint32_t blk = warp + FEW_WARPS * i;
        return blk < nblk ? a.page(b, ((blk0 + blk) * FEW_KEYS) >> a.page_shift) : -1;
    };
    const uint32_t mine = nblk > warp ? (nblk - warp + FEW_WARPS - 1) / FEW_WARPS : 0;
    int ids = page_of(lane);        // of block i: lane i & 31
    int ids_next = page_of(lane + 32);
    auto issue = [&](uint32_t i) {  // lane 0: block i into its stage
        const int pg = __shfl_sync(~0u, (i & 32) ? ids_next : ids, i & 31);
        if (lane == 0) {
            const uint32_t s = i % FEW_ST, blk = blk0 + warp + FEW_WARPS * i;
            const uint32_t dst = smem_u32(ring + s * 2 * G::ROWS);
            const int slot = (int)((blk * FEW_KEYS) & (a.page_size - 1)), p = pg < 0 ? (int)a.n_pages : pg;
            mbar_expect_tx(&full[warp][s], 2 * G::ROWS);
#pragma unroll
            for (int cb = 0; cb < CB; cb++) {
                tma_load_page(dst + cb * FEW_KEYS * 128, &mk, cb * 64, slot, (int)kvh, p, &full[warp][s]);
                tma_load_page(dst + G::ROWS + cb * FEW_KEYS * 128, &mv, cb * 64, slot, (int)kvh, p, &full[warp][s]);
            }
        }
        return pg;
    };
    // `ids` holds blocks [64 h, 64 h + 32) and ids_next the 32 behind them; both
    // move on when the walk has passed them (see the loop)
    int pgs[FEW_ST];
#pragma unroll
    for (int i = 0; i < FEW_ST; i++) pgs[i] = (uint32_t)i < mine ? issue(i) : -1;

    // the queries: 16 rows of [HD] as 64-dim blocks in the swizzle, hi then lo
    uint8_t *sq = smem + G::RING;
    for (uint32_t i = tid; i < 16 * HD / 8; i += FEW_WARPS * 32) {
        const uint32_t r = i / (HD / 8), c = i % (HD / 8);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.f;
        if (r < rows) {
            const uint32_t tok = first + r / q.group, head = kvh * q.group + r % q.group;
            load8(reinterpret_cast<const TQ *>(q.q) + (size_t)tok * q.q_stride + (size_t)head * HD + c * 8, v);
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) split_pack<TC>(v[2 * e], v[2 * e + 1], hi[e], lo[e]);
        const uint32_t at = (c / 8) * 2048 + sw128(r, c & 7);
        *reinterpret_cast<uint4 *>(sq + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (SPLIT) *reinterpret_cast<uint4 *>(sq + G::Q + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    __syncthreads();
    uint32_t qf[HD / 16][4];
    const uint32_t qaddr = smem_u32(sq);
    auto load_q = [&](uint32_t base, int ks, uint32_t(&f)[4]) {
        const uint32_t r = lane & 15, c = ks * 2 + (lane >> 4);
        ldsm4(f, base + (c / 8) * 2048 + sw128(r, c & 7));
    };
#pragma unroll
    for (int ks = 0; ks < HD / 16; ks++) load_q(qaddr, ks, qf[ks]);

    // rows g and g + 8 of the tile are this thread's
    const uint32_t g = lane >> 2, t4 = lane & 3;
    uint32_t rlo[2], rhi[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t r = g + 8 * h;
        rlo[h] = rhi[h] = 0;
        if (r < rows) q.range(pos0 + (int)(r / q.group), n, rlo[h], rhi[h]);
    }
    const float c2 = q.scale * 1.4426950408889634f;  // scores in units of log 2
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float acc[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[i][e] = 0.f;

    bool ok = true;
    uint32_t st = 0, ph = 0;
    for (uint32_t i = 0; i < mine; i++) {
        if (!mbar_wait(&full[warp][st], ph, &abort_flag)) {
            ok = false;
            break;
        }
        int pg = pgs[0];
#pragma unroll
        for (int s = 1; s < FEW_ST; s++) pg = st == (uint32_t)s ? pgs[s] : pg;
        uint8_t *kst = ring + st * 2 * G::ROWS;
        const uint32_t ka = smem_u32(kst), va = ka + G::ROWS;
        const uint32_t s0 = (blk0 + warp + FEW_WARPS * i) * FEW_KEYS;
        if (pg >= 0) {
            if (s0 + FEW_KEYS > n) {  // rows past the sequence's end may hold anything: 0 * inf is not 0
                for (uint32_t x = lane; x < FEW_KEYS * HD / 8; x += 32) {
                    const uint32_t r = x / (HD / 8), c = x % (HD / 8);
                    if (s0 + r >= n)
                        *reinterpret_cast<uint4 *>(kst + G::ROWS + (c / 8) * 2048 + sw128(r, c & 7)) =
                            make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
            float sc[2][4] = {};
#pragma unroll
            for (int ks = 0; ks < HD / 16; ks++) {
                // keys 0-7 | 8-15 x dims 0-7 | 8-15 of this k step
                uint32_t kf[4];
                const uint32_t r = (lane & 7) + ((lane >> 4) << 3), c = ks * 2 + ((lane >> 3) & 1);
                ldsm4(kf, ka + (c / 8) * 2048 + sw128(r, c & 7));
                mma16816<TC>(sc[0], qf[ks], kf[0], kf[1]);
                mma16816<TC>(sc[1], qf[ks], kf[2], kf[3]);
                if (SPLIT) {
                    uint32_t ql[4];
                    load_q(qaddr + G::Q, ks, ql);
                    mma16816<TC>(sc[0], ql, kf[0], kf[1]);
                    mma16816<TC>(sc[1], ql, kf[2], kf[3]);
                }
            }
            uint32_t ph_[4], pl_[4];
            float p[2][4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float x[4], mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t s = s0 + (e >> 1) * 8 + t4 * 2 + (e & 1);
                    x[e] = (s >= rlo[h] && s < rhi[h]) ? sc[e >> 1][2 * h + (e & 1)] * c2 : -INFINITY;
                    mx = fmaxf(mx, x[e]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
                const float mn = fmaxf(m[h], mx);
                const float ms = mn == -INFINITY ? 0.f : mn;
                const float f = ex2(m[h] - ms);
                m[h] = mn;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    p[h][e] = ex2(x[e] - ms);
                    sum += p[h][e];
                }
                l[h] = l[h] * f + sum;
                if (__any_sync(~0u, f != 1.f)) {
#pragma unroll
                    for (int d = 0; d < HD / 8; d++) {
                        acc[d][2 * h] *= f;
                        acc[d][2 * h + 1] *= f;
                    }
                }
            }
            // A operand of the second product: rows g, g + 8 x slots 2 t4, 2 t4 + 8
            split_pack<TC>(p[0][0], p[0][1], ph_[0], pl_[0]);
            split_pack<TC>(p[1][0], p[1][1], ph_[1], pl_[1]);
            split_pack<TC>(p[0][2], p[0][3], ph_[2], pl_[2]);
            split_pack<TC>(p[1][2], p[1][3], ph_[3], pl_[3]);
#pragma unroll
            for (int d = 0; d < HD / 16; d++) {
                uint32_t vf[4];
                const uint32_t r = lane & 15, c = d * 2 + (lane >> 4);
                ldsm4t(vf, va + (c / 8) * 2048 + sw128(r, c & 7));
                mma16816<TC>(acc[2 * d], ph_, vf[0], vf[1]);
                mma16816<TC>(acc[2 * d + 1], ph_, vf[2], vf[3]);
                if (SPLIT) {
                    mma16816<TC>(acc[2 * d], pl_, vf[0], vf[1]);
                    mma16816<TC>(acc[2 * d + 1], pl_, vf[2], vf[3]);
                }
            }
        }
        // the block FEW_ST ahead goes into this stage, once every lane has read it
        const uint32_t nx = i + FEW_ST;
        if (nx < mine) {
            if ((nx & 31) == 0) {  // entering the next 32 page ids
                if (nx & 32)
                    ids = page_of(nx + 32 + lane);  // blocks behind ids_next's
                else
                    ids_next = page_of(nx + 32 + lane);
            }
            __syncwarp();
            const int np = issue(nx);
#pragma unroll
            for (int s = 0; s < FEW_ST; s++)
                if (st == (uint32_t)s) pgs[s] = np;
        }
        if (++st == FEW_ST) st = 0, ph ^= 1;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(~0u, l[h], 1);
        l[h] += __shfl_xor_sync(~0u, l[h], 2);
        if (t4 == 0) {
            s_m[warp][g + 8 * h] = m[h];
            s_l[warp][g + 8 * h] = l[h];
        }
    }
    if (!ok) {  // let the copies in flight land before this block's memory is given back
        if (lane == 0) g_timeout = 1;
        const unsigned long long t0 = now_ns();
        while (now_ns() - t0 < 1000000ull) {
        }
    }
    // join the warps: their outputs through the ring (every stage has been read)
    __syncthreads();
    float *so = reinterpret_cast<float *>(smem);  // [warp][16][HD]
#pragma unroll
    for (int d = 0; d < HD / 8; d++)
#pragma unroll
        for (int h = 0; h < 2; h++)
            *reinterpret_cast<float2 *>(so + (warp * 16 + g + 8 * h) * HD + d * 8 + t4 * 2) =
                make_float2(acc[d][2 * h], acc[d][2 * h + 1]);
    __syncthreads();
    for (uint32_t i = tid; i < rows * (HD / 8); i += FEW_WARPS * 32) {
        const uint32_t r = i / (HD / 8), c = i % (HD / 8);
        float mm = s_m[0][r];
#pragma unroll
        for (int w = 1; w < FEW_WARPS; w++) mm = fmaxf(mm, s_m[w][r]);
        const float ms = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f, v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; w++) {
            const float f = ex2(s_m[w][r] - ms);
            ll += f * s_l[w][r];
            const float *src = so + (w * 16 + r) * HD + c * 8;
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += f * src[e];
        }
        const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);  // NaN stays NaN
        const float lse2 = ll == 0.f ? -INFINITY : mm + log2f(ll);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= inv;
        const uint32_t tok = first + r / q.group, head = kvh * q.group + r % q.group;
        if (direct) {
            store8(reinterpret_cast<TQ *>(o.out) + (size_t)tok * o.out_stride + (size_t)head * HD + c * 8, v);
            if (o.lse && c == 0) o.lse[(size_t)tok * q.heads + head] = lse2 * 0.6931471805599453f;
        } else {
            const size_t row = (((size_t)split * a.n_seqs + b) * a.kv_heads + kvh) * ATTN_FEW + r;
            store8(o.few_o + row * HD + c * 8, v);
            if (c == 0) o.few_lse[row] = lse2;
        }
    }
}

// --------------------------------------------------------------- merge ----
//
// out = sum_s w_s o_s / sum_s w_s, w_s = 2^(lse2_s - max), over the parts that a
// row's kernel wrote.  A warp per (token, head): lanes hold HD / 32 dims.
constexpr int MERGE_WARPS = 4;

template <typename TQ, int HD>
__global__ void __launch_bounds__(MERGE_WARPS * 32) attn_merge_kernel(PagedArgs a, PagedQuery q, AttnOut o) {
    constexpr int E = HD / 32;
    griddep_wait();
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t row = blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5);
    const uint32_t tok = row / q.heads, head = row % q.heads;
    if (tok >= a.n_tok) return;
    uint32_t b = 0;  // sequences that end at or before the token
    for (uint32_t s = 0; s < a.n_seqs; s += 32)
        b += __popc(__ballot_sync(~0u, s + lane < a.n_seqs && __ldg(a.q_start + s + lane + 1) <= (int)tok));
    if (b >= a.n_seqs) return;
    uint32_t first;
    const uint32_t nq = a.tokens(b, first), n = a.len(b);
    if (tok < first || tok - first >= min(nq, a.max_q)) return;
    const uint32_t tq = min(nq, a.max_q), i = tok - first;
    const bool few = o.plan.is_few(tq, q.group);
    uint32_t parts = o.plan.many_splits;
    size_t step = (size_t)a.n_tok * q.heads, at = (size_t)tok * q.heads + head;
    const float *part_o = o.many_o, *part_lse = o.many_lse;
    if (few) {  // the live parts, as attn_few_kernel counts them
        const int pos0 = (int)n - (int)nq;
        const uint32_t chunk = o.plan.few_chunk;
        uint32_t lo0, hi0, lo1, hi1;
        q.range(max(pos0, 0), n, lo0, hi0);
        q.range(pos0 + (int)tq - 1, n, lo1, hi1);
        parts = hi1 > lo0 ? min((hi1 + chunk - 1) / chunk - lo0 / chunk, o.plan.few_splits) : 0;
        step = (size_t)a.n_seqs * a.kv_heads * ATTN_FEW;
        at = ((size_t)b * a.kv_heads + head / q.group) * ATTN_FEW + i * q.group + head % q.group;
        part_o = o.few_o;
        part_lse = o.few_lse;
    }
    if ((few ? o.plan.few_splits : o.plan.many_splits) == 1) return;  // written by its kernel
    float mx = -INFINITY;
    for (uint32_t s = lane; s < parts; s += 32) mx = fmaxf(mx, part_lse[s * step + at]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, d));
    const float ms = mx == -INFINITY ? 0.f : mx;
    float v[E], total = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = 0.f;
    for (uint32_t s = 0; s < parts; s++) {
        const float w = ex2(part_lse[s * step + at] - ms);
        if (w == 0.f) continue;  // a part that saw nothing (NaN goes on)
        total += w;
        const float *src = part_o + (s * step + at) * HD + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] += w * src[e];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    TQ *dst = reinterpret_cast<TQ *>(o.out) + (size_t)tok * o.out_stride + (size_t)head * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) dst[e] = (TQ)(v[e] * inv);
    if (o.lse && lane == 0) o.lse[(size_t)tok * q.heads + head] = total == 0.f ? -INFINITY : (mx + log2f(total)) * 0.6931471805599453f;
}

template <typename TQ, typename TC, int HD>
int launch_few(const AttnPagedCall &c, const AttnOut &o, cudaStream_t s) {
    CUtensorMap mk, mv;
    int rc = make_page_map(&mk, c.a.k, c.a, HD, c.cache_type, FEW_KEYS);
    if (rc == CUQ_OK) rc = make_page_map(&mv, c.a.v, c.a, HD, c.cache_type, FEW_KEYS);
    if (rc) return rc;
    auto kern = attn_few_kernel<TQ, TC, HD>;
    CUQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FewGeo<HD>::SMEM));
    const dim3 grid(c.a.kv_heads, o.plan.few_splits, c.a.n_seqs);
    kern<<<grid, FEW_WARPS * 32, FewGeo<HD>::SMEM, s>>>(c.a, c.q, o, mk, mv);
    CUQ_CUDA_TRY(cudaGetLastError());
    return CUQ_OK;
}

template <typename TQ, typename TC>
int launch_all(const AttnPagedCall &c, const AttnOut &o, cudaStream_t s) {
    int rc = CUQ_OK;
    if (o.plan.many) rc = launch_attention_many(c, o, s);
    if (rc == CUQ_OK && o.plan.few)
        rc = c.hd == 64 ? launch_few<TQ, TC, 64>(c, o, s) : launch_few<TQ, TC, 128>(c, o, s);
    if (rc || (o.plan.few_splits == 1 && o.plan.many_splits == 1)) return rc;
    const uint64_t rows = (uint64_t)c.a.n_tok * c.q.heads;
    const dim3 grid((unsigned)((rows + MERGE_WARPS - 1) / MERGE_WARPS)), block(MERGE_WARPS * 32);
    const cudaError_t e =
        c.hd == 64 ? launch_maybe_pdl(attn_merge_kernel<TQ, 64>, grid, block, 0, s, true, c.a, c.q, o)
                   : launch_maybe_pdl(attn_merge_kernel<TQ, 128>, grid, block, 0, s, true, c.a, c.q, o);
    CUQ_CUDA_TRY(e);
    return CUQ_OK;
}

}  // namespace

namespace ptc {
int make_page_map(CUtensorMap *m, const void *pool, const PagedArgs &a, uint32_t hd, int type, uint32_t rows) {
    const cuuint64_t dims[4] = {hd, a.page_size, a.kv_heads, a.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)a.page_size * hd * 2, a.page_stride * 2};
    const cuuint32_t box[4] = {64, rows, 1, 1}, estr[4] = {1, 1, 1, 1};
    typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn encode = nullptr;
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess || !fn) {
            set_error("paged cache: cuTensorMapEncodeTiled is not available from the driver");
            return CUQ_ECUDA;
        }
        encode = reinterpret_cast<EncodeFn>(fn);
    }
    const CUresult r = encode(m, type == CUQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void *>(pool), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("paged cache: cuTensorMapEncodeTiled failed (%d)", (int)r);
        return CUQ_ECUDA;
    }
    return CUQ_OK;
}
}  // namespace ptc

AttnPlan attention_paged_plan(const AttnPagedCall &c, int sm_count) {
    AttnPlan p{};
    p.few_chunk = 256;
    p.few_splits = p.many_splits = 1;
    if (c.a.n_seqs == 0 || c.a.n_tok == 0 || c.a.max_q == 0) return p;
    const uint64_t g = c.q.group, max_rows = (uint64_t)c.a.max_q * g;
    p.many = max_rows > ATTN_FEW;
    // several sequences may be mixed; one alone is left to the kernel its bound asks for
    p.few = !p.many || (c.a.n_seqs > 1 && g <= ATTN_FEW);
    const uint64_t sms = (uint64_t)sm_count;
    if (p.few) {
        // two CTAs an SM; parts of at least 256 slots, and at most 64 of them
        const uint64_t items = (uint64_t)c.a.n_seqs * c.a.kv_heads;
        uint64_t want = (2 * sms + items - 1) / items, most = ((uint64_t)c.a.max_kv + 255) / 256;
        // many items of unlike lengths: parts of 1024 slots even them out
        if (items > 1 && want < (c.a.max_kv + 1023u) / 1024u) want = (c.a.max_kv + 1023u) / 1024u;
        if (want > most) want = most;
        if (want > 64) want = 64;
        if (want < 1) want = 1;
        uint64_t chunk = (c.a.max_kv + want - 1) / want;
        chunk = (chunk + 63) / 64 * 64;
        if (chunk < 64) chunk = 64;
        p.few_chunk = (uint32_t)chunk;
        p.few_splits = (uint32_t)((c.a.max_kv + chunk - 1) / chunk);
        // a window may start inside a chunk, but spans no more of them
        if (p.few_splits < 1) p.few_splits = 1;
    }
    if (p.many) {
        p.many_tiles = (uint32_t)((c.a.n_tok * g + 255) / 256 + c.a.n_seqs);
        const uint64_t base = ((c.a.n_tok * g + 255) / 256) * c.a.kv_heads;
        uint64_t want = base ? sms / base : 1, most = ((uint64_t)c.a.max_kv + 511) / 512;
        if (want > most) want = most;
        if (want > 64) want = 64;
        p.many_splits = want < 1 ? 1u : (uint32_t)want;
    }
    return p;
}

namespace {
// floats of the few's outputs, the many's outputs, the few's sums, the many's sums
void part_sizes(const AttnPagedCall &c, const AttnPlan &p, size_t (&n)[4]) {
    const size_t few = p.few_splits > 1 ? (size_t)p.few_splits * c.a.n_seqs * c.a.kv_heads * ATTN_FEW : 0;
    const size_t many = p.many_splits > 1 ? (size_t)p.many_splits * c.a.n_tok * c.q.heads : 0;
    n[0] = few * c.hd;
    n[1] = many * c.hd;
    n[2] = few;
    n[3] = many;
}
}  // namespace

size_t attention_paged_workspace(const AttnPagedCall &c, int sm_count) {
    size_t n[4];
    part_sizes(c, attention_paged_plan(c, sm_count), n);
    return (n[0] + n[1] + n[2] + n[3]) * sizeof(float);
}

int launch_attention_paged(const AttnPagedCall &c, int sm_count, cudaStream_t s) {
    AttnOut o{};
    o.out = c.out;
    o.out_stride = c.out_stride;
    o.lse = c.lse;
    o.plan = attention_paged_plan(c, sm_count);
    size_t n[4];
    part_sizes(c, o.plan, n);
    o.few_o = reinterpret_cast<float *>(c.workspace);
    o.many_o = o.few_o + n[0];
    o.few_lse = o.many_o + n[1];
    o.many_lse = o.few_lse + n[2];
    if (c.type == CUQ_F32) return launch_all<float, __half>(c, o, s);
    if (c.type == CUQ_F16) return launch_all<__half, __half>(c, o, s);
    return launch_all<__nv_bfloat16, __nv_bfloat16>(c, o, s);
}

int attention_few_status(cudaStream_t s, int *timed_out) {
    CUQ_CUDA_TRY(cudaMemcpyFromSymbolAsync(timed_out, g_timeout, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
    CUQ_CUDA_TRY(cudaStreamSynchronize(s));
    if (*timed_out) {
        const int zero = 0;
        CUQ_CUDA_TRY(cudaMemcpyToSymbolAsync(g_timeout, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s));
        CUQ_CUDA_TRY(cudaStreamSynchronize(s));
    }
    return CUQ_OK;
}

}  // namespace cuq
