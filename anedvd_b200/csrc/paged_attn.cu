// paged_attn.cu -- attention of a batch's new tokens over a paged KV cache:
//   o = sum_s p_s v_s / sum_s p_s,  p_s = exp(scale q k_s - max),  s over the visible slots.
// This file: how a call is split, the kernel for sequences of few rows (decode
// steps, short drafts) and the merge of split results.  paged_attn_tc.cu has the
// kernel for many rows.
#include "paged_tc.cuh"

namespace cuq {

using namespace ptc;

namespace {

// ------------------------------------------------------------ few rows ----
//
// Bound by HBM: each K and V row is read once for all the rows of its group.  The
// work is the blocks of 16 slots that each (sequence, KV head) sees, one behind the
// other; every warp takes an equal run of them, whatever the lengths, so nothing is
// dealt out unevenly and no two warps wait for each other.  A run may end inside a
// (sequence, KV head), whose warps then each write a part; part `warp + item` is
// free for it, since along the run either the warp or the item steps on.  Beginning
// an item (its queries, its part) costs about what FEW_ITEM blocks do, so every item
// is that much longer than its blocks.
// A warp keeps FEW_ST blocks in flight across item borders, as TMA boxes of 64 dims
// in the 128-byte swizzle, which ldmatrix reads without bank conflicts.  Scores and
// outputs run on mma.sync.m16n8k16 (16 rows x 16 slots, fp32 accumulate); fp32
// queries are two fp16 operands, hi and lo, and so are the probabilities of every type:
// the second operand costs 0 to 5 % (32 requests 39.3 -> 39.6 us, 16 of 600 slots
// 11.8 -> 12.3), and what is left of the error is the output's own rounding (3.5e-4 root
// mean square, with one rounded operand 4.0e-4).
// A decode step of 32 requests up to 8192 slots (32 heads, 8 KV heads, head_dim 128,
// bf16, 186 MB) takes 39.6 us with the merge, 4.7 TB/s, 73 % of a copy's rate; the walk
// itself runs at the rate of HBM, and the rest is the start (three dependent loads
// before the first copy) and the merge.  Larger batches come nearer: 128 requests up to
// 4096 slots 82 us, 5.6 TB/s.  fp32 queries over fp16 take 41.6 us.  Two blocks in
// flight a warp: with three the step took 42.4 us and with four 48.6, since queries and
// page ids then wait behind 28 MB of copies.  With a CTA for each part of 256 to 1024 slots instead of equal runs
// it took 51 to 67 us.
// Where all items are short, a cluster of CTAs takes each instead and joins its parts
// through distributed shared memory: one launch, no workspace (attention_paged_plan has
// the rule and what both forms measured).
constexpr int FEW_WARPS = 4, FEW_ST = 2, FEW_KEYS = 16;
constexpr uint32_t FEW_RUN = 4;   // blocks a warp takes at least
constexpr uint32_t FEW_ITEM = 3;  // blocks' worth of an item's own cost
constexpr uint32_t FEW_NEAR = 8;  // blocks a warp at most where a cluster takes an item

template <int HD>
struct FewGeo {
    static constexpr int ROWS = FEW_KEYS * HD * 2;  // K (or V) bytes of a stage
    static constexpr int SMEM = 1024 + FEW_WARPS * FEW_ST * 2 * ROWS;
    static constexpr int CTAS = HD == 128 ? 2 : 4;  // an SM
};

// A sequence as the few-row kernel sees it: its attended tokens and its blocks.
struct FewSeq {
    uint32_t first, nq, tq, n, blk0, nblk;
    // length of one KV head's item
    __device__ __forceinline__ uint32_t units() const { return nblk ? nblk + FEW_ITEM : 0; }
    __device__ __forceinline__ FewSeq(const PagedArgs &a, const PagedQuery &q, const AttnPlan &plan, uint32_t b) {
        nq = a.tokens(b, first);
        n = a.len(b);
        tq = min(nq, a.max_q);
        blk0 = nblk = 0;
        if (tq == 0 || !plan.is_few(tq, q.group)) return;
        const int pos0 = (int)n - (int)nq;
        uint32_t lo0, hi0, lo1, hi1;
        q.range(max(pos0, 0), n, lo0, hi0);
        q.range(pos0 + (int)tq - 1, n, lo1, hi1);
        if (hi1 <= lo0) return;
        blk0 = lo0 / FEW_KEYS;
        nblk = (hi1 + FEW_KEYS - 1) / FEW_KEYS - blk0;
    }
};

// Units of one warp's run.
__device__ __forceinline__ uint32_t few_run(uint32_t total, uint32_t kv_heads, uint32_t ctas) {
    const uint32_t warps = ctas * FEW_WARPS;
    return max(FEW_RUN, (uint32_t)(((uint64_t)total * kv_heads + warps - 1) / warps));
}

// NEAR: few short items.  A cluster of CTAs takes one item and every warp an equal
// part of its blocks; the parts stay in shared memory and are joined there, so that
// the call is one launch.
template <typename TQ, typename TC, int HD, bool NEAR>
__global__ void __launch_bounds__(FEW_WARPS * 32, FewGeo<HD>::CTAS)
    attn_few_kernel(PagedArgs a, PagedQuery q, AttnOut o, const __grid_constant__ CUtensorMap mk,
                    const __grid_constant__ CUtensorMap mv) {
    using G = FewGeo<HD>;
    constexpr bool SPLIT = std::is_same<TQ, float>::value;
    // probabilities are two 16-bit operands too, hi and lo; as fp16 they are 2^12 larger,
    // so that the low parts keep clear of subnormals
    constexpr float LIFT = std::is_same<TC, __half>::value ? 12.f : 0.f;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[FEW_WARPS][FEW_ST];
    __shared__ int abort_flag;
    __shared__ float s_lse[NEAR ? FEW_WARPS : 1][ATTN_FEW];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = warp_index();
    uint32_t rank = 0, ranks = 1;
    if constexpr (NEAR) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    }
    griddep_wait();
    if (!NEAR) griddep_launch();  // the merge may take its place; it waits for this grid's end
    // units of the sequences [0, 32), one a lane, and of all
    const uint32_t v0 = !NEAR && lane < a.n_seqs ? FewSeq(a, q, o.plan, lane).units() : 0;
    if (tid == 0) {
        prefetch_map(&mk);
        prefetch_map(&mv);
        abort_flag = 0;
        for (int w = 0; w < FEW_WARPS; w++)
            for (int s = 0; s < FEW_ST; s++) mbar_init(&full[w][s], 1);
        mbar_init_fence();
    }
    const uint32_t gw = blockIdx.x * FEW_WARPS + warp;
    uint32_t b0 = 0, h0 = 0, k0 = 0, left = 0;  // the run's first sequence, KV head and unit, and its units
    if constexpr (NEAR) {
        const uint32_t x = blockIdx.x / ranks;
        b0 = x / a.kv_heads;
        h0 = x % a.kv_heads;
        const uint32_t nblk = FewSeq(a, q, o.plan, b0).nblk, warps = ranks * FEW_WARPS, per = (nblk + warps - 1) / warps;
        k0 = min(nblk, (rank * FEW_WARPS + warp) * per);
        left = min(per, nblk - k0);
        if (lane < ATTN_FEW) s_lse[warp][lane] = -INFINITY;
        __syncthreads();
    } else {
        uint32_t total = v0;
        for (uint32_t b = lane + 32; b < a.n_seqs; b += 32) total += FewSeq(a, q, o.plan, b).units();
        total = __reduce_add_sync(~0u, total);
        __syncthreads();
        if (gw == gridDim.x * FEW_WARPS - 1) {  // the last warp, which has the least to do: the table for the merge
            uint32_t before = 0;
            for (uint32_t s0 = 0; s0 < a.n_seqs; s0 += 32) {
                const uint32_t v = s0 + lane < a.n_seqs ? FewSeq(a, q, o.plan, s0 + lane).units() : 0;
                uint32_t upto = v;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t up = __shfl_up_sync(~0u, upto, d);
                    if (lane >= (uint32_t)d) upto += up;
                }
                if (s0 + lane < a.n_seqs) o.few_units[s0 + lane] = before + upto - v;
                before += __shfl_sync(~0u, upto, 31);
            }
            if (lane == 0) o.few_units[a.n_seqs] = total;
        }
        const uint32_t run = few_run(total, a.kv_heads, gridDim.x);
        {
            const uint64_t x0 = (uint64_t)gw * run, all = (uint64_t)total * a.kv_heads;
            left = x0 < all ? (uint32_t)min((uint64_t)run, all - x0) : 0;
        }
        if (!left) return;
        {
            uint32_t x = gw * run;
            for (uint32_t s0 = 0;; s0 += 32) {
                uint32_t v = v0;
                if (s0) v = s0 + lane < a.n_seqs ? FewSeq(a, q, o.plan, s0 + lane).units() : 0;
                v *= a.kv_heads;
                uint32_t upto = v;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t up = __shfl_up_sync(~0u, upto, d);
                    if (lane >= (uint32_t)d) upto += up;
                }
                const uint32_t hit = __ballot_sync(~0u, x < upto);
                if (hit) {
                    const int at = __ffs(hit) - 1;
                    const uint32_t mine = __shfl_sync(~0u, v, at);
                    x -= __shfl_sync(~0u, upto, at) - mine;
                    b0 = s0 + at;
                    h0 = x / (mine / a.kv_heads);
                    k0 = x % (mine / a.kv_heads);
                    break;
                }
                x -= __shfl_sync(~0u, upto, 31);
            }
        }
    }

    uint8_t *ring = smem + warp * (FEW_ST * 2 * G::ROWS);
    // ---- the loading cursor, FEW_ST blocks ahead of the computing one
    uint32_t lb = b0, lh = h0, lk = k0, to_load = left, ist = 0;
    FewSeq ls(a, q, o.plan, lb);
    // lane i: page id, as the table holds it, of block ids_at + i of sequence lb
    uint32_t ids_at = ~0u;
    int ids = 0;
    auto look = [&]() {
        ids_at = lk;
        ids = lk + lane < ls.nblk
                  ? a.pages[(size_t)lb * a.pages_stride + (((ls.blk0 + lk + lane) * FEW_KEYS) >> a.page_shift)]
                  : -1;
    };
    if (lk < ls.nblk) look();  // on its way while the queries are loaded
    auto issue = [&]() -> int {  // the next block into its stage; its page, or -1
        while (to_load && lk >= ls.nblk) {  // past the item's blocks: on to the next one
            const uint32_t skip = min(to_load, ls.nblk + FEW_ITEM - lk);
            to_load -= skip;
            lk = 0;
            if (!to_load) break;
            if (++lh == a.kv_heads) {
                lh = 0;
                do ls = FewSeq(a, q, o.plan, ++lb);
                while (!ls.nblk);  // the run goes on, so there is a later sequence
                ids_at = ~0u;
            }
        }
        if (!to_load) return -1;
        to_load--;
        if (lk < ids_at || lk >= ids_at + 32) look();
        int pg = __shfl_sync(~0u, ids, lk - ids_at);
        if ((uint32_t)pg >= a.n_pages) pg = -1;
        if (lane == 0) {
            const uint32_t dst = smem_u32(ring + ist * 2 * G::ROWS);
            const int slot = (int)(((ls.blk0 + lk) * FEW_KEYS) & (a.page_size - 1)), p = pg < 0 ? (int)a.n_pages : pg;
            mbar_expect_tx(&full[warp][ist], 2 * G::ROWS);
            tma_load_page(dst, &mk, 0, slot, (int)lh, p, &full[warp][ist]);
            tma_load_page(dst + G::ROWS, &mv, 0, slot, (int)lh, p, &full[warp][ist]);
        }
        if (++ist == FEW_ST) ist = 0;
        lk++;
        return pg;
    };
    int pgs[FEW_ST];  // page of the block to compute, of the one behind it, ...
    bool started = false;

    const uint32_t g = lane >> 2, t4 = lane & 3;
    const float c2 = q.scale * 1.4426950408889634f;  // scores in units of log 2
    uint32_t st = 0, ph = 0;
    bool ok = true;
    for (uint32_t b = b0, kvh = h0, k = k0; ok && left;) {
        const FewSeq sq(a, q, o.plan, b);
        if (!sq.nblk) {
            b++;
            continue;
        }
        const uint32_t rows = sq.tq * q.group, blocks = k < sq.nblk ? min(left, sq.nblk - k) : 0;
        if (!blocks) {  // only the end of the item's own cost
            left -= min(left, sq.units() - k);
            k = 0;
            if (++kvh == a.kv_heads) {
                kvh = 0;
                b++;
            }
            continue;
        }
        const int pos0 = (int)sq.n - (int)sq.nq;
        // rows g and g + 8 of the tile are this thread's: their slots and their queries
        uint32_t rlo[2], rhi[2], qf[HD / 16][4], ql[SPLIT ? HD / 16 : 1][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t r = g + 8 * h;
            rlo[h] = rhi[h] = 0;
            const TQ *src = nullptr;
            if (r < rows) {
                const uint32_t i = q.div_group(r);
                q.range(pos0 + (int)i, sq.n, rlo[h], rhi[h]);
                src = reinterpret_cast<const TQ *>(q.q) + (size_t)(sq.first + i) * q.q_stride +
                      (size_t)(kvh * q.group + (r - i * q.group)) * HD + t4 * 2;
            }
#pragma unroll
            for (int ks = 0; ks < HD / 16; ks++)
#pragma unroll
                for (int e = 0; e < 2; e++) {  // dims 2 t4, 2 t4 + 1 and those 8 on
                    if constexpr (SPLIT) {
                        const float2 f = src ? *reinterpret_cast<const float2 *>(src + ks * 16 + e * 8)
                                             : make_float2(0.f, 0.f);
                        split_pack<TC>(f.x, f.y, qf[ks][2 * e + h], ql[ks][2 * e + h]);
                    } else {
                        qf[ks][2 * e + h] = src ? *reinterpret_cast<const uint32_t *>(src + ks * 16 + e * 8) : 0u;
                    }
                }
        }
        if (!started) {  // behind the first queries, which would queue behind it for long
            started = true;
#pragma unroll
            for (int i = 0; i < FEW_ST; i++) pgs[i] = issue();
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float acc[HD / 8][4];
#pragma unroll
        for (int i = 0; i < HD / 8; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][e] = 0.f;

        for (uint32_t i = 0; i < blocks; i++) {
            if (!mbar_wait(&full[warp][st], ph, &abort_flag)) {
                ok = false;
                break;
            }
            const int pg = pgs[0];
#pragma unroll
            for (int s = 1; s < FEW_ST; s++) pgs[s - 1] = pgs[s];
            uint8_t *kst = ring + st * 2 * G::ROWS;
            const uint32_t ka = smem_u32(kst), va = ka + G::ROWS;
            const uint32_t s0 = (sq.blk0 + k + i) * FEW_KEYS;
            if (pg >= 0) {
                const bool tail = s0 + FEW_KEYS > sq.n;
                if (tail) {  // rows past the sequence's end may hold anything: 0 * inf is not 0
                    for (uint32_t x = lane; x < FEW_KEYS * HD / 8; x += 32) {
                        const uint32_t r = x / (HD / 8), c = x % (HD / 8);
                        if (s0 + r >= sq.n)
                            *reinterpret_cast<uint4 *>(kst + G::ROWS + (c / 8) * 2048 + sw128(r, c & 7)) =
                                make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                float sc[2][4] = {}, slo[2][4] = {};
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++) {
                    // keys 0-7 | 8-15 x dims 0-7 | 8-15 of this k step
                    uint32_t kf[4];
                    const uint32_t r = (lane & 7) + ((lane >> 4) << 3), c = ks * 2 + ((lane >> 3) & 1);
                    ldsm4(kf, ka + (c / 8) * 2048 + sw128(r, c & 7));
                    mma16816<TC>(sc[0], qf[ks], kf[0], kf[1]);
                    mma16816<TC>(sc[1], qf[ks], kf[2], kf[3]);
                    if constexpr (SPLIT) {
                        mma16816<TC>(slo[0], ql[ks], kf[0], kf[1]);
                        mma16816<TC>(slo[1], ql[ks], kf[2], kf[3]);
                    }
                }
                if constexpr (SPLIT)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[0][e] += slo[0][e], sc[1][e] += slo[1][e];
                uint32_t phi[4], plo[4];
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
                        p[h][e] = ex2(x[e] - ms + LIFT);
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
                split_pack<TC>(p[0][0], p[0][1], phi[0], plo[0]);
                split_pack<TC>(p[1][0], p[1][1], phi[1], plo[1]);
                split_pack<TC>(p[0][2], p[0][3], phi[2], plo[2]);
                split_pack<TC>(p[1][2], p[1][3], phi[3], plo[3]);
#pragma unroll
                for (int d = 0; d < HD / 16; d++) {
                    uint32_t vf[4];
                    const uint32_t r = lane & 15, c = d * 2 + (lane >> 4);
                    ldsm4t(vf, va + (c / 8) * 2048 + sw128(r, c & 7));
                    mma16816<TC>(acc[2 * d], plo, vf[0], vf[1]);
                    mma16816<TC>(acc[2 * d + 1], plo, vf[2], vf[3]);
                    mma16816<TC>(acc[2 * d], phi, vf[0], vf[1]);
                    mma16816<TC>(acc[2 * d + 1], phi, vf[2], vf[3]);
                }
                if (tail) fence_async_smem();  // the zeros are written before the stage is loaded again
            }
            // the block FEW_ST ahead goes into this stage, once every lane has read it
            __syncwarp();
            pgs[FEW_ST - 1] = issue();
            if (++st == FEW_ST) st = 0, ph ^= 1;
        }
        // this warp's part of the item; NEAR: in the place of its stages, whose last block is done with
        const uint64_t part = NEAR ? 0 : (uint64_t)gw + (uint64_t)b * a.kv_heads + kvh;
        float *const part_o = NEAR ? reinterpret_cast<float *>(ring) : o.few_o;
        float *const part_lse = NEAR ? s_lse[NEAR ? warp : 0] : o.few_lse;
        if (NEAR) __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l[h] += __shfl_xor_sync(~0u, l[h], 1);
            l[h] += __shfl_xor_sync(~0u, l[h], 2);
            const uint32_t r = g + 8 * h;
            if (r >= rows) continue;
            const size_t row = NEAR ? r : part * o.plan.few_rows + r;
            const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];  // NaN stays NaN
            if (t4 == 0) part_lse[row] = l[h] == 0.f ? -INFINITY : m[h] - LIFT + log2f(l[h]);
#pragma unroll
            for (int d = 0; d < HD / 8; d++)
                *reinterpret_cast<float2 *>(part_o + row * HD + d * 8 + t4 * 2) =
                    make_float2(acc[d][2 * h] * inv, acc[d][2 * h + 1] * inv);
        }
        left -= min(left, sq.units() - k);
        k = 0;
        if (++kvh == a.kv_heads) {
            kvh = 0;
            b++;
        }
    }
    if constexpr (NEAR) {
        // a warp a row: a part's sum in each lane, then eight parts on their way at once
        auto sync = [&] {
            __syncwarp();
            if (ranks > 1)
                cluster_sync();
            else
                __syncthreads();
        };
        sync();
        const FewSeq sq(a, q, o.plan, b0);
        constexpr int E = HD / 32;
        const uint32_t parts = ranks * FEW_WARPS, rows = sq.tq * q.group;
        for (uint32_t r = rank * FEW_WARPS + warp; r < rows; r += parts) {
            float ls = -INFINITY;
            if (lane < parts) ls = peer_load(peer_smem(&s_lse[lane % FEW_WARPS][r], lane / FEW_WARPS));
            float top = ls;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
            const float w = ex2(ls - (top == -INFINITY ? 0.f : top));
            float v[E], total = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = 0.f;
            for (uint32_t p0 = 0; p0 < parts; p0 += FEW_WARPS) {
                float src[FEW_WARPS][E];
#pragma unroll
                for (int i = 0; i < FEW_WARPS; i++)
#pragma unroll
                    for (int e = 0; e < E; e++)
                        src[i][e] = peer_load(peer_smem(smem + i * (FEW_ST * 2 * G::ROWS) + (r * HD + e * 32 + lane) * 4,
                                                        p0 / FEW_WARPS));
#pragma unroll
                for (int i = 0; i < FEW_WARPS; i++) {
                    const float wi = __shfl_sync(~0u, w, (p0 + i) & 31);
                    if (wi == 0.f) continue;  // a part that saw nothing may hold anything
                    total += wi;
#pragma unroll
                    for (int e = 0; e < E; e++) v[e] += wi * src[i][e];
                }
            }
            const float inv = total == 0.f ? 0.f : 1.f / total;
            const uint32_t i = q.div_group(r), tok = sq.first + i, head = h0 * q.group + (r - i * q.group);
            TQ *dst = reinterpret_cast<TQ *>(o.out) + (size_t)tok * o.out_stride + (size_t)head * HD + lane;
#pragma unroll
            for (int e = 0; e < E; e++) dst[e * 32] = (TQ)(v[e] * inv);
            if (o.lse && lane == 0)
                o.lse[(size_t)tok * q.heads + head] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
        }
        sync();  // the others may still read this CTA's parts
    }
    if (!ok) give_up(lane == 0);
}

// --------------------------------------------------------------- merge ----
//
// out = sum_s w_s o_s / sum_s w_s, w_s = 2^(lse2_s - max), over the parts that a
// row's kernel wrote.  A warp per (token, head): lanes hold HD / 32 dims.  Bound by the
// latency of its dependent loads (sequence, lengths and units, sums, outputs): 9.8 us
// alone under a profiler for the 26 parts an item of a decode step of 32 requests, of
// which 5 show behind the walk.  Reading one part after the other it took twice as long.
constexpr int MERGE_WARPS = 4;

template <typename TQ, int HD>
__global__ void __launch_bounds__(MERGE_WARPS * 32) attn_merge_kernel(PagedArgs a, PagedQuery q, AttnOut o) {
    constexpr int E = HD / 32;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t row = blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5);
    griddep_wait();
    const uint32_t tok = row / q.heads, head = row % q.heads;
    const uint32_t b = tok < a.n_tok ? a.sequence_of((int)tok) : a.n_seqs;
    uint32_t first = 0, nq = 0, before = 0, total_units = 0;
    if (o.plan.few && b < a.n_seqs) {  // on their way beside the batch's
        before = o.few_units[b];
        total_units = o.few_units[a.n_seqs];
    }
    if (b < a.n_seqs) nq = a.tokens(b, first);
    const uint32_t tq = min(nq, a.max_q), i = tok - first;
    const bool few = o.plan.is_few(tq, q.group);
    // a row of no sequence, past max_q, or written by its kernel
    const bool none = b >= a.n_seqs || tok < first || i >= tq || (!few && o.plan.many_splits == 1);
    const FewSeq sq(a, q, o.plan, none ? 0 : b);
    if (none) return;
    uint32_t parts = o.plan.many_splits;
    size_t step = (size_t)a.n_tok * q.heads, at = (size_t)tok * q.heads + head;
    const float *part_o = o.many_o, *part_lse = o.many_lse;
    if (few) {  // the warps whose runs hold blocks of this item
        const uint32_t run = few_run(total_units, a.kv_heads, o.plan.few_ctas);
        const uint32_t kvh = head / q.group;
        const uint64_t x0 = (uint64_t)before * a.kv_heads + (uint64_t)kvh * sq.units();
        const uint32_t w0 = (uint32_t)(x0 / run), w1 = (uint32_t)((x0 + sq.nblk + run - 1) / run);
        parts = sq.nblk ? w1 - w0 : 0;
        step = o.plan.few_rows;
        at = (w0 + (size_t)b * a.kv_heads + kvh) * step + i * q.group + head % q.group;
        part_o = o.few_o;
        part_lse = o.few_lse;
    }
    float v[E], total = 0.f, top = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = 0.f;
    for (uint32_t s0 = 0; s0 < parts; s0 += 32) {  // a part's sum in each lane
        const float ls = s0 + lane < parts ? part_lse[(s0 + lane) * step + at] : -INFINITY;
        float mx = ls;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, d));
        const float up = fmaxf(top, mx), ms = up == -INFINITY ? 0.f : up;
        const float f = ex2(top - ms), w = ex2(ls - ms);
        top = up;
        total *= f;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] *= f;
        const uint32_t n32 = min(32u, parts - s0);
        for (uint32_t i0 = 0; i0 < n32; i0 += 8) {  // eight parts on their way at once
            float src[8][E];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float *from = part_o + ((s0 + min(i0 + i, n32 - 1)) * step + at) * HD + lane * E;
                if constexpr (E == 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(from);
                    src[i][0] = f.x, src[i][1] = f.y, src[i][2] = f.z, src[i][3] = f.w;
                } else {
                    const float2 f = *reinterpret_cast<const float2 *>(from);
                    src[i][0] = f.x, src[i][1] = f.y;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float wi = __shfl_sync(~0u, w, (i0 + i) & 31);
                if (i0 + i >= n32 || wi == 0.f) continue;  // a part that saw nothing may hold anything
                total += wi;
#pragma unroll
                for (int e = 0; e < E; e++) v[e] += wi * src[i][e];
            }
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    TQ *dst = reinterpret_cast<TQ *>(o.out) + (size_t)tok * o.out_stride + (size_t)head * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) dst[e] = (TQ)(v[e] * inv);
    if (o.lse && lane == 0) o.lse[(size_t)tok * q.heads + head] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
}

template <typename TQ, typename TC, int HD>
int launch_few(const AttnPagedCall &c, const AttnOut &o, cudaStream_t s) {
    CUtensorMap mk, mv;
    int rc = make_page_map(&mk, c.a.k, c.a, HD, c.cache_type, FEW_KEYS, HD / 64);
    if (rc == CUQ_OK) rc = make_page_map(&mv, c.a.v, c.a, HD, c.cache_type, FEW_KEYS, HD / 64);
    if (rc) return rc;
    auto launch = [&](auto kern, uint32_t ctas, uint32_t cluster, std::atomic<uint64_t> &allowed) -> int {
        CUQ_CUDA_TRY(allow_smem(kern, FewGeo<HD>::SMEM, allowed));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas);
        cfg.blockDim = dim3(FEW_WARPS * 32);
        cfg.dynamicSmemBytes = FewGeo<HD>::SMEM;
        cfg.stream = s;
        cudaLaunchAttribute attrs[2];
        attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[0].val.programmaticStreamSerializationAllowed = 1;
        attrs[1].id = cudaLaunchAttributeClusterDimension;
        attrs[1].val.clusterDim.x = cluster;
        attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
        cfg.attrs = attrs;
        cfg.numAttrs = cluster ? 2 : 1;
        CUQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, c.a, c.q, o, mk, mv));
        return CUQ_OK;
    };
    static std::atomic<uint64_t> allowed, allowed_near;
    const AttnPlan &p = o.plan;
    if (p.few_cluster)
        return launch(attn_few_kernel<TQ, TC, HD, true>, c.a.n_seqs * c.a.kv_heads * p.few_cluster, p.few_cluster,
                      allowed_near);
    return launch(attn_few_kernel<TQ, TC, HD, false>, p.few_ctas, 0, allowed);
}

template <typename TQ, typename TC>
int launch_all(const AttnPagedCall &c, const AttnOut &o, cudaStream_t s) {
    int rc = CUQ_OK;
    if (o.plan.many) rc = launch_attention_many(c, o, s);
    if (rc == CUQ_OK && o.plan.few)
        rc = c.hd == 64 ? launch_few<TQ, TC, 64>(c, o, s) : launch_few<TQ, TC, 128>(c, o, s);
    if (rc || o.plan.few_cluster || (!o.plan.few && o.plan.many_splits == 1)) return rc;
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
int make_page_map(CUtensorMap *m, const void *pool, const PagedArgs &a, uint32_t hd, int type, uint32_t rows,
                  uint32_t blocks) {
    const cuuint64_t dims[5] = {64, a.page_size, hd / 64, a.kv_heads, a.n_pages};
    const cuuint64_t strides[4] = {(cuuint64_t)hd * 2, 128, (cuuint64_t)a.page_size * hd * 2, a.page_stride * 2};
    const cuuint32_t box[5] = {64, rows, blocks, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
    typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const EncodeFn encode = []() -> EncodeFn {  // the driver's, looked up through the runtime
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return nullptr;
        return reinterpret_cast<EncodeFn>(fn);
    }();
    if (!encode) {
        set_error("paged cache: cuTensorMapEncodeTiled is not available from the driver");
        return CUQ_ECUDA;
    }
    const CUresult r = encode(m, type == CUQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
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
    p.many_splits = 1;
    if (c.a.n_seqs == 0 || c.a.n_tok == 0 || c.a.max_q == 0) return p;
    const uint64_t g = c.q.group, max_rows = (uint64_t)c.a.max_q * g;
    p.many = max_rows > ATTN_FEW;
    // several sequences may be mixed; one alone is left to the kernel its bound asks for
    p.few = !p.many || (c.a.n_seqs > 1 && g <= ATTN_FEW);
    const uint64_t sms = (uint64_t)sm_count;
    if (p.few) {
        // as many CTAs as fit at once, but no more than have blocks to take
        const uint64_t blocks = (uint64_t)c.a.n_seqs * c.a.kv_heads * ((c.a.max_kv + FEW_KEYS - 1) / FEW_KEYS);
        const uint64_t most = sms * (c.hd == 64 ? FewGeo<64>::CTAS : FewGeo<128>::CTAS);
        const uint64_t want = (blocks + FEW_RUN * FEW_WARPS - 1) / (FEW_RUN * FEW_WARPS);
        p.few_ctas = (uint32_t)(want < 1 ? 1 : want < most ? want : most);
        p.few_rows = max_rows < ATTN_FEW ? (uint32_t)max_rows : ATTN_FEW;
        const uint64_t items = (uint64_t)c.a.n_seqs * c.a.kv_heads;
        if (!p.many && items <= most) {
            // As few blocks a warp as 8 CTAs an item, all of the call's at once on the GPU, come
            // to, in as few CTAs; up to FEW_NEAR.  One token over 40, 600, 2000, 4000 and 8000
            // slots (9 heads, 3 KV heads, head_dim 64, fp32, in a graph) takes 4.3, 6.6, 8.6, 12.1
            // and 19.1 us this way, 8.7, 9.5, 10.7, 13.5 and 16.2 with runs and the merge; 16
            // over 600 (32 heads, 8 KV heads, head_dim 128, bf16) 12.2 instead of 15.7.
            uint64_t seen = c.a.max_kv;
            if (c.q.window && c.q.window + (uint64_t)c.a.max_q < seen) seen = c.q.window + (uint64_t)c.a.max_q;
            const uint64_t longest = seen / FEW_KEYS + 1, warps = (most / items < 8 ? most / items : 8) * FEW_WARPS;
            const uint64_t each = (longest + warps - 1) / warps;
            if (each <= FEW_NEAR) p.few_cluster = (uint32_t)((longest + each * FEW_WARPS - 1) / (each * FEW_WARPS));
        }
    }
    if (p.many) {
        p.many_tiles = (uint32_t)((c.a.n_tok * g + 255) / 256 + c.a.n_seqs);
        const uint64_t base = ((c.a.n_tok * g + 255) / 256) * c.a.kv_heads;
        // as many parts of the slots as leave all CTAs on the GPU at once (one an SM), of 512
        // slots at least.  With one part, this many and twice as many (12 heads, 2 KV heads,
        // head_dim 128, bf16, in a graph): 64 tokens over 2048 slots 34, 19 and 19 us, over
        // 32768 410, 33 and 48; 512 over 8192 109, 36 and 49, over 32768 414, 87 and 98; 1024
        // over 32768 413, 161 and 168.  Where half a wave or more is there without parts a
        // second wave may pay (2048 over 32768 425 and 314 us) or not (over 2048 35 and 51);
        // the window is left out of account, and its empty parts cost little: 64 tokens with a
        // window of 128 over 32768 slots take 23 us.
        uint64_t want = base ? sms / base : 1, most = ((uint64_t)c.a.max_kv + 511) / 512;
        if (want > most) want = most;
        if (want > 64) want = 64;
        p.many_splits = want < 1 ? 1u : (uint32_t)want;
    }
    return p;
}

namespace {
// floats of the few's outputs, the many's outputs, the few's sums, the many's sums, and the few's table
void part_sizes(const AttnPagedCall &c, const AttnPlan &p, size_t (&n)[5]) {
    const size_t few = p.few && !p.few_cluster ? ((size_t)p.few_ctas * FEW_WARPS + (size_t)c.a.n_seqs * c.a.kv_heads) * p.few_rows : 0;
    const size_t many = p.many_splits > 1 ? (size_t)p.many_splits * c.a.n_tok * c.q.heads : 0;
    n[0] = few * c.hd;
    n[1] = many * c.hd;
    n[2] = few;
    n[3] = many;
    n[4] = p.few && !p.few_cluster ? (size_t)c.a.n_seqs + 1 : 0;
}
}  // namespace

size_t attention_paged_workspace(const AttnPagedCall &c, int sm_count) {
    size_t n[5];
    part_sizes(c, attention_paged_plan(c, sm_count), n);
    return (n[0] + n[1] + n[2] + n[3] + n[4]) * sizeof(float);
}

int launch_attention_paged(const AttnPagedCall &c, int sm_count, cudaStream_t s) {
    AttnOut o{};
    o.out = c.out;
    o.out_stride = c.out_stride;
    o.lse = c.lse;
    o.plan = attention_paged_plan(c, sm_count);
    size_t n[5];
    part_sizes(c, o.plan, n);
    o.few_o = reinterpret_cast<float *>(c.workspace);
    o.many_o = o.few_o + n[0];
    o.few_lse = o.many_o + n[1];
    o.many_lse = o.few_lse + n[2];
    o.few_units = reinterpret_cast<uint32_t *>(o.many_lse + n[3]);
    if (c.type == CUQ_F32) return launch_all<float, __half>(c, o, s);
    if (c.type == CUQ_F16) return launch_all<__half, __half>(c, o, s);
    return launch_all<__nv_bfloat16, __nv_bfloat16>(c, o, s);
}

namespace {
// A bounded wait that nothing ends, given up and counted as the kernels' own are.
__global__ void __launch_bounds__(32) wait_probe_kernel(unsigned long long limit_ns) {
    __shared__ uint64_t bar;
    __shared__ int abort_flag;
    griddep_wait();
    if (threadIdx.x == 0) {
        abort_flag = 0;
        mbar_init(&bar, 1);
        mbar_init_fence();
    }
    __syncthreads();
    if (!mbar_wait_slow(&bar, 0, &abort_flag, limit_ns)) give_up(threadIdx.x == 0);
}
}  // namespace

int launch_wait_probe(uint32_t limit_us, cudaStream_t s) {
    CUQ_CUDA_TRY(launch_maybe_pdl(wait_probe_kernel, dim3(1), dim3(32), 0, s, true, limit_us * 1000ull));
    return CUQ_OK;
}

int attention_few_gave_up(cudaStream_t s, unsigned int *n) { return gave_up_count(s, n); }

}  // namespace cuq
