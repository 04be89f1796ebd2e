// paged_attn_tc.cu -- attention of many new tokens over a paged KV cache on the
// 5th-generation tensor cores (the rows and the split: paged_attn.cu).
//
// A CTA takes 256 rows of one KV head as two streams of 128 (a row is a TMEM
// lane) and walks its part of the slots in tiles of 128 keys:
//   * warp 9 loads each tile's K and V pages by TMA (128-byte swizzle) into a ring;
//   * one lane of warp 8 issues S = Q K^T (both operands in shared memory) and
//     O += P V (P in tensor memory, V with its dims contiguous) for both streams;
//   * warps 0-3 and 4-7 are the streams' softmax: a thread owns a row, reads its
//     128 scores from tensor memory, keeps the running maximum and sum in
//     registers and writes P over S as 16-bit pairs.
// While one stream is in its softmax the other's products run.  S of tile j + 1 is
// issued behind O += P V of tile j, so when S is there, O is complete: the softmax
// threads rescale O themselves, and only when a row's maximum has grown by more
// than 2^8 (until then P stays below 2^8 and the sum takes it as it is).
// fp32 queries are two fp16 operands, and P is then two, which together fill S.  The
// tensor cores cut off what falls below the accumulator's last place, always towards
// zero: over a long context that is 2e-6 of an fp32 output.  So with fp32 queries O is
// of one tile only and the softmax threads sum the tiles in registers (4e-7).
// 16-bit queries have one 16-bit P; the row's sum takes it unrounded.  Two operands as
// for fp32 queries would add half of the products again.  Sums of the rounded
// probabilities beside the unrounded ones, which lse needs, took a prompt of 4096 tokens
// from 151 to 158 us for an error of 2.74e-5 instead of 2.79e-5 (root mean square).
// What bounds it: per 128 x 128 tile the two products take 1024 cycles of the
// tensor pipe at head_dim 128 (512 at 64) and the exponentials 1024 of the MUFU; but
// Q K^T reads both operands from shared memory, 8 KB a product of 64 cycles, and runs
// at 86, so that a pair of tiles takes at least 2400 cycles and is measured at 2900.
// Start and end of a CTA cost 11 000 more.  4096 tokens of 32 heads (8 KV heads,
// head_dim 128, fp16, causal) take 151 us, 912 TFLOP/s, 53 % of the measured product
// rate; 512 tokens over 32768 slots (12 heads, 2 KV heads, bf16) 101 us, 1.01 PFLOP/s.
// With fp32 queries over fp16, twice the products: 246 us, and the chunk 166.
// Tried and not kept: a quarter of the exponentials as polynomials on the FMA pipe
// (155 us), queries and first tile loaded before the first barrier (162 us), P handed
// over as 96 + 32 keys (158 us), two softmax threads a row (166 us).
#include "paged_tc.cuh"

namespace cuq {

using namespace ptc;

namespace {

constexpr int NT = 384;  // warps 0-3, 4-7 softmax, 8 MMA, 9 TMA, 10-11 idle
constexpr int KEYS = 128;

template <int HD, bool SPLIT>
struct ManyGeo {
    static constexpr int CB = HD / 64;
    static constexpr int TILE = KEYS * HD * 2;                  // bytes of a K or V tile
    static constexpr int Q = 128 * HD * 2 * (SPLIT ? 2 : 1);    // bytes of one stream's queries
    static constexpr int ST = (HD == 128) ? (SPLIT ? 3 : 5) : 6;
    static constexpr int SMEM = 1024 + 2 * Q + ST * TILE;
};

struct ManyBars {
    uint64_t q_full[2], kv_full[6], kv_empty[6], s_full[2], p_full[2][2], o_full[2], clean;
};

template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(NT, 1) attn_many_kernel(PagedArgs a, PagedQuery q, AttnOut o,
                                                           const __grid_constant__ CUtensorMap mk,
                                                           const __grid_constant__ CUtensorMap mv) {
    constexpr bool SPLIT = std::is_same<TQ, float>::value;
    using G = ManyGeo<HD, SPLIT>;
    // probabilities of fp32 queries are 2^7 larger (below 2^15 with the 2^8 that a
    // maximum may lag), so that their low fp16 parts keep clear of subnormals
    constexpr float LIFT = SPLIT ? 7.f : 0.f;
    constexpr int ST = G::ST;
    extern __shared__ uint8_t smem_raw[];
    __shared__ ManyBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, s_hole[2];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = warp_index();
    const uint32_t kvh = blockIdx.x % a.kv_heads, split = blockIdx.y;
    griddep_wait();
    griddep_launch();  // the few-row kernel or the merge may follow into free SMs; it waits for this grid's end

    // the tile: tiles are counted over the sequences that are this kernel's
    uint32_t b = 0, tile = blockIdx.x / a.kv_heads, ntile = 0;
    {
        bool found = false;
        for (uint32_t s0 = 0; s0 < a.n_seqs && !found; s0 += 32) {
            uint32_t cnt = 0, f;
            if (s0 + lane < a.n_seqs) {
                const uint32_t tq = min(a.tokens(s0 + lane, f), a.max_q);
                if (tq && !o.plan.is_few(tq, q.group)) cnt = (tq * q.group + 255) / 256;
            }
            uint32_t incl = cnt;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t up = __shfl_up_sync(~0u, incl, d);
                if (lane >= (uint32_t)d) incl += up;
            }
            const uint32_t hit = __ballot_sync(~0u, tile < incl);
            if (hit) {
                const int l = __ffs(hit) - 1;
                b = s0 + l;
                ntile = __shfl_sync(~0u, cnt, l);
                tile -= __shfl_sync(~0u, incl, l) - ntile;
                found = true;
            } else {
                tile -= __shfl_sync(~0u, incl, 31);
            }
        }
        if (!found) return;  // the same for every warp
    }
    tile = ntile - 1 - tile;  // a causal sequence's last tiles see the most slots: first
    uint32_t first;
    const uint32_t nq = a.tokens(b, first), n = a.len(b), tq = min(nq, a.max_q);
    const uint32_t rows = tq * q.group, row0 = tile * 256;
    const uint32_t my_rows = min(rows - row0, 256u);
    const int pos0 = (int)n - (int)nq;
    const bool two = my_rows > 128;
    // the slots that any of the rows sees, in tiles, and this split's part of them
    uint32_t j0, j1;
    {
        uint32_t lo0, hi0, lo1, hi1;
        q.range(max(pos0 + (int)(row0 / q.group), 0), n, lo0, hi0);
        q.range(pos0 + (int)((row0 + my_rows - 1) / q.group), n, lo1, hi1);
        j0 = lo0 / KEYS;
        j1 = hi1 > lo0 ? (hi1 + KEYS - 1) / KEYS : j0;
        const uint32_t per = (j1 - j0 + o.plan.many_splits - 1) / o.plan.many_splits;
        j0 = min(j1, j0 + split * per);
        j1 = min(j1, j0 + per);
    }
    const uint32_t nt = j1 - j0;

    if (warp == 8) tmem_alloc512(&tmem_slot);
    if (tid == 0) {
        abort_flag = s_hole[0] = s_hole[1] = 0;
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.q_full[i], 128);
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_full[i][0], 128);
            mbar_init(&bars.p_full[i][1], 128);
            mbar_init(&bars.o_full[i], 1);
        }
        for (int i = 0; i < ST; i++) {
            mbar_init(&bars.kv_full[i], 1);
            mbar_init(&bars.kv_empty[i], 1);
        }
        mbar_init(&bars.clean, 1);
        mbar_init_fence();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    uint8_t *ring = smem + 2 * G::Q;

    // 384 threads of 168 registers: the softmax's 256 take 208 (224), the others' 128 keep 88 (56)
    if (warp >= 8) {
        if constexpr (SPLIT)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        else
            asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            // ------------------------------------------------------ MMA issuer
            if (nt) {
                const uint32_t leader = elect_one();
                const uint32_t id_s = idesc<TC>(128, KEYS, false), id_o = idesc<TC>(128, HD, true);
                const uint64_t qd = sdesc_sw128(smem_u32(smem), 16, 1024), kd = sdesc_sw128(smem_u32(ring), 16, 1024),
                               vd = sdesc_sw128(smem_u32(ring), KEYS * 128, 1024);
                const uint32_t ns = two ? 2 : 1;
                auto wait_kv = [&](uint32_t x) { return mbar_wait(&bars.kv_full[x % ST], (x / ST) & 1, &abort_flag); };
                auto qk = [&](uint32_t s, uint32_t x) {  // S_s = Q_s K^T with K in stage x
                    const uint64_t kb = kd + (x % ST) * (G::TILE >> 4), qb = qd + s * (G::Q >> 4);
#pragma unroll
                    for (int part = 0; part < (SPLIT ? 2 : 1); part++)
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ks++) {
                            const uint32_t off = ((ks / 4) * (128 * 128) + (ks % 4) * 32) >> 4;
                            // (the low parts first: what the accumulator cuts off is then small against the sum)
                        umma_ss(leader, tmem + s * 128, qb + (SPLIT ? 1 - part : 0) * (128 * HD * 2 >> 4) + off, kb + off, id_s,
                                part | ks ? 1u : 0u);
                        }
                };
                auto pv = [&](uint32_t s, uint32_t x, int half, bool acc) {  // O_s += P_s V, 64 keys of V in stage x
                    const uint64_t vb = vd + (x % ST) * (G::TILE >> 4) + half * (KEYS * 64 >> 4);
                    const uint32_t d = tmem + 256 + s * 128, pa = tmem + s * 128 + half * (SPLIT ? 64 : 32);
#pragma unroll
                    for (int part = 0; part < (SPLIT ? 2 : 1); part++)
#pragma unroll
                        for (int i = 0; i < KEYS / 32; i++)
                            umma_ts(leader, d, SPLIT ? pa + (i / 2) * 32 + (1 - part) * 16 + (i & 1) * 8 : pa + i * 8, vb + (i * 2048 >> 4), id_o, (acc || part || i) ? 1u : 0u);
                };
                // stage x may be loaded again; only where it will be, so that no arrival is left in flight at the end
                auto freed = [&](uint32_t x) {
                    if (x + ST < 2 * nt) umma_commit(leader, &bars.kv_empty[x % ST]);
                };
                const bool tail = j1 * KEYS > n;
                bool ok = mbar_wait(&bars.q_full[0], 0, &abort_flag) && (!two || mbar_wait(&bars.q_full[1], 0, &abort_flag)) &&
                          wait_kv(0);
                if (ok) {
                    tc_fence_after();
                    for (uint32_t s = 0; s < ns; s++) {
                        qk(s, 0);
                        umma_commit(leader, &bars.s_full[s]);
                    }
                    freed(0);
                }
                for (uint32_t j = 0; ok && j < nt; j++) {
                    const uint32_t xv = 2 * j + 1, xk = 2 * j + 2;
                    const bool more = j + 1 < nt;
                    ok = wait_kv(xv) && (!more || wait_kv(xk)) &&
                         (more || !tail || mbar_wait(&bars.clean, 0, &abort_flag));
                    for (uint32_t s = 0; ok && s < ns; s++) {
                        ok = mbar_wait(&bars.p_full[s][0], j & 1, &abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        pv(s, xv, 0, !SPLIT && j > 0);
                        ok = mbar_wait(&bars.p_full[s][1], j & 1, &abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        pv(s, xv, 1, true);
                        if (more) {
                            qk(s, xk);
                            umma_commit(leader, &bars.s_full[s]);
                        } else {
                            umma_commit(leader, &bars.o_full[s]);
                        }
                    }
                    if (ok) {
                        freed(xv);
                        if (more) freed(xk);
                    }
                }
            }
        } else if (warp == 9) {
            // ------------------------------------------------------ TMA: K and V pages
            const uint32_t box = min(a.page_size, (uint32_t)KEYS), nbox = KEYS / box;
            auto page_of = [&](uint32_t j) -> int {  // of this lane's box of tile j; past the end: a hole
                const uint32_t slot = j * KEYS + lane * box;
                if (lane >= nbox || slot >= n) return (int)a.n_pages;
                const int pg = a.page(b, slot >> a.page_shift);
                return pg < 0 ? (int)a.n_pages : pg;
            };
            int pg = page_of(j0);
            bool ok = true;
            for (uint32_t j = 0; ok && j < nt; j++) {
                const int next = j + 1 < nt ? page_of(j0 + j + 1) : 0;
                const int slot = (int)(((j0 + j) * KEYS + lane * box) & (a.page_size - 1));
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const uint32_t x = 2 * j + v, st = x % ST;
                    if (x >= (uint32_t)ST && !mbar_wait(&bars.kv_empty[st], ((x / ST) - 1) & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) mbar_expect_tx(&bars.kv_full[st], G::TILE);
                    __syncwarp();
                    if (lane < nbox) {
                        const uint32_t dst = smem_u32(ring + st * G::TILE) + lane * box * 128;
#pragma unroll
                        for (int cb = 0; cb < G::CB; cb++)
                            tma_load_page(dst + cb * (KEYS * 128), v ? &mv : &mk, cb, slot, (int)kvh, pg,
                                          &bars.kv_full[st]);
                    }
                }
                pg = next;
            }
            // V rows past the sequence's end may hold anything, and 0 * inf is not 0
            if (ok && nt && j1 * KEYS > n) {
                const uint32_t x = 2 * nt - 1, st = x % ST;
                if (mbar_wait(&bars.kv_full[st], (x / ST) & 1, &abort_flag)) {
                    const uint32_t r0 = n - (j1 - 1) * KEYS;
                    for (uint32_t i = lane; i < (KEYS - r0) * (HD / 8); i += 32) {
                        const uint32_t r = r0 + i / (HD / 8), c = i % (HD / 8);
                        *reinterpret_cast<uint4 *>(ring + st * G::TILE + (c / 8) * (KEYS * 128) + sw128(r, c & 7)) =
                            make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.clean);
                }
            }
        }
    } else {
        if constexpr (SPLIT)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        else
            asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ------------------------------------------------------ softmax
        const uint32_t s = warp >> 2, t = tid & 127;
        if (s == 0 || two) {
            // are there holes among the slots?  (then the softmax looks each tile's pages up)
            bool hole = false;
            for (uint32_t x = (j0 * KEYS >> a.page_shift) + t; ((uint64_t)x << a.page_shift) < min(n, j1 * KEYS); x += 128)
                hole |= a.page(b, x) < 0;
            if (hole) s_hole[s] = 1;
            // queries, all of a thread's 16-byte chunks in flight; a negative scale goes
            // into their sign, so that the largest score has the largest weight
            uint8_t *sq = smem + s * G::Q;
            constexpr int CH = HD / 8, W = SPLIT ? 2 : 1, BATCH = SPLIT ? 8 : CH;  // chunks of 8 values a row
            const uint32_t flip = q.scale < 0.f ? 0x80008000u : 0u;
            const uint32_t tok0 = row0 / q.group, rem0 = row0 - tok0 * q.group + s * 128;
            const TQ *qb = reinterpret_cast<const TQ *>(q.q) + (size_t)(first + tok0) * q.q_stride +
                           (size_t)kvh * q.group * HD;
            // local row r: token tok0 + (rem0 + r) / group
            auto row_of = [&](uint32_t r, uint32_t &tok, uint32_t &head) {
                const uint32_t x = rem0 + r;
                tok = q.div_group(x);
                head = x - tok * q.group;
            };
#pragma unroll 1
            for (uint32_t i0 = t; i0 < 128 * CH; i0 += 128 * BATCH) {
                uint4 raw[BATCH][W];
#pragma unroll
                for (int e = 0; e < BATCH; e++) {
                    const uint32_t i = i0 + e * 128, r = i / CH, c = i % CH;
                    uint32_t tok, head;
                    row_of(r, tok, head);
                    const bool in = s * 128 + r < my_rows;
                    const uint4 *src = reinterpret_cast<const uint4 *>(qb + (size_t)tok * q.q_stride + head * HD + c * 8);
#pragma unroll
                    for (int w = 0; w < W; w++) raw[e][w] = in ? src[w] : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < BATCH; e++) {
                    const uint32_t i = i0 + e * 128, r = i / CH, c = i % CH;
                    const uint32_t at = (c / 8) * (128 * 128) + sw128(r, c & 7);
                    uint4 h = raw[e][0];
                    if (SPLIT) {
                        const uint4 g = raw[e][W - 1];
                        uint32_t lo[4];
                        split_pack<TC>(__uint_as_float(raw[e][0].x), __uint_as_float(raw[e][0].y), h.x, lo[0]);
                        split_pack<TC>(__uint_as_float(raw[e][0].z), __uint_as_float(raw[e][0].w), h.y, lo[1]);
                        split_pack<TC>(__uint_as_float(g.x), __uint_as_float(g.y), h.z, lo[2]);
                        split_pack<TC>(__uint_as_float(g.z), __uint_as_float(g.w), h.w, lo[3]);
                        *reinterpret_cast<uint4 *>(sq + 128 * HD * 2 + at) =
                            make_uint4(lo[0] ^ flip, lo[1] ^ flip, lo[2] ^ flip, lo[3] ^ flip);
                    }
                    *reinterpret_cast<uint4 *>(sq + at) = make_uint4(h.x ^ flip, h.y ^ flip, h.z ^ flip, h.w ^ flip);
                }
            }
            fence_async_smem();
            mbar_arrive(&bars.q_full[s]);
            group_sync<128>(s + 1);
            hole = s_hole[s];

            const uint32_t rr = row0 + s * 128 + t;
            const bool live = s * 128 + t < my_rows;
            uint32_t lo = 0, hi = 0;
            if (live) q.range(pos0 + (int)(rr / q.group), n, lo, hi);
            // a tile inside every row's range needs no mask
            const uint32_t all_lo = __reduce_max_sync(~0u, live ? lo : 0u);
            const uint32_t all_hi = __reduce_min_sync(~0u, live ? hi : 0xFFFFFFFFu);
            const float c2 = fmaxf(fabsf(q.scale) * 1.4426950408889634f, 1e-30f);
            const float grow = 8.f / c2;
            const uint32_t lane_base = (warp & 3) << 21;  // this warp's TMEM lanes
            const uint32_t ts = tmem + s * 128 + lane_base, to = tmem + 256 + s * 128 + lane_base;
            float m = -INFINITY, l = 0.f;
            float osum[SPLIT ? HD : 1];  // fp32 queries: the output so far
#pragma unroll
            for (int i = 0; i < (SPLIT ? HD : 1); i++) osum[i] = 0.f;
            bool ok = true;
            for (uint32_t j = 0; j < nt; j++) {
                if (!mbar_wait(&bars.s_full[s], j & 1, &abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t k0 = (j0 + j) * KEYS;
                const bool masked = hole || k0 < all_lo || k0 + KEYS > all_hi;
                uint32_t gone = 0;  // 16-slot units on a hole
                if (hole) {
                    const uint32_t slot = k0 + (lane & 7) * 16;
                    gone = __ballot_sync(~0u, lane < 8 && slot < n && a.page(b, slot >> a.page_shift) < 0);
                }
                const int rlo = (int)lo - (int)k0, rhi = (int)hi - (int)k0;
                f32x2 sum = pack2(0.f, 0.f);
                if constexpr (SPLIT) {
                    float x[32], mt = -INFINITY;
                    auto scores = [&](int ch) {  // 32 scores, masked
                        tmem_ld32(ts + ch * 32, x);
                        tmem_wait_ld();
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 32; i++) {
                                const int c = ch * 32 + i;
                                if (c < rlo || c >= rhi || ((gone >> (c / 16)) & 1u)) x[i] = -INFINITY;
                            }
                        }
                    };
#pragma unroll
                    for (int ch = 0; ch < 4; ch++) {
                        scores(ch);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) mt = max3(mt, x[i], x[i + 1]);
                    }
                    if (j > 0) {  // the last tile's O is complete: S was issued behind it
#pragma unroll
                        for (int ch = 0; ch < HD / 32; ch++) {
                            tmem_ld32(to + ch * 32, x);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) osum[ch * 32 + i] += x[i];
                        }
                    }
                    if (mt > m + grow) {
                        const float f = ex2((m - mt) * c2);  // 0 from -inf
                        m = mt;
                        l *= f;
#pragma unroll
                        for (int i = 0; i < HD; i++) osum[i] *= f;
                    }
                    const float mc = LIFT - (m == -INFINITY ? 0.f : m) * c2;
                    const f32x2 cc = pack2(c2, c2), nm = pack2(mc, mc);
                    // P takes the place of its own 32 scores: 16 columns hi, 16 lo
#pragma unroll
                    for (int ch = 0; ch < 4; ch++) {
                        scores(ch);
                        uint32_t ph[16], pl[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float u, v;
                            unpack2(fma2(pack2(x[e], x[e + 1]), cc, nm), u, v);
                            u = ex2(u);
                            v = ex2(v);
                            sum = add2(sum, pack2(u, v));
                            split_pack<TC>(u, v, ph[e / 2], pl[e / 2]);
                        }
                        tmem_st16(ts + ch * 32, ph);
                        tmem_st16(ts + ch * 32 + 16, pl);
                        if (ch & 1) {
                            tmem_wait_st();
                            tc_fence_before();
                            mbar_arrive(&bars.p_full[s][ch / 2]);
                        }
                    }
                } else {
                    float x[128];
                    tmem_ld32(ts, x);
                    tmem_ld32(ts + 32, x + 32);
                    tmem_wait_ld();
                    tmem_ld32(ts + 64, x + 64);
                    tmem_ld32(ts + 96, x + 96);
                    float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int i = 4; i < 60; i += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], x[i + e], x[i + 4 + e]);
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e] = fmaxf(mx[e], x[60 + e]);
                    tmem_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 128; i++)
                            if (i < rlo || i >= rhi || ((gone >> (i / 16)) & 1u)) x[i] = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 4; e++) mx[e] = -INFINITY;  // over the visible ones only
#pragma unroll
                        for (int i = 0; i < 64; i += 8)
#pragma unroll
                            for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], x[i + e], x[i + 4 + e]);
                    }
#pragma unroll
                    for (int i = 64; i < 128; i += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], x[i + e], x[i + 4 + e]);
                    const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    const bool up = mt > m + grow || (m == -INFINITY && mt > m);
                    if (__any_sync(~0u, up)) {
                        const float mn = up ? mt : m;
                        const float f = up ? ex2((m - mn) * c2) : 1.f;  // 0 from -inf
                        m = mn;
                        l *= f;
                        if (j > 0) {  // O is complete: S was issued behind it
#pragma unroll 1
                            for (int i = 0; i < HD / 16; i++) {
                                float ov[16];
                                asm volatile(
                                    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
                                    "%14,%15}, [%16];"
                                    : "=f"(ov[0]), "=f"(ov[1]), "=f"(ov[2]), "=f"(ov[3]), "=f"(ov[4]), "=f"(ov[5]),
                                      "=f"(ov[6]), "=f"(ov[7]), "=f"(ov[8]), "=f"(ov[9]), "=f"(ov[10]), "=f"(ov[11]),
                                      "=f"(ov[12]), "=f"(ov[13]), "=f"(ov[14]), "=f"(ov[15])
                                    : "r"(to + i * 16));
                                tmem_wait_ld();
                                uint32_t r[16];
#pragma unroll
                                for (int e = 0; e < 16; e++) r[e] = __float_as_uint(ov[e] * f);
                                tmem_st16(to + i * 16, r);
                            }
                        }
                    }
                    const float mm = m == -INFINITY ? 0.f : m;
                    const float mc = -mm * c2;
                    const f32x2 cc = pack2(c2, c2), nm = pack2(mc, mc);
#pragma unroll
                    for (int half = 0; half < 2; half++) {
#pragma unroll
                        for (int q16 = 0; q16 < 2; q16++) {
                            uint32_t ph[16];
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                const int i = half * 64 + q16 * 32 + e;
                                float u, v;
                                unpack2(fma2(pack2(x[i], x[i + 1]), cc, nm), u, v);
                                u = ex2(u);
                                v = ex2(v);
                                sum = add2(sum, pack2(u, v));
                                ph[e / 2] = Pair<TC>::pack(u, v);
                            }
                            tmem_st16(ts + half * 32 + q16 * 16, ph);
                        }
                        tmem_wait_st();
                        tc_fence_before();
                        mbar_arrive(&bars.p_full[s][half]);
                    }
                }
                float u, v;
                unpack2(sum, u, v);
                l += u + v;
            }
            // ---------------------------------------------------- output
            float inv = 0.f, lse2 = -INFINITY;
            if (nt && ok) {
                ok = mbar_wait(&bars.o_full[s], 0, &abort_flag);
                tc_fence_after();
                inv = l == 0.f ? 0.f : 1.f / l;
                if (l != 0.f) lse2 = m * c2 - LIFT + log2f(l);
            }
            ok = group_all<128>(s + 1, ok);
            const bool direct = o.plan.many_splits == 1;
            uint32_t tok, head;
            row_of(t, tok, head);
            tok += first + tok0;
            head += kvh * q.group;
            const size_t part0 = (size_t)split * a.n_tok * q.heads;
            if (ok && live) {
                if (direct && o.lse) o.lse[(size_t)tok * q.heads + head] = lse2 * 0.6931471805599453f;
                if (!direct) o.many_lse[part0 + (size_t)tok * q.heads + head] = lse2;
            }
            // rows leave through shared memory (this stream's queries are done with), 128
            // bytes of each at a time, so that stores cover whole lines
            auto leave = [&](auto *dst0, size_t stride, size_t row_step) {
                using TO = typename std::remove_pointer<decltype(dst0)>::type;
                constexpr int COLS = 128 / sizeof(TO);
#pragma unroll(SPLIT ? HD : 1)
                for (int c0 = 0; c0 < HD; c0 += COLS) {
                    float ov[COLS];
#pragma unroll
                    for (int i = 0; i < COLS; i += 32) tmem_ld32(to + c0 + i, ov + i);
                    tmem_wait_ld();
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int i = 0; i < COLS; i++) ov[i] += osum[c0 + i];
                    }
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        uint4 u;
                        if constexpr (sizeof(TO) == 4) {
                            const float *w = ov + c * 4;
                            u = make_uint4(__float_as_uint(nt ? w[0] * inv : 0.f), __float_as_uint(nt ? w[1] * inv : 0.f),
                                           __float_as_uint(nt ? w[2] * inv : 0.f), __float_as_uint(nt ? w[3] * inv : 0.f));
                        } else {
                            const float *w = ov + c * 8;
                            u = make_uint4(Pair<TO>::pack(w[0] * inv, w[1] * inv), Pair<TO>::pack(w[2] * inv, w[3] * inv),
                                           Pair<TO>::pack(w[4] * inv, w[5] * inv), Pair<TO>::pack(w[6] * inv, w[7] * inv));
                            if (!nt) u = make_uint4(0, 0, 0, 0);  // no tile: tensor memory holds anything
                        }
                        *reinterpret_cast<uint4 *>(sq + sw128(t, c)) = u;
                    }
                    group_sync<128>(s + 1);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint32_t r = e * 16 + t / 8, c = t & 7;
                        uint32_t tk, hd;
                        row_of(r, tk, hd);
                        if (s * 128 + r < my_rows)
                            *reinterpret_cast<uint4 *>(dst0 + (size_t)(first + tok0 + tk) * stride +
                                                       (size_t)(kvh * q.group + hd) * row_step + c0 + c * (16 / sizeof(TO))) =
                                *reinterpret_cast<const uint4 *>(sq + sw128(r, c));
                    }
                    group_sync<128>(s + 1);
                }
            };
            if (ok && direct) leave(reinterpret_cast<TQ *>(o.out), o.out_stride, (size_t)HD);
            if (ok && !direct && nt) leave(o.many_o + part0 * HD, (size_t)q.heads * HD, (size_t)HD);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) give_up(tid == 0);
    if (warp == 8) {
        tc_fence_after();
        tmem_free512(tmem);
    }
}

template <typename TQ, typename TC, int HD>
int launch_many(const AttnPagedCall &c, const AttnOut &o, cudaStream_t s) {
    using G = ManyGeo<HD, std::is_same<TQ, float>::value>;
    const uint32_t box = c.a.page_size < KEYS ? c.a.page_size : KEYS;
    CUtensorMap mk, mv;
    int rc = make_page_map(&mk, c.a.k, c.a, HD, c.cache_type, box, 1);
    if (rc == CUQ_OK) rc = make_page_map(&mv, c.a.v, c.a, HD, c.cache_type, box, 1);
    if (rc) return rc;
    auto kern = attn_many_kernel<TQ, TC, HD>;
    static std::atomic<uint64_t> allowed;
    CUQ_CUDA_TRY(allow_smem(kern, G::SMEM, allowed));
    CUQ_CUDA_TRY(launch_maybe_pdl(kern, dim3(c.a.kv_heads * o.plan.many_tiles, o.plan.many_splits), dim3(NT), G::SMEM, s,
                                  true, c.a, c.q, o, mk, mv));
    return CUQ_OK;
}

}  // namespace

int launch_attention_many(const AttnPagedCall &c, const AttnOut &o, cudaStream_t s) {
    if (c.type == CUQ_F32)
        return c.hd == 64 ? launch_many<float, __half, 64>(c, o, s) : launch_many<float, __half, 128>(c, o, s);
    if (c.type == CUQ_F16)
        return c.hd == 64 ? launch_many<__half, __half, 64>(c, o, s) : launch_many<__half, __half, 128>(c, o, s);
    return c.hd == 64 ? launch_many<__nv_bfloat16, __nv_bfloat16, 64>(c, o, s)
                      : launch_many<__nv_bfloat16, __nv_bfloat16, 128>(c, o, s);
}

int attention_many_gave_up(cudaStream_t s, unsigned int *n) { return gave_up_count(s, n); }

}  // namespace cuq
