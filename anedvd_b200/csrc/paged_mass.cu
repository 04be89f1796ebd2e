// paged_mass.cu -- the attention weight that each cached slot gathers:
//   mass[b][kv head][s] = decay mass + sum over queries and heads of exp(scale q k_s - lse).
//
// With lse known this is a column sum of a softmax, so the product is taken the
// other way round: S^T = K Q^T on tcgen05, a slot is a TMEM lane and a thread, and
// the sum over queries stays in that thread's registers: no maximum, no exchange
// between lanes, no atomics, one fixed order.
//
// An item is 256 slots of one KV head of one sequence, two 128-slot streams that
// share the query tiles (128 (token, head) rows).  Persistent CTAs walk items:
//   * warp 17 loads K pages by TMA (a ring of two items);
//   * warps 18-21 gather query rows and their lse into a ring of query tiles; a
//     tile that the next item uses again stays where it is;
//   * warp 16 issues S^T into two TMEM buffers per stream;
//   * warps 0-15 sum 2^(S c - lse log2 e) over the columns, two threads a slot, 64
//     columns each: four warps a scheduler hide one another's waits.
// Few queries: bound by the bytes of K, with only the columns that hold queries
// computed.  Many: by the exponentials (16 a cycle and SM); then the query tiles of
// an item are dealt out over a cluster, whose CTAs' sums are joined in rank order
// through distributed shared memory.  The last 32 queries of 4 sequences up to 16384
// slots (32 heads, 8 KV heads, head_dim 128) take 18.4 us, 3.15 TB/s: six items a CTA of
// 2450 cycles (2048 of them exponentials) and 1200 between two items, after 8700 to
// the first.  2048 queries over 4096 slots (12 heads, 2 KV heads) take 43 us, 2700
// cycles a step of 256 slots x 128 rows.  Six of 16 exponential pairs as polynomials on
// the FMA pipe made it slower (51 us); eight summing warps instead of sixteen, 53 us;
// two items a cluster, one of many queries and one of few, no faster (43 us).  With fp32
// queries the two take 24.1 and 76.8 us.
// The sums of the second case are off by 2.5e-7 of the largest (6e-8 in plain fp32): the
// tensor cores cut the score sums towards zero.  The exponent as (scale s - lse) log2 e,
// whose rounding is smaller, changed nothing and took 44 us.
#include "paged_tc.cuh"

namespace cuq {

using namespace ptc;

namespace {

constexpr int NT = 704;  // warps 0-15 sums, 16 MMA, 17 TMA, 18-21 query tiles
constexpr int ITEM = 256;         // slots
constexpr int LISTED = 64;        // items of a CTA that are worked out at its start
constexpr int MAX_SEQS = 1024;    // sequences of one launch (the table in shared memory)

template <int HD, bool SPLIT>
struct MassGeo {
    static constexpr int CB = HD / 64;
    static constexpr int TILE = 128 * HD * 2;
    static constexpr int Q = TILE * (SPLIT ? 2 : 1);
    static constexpr int UNITS = 6;  // tiles of shared memory, dealt out to keys and queries (see KQ)
    static constexpr int SMEM = 1024 + UNITS * TILE + MAX_SEQS * 16;
};

// How the tiles are dealt out: few queries stay while keys stream, two items of
// keys (4 tiles) and 2 of queries; many stream over one item's keys, 2 and 4.
// A query tile of fp32 takes two.
struct KQ {
    uint32_t k_items, q_log;  // stages: items of keys, log2 of query tiles
    __device__ __forceinline__ KQ(bool near, bool split) : k_items(near ? 2 : 1), q_log((near ? 1 : 2) - (split ? 1 : 0)) {}
    __device__ __forceinline__ uint32_t k_stage(uint32_t x) const { return k_items == 2 ? x & 1 : 0; }
    __device__ __forceinline__ uint32_t k_phase(uint32_t x) const { return (k_items == 2 ? x >> 1 : x) & 1; }
    __device__ __forceinline__ uint32_t q_stage(uint32_t x) const { return x & ((1u << q_log) - 1); }
    __device__ __forceinline__ uint32_t q_phase(uint32_t x) const { return (x >> q_log) & 1; }
    __device__ __forceinline__ bool q_reused(uint32_t x) const { return x >= (1u << q_log); }
};

struct MassArgs {
    PagedArgs a;
    PagedQuery q;
    float *mass;
    size_t mass_stride;
    const float *lse;
    uint32_t last_q, seq0, seqs;  // this launch's sequences
    float decay;
};

// One item as every role sees it.
struct Item {
    uint32_t b, h, k0, n;        // sequence, KV head, first slot, slots of the sequence
    uint32_t first;              // first token row
    int pos0;                    // slot of token 0
    uint32_t i0, tq;             // tokens [i0, tq) count
    uint32_t qt0, steps;         // first query tile and this CTA's number of them
};

template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(NT, 1) mass_kernel(MassArgs p, const __grid_constant__ CUtensorMap mk) {
    constexpr bool SPLIT = std::is_same<TQ, float>::value;
    using G = MassGeo<HD, SPLIT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t k_full[2], k_empty[2], q_full[4], q_empty[4], s_full[2][2], s_empty[2][2];
    // -lse log2 e of the rows of query tile i at [i % 8]; -inf where a row counts
    // nothing.  A tile is written once the products of the tile 4 (or fewer) before it
    // are done, and those are at most two steps ahead of the sums: 4 + 2 < 8 tiles.
    __shared__ float s_nlse[8][128];
    __shared__ float s_red[2][ITEM];
    __shared__ const void *s_row[2][128];  // the rows of a query tile; null where a row counts nothing
    __shared__ Item s_items[LISTED];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t most = p.last_q ? min(p.last_q, p.a.max_q) : p.a.max_q;
    const bool near = (uint64_t)most * p.q.group <= 128;
    const KQ ring(near, SPLIT);
    uint8_t *kring = smem, *qring = smem + 2 * ring.k_items * G::TILE;
    // per sequence: items of the sequences up to it (per KV head), slots, first token row, tokens
    uint4 *s_seq = reinterpret_cast<uint4 *>(smem + G::UNITS * G::TILE);
    const PagedArgs &a = p.a;
    const PagedQuery &q = p.q;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = warp_index();
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));

    griddep_wait();
    if (warp == 16) tmem_alloc512(&tmem_slot);
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            for (int s = 0; s < 2; s++) {
                mbar_init(&s_full[s][i], 2);
                mbar_init(&s_empty[s][i], 256);
            }
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(&q_full[i], 128);
            mbar_init(&q_empty[i], 1);
        }
        mbar_init_fence();
    }
    // the sequence table: running sums of ceil(len / 256)
    if (warp == 0) {
        uint32_t run = 0;
        for (uint32_t s0 = 0; s0 < p.seqs; s0 += 32) {
            const uint32_t i = s0 + lane;
            uint32_t len = 0, nq = 0, first = 0;
            if (i < p.seqs) {
                len = a.len(p.seq0 + i);
                nq = a.tokens(p.seq0 + i, first);
            }
            uint32_t v = (len + ITEM - 1) / ITEM;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t up = __shfl_up_sync(~0u, v, d);
                if (lane >= (uint32_t)d) v += up;
            }
            if (i < p.seqs) s_seq[i] = make_uint4(run + v, len, first, nq);
            run += __shfl_sync(~0u, v, 31);
        }
    }
    __syncthreads();
    const uint32_t run = s_seq[p.seqs - 1].x;
    const uint32_t total = run * a.kv_heads;
    // few queries: neighbouring items, which share their query tile; else dealt out,
    // since a causal mask gives the first slots the most queries
    const uint32_t cluster = blockIdx.x / ranks, clusters = gridDim.x / ranks;
    const uint32_t per = near ? (total + clusters - 1) / clusters : 1;
    const uint32_t x0 = cluster * per, x1 = near ? min(total, x0 + per) : total, xs = near ? 1 : clusters;

    auto find = [&](uint32_t x, Item &t) {
        // sequence-major: find the sequence in the table, then its KV head and slots
        uint32_t lo = 0, hi = p.seqs - 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if ((uint64_t)s_seq[mid].x * a.kv_heads > x)
                hi = mid;
            else
                lo = mid + 1;
        }
        const uint4 seq = s_seq[lo];
        const uint32_t base = lo ? s_seq[lo - 1].x : 0, cnt = seq.x - base, y = x - base * a.kv_heads;
        t.b = p.seq0 + lo;
        t.h = y / cnt;
        t.k0 = (y % cnt) * ITEM;
        t.n = seq.y;
        t.first = seq.z;
        const uint32_t nq = seq.w;
        t.pos0 = (int)t.n - (int)nq;
        t.tq = min(nq, a.max_q);
        t.i0 = (p.last_q && nq > p.last_q) ? nq - p.last_q : 0;
        if (t.pos0 < 0) t.i0 = max(t.i0, (uint32_t)-t.pos0);  // tokens before slot 0 see nothing
        t.qt0 = t.steps = 0;
        if (t.i0 < t.tq) {
            uint32_t ia = t.i0, ib = t.tq;
            if (q.causal) {
                ia = (uint32_t)max((int)ia, (int)t.k0 - t.pos0);
                if (q.window) ib = (uint32_t)max(0ll, min((long long)ib, (long long)t.k0 + ITEM - 1 + q.window - t.pos0));
            }
            if (ia < ib) {
                t.qt0 = (ia - t.i0) * q.group / 128;
                const uint32_t tiles = ((ib - t.i0) * q.group + 127) / 128 - t.qt0;
                t.steps = tiles > rank ? (tiles - rank + ranks - 1) / ranks : 0;
            }
        }
    };
    for (uint32_t i = tid; i < (uint32_t)LISTED && x0 + (uint64_t)i * xs < x1; i += NT) find(x0 + i * xs, s_items[i]);
    auto item = [&](uint32_t x, Item &t) {
        const uint32_t i = near ? x - x0 : (x - x0) / xs;
        if (i < (uint32_t)LISTED)
            t = s_items[i];
        else
            find(x, t);
    };
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // rows of query tile qt of item t
    auto tile_rows = [&](const Item &t, uint32_t qt) { return min(128u, (t.tq - t.i0) * q.group - qt * 128); };

    if (warp == 16) {
        // ------------------------------------------------------ MMA issuer
        {
            const uint32_t leader = elect_one();
            const uint32_t ka = smem_u32(kring), qa = smem_u32(qring);
            uint32_t kx = 0, qx = 0, st = 0, ob = ~0u, oh = 0, oq = 0;
            bool ok = true, held = false;
            for (uint32_t x = x0; ok && x < x1; x += xs) {
                Item t;
                item(x, t);
                if (!t.steps) continue;
                ok = mbar_wait(&k_full[ring.k_stage(kx)], ring.k_phase(kx), &abort_flag);
                for (uint32_t e = 0; ok && e < t.steps; e++, st++) {
                    const uint32_t qt = t.qt0 + rank + e * ranks;
                    if (!held || t.b != ob || t.h != oh || qt != oq) {
                        if (held) {
                            umma_commit(leader, &q_empty[ring.q_stage(qx)]);
                            qx++;
                        }
                        held = true;
                        ob = t.b, oh = t.h, oq = qt;
                        ok = mbar_wait(&q_full[ring.q_stage(qx)], ring.q_phase(qx), &abort_flag);
                        if (!ok) break;
                    }
                    const uint32_t nr = tile_rows(t, qt), id = idesc<TC>(128, (nr + 31) / 32 * 32, false);
                    const uint32_t buf = st & 1, qb = qa + ring.q_stage(qx) * G::Q;
                    for (uint32_t s = 0; s < 2; s++) {
                        if (st >= 2 && !mbar_wait(&s_empty[s][buf], ((st >> 1) - 1) & 1, &abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t kb = ka + (ring.k_stage(kx) * 2 + s) * G::TILE;
#pragma unroll
                        for (int part = 0; part < (SPLIT ? 2 : 1); part++)
#pragma unroll
                            for (int ks = 0; ks < HD / 16; ks++) {
                                const uint32_t off = (ks / 4) * (128 * 128) + (ks % 4) * 32;
                                umma_ss(leader, tmem + (s * 2 + buf) * 128, sdesc_sw128(kb + off, 16, 1024),
                                        sdesc_sw128(qb + (SPLIT ? 1 - part : 0) * G::TILE + off, 16, 1024), id,
                                        part | ks ? 1u : 0u);  // the low parts first
                            }
                        umma_commit(leader, &s_full[s][buf]);
                        if (leader) mbar_arrive(&s_full[s][buf]);  // hands on what the query warps wrote to s_nlse
                    }
                }
                if (ok) umma_commit(leader, &k_empty[ring.k_stage(kx)]);
                kx++;
            }
            if (ok && held) umma_commit(leader, &q_empty[ring.q_stage(qx)]);
        }
    } else if (warp == 17) {
        // ------------------------------------------------------ TMA: K pages
        const uint32_t box = min(a.page_size, 128u), nbox = ITEM / box;
        uint32_t kx = 0;
        bool ok = true;
        for (uint32_t x = x0; ok && x < x1; x += xs) {
            Item t;
            item(x, t);
            if (!t.steps) continue;
            const uint32_t st = ring.k_stage(kx), slot = t.k0 + lane * box;
            int pg = (int)a.n_pages;  // outside the pool: zeros
            if (lane < nbox && slot < t.n) {
                pg = a.page(t.b, slot >> a.page_shift);
                if (pg < 0) pg = (int)a.n_pages;
            }
            if (kx >= ring.k_items) ok = mbar_wait(&k_empty[st], ring.k_phase(kx) ^ 1, &abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(&k_full[st], 2 * G::TILE);
            __syncwarp();
            if (lane < nbox) {
                const uint32_t row = lane * box;
                const uint32_t dst = smem_u32(kring) + (st * 2 + row / 128) * G::TILE + (row & 127) * 128;
#pragma unroll
                for (int cb = 0; cb < G::CB; cb++)
                    tma_load_page(dst + cb * (128 * 128), &mk, cb, (int)(slot & (a.page_size - 1)), (int)t.h, pg,
                                  &k_full[st]);
            }
            kx++;
        }
        for (uint32_t i = kx > ring.k_items ? kx - ring.k_items : 0; ok && i < kx; i++)  // drain
            ok = mbar_wait(&k_empty[ring.k_stage(i)], ring.k_phase(i), &abort_flag);
    } else if (warp >= 18) {
        // ------------------------------------------------------ query tiles
        const uint32_t t128 = tid - 18 * 32;
        uint32_t qx = 0, ob = ~0u, oh = 0, oq = 0;
        bool ok = true, pending = false;
        auto send = [&]() {  // hand over the tile whose copies were issued last
            if (!pending) return;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            fence_async_smem();
            mbar_arrive(&q_full[ring.q_stage(qx - 1)]);
            pending = false;
        };
        for (uint32_t x = x0; ok && x < x1; x += xs) {
            Item t;
            item(x, t);
            for (uint32_t e = 0; ok && e < t.steps; e++) {
                const uint32_t qt = t.qt0 + rank + e * ranks;
                if (qx && t.b == ob && t.h == oh && qt == oq) continue;
                ob = t.b, oh = t.h, oq = qt;
                const uint32_t st = ring.q_stage(qx), nr = tile_rows(t, qt), r0 = t.i0 * q.group + qt * 128;
                // thread r: where row r of the tile lies, and its lse
                float ls = -INFINITY;
                const TQ *src = nullptr;
                if (t128 < nr) {
                    const uint32_t tok = t.first + (r0 + t128) / q.group;
                    const uint32_t head = t.h * q.group + (r0 + t128) % q.group;
                    ls = p.lse[(size_t)tok * q.heads + head];
                    src = reinterpret_cast<const TQ *>(q.q) + (size_t)tok * q.q_stride + (size_t)head * HD;
                }
                constexpr int CH = HD / 8, BATCH = 4;
                uint8_t *dst = qring + st * G::Q;
                if (ring.q_reused(qx) && !mbar_try_wait(&q_empty[st], ring.q_phase(qx) ^ 1)) {
                    send();  // rather than hold the last tile back
                    ok = mbar_wait(&q_empty[st], ring.q_phase(qx) ^ 1, &abort_flag);
                }
                // a row that saw nothing counts nothing, and its products are kept finite
                s_nlse[qx & 7][t128] = ls == -INFINITY ? -INFINITY : -ls * 1.4426950408889634f;
                s_row[qx & 1][t128] = ls == -INFINITY ? nullptr : src;
                ok = group_all<128>(1, ok);
                if (!ok) break;
                // this thread's chunk of rows r1, r1 + 128 / CH, ...
                const uint32_t r1 = t128 / CH, c = t128 % CH;
                if constexpr (!SPLIT) {
#pragma unroll
                    for (int k = 0; k < CH; k++) {
                        const uint32_t r = r1 + k * (128 / CH);
                        const TQ *row = reinterpret_cast<const TQ *>(s_row[qx & 1][r]);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         smem_u32(dst) + (c / 8) * (128 * 128) + sw128(r, c & 7)),
                                     "l"(row ? row + c * 8 : reinterpret_cast<const TQ *>(q.q)), "r"(row ? 16 : 0)
                                     : "memory");
                    }
                    // the tile before this one goes out while this one is on its way
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (pending) {
                        asm volatile("cp.async.wait_group 1;" ::: "memory");
                        fence_async_smem();
                        mbar_arrive(&q_full[ring.q_stage(qx - 1)]);
                    }
                    pending = true;
                } else {
#pragma unroll 1
                    for (int part = 0; part < CH / BATCH; part++) {
                        uint4 raw[BATCH][2];
#pragma unroll
                        for (int k = 0; k < BATCH; k++) {
                            const uint32_t r = r1 + (part * BATCH + k) * (128 / CH);
                            const TQ *row = reinterpret_cast<const TQ *>(s_row[qx & 1][r]);
                            const uint4 *from = reinterpret_cast<const uint4 *>(row + c * 8);
                            raw[k][0] = row ? *from : make_uint4(0, 0, 0, 0);
                            raw[k][1] = row ? from[1] : make_uint4(0, 0, 0, 0);
                        }
#pragma unroll
                        for (int k = 0; k < BATCH; k++) {
                            const uint32_t r = r1 + (part * BATCH + k) * (128 / CH);
                            const uint32_t at = (c / 8) * (128 * 128) + sw128(r, c & 7);
                            const uint4 f = raw[k][0], g = raw[k][1];
                            uint4 hi, lo;
                            split_pack<TC>(__uint_as_float(f.x), __uint_as_float(f.y), hi.x, lo.x);
                            split_pack<TC>(__uint_as_float(f.z), __uint_as_float(f.w), hi.y, lo.y);
                            split_pack<TC>(__uint_as_float(g.x), __uint_as_float(g.y), hi.z, lo.z);
                            split_pack<TC>(__uint_as_float(g.z), __uint_as_float(g.w), hi.w, lo.w);
                            *reinterpret_cast<uint4 *>(dst + at) = hi;
                            *reinterpret_cast<uint4 *>(dst + G::TILE + at) = lo;
                        }
                    }
                }
                if constexpr (SPLIT) {
                    fence_async_smem();
                    mbar_arrive(&q_full[st]);
                }
                qx++;
            }
        }
        send();
        const uint32_t q_tiles = 1u << ring.q_log;
        for (uint32_t i = qx > q_tiles ? qx - q_tiles : 0; ok && i < qx; i++)  // drain
            ok = mbar_wait(&q_empty[ring.q_stage(i)], ring.q_phase(i), &abort_flag);
    } else {
        // ------------------------------------------------------ column sums
        const uint32_t s = warp >> 3, half = (warp >> 2) & 1, t128 = tid & 127;
        const int col0 = (int)half * 64;  // this thread's columns
        const uint32_t ts = tmem + s * 256 + col0 + ((warp & 3) << 21);
        const float c2 = q.scale * 1.4426950408889634f;
        const f32x2 cc = pack2(c2, c2);
        uint32_t qx = 0, st = 0, ob = ~0u, oh = 0, oq = 0, flip = 0;
        bool ok = true, held = false;
        for (uint32_t x = x0; ok && x < x1; x += xs) {
            Item t;
            item(x, t);
            const uint32_t k = t.k0 + s * 128 + t128;       // this thread's slot
            // rows (of those that count) [vlo, vhi) see slot k; all the warp's slots are seen by [wlo, whi)
            const int T = (int)t.tq - (int)t.i0, R = max(T, 0) * (int)q.group;
            int vlo = 0, vhi = R, wlo = 0, whi = R;
            if (q.causal && T > 0) {
                const int at = (int)k - (t.pos0 + (int)t.i0), w0 = at - (int)lane;  // against the first one's slot
                auto row = [&](int i) { return max(0, min(T, i)) * (int)q.group; };
                vlo = row(at);
                wlo = row(w0 + 31);
                if (q.window) {
                    vhi = row(at + (int)q.window);
                    whi = row(w0 + (int)q.window);
                }
            }
            float *const m = p.mass + ((size_t)t.b * a.kv_heads + t.h) * p.mass_stride + k;
            float old = 0.f, sum = 0.f;
            int page_id = -1;  // looked at when the sums are there
            if (half == 0 && k < t.n) {
                page_id = a.pages[(size_t)t.b * a.pages_stride + (k >> a.page_shift)];
                if (ranks == 1 && p.decay != 0.f) old = p.decay * *m;
            }
            for (uint32_t e = 0; e < t.steps; e++, st++) {
                const uint32_t qt = t.qt0 + rank + e * ranks;
                if (!held || t.b != ob || t.h != oh || qt != oq) {
                    if (held) qx++;
                    held = true;
                    ob = t.b, oh = t.h, oq = qt;
                }
                const uint32_t buf = st & 1, nr = tile_rows(t, qt);
                ok = mbar_wait(&s_full[s][buf], (st >> 1) & 1, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                const int r_tile = (int)(qt * 128) + col0, clo = vlo - r_tile, chi = vhi - r_tile;
                const int cols = (int)nr - col0;  // may be none
                const bool masked = wlo > r_tile || whi < r_tile + min(cols, 64);
                const float *nl = s_nlse[qx & 7] + col0;
                f32x2 acc = pack2(0.f, 0.f), acc1 = acc;
#pragma unroll
                for (int ch = 0; ch < 2; ch++) {
                    const int c0 = ch * 32;
                    if (c0 >= cols) break;
                    float w[32];
                    tmem_ld32(ts + buf * 128 + c0, w);
                    tmem_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 l4 = *reinterpret_cast<const float4 *>(nl + c0 + i);
                            float u[4];
                            unpack2(fma2(pack2(w[i], w[i + 1]), cc, pack2(l4.x, l4.y)), u[0], u[1]);
                            unpack2(fma2(pack2(w[i + 2], w[i + 3]), cc, pack2(l4.z, l4.w)), u[2], u[3]);
#pragma unroll
                            for (int k4 = 0; k4 < 4; k4++)
                                u[k4] = (c0 + i + k4 >= clo && c0 + i + k4 < chi) ? u[k4] : -INFINITY;
                            acc = add2(acc, pack2(ex2(u[0]), ex2(u[1])));
                            acc1 = add2(acc1, pack2(ex2(u[2]), ex2(u[3])));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 l4 = *reinterpret_cast<const float4 *>(nl + c0 + i);
                            float u0, u1, u2, u3;
                            unpack2(fma2(pack2(w[i], w[i + 1]), cc, pack2(l4.x, l4.y)), u0, u1);
                            unpack2(fma2(pack2(w[i + 2], w[i + 3]), cc, pack2(l4.z, l4.w)), u2, u3);
                            acc = add2(acc, pack2(ex2(u0), ex2(u1)));
                            acc1 = add2(acc1, pack2(ex2(u2), ex2(u3)));
                        }
                    }
                }
                acc = add2(acc, acc1);
                tc_fence_before();
                mbar_arrive(&s_empty[s][buf]);
                float even, odd;
                unpack2(acc, even, odd);
                sum += even + odd;
            }
            // the second half's sum goes to the first half's thread
            float *red = s_red[flip] + s * 128 + t128;  // the other buffer next time
            flip ^= 1;
            if (half) *red = sum;
            ok = group_all<256>(s + 2, ok);  // the stream's threads go on or stop together
            if (!half) {
                sum = (uint32_t)page_id < a.n_pages ? sum + *red : 0.f;  // a hole gathers nothing
                if (ranks > 1)
                    s_red[1][s * 128 + t128] = sum;
                else if (k < t.n && ok)
                    *m = old + sum;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) give_up(tid == 0);
    if (warp == 16) {
        tc_fence_after();
        tmem_free512(tmem);
    }
    if (ranks > 1) {  // one item per cluster: rank 0 joins the sums in rank order
        cluster_sync();
        if (rank == 0 && tid < ITEM && x0 < x1) {
            Item t;
            item(x0, t);
            const uint32_t k = t.k0 + tid;
            float sum = 0.f;
            for (uint32_t r = 0; r < ranks; r++) sum += peer_load(peer_smem(&s_red[1][tid], r));
            if (k < t.n) {
                float *m = p.mass + ((size_t)t.b * a.kv_heads + t.h) * p.mass_stride + k;
                *m = p.decay == 0.f ? sum : p.decay * *m + sum;
            }
        }
        cluster_sync();
    }
}

template <typename TQ, typename TC, int HD>
int launch_mass(const MassPagedCall &c, int sm_count, cudaStream_t s) {
    using G = MassGeo<HD, std::is_same<TQ, float>::value>;
    CUtensorMap mk;
    int rc = make_page_map(&mk, c.a.k, c.a, HD, c.cache_type, c.a.page_size < 128 ? c.a.page_size : 128, 1);
    if (rc) return rc;
    auto kern = mass_kernel<TQ, TC, HD>;
    static std::atomic<uint64_t> allowed;
    CUQ_CUDA_TRY(allow_smem(kern, G::SMEM, allowed));
    MassArgs p{};
    p.a = c.a;
    p.q = c.q;
    p.mass = c.mass;
    p.mass_stride = c.mass_stride;
    p.lse = c.lse;
    p.last_q = c.last_q;
    p.decay = c.decay;
    const uint64_t tokens = c.last_q && c.last_q < c.a.max_q ? c.last_q : c.a.max_q;
    const uint64_t tiles = (tokens * c.q.group + 127) / 128;
    for (uint32_t seq0 = 0; seq0 < c.a.n_seqs; seq0 += MAX_SEQS) {
        p.seq0 = seq0;
        p.seqs = c.a.n_seqs - seq0 < (uint32_t)MAX_SEQS ? c.a.n_seqs - seq0 : (uint32_t)MAX_SEQS;
        const uint64_t items = (uint64_t)p.seqs * c.a.kv_heads * ((c.a.max_kv + ITEM - 1) / ITEM);
        uint32_t ranks = 1;
        while (ranks < 8 && ranks * 2 <= tiles && items * ranks * 2 <= (uint64_t)sm_count) ranks *= 2;
        const uint64_t want = items * ranks;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(ranks > 1 || want < (uint64_t)sm_count ? want : (uint64_t)sm_count));
        cfg.blockDim = dim3(NT);
        cfg.dynamicSmemBytes = G::SMEM;
        cfg.stream = s;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
        CUQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, mk));
    }
    return CUQ_OK;
}

}  // namespace

int launch_attention_mass(const MassPagedCall &c, int sm_count, cudaStream_t s) {
    if (c.type == CUQ_F32)
        return c.hd == 64 ? launch_mass<float, __half, 64>(c, sm_count, s) : launch_mass<float, __half, 128>(c, sm_count, s);
    if (c.type == CUQ_F16)
        return c.hd == 64 ? launch_mass<__half, __half, 64>(c, sm_count, s)
                          : launch_mass<__half, __half, 128>(c, sm_count, s);
    return c.hd == 64 ? launch_mass<__nv_bfloat16, __nv_bfloat16, 64>(c, sm_count, s)
                      : launch_mass<__nv_bfloat16, __nv_bfloat16, 128>(c, sm_count, s);
}

int attention_mass_gave_up(cudaStream_t s, unsigned int *n) { return gave_up_count(s, n); }

}  // namespace cuq
