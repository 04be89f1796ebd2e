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
//   * warp 9 loads K pages by TMA (a ring of two items);
//   * warps 10-13 gather query rows and their lse into a ring of query tiles; a
//     tile that the next item uses again stays where it is;
//   * one lane of warp 8 issues S^T into two TMEM buffers per stream;
//   * warps 0-3 and 4-7 sum 2^(S c - lse log2 e) over the columns.
// Few queries: bound by the bytes of K, with only the columns that hold queries
// computed.  Many: by the exponentials (16 a cycle and SM); then the query tiles of
// an item are dealt out over a cluster, whose CTAs' sums are joined in rank order
// through distributed shared memory.
#include "paged_tc.cuh"

namespace cuq {

using namespace ptc;

namespace {

__device__ int g_timeout;

constexpr int NT = 448;
constexpr int ITEM = 256;         // slots
constexpr int MAX_SEQS = 1024;    // sequences of one launch (the table in shared memory)

template <int HD, bool SPLIT>
struct MassGeo {
    static constexpr int CB = HD / 64;
    static constexpr int TILE = 128 * HD * 2;
    static constexpr int Q = TILE * (SPLIT ? 2 : 1);
    static constexpr int QST = (HD == 128 ? 2 : 4) / (SPLIT ? 2 : 1);
    static constexpr int SMEM = 1024 + 4 * TILE + QST * Q + MAX_SEQS * 16;
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
    constexpr int QST = G::QST;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t k_full[2], k_empty[2], q_full[QST], q_empty[QST], s_full[2][2], s_empty[2][2];
    __shared__ float s_nlse[QST][128];  // -lse log2 e; -inf where a row counts nothing
    __shared__ float s_red[ITEM];
    __shared__ uint32_t s_scan[NT / 32], tmem_slot;
    __shared__ int abort_flag;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *kring = smem, *qring = smem + 4 * G::TILE;
    // per sequence: items of the sequences up to it (per KV head), slots, first token row, tokens
    uint4 *s_seq = reinterpret_cast<uint4 *>(qring + QST * G::Q);
    const PagedArgs &a = p.a;
    const PagedQuery &q = p.q;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = warp_index();
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));

    if (warp == 8) tmem_alloc512(&tmem_slot);
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            for (int s = 0; s < 2; s++) {
                mbar_init(&s_full[s][i], 1);
                mbar_init(&s_empty[s][i], 128);
            }
        }
        for (int i = 0; i < QST; i++) {
            mbar_init(&q_full[i], 128);
            mbar_init(&q_empty[i], 1 + 256);
        }
        mbar_init_fence();
    }
    // the item table: running sums of ceil(len / 256)
    uint32_t run = 0;
    for (uint32_t s0 = 0; s0 < p.seqs; s0 += NT) {
        const uint32_t i = s0 + tid;
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
        if (lane == 31) s_scan[warp] = v;
        __syncthreads();
        uint32_t before = run;
        for (uint32_t w = 0; w < NT / 32; w++) {
            if (w < warp) before += s_scan[w];
            run += s_scan[w];
        }
        if (i < p.seqs) s_seq[i] = make_uint4(before + v, len, first, nq);
        __syncthreads();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t total = run * a.kv_heads;
    // few queries: neighbouring items, which share their query tile; else dealt out,
    // since a causal mask gives the first slots the most queries
    const uint32_t cluster = blockIdx.x / ranks, clusters = gridDim.x / ranks;
    const uint32_t most = p.last_q ? min(p.last_q, a.max_q) : a.max_q;
    const bool near = (uint64_t)most * q.group <= 128;
    const uint32_t per = near ? (total + clusters - 1) / clusters : 1;
    const uint32_t x0 = cluster * per, x1 = near ? min(total, x0 + per) : total, xs = near ? 1 : clusters;

    auto item = [&](uint32_t x, Item &t) {
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
    // rows of query tile qt of item t
    auto tile_rows = [&](const Item &t, uint32_t qt) { return min(128u, (t.tq - t.i0) * q.group - qt * 128); };

    if (warp == 8) {
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
                ok = mbar_wait(&k_full[kx & 1], (kx >> 1) & 1, &abort_flag);
                for (uint32_t e = 0; ok && e < t.steps; e++, st++) {
                    const uint32_t qt = t.qt0 + rank + e * ranks;
                    if (!held || t.b != ob || t.h != oh || qt != oq) {
                        if (held) {
                            umma_commit(leader, &q_empty[qx % QST]);
                            qx++;
                        }
                        held = true;
                        ob = t.b, oh = t.h, oq = qt;
                        ok = mbar_wait(&q_full[qx % QST], (qx / QST) & 1, &abort_flag);
                        if (!ok) break;
                    }
                    const uint32_t nr = tile_rows(t, qt), id = idesc<TC>(128, (nr + 31) / 32 * 32, false);
                    const uint32_t buf = st & 1, qb = qa + (qx % QST) * G::Q;
                    for (uint32_t s = 0; s < 2; s++) {
                        if (st >= 2 && !mbar_wait(&s_empty[s][buf], ((st >> 1) - 1) & 1, &abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t kb = ka + ((kx & 1) * 2 + s) * G::TILE;
#pragma unroll
                        for (int part = 0; part < (SPLIT ? 2 : 1); part++)
#pragma unroll
                            for (int ks = 0; ks < HD / 16; ks++) {
                                const uint32_t off = (ks / 4) * (128 * 128) + (ks % 4) * 32;
                                umma_ss(leader, tmem + (s * 2 + buf) * 128, sdesc_sw128(kb + off, 16, 1024),
                                        sdesc_sw128(qb + part * G::TILE + off, 16, 1024), id, part | ks ? 1u : 0u);
                            }
                        umma_commit(leader, &s_full[s][buf]);
                    }
                }
                if (ok) umma_commit(leader, &k_empty[kx & 1]);
                kx++;
            }
            if (ok && held) umma_commit(leader, &q_empty[qx % QST]);
        }
    } else if (warp == 9) {
        // ------------------------------------------------------ TMA: K pages
        const uint32_t box = min(a.page_size, 128u), nbox = ITEM / box;
        uint32_t kx = 0;
        bool ok = true;
        for (uint32_t x = x0; ok && x < x1; x += xs) {
            Item t;
            item(x, t);
            if (!t.steps) continue;
            const uint32_t st = kx & 1, slot = t.k0 + lane * box;
            int pg = (int)a.n_pages;  // outside the pool: zeros
            if (lane < nbox && slot < t.n) {
                pg = a.page(t.b, slot >> a.page_shift);
                if (pg < 0) pg = (int)a.n_pages;
            }
            if (kx >= 2) ok = mbar_wait(&k_empty[st], ((kx >> 1) - 1) & 1, &abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(&k_full[st], 2 * G::TILE);
            __syncwarp();
            if (lane < nbox) {
                const uint32_t row = lane * box;
                const uint32_t dst = smem_u32(kring) + (st * 2 + row / 128) * G::TILE + (row & 127) * 128;
#pragma unroll
                for (int cb = 0; cb < G::CB; cb++)
                    tma_load_page(dst + cb * (128 * 128), &mk, cb * 64, (int)(slot & (a.page_size - 1)), (int)t.h, pg,
                                  &k_full[st]);
            }
            kx++;
        }
        for (uint32_t i = kx > 2 ? kx - 2 : 0; ok && i < kx; i++)  // drain
            ok = mbar_wait(&k_empty[i & 1], (i >> 1) & 1, &abort_flag);
    } else if (warp >= 10) {
        // ------------------------------------------------------ query tiles
        const uint32_t t128 = tid - 320;
        uint32_t qx = 0, ob = ~0u, oh = 0, oq = 0;
        bool ok = true;
        for (uint32_t x = x0; ok && x < x1; x += xs) {
            Item t;
            item(x, t);
            for (uint32_t e = 0; ok && e < t.steps; e++) {
                const uint32_t qt = t.qt0 + rank + e * ranks;
                if (qx && t.b == ob && t.h == oh && qt == oq) continue;
                ob = t.b, oh = t.h, oq = qt;
                const uint32_t st = qx % QST, nr = tile_rows(t, qt), r0 = t.i0 * q.group + qt * 128;
                const uint32_t tok0 = r0 / q.group, rem0 = r0 - tok0 * q.group;  // row r: (rem0 + r) / group tokens on
                auto row_of = [&](uint32_t r, uint32_t &tok, uint32_t &head) {
                    const uint32_t y = rem0 + r;
                    tok = q.div_group(y);
                    head = y - tok * q.group;
                };
                const TQ *qb = reinterpret_cast<const TQ *>(q.q) + (size_t)(t.first + tok0) * q.q_stride +
                               (size_t)t.h * q.group * HD;
                float ls = -INFINITY;
                if (t128 < nr) {
                    uint32_t tok, head;
                    row_of(t128, tok, head);
                    ls = __ldg(p.lse + (size_t)(t.first + tok0 + tok) * q.heads + t.h * q.group + head);
                }
                // all of a thread's 16-byte chunks in flight, before the wait for the stage
                constexpr int CH = HD / 8, W = SPLIT ? 2 : 1, BATCH = SPLIT ? CH / 2 : CH;
                uint8_t *dst = qring + st * G::Q;
#pragma unroll 1
                for (int part = 0; part < CH / BATCH; part++) {
                    uint4 raw[BATCH][W];
#pragma unroll
                    for (int k = 0; k < BATCH; k++) {
                        const uint32_t i = t128 + (part * BATCH + k) * 128, r = i / CH, c = i % CH;
                        uint32_t tok, head;
                        row_of(r, tok, head);
                        const uint4 *src = reinterpret_cast<const uint4 *>(qb + (size_t)tok * q.q_stride + head * HD + c * 8);
#pragma unroll
                        for (int w = 0; w < W; w++) raw[k][w] = r < nr ? __ldg(src + w) : make_uint4(0, 0, 0, 0);
                    }
                    if (part == 0) {
                        if (qx >= (uint32_t)QST) ok = mbar_wait(&q_empty[st], ((qx / QST) - 1) & 1, &abort_flag);
                        // a row that saw nothing counts nothing
                        s_nlse[st][t128] = ls == -INFINITY ? -INFINITY : -ls * 1.4426950408889634f;
                        ok = group_all(1, ok);
                    }
#pragma unroll
                    for (int k = 0; k < BATCH; k++) {
                        const uint32_t i = t128 + (part * BATCH + k) * 128, r = i / CH, c = i % CH;
                        const uint32_t at = (c / 8) * (128 * 128) + sw128(r, c & 7);
                        uint4 hi = raw[k][0], lo = make_uint4(0, 0, 0, 0);
                        if (SPLIT) {
                            const uint4 g = raw[k][W - 1];
                            split_pack<TC>(__uint_as_float(raw[k][0].x), __uint_as_float(raw[k][0].y), hi.x, lo.x);
                            split_pack<TC>(__uint_as_float(raw[k][0].z), __uint_as_float(raw[k][0].w), hi.y, lo.y);
                            split_pack<TC>(__uint_as_float(g.x), __uint_as_float(g.y), hi.z, lo.z);
                            split_pack<TC>(__uint_as_float(g.z), __uint_as_float(g.w), hi.w, lo.w);
                        }
                        // where nothing counts the products are kept finite
                        if (s_nlse[st][r] == -INFINITY) hi = lo = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4 *>(dst + at) = hi;
                        if (SPLIT) *reinterpret_cast<uint4 *>(dst + G::TILE + at) = lo;
                    }
                }
                if (!ok) break;
                fence_async_smem();
                mbar_arrive(&q_full[st]);
                qx++;
            }
        }
        for (uint32_t i = qx > (uint32_t)QST ? qx - QST : 0; ok && i < qx; i++)  // drain
            ok = mbar_wait(&q_empty[i % QST], (i / QST) & 1, &abort_flag);
    } else {
        // ------------------------------------------------------ column sums
        const uint32_t s = warp >> 2, t128 = tid & 127;
        const uint32_t ts = tmem + s * 256 + ((warp & 3) << 21);
        const float c2 = q.scale * 1.4426950408889634f;
        const f32x2 cc = pack2(c2, c2);
        uint32_t qx = 0, st = 0, ob = ~0u, oh = 0, oq = 0;
        bool ok = true, held = false;
        for (uint32_t x = x0; ok && x < x1; x += xs) {
            Item t;
            item(x, t);
            const uint32_t k = t.k0 + s * 128 + t128;       // this thread's slot
            const uint32_t kw = k - lane;                   // its warp's first
            // rows (of those that count) [vlo, vhi) see slot k; all the warp's slots are seen by [wlo, whi)
            const int R = (int)((t.tq - min(t.i0, t.tq)) * q.group);
            int vlo = 0, vhi = R, wlo = 0, whi = R;
            if (q.causal) {
                auto row = [&](long long i) { return (int)max(0ll, min((long long)R, (i - t.i0) * q.group)); };
                vlo = row((long long)k - t.pos0);
                wlo = row((long long)kw + 31 - t.pos0);
                if (q.window) {
                    vhi = row((long long)k + q.window - t.pos0);
                    whi = row((long long)kw + q.window - t.pos0);
                }
            }
            float *const m = p.mass + ((size_t)t.b * a.kv_heads + t.h) * p.mass_stride + k;
            float old = 0.f;
            bool there = false;  // a hole gathers nothing
            if (k < t.n) {
                there = a.page(t.b, k >> a.page_shift) >= 0;
                if (ranks == 1 && p.decay != 0.f) old = p.decay * *m;
            }
            float sum = 0.f;
            for (uint32_t e = 0; e < t.steps; e++, st++) {
                const uint32_t qt = t.qt0 + rank + e * ranks;
                if (!held || t.b != ob || t.h != oh || qt != oq) {
                    if (held) {
                        mbar_arrive(&q_empty[qx % QST]);
                        qx++;
                    }
                    held = true;
                    ob = t.b, oh = t.h, oq = qt;
                    ok = mbar_wait(&q_full[qx % QST], (qx / QST) & 1, &abort_flag);
                    if (!ok) break;
                }
                const uint32_t buf = st & 1, nr = tile_rows(t, qt), r0 = t.i0 * q.group + qt * 128;
                ok = mbar_wait(&s_full[s][buf], (st >> 1) & 1, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                const int r_tile = (int)(qt * 128), clo = vlo - r_tile, chi = vhi - r_tile;
                const bool masked = wlo > r_tile || whi < r_tile + (int)nr;
                const float *nl = s_nlse[qx % QST];
                f32x2 acc = pack2(0.f, 0.f), acc1 = acc;
                // 32 columns at a time, the next 32 on their way from tensor memory
                float v[2][32];
                tmem_ld32(ts + buf * 128, v[0]);
#pragma unroll
                for (int ch = 0; ch < 4; ch++) {
                    const int c0 = ch * 32;
                    if (c0 >= (int)nr) break;
                    tmem_wait_ld();
                    if (ch < 3 && c0 + 32 < (int)nr) tmem_ld32(ts + buf * 128 + c0 + 32, v[(ch + 1) & 1]);
                    float *w = v[ch & 1];
                    f32x2 n2[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 l4 = *reinterpret_cast<const float4 *>(nl + c0 + i);
                        n2[i / 2] = pack2(l4.x, l4.y);
                        n2[i / 2 + 1] = pack2(l4.z, l4.w);
                    }
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float u0, u1;
                            unpack2(fma2(pack2(w[i], w[i + 1]), cc, n2[i / 2]), u0, u1);
                            u0 = (c0 + i >= clo && c0 + i < chi) ? u0 : -INFINITY;
                            u1 = (c0 + i + 1 >= clo && c0 + i + 1 < chi) ? u1 : -INFINITY;
                            acc = add2(acc, pack2(ex2(u0), ex2(u1)));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            float u0, u1, u2, u3;
                            unpack2(fma2(pack2(w[i], w[i + 1]), cc, n2[i / 2]), u0, u1);
                            unpack2(fma2(pack2(w[i + 2], w[i + 3]), cc, n2[i / 2 + 1]), u2, u3);
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
            if (!there) sum = 0.f;
            if (ok && ranks == 1 && k < t.n) *m = old + sum;
            if (ranks > 1) s_red[s * 128 + t128] = sum;
        }
        if (ok && held) mbar_arrive(&q_empty[qx % QST]);
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        if (tid == 0) g_timeout = 1;
        const unsigned long long t0 = now_ns();
        while (now_ns() - t0 < 1000000ull) {
        }
    }
    if (warp == 8) {
        tc_fence_after();
        tmem_free512(tmem);
    }
    if (ranks > 1) {  // one item per cluster: rank 0 joins the sums in rank order
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank == 0 && tid < ITEM && x0 < x1) {
            Item t;
            item(x0, t);
            const uint32_t k = t.k0 + tid;
            float sum = 0.f;
            for (uint32_t r = 0; r < ranks; r++) {
                uint32_t at;
                float v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&s_red[tid])), "r"(r));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
                sum += v;
            }
            if (k < t.n) {
                float *m = p.mass + ((size_t)t.b * a.kv_heads + t.h) * p.mass_stride + k;
                *m = p.decay == 0.f ? sum : p.decay * *m + sum;
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <typename TQ, typename TC, int HD>
int launch_mass(const MassPagedCall &c, int sm_count, cudaStream_t s) {
    using G = MassGeo<HD, std::is_same<TQ, float>::value>;
    CUtensorMap mk;
    int rc = make_page_map(&mk, c.a.k, c.a, HD, c.cache_type, c.a.page_size < 128 ? c.a.page_size : 128);
    if (rc) return rc;
    auto kern = mass_kernel<TQ, TC, HD>;
    CUQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
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
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
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

int attention_mass_status(cudaStream_t s, int *timed_out) {
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
