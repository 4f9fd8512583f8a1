// Attention weight per cached slot (b2_attention_paged_weights):
//
//   weights[g][j] = prev[g][j] + sum_{i, h in g} exp(s_ijh - lse_ih)
//
// over the new rows i that see slot j, from q, K and the row sums that the
// attention left.  Every slot belongs to one warp, which adds its rows in
// their order: no atomics, and the result does not depend on timing.
#include <type_traits>

#include "b2_tc.cuh"

namespace {

using namespace b2p;

struct WeightParams {
    Batch bt;
    const uint16_t* k;
    long long page_stride, head_stride, row_stride;
    const __half* q16;
    int ldq;
    const float* lse;
    int max_q, nq, nkv, G;
    float* weights;
    const float* prev;
    long long ldw;
    int short_rows;  // sequences with at most this many (token, head) rows per kv head are the short kernel's
    int* err;
    int limit;       // polls of a wait
};

// ─── few rows per sequence ───
//
// Bound by reading K once.  A warp owns 32 slots, two groups of 16: S = K Q^T on
// mma m16n8k16 with the slots as M rows and eight (token, head) rows as N columns.
// The dims of the sum may go in any order as long as K and Q agree, so a lane takes
// 16 consecutive bytes of its row for two k steps and the fragments come straight
// from global memory, a row's four lanes reading 64 consecutive bytes.  Everything
// a block needs is asked for before any of it is used.  64 sequences of 128 to 4096
// slots (70 thousand in all) with 8 kv heads, hd 128, take 32.7 us: 0.69 of the measured
// copy rate.
constexpr int kThreads = 128;
constexpr int kBlk = 128;

// (not the read-only path: the kernel may have started while K was being appended)
__device__ __forceinline__ uint4 ld_k16(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 4) weights_short_kernel(const WeightParams p) {
    __shared__ int pre[B2_PAGED_MAX_SEQS + 1];
    b2::pdl_trigger();
    b2::pdl_wait();  // (behind the long kernel too: there is no workspace to hand over what that one waited for)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c4 = lane & 3;
    prefix_work(pre, p.bt.n_seqs, [&](int s) {
        const Seq q = p.bt.seq(s);
        return min(q.Q, p.max_q) * p.G > p.short_rows ? 0 : cdiv(q.len, kBlk) * p.nkv;
    });
    const int W = pre[p.bt.n_seqs];
    const float scale = kLog2e / sqrtf((float)HD);
    const int slot_mask = (1 << p.bt.page_shift) - 1;
    for (int x = blockIdx.x; x < W; x += gridDim.x) {
        const int s = prefix_find(pre, p.bt.n_seqs, x);
        const Seq sq = p.bt.seq(s);
        const int nb = cdiv(sq.len, kBlk), g = (x - pre[s]) / nb, j0 = (x - pre[s]) % nb * kBlk + warp * 32;
        if (j0 >= sq.len) continue;
        const int rows = min(sq.Q, p.max_q) * p.G;
        // first row that may see a slot of this warp, down to a column tile's start
        const int r_first = max(0, j0 - sq.base) * p.G / 8 * 8;
        const size_t o = ((size_t)s * p.nkv + g) * p.ldw + j0 + lane;
        const bool out = j0 + lane < sq.len && j0 + lane < p.ldw;
        const float was = out && p.prev ? p.prev[o] : 0.f;  // lane = slot
        int page[2];
#pragma unroll
        for (int t = 0; t < 2; t++) page[t] = j0 + 16 * t < sq.len ? p.bt.page(s, j0 + 16 * t) : -1;
        float acc[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
        if (r_first < rows && (page[0] >= 0 || page[1] >= 0)) {
            uint4 a[2][2][HD / 32];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint16_t* kp = p.k + max(page[t], 0) * p.page_stride + g * p.head_stride +
                                     (long long)(((j0 + 16 * t) & slot_mask) + n) * p.row_stride + 8 * c4;
#pragma unroll
                for (int u = 0; u < HD / 32; u++) {
                    a[t][0][u] = page[t] >= 0 ? ld_k16(kp + 32 * u) : make_uint4(0, 0, 0, 0);
                    a[t][1][u] = page[t] >= 0 ? ld_k16(kp + 8 * p.row_stride + 32 * u) : make_uint4(0, 0, 0, 0);
                }
            }
            for (int r0 = r_first; r0 < rows; r0 += 8) {
                const int rq = r0 + n;
                uint4 b[HD / 32];
                const __half* qp = p.q16 + (size_t)(sq.row0 + rq / p.G) * p.ldq + (size_t)(g * p.G + rq % p.G) * HD + 8 * c4;
#pragma unroll
                for (int u = 0; u < HD / 32; u++)
                    b[u] = rq < rows ? *reinterpret_cast<const uint4*>(qp + 32 * u) : make_uint4(0, 0, 0, 0);
                float l[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = r0 + 2 * c4 + e;
                    l[e] = r < rows ? p.lse[(size_t)(sq.row0 + r / p.G) * p.nq + g * p.G + r % p.G] : -INFINITY;
                }
                __syncwarp();  // no load moves behind this
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < HD / 32; u++) {
                        const uint32_t f0[4] = {a[t][0][u].x, a[t][1][u].x, a[t][0][u].y, a[t][1][u].y};
                        const uint32_t f1[4] = {a[t][0][u].z, a[t][1][u].z, a[t][0][u].w, a[t][1][u].w};
                        mma16816(sc, f0, b[u].x, b[u].y);
                        mma16816(sc, f1, b[u].z, b[u].w);
                    }
                    const int ja = j0 + 16 * t + n;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int lim = page[t] < 0 || l[e] == -INFINITY ? -1
                                                                         : min(sq.len - 1, sq.base + (r0 + 2 * c4 + e) / p.G);
                        const float l2 = l[e] * kLog2e;
                        if (ja <= lim) acc[t][0] += ex2(fmaf(sc[e], scale, -l2));
                        if (ja + 8 <= lim) acc[t][1] += ex2(fmaf(sc[e + 2], scale, -l2));
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                acc[t][e] += __shfl_xor_sync(0xffffffffu, acc[t][e], 1);
                acc[t][e] += __shfl_xor_sync(0xffffffffu, acc[t][e], 2);
            }
        // slot j0 + lane: group lane / 16, row lane % 16, held by the lanes of row (lane % 8)
        const float v00 = __shfl_sync(0xffffffffu, acc[0][0], (lane & 7) * 4), v01 = __shfl_sync(0xffffffffu, acc[0][1], (lane & 7) * 4);
        const float v10 = __shfl_sync(0xffffffffu, acc[1][0], (lane & 7) * 4), v11 = __shfl_sync(0xffffffffu, acc[1][1], (lane & 7) * 4);
        const float v = lane < 16 ? (lane < 8 ? v00 : v01) : (lane < 24 ? v10 : v11);
        if (out) p.weights[o] = was + v;
    }
}

// ─── many rows per sequence: chunks ───
//
// Bound by the exponentials (16 per clock and SM), before the product (2 hd FLOP
// per pair).  A unit is 256 slots of one kv head: two K tiles of 128 slots, each
// the A operand of S^T_t = K_t Q^T (tcgen05, N = 128 rows: T tokens x the G heads
// of the group), so a thread owns a slot and adds its columns in registers, and a
// Q tile brought in once serves both K tiles.  Where there are too few units to
// go round, S CTAs of a cluster take every S-th Q tile of one; their sums meet in
// the first one's shared memory and are added in rank order.
// 2048 rows after 6144, 16 q heads, hd 128: 97 us at 1.93 GHz, where the exponentials
// alone would fill the unit for 52 and the product takes 37.  (16 warps of half the columns
// each in place of 8: the same, and 3 to 19 % slower with chunks of 60 to 1000 rows.
// Telling tiles with excluded rows apart costs 2 of the 97.)
//   warp 8      producer: the unit's K tiles, Q tiles and their rows' -lse;
//   warp 9      tensor cores;
//   warps 0-3, 4-7   the exponentials of K tile 0 and 1, one slot per thread.
constexpr int kUnit = 256;
constexpr int kLongThreads = 320;
constexpr int kRowsT = 128;  // rows of a Q tile
constexpr int kMaxCluster = 4;
constexpr int kMaxRounds = 16;  // units per CTA up to which several CTAs may share one
// One pair of exponentials in kPoly takes a polynomial instead of the exponential
// unit: 2048 rows after 6144, 16 q heads, took 101 us with 3, 104 with 4, 108 without
// (before units were dealt out as below).
constexpr int kPoly = 3;

template <int HD>
struct LongSmem {
    static constexpr int kTile = 128 * HD * 2;
    static constexpr int kQStages = HD == 128 ? 4 : 8;
    alignas(1024) unsigned char k[2][kTile];  // [tile]
    alignas(1024) unsigned char q[kQStages][kTile];
    alignas(16) float nl[16][kRowsT];            // -lse log2(e) of the rows of Q tile (count % 16)
    int none[16];                                // some of them are -infinity: rows without weight
    float part[2][kMaxCluster - 1][kUnit];       // first CTA: the others' sums, by unit parity
    uint64_t k_full, k_empty, q_full[kQStages], q_empty[kQStages];
    uint64_t s_full[2][2], s_free[2][2];         // [K tile][buffer]
    uint64_t sum_full[2], sum_free[2];
    uint64_t drain;
    uint32_t tmem;
    volatile int failed[2];          // some warp's wait ran out; polls after which one does
    volatile int k_issued, q_issued; // units whose K, and Q tiles, that the producer has asked for
    int pre[B2_PAGED_MAX_SEQS + 1];
};

struct Unit {
    int s, g, j0;       // sequence, kv head, first slot
    int tiles, first;   // Q tiles of the sequence, and the first that sees a slot of the unit
    int rows;           // (token, head) rows
    Seq sq;
};

__device__ __forceinline__ Unit find_unit(const WeightParams& p, const int* pre, int T, int x) {
    Unit u;
    u.s = prefix_find(pre, p.bt.n_seqs, x);
    u.sq = p.bt.seq(u.s);
    // heads of the same slots side by side: a sequence's last units, which its early rows do
    // not see, come last
    const int off = x - pre[u.s];
    u.g = off % p.nkv;
    u.j0 = off / p.nkv * kUnit;
    const int toks = min(u.sq.Q, p.max_q);
    u.rows = toks * p.G;
    u.tiles = cdiv(toks, T);
    u.first = max(0, u.j0 - u.sq.base) / T;
    return u;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t in_rank(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void remote_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// warp_wait for a barrier that other CTAs of the cluster arrive on.
__device__ __forceinline__ bool cluster_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
    for (int it = 0;; it++) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, "
            "0, p;\n}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
        if (__any_sync(0xffffffffu, it > failed[1] || failed[0])) {
            failed[0] = 1;
            return false;
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kLongThreads, 1)
    weights_long_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const WeightParams p,
                        int cluster) {
    using Sm = LongSmem<HD>;
    constexpr int kHalves = HD / 64;
    extern __shared__ unsigned char smem_raw[];
    Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    volatile int* failed = sm.failed;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            for (int t = 0; t < 2; t++) {
                mbar_init(&sm.s_full[t][i], 1);
                mbar_init(&sm.s_free[t][i], 4);
            }
            mbar_init(&sm.sum_free[i], 256);
        }
        for (int i = 0; i < Sm::kQStages; i++) {
            mbar_init(&sm.q_full[i], 1);
            mbar_init(&sm.q_empty[i], 1);
        }
        mbar_init(&sm.k_full, 1);
        mbar_init(&sm.k_empty, 1);
        mbar_init(&sm.drain, 1);
        sm.failed[0] = 0;
        sm.failed[1] = p.limit;
        sm.k_issued = sm.q_issued = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tq) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
    }
    if (warp == 9) tmem_alloc512(&sm.tmem);
    b2::pdl_wait();
    b2::pdl_trigger();
    const int T = kRowsT / p.G;
    prefix_work(sm.pre, p.bt.n_seqs, [&](int s) {
        const Seq q = p.bt.seq(s);
        return min(q.Q, p.max_q) * p.G > p.short_rows ? cdiv(q.len, kUnit) * p.nkv : 0;
    });
    // Units go round the groups of S CTAs and back, as later ones of a sequence cost
    // less.  S: the fewest that give the shortest schedule, a unit costing its Q tiles
    // and about one more for its K tiles, judged by the first group and the last.  Many
    // rounds are even enough.  (2048 rows after 6144, 8 kv heads, before excluded rows were told
    // apart: 90 us with two CTAs, 96 with one, 98 with one and the groups always in the same order.)
    const int W = sm.pre[p.bt.n_seqs];
    auto place = [](int round, int c, int n) { return round * n + (round & 1 ? n - 1 - c : c); };
    int S = 1;
    if (cdiv(W, gridDim.x) <= kMaxRounds) {
        int best = 0;
        for (int c = 1; c <= cluster; c *= 2) {
            const int n = gridDim.x / c;
            int sum[2] = {0, 0};
            for (int r = lane; r * n < W; r += 32) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int x = place(r, e ? n - 1 : 0, n);
                    if (x >= W) continue;
                    const Unit u = find_unit(p, sm.pre, T, x);
                    sum[e] += cdiv(max(0, u.tiles - u.first), c) + 1;
                }
            }
            const int cost = max(__reduce_add_sync(0xffffffffu, sum[0]), __reduce_add_sync(0xffffffffu, sum[1]));
            if (c == 1 || cost < best) best = cost, S = c;
        }
    }
    const int step = gridDim.x / S, group = (int)blockIdx.x / S, rank = (int)blockIdx.x % S;
    const uint32_t lead_cta = cluster > 1 ? cluster_rank() - rank : 0;  // this unit's first CTA, in the cluster
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) mbar_init(&sm.sum_full[i], S > 1 ? 256 * (S - 1) : 1);
        mbar_init_fence();
    }
    tc_fence_before();
    __syncthreads();
    if (cluster > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    bool ok = true;

    if (warp == 8) {
        // ── producer ──
        const int page_rows = 1 << p.bt.page_shift, box_rows = min(page_rows, 128), boxes = 128 / box_rows;
        const int box = lane / kHalves, half = lane % kHalves;
        int nu = 0, nq = 0;  // units and Q tiles loaded
        // this lane's four rows of a Q tile
        int tok[4], head[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            tok[e] = (32 * e + lane) / p.G;
            head[e] = (32 * e + lane) % p.G;
        }
        for (int r = 0, x; ok && (x = place(r, group, step)) < W; r++) {
            const Unit u = find_unit(p, sm.pre, T, x);
            const int first = uniform(u.first) + rank, tiles = uniform(u.tiles), toks = u.rows / p.G;
            if (first >= tiles) continue;
            const float* lse = p.lse + (size_t)u.sq.row0 * p.nq + u.g * p.G;
            float next[4];
            auto load_lse = [&](int i) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    next[e] = tok[e] < T && i * T + tok[e] < toks ? lse[(size_t)(i * T + tok[e]) * p.nq + head[e]] : -INFINITY;
            };
            load_lse(first);
            // K of the unit before is done with; its pages
            int page[2] = {-1, -1};
            if (box < boxes)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int j = u.j0 + t * 128 + box * box_rows;
                    page[t] = j < u.sq.len ? p.bt.page(u.s, j) : -1;
                }
            if (nu) ok = warp_wait(&sm.k_empty, (nu - 1) & 1, failed);
            if (!ok) break;
            nu++;
            if (lane == 0) {
                mbar_expect_tx(&sm.k_full, 2 * Sm::kTile);
                sm.k_issued = nu;
            }
            __syncwarp();
            if (box < boxes)
#pragma unroll
                for (int t = 0; t < 2; t++)
                    tma_load_5d(sm.k[t] + half * 16384 + box * box_rows * 128, &tk, 0, (u.j0 + box * box_rows) & (page_rows - 1),
                                half, u.g, page[t] >= 0 ? page[t] : p.bt.n_pages, &sm.k_full);
            for (int i = first; i < tiles; i += S, nq++) {
                const int qb = nq % Sm::kQStages;
                if (nq >= Sm::kQStages) ok = warp_wait(&sm.q_empty[qb], (nq / Sm::kQStages - 1) & 1, failed);
                if (!ok) break;
                bool none = false;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    none |= next[e] == -INFINITY;
                    sm.nl[nq & 15][32 * e + lane] = next[e] == -INFINITY ? -INFINITY : -next[e] * kLog2e;
                }
                none = __any_sync(0xffffffffu, none);
                if (lane == 0) sm.none[nq & 15] = none;
                __syncwarp();
                if (lane == 0) {
                    mbar_expect_tx(&sm.q_full[qb], T * p.G * HD * 2);
                    sm.q_issued = nq + 1;
                }
                __syncwarp();
                if (lane < kHalves)
                    tma_load_5d(sm.q[qb] + lane * 16384, &tq, 0, 0, u.sq.row0 + i * T, lane, u.g, &sm.q_full[qb]);
                if (i + S < tiles) load_lse(i + S);
            }
        }
    } else if (warp == 9) {
        // ── tensor cores ──
        constexpr uint32_t id = idesc_f16(128, kRowsT, false);
        const uint32_t lead = lane == 0, tm = (uint32_t)uniform((int)tmem);
        auto wait = [&](uint64_t* bar, int parity) {
            ok = warp_wait(bar, parity, failed);
            tc_fence_after();
            return ok;
        };
        // descriptors of the first element; later ones add to the 14-bit address field
        const uint64_t dk = sw128_desc(smem_u32(sm.k[0]), 16), dq = sw128_desc(smem_u32(sm.q[0]), 16);
        int nu = 0, nq = 0;
        for (int r = 0, x; ok && (x = place(r, group, step)) < W; r++) {
            const Unit u = find_unit(p, sm.pre, T, x);
            const int first = uniform(u.first) + rank, tiles = uniform(u.tiles);
            if (first >= tiles) continue;
            if (!wait(&sm.k_full, nu & 1)) break;
            nu++;
            for (int i = first; i < tiles && ok; i += S, nq++) {
                const int b = nq & 1, st = nq % Sm::kQStages;
                if (!wait(&sm.q_full[st], (nq / Sm::kQStages) & 1)) break;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if (nq >= 2 && !wait(&sm.s_free[t][b], (nq / 2 - 1) & 1)) break;
                    const uint64_t a = dk + t * (Sm::kTile >> 4), q = dq + st * (Sm::kTile >> 4);
#pragma unroll
                    for (int e = 0; e < HD / 16; e++) {
                        const uint32_t o = ((e >> 2) * 16384 + (e & 3) * 32) >> 4;
                        umma_ss(tm + (2 * t + b) * 128, a + o, q + o, id, e != 0, lead);
                    }
                    umma_commit(&sm.s_full[t][b], lead);
                }
                umma_commit(&sm.q_empty[st], lead);
            }
            umma_commit(&sm.k_empty, lead);
        }
        umma_commit(&sm.drain, lead);  // the CTA ends behind its products and their arrivals
        __syncwarp();
        copies_land(&sm.drain, 1, 1);
    } else {
        // ── exponentials of K tile t: thread = slot ──
        const int t = warp >> 2, slot = threadIdx.x;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const float scale = kLog2e / sqrtf((float)HD);
        const uint64_t scale2 = pack_f2(scale, scale);
        int nq = 0, done = 0;  // Q tiles; units (all of them, with work here or not)
        for (int x; ok && (x = place(done, group, step)) < W; done++) {
            const Unit u = find_unit(p, sm.pre, T, x);
            const int j = u.j0 + slot;
            uint64_t acc[2] = {pack_f2(0.f, 0.f), pack_f2(0.f, 0.f)};
            const int first = uniform(u.first) + rank, tiles = uniform(u.tiles);
            // One Q tile; edge: with columns that the slot is not seen by, or of rows without weight, whose
            // product with K may be anything.  Two copies, because a path beside the common one costs that one
            // time even where it is not taken.
            // (its first 32 columns are on their way)
            auto step = [&](auto edge, uint32_t ts, uint32_t (&va)[32], int c0, int c1) {
                const int b = nq & 1;
                const float4* nl = reinterpret_cast<const float4*>(sm.nl[nq & 15]);
                uint32_t vb[32];
                // 32 columns from c0 on, the next ones on their way
                auto add = [&](uint32_t (&v)[32], int col) {
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        const float4 n4 = nl[(col + c) / 4];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float x, y;
                            unpack_f2(fma_f2(pack_f2(__uint_as_float(v[c + 2 * e]), __uint_as_float(v[c + 2 * e + 1])), scale2,
                                             e ? pack_f2(n4.z, n4.w) : pack_f2(n4.x, n4.y)),
                                      x, y);
                            if constexpr (decltype(edge)::value) {  // (here, where a row's NaN sum is in it too)
                                const int r = col + c + 2 * e;
                                if (r < c0 || r >= c1 || (e ? n4.z : n4.x) == -INFINITY) x = -INFINITY;
                                if (r + 1 < c0 || r + 1 >= c1 || (e ? n4.w : n4.y) == -INFINITY) y = -INFINITY;
                            }
                            const bool poly = (c / 2 + e) % kPoly == kPoly - 1;
                            acc[e] = add_f2(acc[e], poly ? ex2_f2(x, y) : pack_f2(ex2(x), ex2(y)));
                        }
                    }
                };
                tmem_wait_ld();
                tmem_ld32<0>(ts + 32, vb);
                add(va, 0);
                tmem_wait_ld();
                tmem_ld32<0>(ts + 64, va);
                add(vb, 32);
                tmem_wait_ld();
                tmem_ld32<0>(ts + 96, vb);
                add(va, 64);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.s_free[t][b]);
                add(vb, 96);
            };
            for (int i = first; i < tiles; i += S, nq++) {
                // columns of tokens from the slot's own on, and rows that exist (bounded before the product:
                // a slot may lie 2^31 before the new rows)
                const int c0 = max(0, min(j - u.sq.base - i * T, kRowsT)) * p.G, c1 = min(T * p.G, u.rows - i * T * p.G);
                const uint32_t ts = tmem + lanes + (2 * t + (nq & 1)) * 128;
                uint32_t va[32];
                ok = warp_wait(&sm.s_full[t][nq & 1], (nq / 2) & 1, failed);
                tc_fence_after();
                tmem_ld32<0>(ts, va);
                const int none = *(volatile int*)&sm.none[nq & 15];
                if (B2_RARE(__any_sync(0xffffffffu, c0 > 0 || c1 < kRowsT || none))) step(std::true_type{}, ts, va, c0, c1);
                else step(std::false_type{}, ts, va, c0, c1);
                if (B2_RARE(!ok)) break;
            }
            if (!ok) break;
            float total, odd;
            unpack_f2(add_f2(acc[0], acc[1]), total, odd);
            total += odd;
            const int par = done & 1;
            if (rank > 0) {
                // to the first CTA, once it has read what this buffer held two units ago
                if (done >= 2) ok = cluster_wait(&sm.sum_free[par], (done / 2 - 1) & 1, failed);
                if (!ok) break;
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(in_rank(&sm.part[par][rank - 1][slot], lead_cta)), "f"(total)
                             : "memory");
                remote_arrive(in_rank(&sm.sum_full[par], lead_cta));
                continue;
            }
            if (S > 1) {
                ok = cluster_wait(&sm.sum_full[par], (done / 2) & 1, failed);
                if (!ok) break;
                for (int e = 1; e < S; e++) total += sm.part[par][e - 1][slot];
                for (int e = 1; e < S; e++) remote_arrive(in_rank(&sm.sum_free[par], lead_cta + e));
            }
            if (j < u.sq.len && j < p.ldw) {
                const size_t o = ((size_t)u.s * p.nkv + u.g) * p.ldw + j;
                p.weights[o] = (p.prev ? p.prev[o] : 0.f) + (p.bt.page(u.s, j) >= 0 ? total : 0.f);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (B2_RARE(*failed)) {
        // Some warp gave up: the CTA must not end before the copies that it has asked for have landed.
        if (threadIdx.x == 0) atomicExch(p.err, 1);
        if (warp == 8 && lane == 0) {
            copies_land(&sm.k_full, 1, sm.k_issued);
            copies_land(sm.q_full, Sm::kQStages, sm.q_issued);
        }
        __syncthreads();
    }
    // the others may still write to or arrive at this CTA's shared memory
    if (cluster > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    if (warp == 9) {
        tc_fence_after();
        tmem_free512(tmem);
    }
}

// Clusters of S CTAs that fit the device at once.
template <int HD>
int max_clusters(int S, int dev, int sms, size_t smem) {
    if (S == 1) return sms;
    static std::atomic<int> known[64][kMaxCluster + 1];
    std::atomic<int>& c = known[dev & 63][S];
    int n = c.load(std::memory_order_relaxed);
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(S);
        cfg.blockDim = dim3(kLongThreads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = S;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, weights_long_kernel<HD>, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            return 0;
        }
        c.store(n, std::memory_order_relaxed);
    }
    return n;
}

template <int HD>
int launch_long(const WeightParams& p, const B2PagedKV* kv, int dev, int sms, cudaStream_t s) {
    static std::atomic<unsigned long long> allowed{0};
    constexpr size_t smem = sizeof(LongSmem<HD>) + 1024;
    cudaError_t e = allow_smem(weights_long_kernel<HD>, smem, allowed, dev);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged_weights smem: %s", cudaGetErrorString(e));
    CUtensorMap tq, tk;
    const int box = kv->page_size < 128 ? kv->page_size : 128, T = kRowsT / p.G;
    int rc = b2_paged_map(&tk, kv->k_pages, kv, p.nkv, HD, box, 1);
    if (!rc) rc = q_map(&tq, p.q16, p.ldq, p.bt.M, p.nkv, p.G, HD, T);
    if (rc) return rc;
    // Clusters of as many CTAs as the Q tiles of a unit can keep busy, and of four only where
    // the units could not fill the SMs: they leave some SMs without work (98 us instead of 90,
    // for the call above).
    const int tiles = cdiv(p.max_q, T);
    const long long units = ((long long)kv->max_pages * kv->page_size + kUnit - 1) / kUnit * p.nkv * kv->n_seqs;
    int S = tiles >= 4 && units <= sms ? 4 : tiles >= 2 ? 2 : 1, clusters = max_clusters<HD>(S, dev, sms, smem);
    if (clusters == 0) clusters = sms, S = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(clusters * S);
    cfg.blockDim = dim3(kLongThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = S;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = S > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, weights_long_kernel<HD>, tq, tk, p, S);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged_weights: %s", cudaGetErrorString(e));
    return 0;
}

// (token, head) rows of a kv head up to which the kernel of few rows takes a sequence:
// it costs a product with every eight rows, the other one a tile of 128 at least.  Two q
// heads each, 8 kv heads, hd 128, 128 to 4096 slots: 16 tokens, 32 rows, take 71 us for
// 64 sequences (11 for 8, 186 for 200) here and 83 (17, 214) there; 20 tokens 84 (13, 221)
// and 83 (17, 215); 24 tokens 97 (14, 256) and 83 (17, 216).
constexpr int kShortRows = 40;

}  // namespace

extern "C" int b2_attention_paged_weights(float* weights, const float* prev, long long ldw, const uint16_t* q16, int ldq,
                                          const float* lse, int M, int max_q, int nq, int nkv, int hd,
                                          const B2PagedKV* kv, int* err, b2_stream_t s) {
    int rc = b2_paged_check("b2_attention_paged_weights", kv, nkv, hd, true);
    if (rc) return rc;
    if ((kv->n_seqs > 0 && !weights) || (M > 0 && (!q16 || !lse)) || !err || ldw < 0 || M < 0 || max_q < 0 || nq <= 0 || nq % nkv || nq / nkv > 16)
        return b2_set_error(B2_ERR_INVALID_ARG,
                            "b2_attention_paged_weights: bad arguments (nq a multiple of nkv, at most 16)");
    if (ldq < (long long)nq * hd || ldq % 8 || (reinterpret_cast<uintptr_t>(q16) & 15))
        return b2_set_error(B2_ERR_INVALID_ARG,
                            "b2_attention_paged_weights: q16 must be 16-byte aligned, ldq a multiple of 8 that holds "
                            "every head");
    if (kv->n_seqs == 0) return 0;
    const long long cap = ((long long)kv->max_pages * kv->page_size + kBlk - 1) / kBlk;
    const long long blocks = cap * kv->n_seqs * nkv;
    if (blocks >= (1ll << 31) - 65536)
        return b2_set_error(B2_ERR_INVALID_ARG, "b2_attention_paged_weights: %lld blocks of work in one call", blocks);
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (max_q > M) max_q = M;
    const WeightParams p{make_batch(kv, M), kv->k_pages, kv->page_stride, kv->head_stride, kv->row_stride,
                         reinterpret_cast<const __half*>(q16), ldq, lse, max_q, nq, nkv, nq / nkv, weights, prev, ldw,
                         kShortRows, err, wait_limit()};
    if ((long long)max_q * p.G > kShortRows) {
        rc = hd == 128 ? launch_long<128>(p, kv, dev, sms, (cudaStream_t)s) : launch_long<64>(p, kv, dev, sms, (cudaStream_t)s);
        if (rc) return rc;
    }
    const long long grid = blocks < sms * 4 ? blocks : sms * 4;  // what is resident
    const cudaError_t e = b2::launch_pdl(hd == 128 ? weights_short_kernel<128> : weights_short_kernel<64>,
                                         dim3((unsigned)grid), dim3(kThreads), 0, (cudaStream_t)s, p);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged_weights: %s", cudaGetErrorString(e));
    return 0;
}
