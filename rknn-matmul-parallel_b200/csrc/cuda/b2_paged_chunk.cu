// Attention of chunks of new rows over a paged KV cache: the part of
// b2_attention_paged for sequences that bring many rows (prompts, drafted
// tokens of wide GQA groups), on the 5th-generation tensor cores.
//
// A tile is 128 rows of one kv head: T = 128 / G tokens times the G q heads of
// its group, so K and V are read once for the whole group.  A CTA works on a
// pair of tiles (2 T tokens) against blocks of 64 slots:
//
//   warp 8      producer: Q tiles, then K and V blocks by TMA through the page
//               table into a ring of shared-memory stages; unmapped pages and
//               pages past kv_len are fetched from outside the tensor, which
//               fills zeros;
//   warps 9, 10 the tensor cores for tile 0 and tile 1: S_t = Q_t K^T (128 x 64,
//               FP32 in tensor memory) and O_t += P_t V with P_t read from tensor
//               memory;
//   warp 11     looks for infinities and NaN in V where some rows may not see it;
//   warps 0-3, 4-7   the softmax of tile 0 and of tile 1, one row per thread:
//               maximum, exponentials, sum, P_t as FP16 over S_t's columns.
//
// S_t has two buffers, so that a tile's next scores are there when its softmax has
// done the block before (blocks of 128 slots with one buffer: 534 us where this takes
// 512, for 4096 new rows after 12288 at 16 q heads, 8 kv heads, hd 128).  O_t is
// rescaled only when a row's maximum has grown by more than 2^8 since the last
// time: until then the weights are taken relative to the older maximum, which
// changes no result (the sum carries the same factor).
//
// Bound by the two products (4 hd FLOP per row and slot) and, at hd 128 just as
// much, by the exponentials: 16 per clock and SM.  Those 4096 rows take 566 us (502 at
// best) called again and again, 850 TFLOP/s, 0.51 of a library product's rate, the SM clock
// at 1.72 GHz under the power cap; in shorter runs, at a higher clock, 491.  In those the
// products and their barriers alone took 468, the softmax without the products 460, and
// every fourth exponential by a polynomial instead 501: the softmax waits for the order of
// its steps, not for the exponential unit.
//
// The work of the call is one line of blocks, cut into equal stretches for the
// CTAs; pairs that a cut divides leave pieces (maximum, sum, unnormalised O) in
// the workspace, which the kernel launched behind this one merges.
#include <type_traits>

#include "b2_tc.cuh"

namespace {

using namespace b2p;

constexpr int kBlk = 64;
// Three warpgroups, launched with 168 registers a thread; those of the softmax, which
// hold a row's 64 scores and weights, go to 208 and the third gives them up:
// 208 + 208 + 88 = 3 x 168.
constexpr int kThreads = 384;
constexpr int kMaxItems = 2048;  // entries of the line's prefix in shared memory
constexpr int kMinBlocks = 4;    // shortest stretch of a CTA
constexpr float kLazy = 8.f;     // growth of the maximum (log2) that O tolerates without rescaling
// Weights are 2^(s - m + kUp) <= 2^(kLazy + kUp) = 2^15 in FP16; kUp keeps small
// ones out of FP16's subnormals down to 2^-21 of the reference.
constexpr float kUp = 7.f;

template <int HD>
struct Cfg {
    static constexpr int kHalves = HD / 64;
    static constexpr int kQTile = 128 * HD * 2;  // bytes
    static constexpr int kTile = kBlk * HD * 2;  // K block or V block, bytes
    static constexpr int kStages = HD == 128 ? 4 : 8;  // of a K block and its V block
    static constexpr int kQHalf = 128 * 128, kHalf = kBlk * 128;  // 64 dims of a Q tile, of a block
    // tensor-memory columns: buffer i of S_t at 128 t + 64 i (P_t over its first half), O_t at 256 + HD t
    static constexpr uint32_t kS = 0, kO = 256;
};

template <int HD>
struct Smem {
    alignas(1024) unsigned char q[2][Cfg<HD>::kQTile];
    alignas(1024) unsigned char ring[Cfg<HD>::kStages][2][Cfg<HD>::kTile];  // [stage][K, V]
    uint64_t full[Cfg<HD>::kStages], empty[Cfg<HD>::kStages];
    uint64_t q_full, q_empty;
    // [tile][buffer of S and P]; o_done too: two products may be under way, and a wait tells two phases apart
    uint64_t s_full[2][2], p_ready[2][2], o_done[2][2];
    uint64_t o_free[2], drain[2];
    uint32_t tmem;
    volatile int failed[2];  // some warp's wait ran out; polls after which one does
    volatile int issued;     // blocks that the producer has asked for
    volatile int q_issued;   // segments whose Q it has asked for
    int skip[2][2];  // [tile][buffer]: block count of a block whose product with V the softmax did itself
    unsigned last_bad[16];  // entry (block count % 16): the count, and 1 + the last slot whose V is not finite
    int mapped[16];  // bit w of entry (block count % 16): slots 16 w .. 16 w + 15 are mapped
    int pre_seq[B2_PAGED_MAX_SEQS + 1];
    int pre[kMaxItems + 1];
};

// A stretch's part of one tile pair: blocks [b0, b1) of its nb.
struct Seg {
    int s, g, i0;
    int tok0, tok1;    // tokens of each tile
    int live0, live1;  // end of the stretch's blocks that some row of the tile sees
    int b0, b1, nb, x0;
    Seq sq;
    __device__ __forceinline__ int end() const { return max(live0, live1); }
    // (selected, not indexed: an indexed member lives in local memory, a load in every block)
    __device__ __forceinline__ int tok(int t) const { return t ? tok1 : tok0; }
    __device__ __forceinline__ int live(int t) const { return t ? live1 : live0; }
};

struct LongParams {
    AttnParams a;
    int T;      // tokens of one tile
    int group;  // tile pairs of one entry of the line's prefix
};

// Slots that every row of tile t sees, as far as they are mapped: those of its first token.
__device__ __forceinline__ int seen_by_all(const LongParams& p, const Seg& g, int t) {
    return max(0, min(g.sq.len, g.sq.base + g.i0 + t * p.T + 1));
}

// Tile pairs of a sequence (none when the short kernel takes it) and the blocks
// that its pair t reaches.
__device__ __forceinline__ int pairs_of(const LongParams& p, const Seq& q) {
    const int n = min(q.Q, p.a.max_q);
    return n * p.a.G <= p.a.short_rows ? 0 : cdiv(n, 2 * p.T);
}
__device__ __forceinline__ int blocks_of(const LongParams& p, const Seq& q, int t) {
    const int last = min(min(q.Q, p.a.max_q), (t + 1) * 2 * p.T);
    return max(1, cdiv(min(q.len, max(0, q.base + last)), kBlk));
}

// Where the stretch of CTA c begins.
template <int HD>
__device__ __forceinline__ int stretch_start(const LongParams& p, const Smem<HD>& sm, int items, int W, int per, int c) {
    const long long at = (long long)c * per;
    if (at >= W) return W;
    const int x = (int)at, e = prefix_find(sm.pre, items, x), s = prefix_find(sm.pre_seq, p.a.bt.n_seqs, e);
    const Seq q = p.a.bt.seq(s);
    const int first = (e - sm.pre_seq[s]) * p.group, nb = blocks_of(p, q, first + min(p.group, pairs_of(p, q) - first) - 1);
    return snap_to(x, (x - sm.pre[e]) % nb, nb, per);
}

template <int HD>
__device__ __forceinline__ Seg find_seg(const LongParams& p, const Smem<HD>& sm, int items, int x, int x1) {
    Seg r;
    const int e = prefix_find(sm.pre, items, x);
    r.s = prefix_find(sm.pre_seq, p.a.bt.n_seqs, e);
    r.sq = p.a.bt.seq(r.s);
    const int first = (e - sm.pre_seq[r.s]) * p.group, n = min(p.group, pairs_of(p, r.sq) - first);
    r.nb = blocks_of(p, r.sq, first + n - 1);
    const int off = x - sm.pre[e], item = off / r.nb;
    r.b0 = off - item * r.nb;
    r.b1 = min(r.nb, r.b0 + (x1 - x));
    r.x0 = x - r.b0;
    r.g = item % p.a.nkv;
    r.i0 = (first + item / p.a.nkv) * 2 * p.T;
    const int rest = min(r.sq.Q, p.a.max_q) - r.i0;
    r.tok0 = min(p.T, rest);
    r.tok1 = max(0, min(p.T, rest - p.T));
    r.live0 = min(r.b1, cdiv(min(r.sq.len, max(0, r.sq.base + r.i0 + r.tok0)), kBlk));
    r.live1 = r.tok1 ? min(r.b1, cdiv(min(r.sq.len, max(0, r.sq.base + r.i0 + p.T + r.tok1)), kBlk)) : 0;
    return r;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    attn_long_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const LongParams p) {
    using C = Cfg<HD>;
    extern __shared__ unsigned char smem_raw[];
    Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Batch& bt = p.a.bt;
    volatile int* failed = sm.failed;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 2);
        }
        mbar_init(&sm.q_full, 1);
        mbar_init(&sm.q_empty, 2);
        for (int t = 0; t < 2; t++) {
            mbar_init(&sm.drain[t], 1);
            for (int i = 0; i < 2; i++) {
                mbar_init(&sm.s_full[t][i], 1);
                mbar_init(&sm.p_ready[t][i], 4);
                mbar_init(&sm.o_done[t][i], 1);
            }
            mbar_init(&sm.o_free[t], 4);
        }
        sm.failed[0] = 0;
        sm.failed[1] = p.a.limit;
        sm.issued = sm.q_issued = 0;
        for (int i = 0; i < 4; i++) sm.skip[i >> 1][i & 1] = -1;
        for (int i = 0; i < 16; i++) sm.last_bad[i] = ~0u;
        mbar_init_fence();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tq) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
    }
    if (warp == 9) tmem_alloc512(&sm.tmem);
    b2::pdl_wait();
    // The kernel behind this one works on other rows and waits for this grid only before
    // it merges: it may start now that the kernels before this one are done, and is told so.
    if (blockIdx.x == 0 && threadIdx.x == 0) tell_waited(p.a);
    b2::pdl_trigger();
    prefix_work(sm.pre_seq, bt.n_seqs, [&](int s) { return cdiv(pairs_of(p, bt.seq(s)), p.group); });
    const int items = min(sm.pre_seq[bt.n_seqs], kMaxItems);  // (more only when sequences share rows)
    prefix_work(sm.pre, items, [&](int e) {
        const int s = prefix_find(sm.pre_seq, bt.n_seqs, e);
        const Seq q = bt.seq(s);
        const int first = (e - sm.pre_seq[s]) * p.group, n = min(p.group, pairs_of(p, q) - first);
        return n * p.a.nkv * blocks_of(p, q, first + n - 1);
    });
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    const int W = items ? sm.pre[items] : 0;
    const int per = max(kMinBlocks, cdiv(W, gridDim.x));
    const int x0 = stretch_start<HD>(p, sm, items, W, per, blockIdx.x),
              x1 = stretch_start<HD>(p, sm, items, W, per, blockIdx.x + 1);
    bool ok = true;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;" ::: "memory");
        if (warp == 8) {
            // ── producer ──
            // Lanes copy the boxes of a block: K's, then V's, a box holding every half of the head's dims
            // where a page has all rows of the block.
            const int page_rows = 1 << bt.page_shift, box_rows = min(page_rows, kBlk), boxes = kBlk / box_rows;
            const int halves = boxes == 1 ? 1 : C::kHalves, per_kv = boxes * halves;
            const int is_v = lane >= per_kv, box = (lane - is_v * per_kv) / halves, half = lane % halves;
            const CUtensorMap* map = is_v ? &tv : &tk;
            unsigned char* to = sm.ring[0][is_v] + half * C::kHalf + box * box_rows * 128;
            int n = 0, seg = 0;  // blocks, segments with work
            for (int x = x0; x < x1 && ok;) {
                const Seg g = find_seg<HD>(p, sm, items, x, x1);
                x = uniform(x + g.b1 - g.b0);
                const int b0 = uniform(g.b0), e = uniform(g.end());
                if (e <= b0) continue;
                // page ids of the next 32 boxes, one per lane, asked for before they are needed
                int ids_from = b0, id = -1, next = -1;
                auto load_ids = [&](int from) {
                    const int j = from * kBlk + lane * box_rows;
                    return j < g.sq.len && from + lane / boxes < e ? bt.page(g.s, j) : -1;
                };
                id = load_ids(b0);
                next = load_ids(b0 + 32 / boxes);
                if (seg) ok = warp_wait(&sm.q_empty, (seg - 1) & 1, failed);
                if (!ok) break;
                const int tiles = g.tok1 ? 2 : 1, rows = p.T * p.a.G;
                if (lane == 0) {
                    mbar_expect_tx(&sm.q_full, tiles * rows * HD * 2);
                    sm.q_issued = seg + 1;
                }
                __syncwarp();
                if (lane < tiles * C::kHalves) {
                    const int t = lane / C::kHalves, h = lane % C::kHalves;
                    // (64 dims, q heads of the group, tokens, halves, kv heads): rows land as token * G + head
                    tma_load_5d(sm.q[t] + h * C::kQHalf, &tq, 0, 0, g.sq.row0 + g.i0 + t * p.T, h, g.g, &sm.q_full);
                }
                seg++;
                for (int b = b0; b < e; b++, n++) {
                    if ((b - ids_from) * boxes == 32) {
                        ids_from = b;
                        id = next;
                        next = load_ids(b + 32 / boxes);
                    }
                    const int at = (b - ids_from) * boxes, st = n % C::kStages;
                    const unsigned have = __ballot_sync(0xffffffffu, id >= 0) >> at;
                    const int page = __shfl_sync(0xffffffffu, id, (at + box) & 31);
                    if (n >= C::kStages) ok = warp_wait(&sm.empty[st], (n / C::kStages - 1) & 1, failed);
                    if (!ok) break;
                    if (lane == 0) {
                        int bits = 0;
                        for (int w = 0; w < kBlk / 16; w++) bits |= (have >> (w * 16 / box_rows) & 1) << w;
                        sm.mapped[n & 15] = bits;
                        mbar_expect_tx(&sm.full[st], 2 * C::kTile);
                        sm.issued = n + 1;
                    }
                    __syncwarp();
                    if (lane < 2 * per_kv)
                        tma_load_5d(to + st * 2 * C::kTile, map, 0, (b * kBlk + box * box_rows) & (page_rows - 1), half, g.g,
                                    page >= 0 ? page : bt.n_pages, &sm.full[st]);
                }
            }
        } else if (warp < 11) {
            // ── tensor cores, for tile t ──
            constexpr uint32_t id_s = idesc_f16(128, kBlk, false), id_o = idesc_f16(128, HD, true);
            const int t = uniform(warp - 9);
            const uint32_t lead = lane == 0, tm = (uint32_t)uniform((int)tmem);
            const uint32_t ts = tm + C::kS + 128 * t, to = tm + C::kO + HD * t;
            int k = 0, seg = 0;  // blocks, segments with work
            int np = 0;  // P tiles consumed
            int no = 0;  // segments whose O has been summed
            auto wait = [&](uint64_t* bar, int parity) {
                ok = warp_wait(bar, parity, failed);
                tc_fence_after();
                return ok;
            };
            // descriptors of the first element; later ones add to the 14-bit address field
            const uint64_t dq = sw128_desc(smem_u32(sm.q[t]), 16), dk = sw128_desc(smem_u32(sm.ring[0][0]), 16),
                           dv = sw128_desc(smem_u32(sm.ring[0][1]), C::kHalf);
            int ns = 0;  // S tiles made
            auto mma_s = [&](int st) {
                const uint64_t k0 = dk + st * (2 * C::kTile >> 4);
                const uint32_t d = ts + 64 * (ns & 1);
#pragma unroll
                for (int i = 0; i < HD / 16; i++)
                    umma_ss(d, dq + (((i >> 2) * C::kQHalf + (i & 3) * 32) >> 4), k0 + (((i >> 2) * C::kHalf + (i & 3) * 32) >> 4),
                            id_s, i != 0, lead);
                umma_commit(&sm.s_full[t][ns & 1], lead);
                ns++;
            };
            for (int x = x0; x < x1 && ok;) {
                const Seg g = find_seg<HD>(p, sm, items, x, x1);
                x = uniform(x + g.b1 - g.b0);
                const int b0 = uniform(g.b0), live = uniform(g.live(t)), e = uniform(g.end());
                const int edge_from = uniform(seen_by_all(p, g, t)) / kBlk;
                if (e <= b0) continue;
                if (!wait(&sm.q_full, seg & 1)) break;
                seg++;
                if (!wait(&sm.full[k % C::kStages], (k / C::kStages) & 1)) break;
                if (b0 < live) mma_s(k % C::kStages);
                if (b0 + 1 == e) umma_commit(&sm.q_empty, lead);
                for (int b = b0; b < e; b++, k++) {
                    const int st = k % C::kStages;
                    if (b + 1 < e) {
                        // The next scores, into the buffer of the last P: the products of one tile run in
                        // order, so that P has been read by then.
                        const int next = (k + 1) % C::kStages;
                        if (B2_RARE(!wait(&sm.full[next], ((k + 1) / C::kStages) & 1))) break;
                        if (b + 1 < live) mma_s(next);
                        if (b + 2 == e) umma_commit(&sm.q_empty, lead);
                    }
                    if (b < live) {
                        const bool first = b == b0;
                        // the segment before's O has been read
                        if (B2_RARE(first && no++ && !wait(&sm.o_free[t], no & 1))) break;
                        const uint64_t v = dv + st * (2 * C::kTile >> 4);
                        if (B2_RARE(!wait(&sm.p_ready[t][np & 1], (np >> 1) & 1))) break;
                        const uint32_t pt = ts + 64 * (np & 1);
                        const bool skip = B2_RARE(b >= edge_from) && *(volatile int*)&sm.skip[t][np & 1] == k;
#pragma unroll
                        for (int i = 0; i < kBlk / 16 && !skip; i++)
                            umma_ts(to, pt + 8 * i, v + i * (2048 >> 4), id_o, !first || i > 0, lead);
                        umma_commit(&sm.o_done[t][np & 1], lead);
                        np++;
                    }
                    umma_commit(&sm.empty[st], lead);
                }
            }
            umma_commit(&sm.drain[t], lead);  // the CTA ends behind its products and their arrivals
            __syncwarp();
            copies_land(&sm.drain[t], 1, 1);
        } else {
            // ── the last slot of each block that some rows may not see whose V is not finite ──
            // (a stage of such a block is not given back before the softmax has this)
            int n = 0;
            for (int x = x0; x < x1 && ok;) {
                const Seg g = find_seg<HD>(p, sm, items, x, x1);
                x += g.b1 - g.b0;
                const int e = uniform(g.end()), b0 = uniform(g.b0), len = uniform(g.sq.len);
                const int seen_all = uniform(seen_by_all(p, g, 0));
                for (int b = max(b0, seen_all / kBlk); b < e && b * kBlk < len; b++) {
                    const int k = n + b - b0, from = max(0, seen_all - b * kBlk), to = min(kBlk, len - b * kBlk);
                    // This warp waits for few of a stage's phases, so it first has to know that the one it
                    // means has begun.  (The limit starts again with every block: it may be far away.)
                    for (int it = 0, was = 0, now; (now = sm.issued) <= k && ok; it++) {
                        if (now != was) was = now, it = 0;
                        if (it > failed[1] || failed[0]) failed[0] = 1, ok = false;
                        __nanosleep(32);
                    }
                    ok = __all_sync(0xffffffffu, ok) && warp_wait(&sm.full[k % C::kStages], (k / C::kStages) & 1, failed);
                    if (!ok) break;
                    const unsigned char* v = sm.ring[k % C::kStages][1];
                    int last = 0;  // slot + 1
#pragma unroll 4
                    for (int i = from * (HD / 8) + lane; i < to * (HD / 8); i += 32)
                        if (non_finite8(*reinterpret_cast<const uint4*>(v + (i % (HD / 8) >> 3) * C::kHalf +
                                                                        i / (HD / 8) * 128 + (i & 7) * 16)))
                            last = i / (HD / 8) + 1;
                    last = __reduce_max_sync(0xffffffffu, last);
                    if (lane == 0) *(volatile unsigned*)&sm.last_bad[k & 15] = (unsigned)k << 8 | (unsigned)last;
                }
                n += max(0, e - b0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;" ::: "memory");
        // ── softmax of tile t: thread = row ──
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s0 = tmem + lanes + C::kS + 128 * t, to = tmem + lanes + C::kO + HD * t;
        const float scale = kLog2e / sqrtf((float)HD);
        int nblk = 0;  // blocks of all segments so far (the producer's count)
        int ns = 0;    // of them this tile's
        bool owns = false;
        for (int x = x0; x < x1 && ok;) {
            const Seg g = find_seg<HD>(p, sm, items, x, x1);
            x += g.b1 - g.b0;
            const int tok = r / p.a.G, first = uniform(g.b0), last = uniform(g.live(t)), len = uniform(g.sq.len);
            const bool live = tok < g.tok(t);
            const int lim = live ? min(len - 1, g.sq.base + g.i0 + t * p.T + tok) : -1;
            float m = -INFINITY;
            uint64_t l2 = pack_f2(0.f, 0.f);  // sum of even and of odd slots
            uint32_t sv[kBlk];
            // the scores of block number i of this tile, asked for while the block before is put away
            auto load_s = [&](int i) {
                ok = warp_wait(&sm.s_full[t][i & 1], (i >> 1) & 1, failed);
                if (!ok) return;
                tc_fence_after();
                tmem_ld32<0>(s0 + 64 * (i & 1), sv);
                tmem_ld32<32>(s0 + 64 * (i & 1) + 32, sv);
            };
            if (first < last) load_s(ns);
            if (!ok) break;
            // blocks from here on hold slots that some row of the tile does not see, or that are not
            // cached (whose V rows the four warps zero together)
            const int seen_all = uniform(seen_by_all(p, g, t)), edge_from = seen_all / kBlk;
            const uint64_t scale2 = pack_f2(scale, scale);
            // One block; edge: with slots that are not seen.  Two copies, because a path beside the common
            // one costs that one a fifth of its time even where it is not taken.
            auto step = [&](auto edge, int b, int bits) {
                const int j0 = b * kBlk, n = nblk + (b - first);
                const uint32_t ts = s0 + 64 * (ns & 1);
                uint32_t lo = 0, hi = 0;  // bit c of the pair: the row sees slot j0 + c
                bool by_hand = false;
                tmem_wait_ld();
                if constexpr (decltype(edge)::value) {
                    const int seen = lim - j0 + 1;
                    lo = (bits & 1 ? 0xffffu : 0u) | (bits & 2 ? 0xffff0000u : 0u);
                    hi = (bits & 4 ? 0xffffu : 0u) | (bits & 8 ? 0xffff0000u : 0u);
                    if (seen < 32) lo &= (1u << max(seen, 0)) - 1;
                    if (seen < 64) hi &= (1u << max(seen - 32, 0)) - 1;
#pragma unroll
                    for (int c = 0; c < kBlk; c++)
                        if (!((c < 32 ? lo : hi) >> (c & 31) & 1)) sv[c] = 0xff800000u;  // -inf
                    if (len < j0 + kBlk) {
                        // V rows past kv_len may hold anything: zero them (their P is zero, and 0 x inf is not)
                        // (S from this stage's K is there, so its V is)
                        unsigned char* v = sm.ring[n % C::kStages][1];
                        for (int i = r; i < (j0 + kBlk - len) * (HD / 8); i += 128) {
                            const int row = len - j0 + i / (HD / 8), c = i % (HD / 8);
                            *reinterpret_cast<uint4*>(v + (c >> 3) * C::kHalf + row * 128 + (c & 7) * 16) =
                                make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    // An infinite or NaN V at a slot that some row does not see would reach that row
                    // too (0 x inf): such a block is summed by its rows themselves.
                    // (This costs 1 us of 23 with 8 x 60 rows, 5 of 491 with 4096 rows.)
                    if (b >= edge_from && j0 < len) {
                        unsigned w = 0;
                        for (int it = 0; ok && ((w = *(volatile unsigned*)&sm.last_bad[n & 15]) >> 8) != (n & 0xffffffu); it++)
                            if (it > failed[1] || failed[0]) failed[0] = 1, ok = false;
                        ok = __all_sync(0xffffffffu, ok);
                        by_hand = ok && uniform((int)(w & 255)) > max(0, seen_all - j0);
                    }
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kBlk / 2; i++)
                    mx4[i & 3] = max3(mx4[i & 3], __uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1]));
                const float mx = max3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]) * scale;
                // a new reference for rows that outgrew theirs
                const bool grow = live && (mx > m + kLazy || (m == -INFINITY && mx > m));
                if (B2_RARE(__any_sync(0xffffffffu, grow))) {
                    const float f = grow ? ex2(m - mx) : 1.f;
                    if (grow) m = mx;
                    if (b > first) {
                        l2 = fma_f2(l2, pack_f2(f, f), pack_f2(0.f, 0.f));
                        ok = warp_wait(&sm.o_done[t][(ns - 1) & 1], ((ns - 1) >> 1) & 1, failed);
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD && ok; c += 32) {
                            uint32_t ov[32];
                            tmem_ld32<0>(to + c, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
                            tmem_st32(to + c, ov);
                        }
                    }
                }
                uint32_t pk[kBlk / 2];
                uint64_t add[2] = {pack_f2(0.f, 0.f), pack_f2(0.f, 0.f)};
                const float bias = m == -INFINITY ? 0.f : kUp - m;
                const uint64_t bias2 = pack_f2(bias, bias);
#pragma unroll
                for (int i = 0; i < kBlk / 2; i++) {
                    float x, y;
                    unpack_f2(fma_f2(pack_f2(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1])), scale2, bias2), x, y);
                    x = ex2(x);
                    y = ex2(y);
                    add[i & 1] = add_f2(add[i & 1], pack_f2(x, y));
                    pk[i] = pack_h2(x, y);
                }
                tmem_st32(ts, pk);
                if constexpr (decltype(edge)::value) {
                    if (B2_RARE(by_hand)) {
                        tmem_wait_st();
                        // (V is there: the warp that looked has seen it; this wait makes it visible here)
                        ok = ok && warp_wait(&sm.full[n % C::kStages], (n / C::kStages) & 1, failed);
                        if (b > first) {
                            ok = ok && warp_wait(&sm.o_done[t][(ns - 1) & 1], ((ns - 1) >> 1) & 1, failed);
                            tc_fence_after();
                        }
                        const unsigned char* v = sm.ring[n % C::kStages][1];
#pragma unroll 1
                        for (int c = 0; c < HD && ok; c += 32) {
                            uint32_t ov[32];
#pragma unroll
                            for (int i = 0; i < 32; i++) ov[i] = 0u;
                            if (b > first) {
                                tmem_ld32<0>(to + c, ov);
                                tmem_wait_ld();
                            }
#pragma unroll 1
                            for (int s = 0; s < kBlk; s++) {
                                __syncwarp();
                                const uint32_t w = tmem_ld1(ts + s / 2);
                                tmem_wait_ld();
                                const float ps = __half2float(__ushort_as_half((unsigned short)(s & 1 ? w >> 16 : w)));
                                const bool see = (s < 32 ? lo : hi) >> (s & 31) & 1;
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const uint4 u = *reinterpret_cast<const uint4*>(
                                        v + (c >> 6) * C::kHalf + s * 128 + ((((c & 63) >> 3) + i) ^ (s & 7)) * 16);
                                    const uint32_t h[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                                    for (int e = 0; e < 8; e++) {
                                        const float x = __half2float(
                                            __ushort_as_half((unsigned short)(e & 1 ? h[e / 2] >> 16 : h[e / 2])));
                                        if (see) ov[8 * i + e] = __float_as_uint(fmaf(ps, x, __uint_as_float(ov[8 * i + e])));
                                    }
                                }
                            }
                            __syncwarp();
                            tmem_st32(to + c, ov);
                        }
                        if ((threadIdx.x & 127) == 0) sm.skip[t][ns & 1] = n;
                    }
                }
                l2 = add_f2(l2, add_f2(add[0], add[1]));
                if (b + 1 < last) load_s(ns + 1);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_ready[t][ns & 1]);
            };
            for (int b = first; b < last; b++, ns++) {
                const int bits = *(volatile int*)&sm.mapped[(nblk + b - first) & 15];
                if (B2_RARE(b >= edge_from || bits != (1 << kBlk / 16) - 1)) step(std::true_type{}, b, bits);
                else step(std::false_type{}, b, bits);
                if (B2_RARE(!ok)) break;
            }
            if (!ok) break;
            nblk += max(0, g.end() - first);
            // the pair's result, or this stretch's piece of it
            int own, end;  // CTAs of the pair's pieces
            cut_of(g.x0, g.nb, per, own, end);
            const bool whole = own >= end, any = last > first;
            if (any) {
                ok = warp_wait(&sm.o_done[t][(ns - 1) & 1], ((ns - 1) >> 1) & 1, failed);
                if (!ok) break;
                tc_fence_after();
            }
            float la, lb;
            unpack_f2(l2, la, lb);
            const float l = la + lb;
            const size_t row = (size_t)(g.sq.row0 + g.i0 + t * p.T + tok);
            const int h = g.g * p.a.G + r % p.a.G;
            float* part = p.a.long_part + (size_t)(2 * blockIdx.x + (g.b0 == 0 ? 1 : 0)) * long_piece_floats(HD);
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t ov[32];
                if (any) {
                    tmem_ld32<0>(to + c, ov);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) ov[i] = 0u;
                }
                if (live && whole) {
                    uint4* dst = reinterpret_cast<uint4*>(p.a.out16 + (row * p.a.nq + h) * HD + c);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint4 u;
                        uint32_t* w = &u.x;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            w[e] = pack_h2(__uint_as_float(ov[8 * i + 2 * e]) * inv, __uint_as_float(ov[8 * i + 2 * e + 1]) * inv);
                        dst[i] = u;
                    }
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        *reinterpret_cast<uint4*>(part + ((size_t)(t * (HD / 4) + c / 4 + i) * kLongRows + r) * 4) =
                            make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
                }
                __syncwarp();
            }
            if (live) {
                if (!whole)
                    *reinterpret_cast<float2*>(part + 2 * kLongRows * HD + 2 * (t * kLongRows + r)) = make_float2(m - kUp, l);
                else if (p.a.lse)
                    p.a.lse[row * p.a.nq + h] = l == 0.f ? -INFINITY : (m - kUp) * kLn2 + logf(l);
            }
            tc_fence_before();
            __syncwarp();
            if (any && lane == 0) mbar_arrive(&sm.o_free[t]);
            if (!whole && g.b0 == 0) {
                owns = true;
                if (threadIdx.x == 0)
                    p.a.cuts[blockIdx.x] =
                        Cut{end - own + 1, g.sq.row0 + g.i0, g.tok0 + g.tok1, g.g};
            }
        }
        if (threadIdx.x == 0 && !owns) p.a.cuts[blockIdx.x] = Cut{0, 0, 0, 0};
        tmem_wait_ld();  // (a wait that ran out may have left a load on its way)
        tmem_wait_st();
    }
    tc_fence_before();
    __syncthreads();
    if (B2_RARE(*failed)) {
        // Some warp gave up: the CTA must not end before the copies that it has asked for have landed.
        if (threadIdx.x == 0) atomicExch(p.a.err, 1);
        if (warp == 8 && lane == 0) {
            copies_land(sm.full, C::kStages, sm.issued);
            copies_land(&sm.q_full, 1, sm.q_issued);
        }
        __syncthreads();
    }
    if (warp == 9) {
        tc_fence_after();
        tmem_free512(tmem);
    }
}

template <int HD>
int launch_long(LongParams& p, const B2PagedKV* kv, int dev, int sms, cudaStream_t s) {
    static std::atomic<unsigned long long> done{0};
    constexpr size_t smem = sizeof(Smem<HD>) + 1024;
    cudaError_t e = allow_smem(attn_long_kernel<HD>, smem, done, dev);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged smem: %s", cudaGetErrorString(e));
    CUtensorMap tq, tk, tv;
    const int box = kv->page_size < kBlk ? kv->page_size : kBlk;
    const int halves = box == kBlk ? HD / 64 : 1;
    int rc = b2_paged_map(&tk, kv->k_pages, kv, p.a.nkv, HD, box, halves);
    if (!rc) rc = b2_paged_map(&tv, kv->v_pages, kv, p.a.nkv, HD, box, halves);
    if (!rc) rc = q_map(&tq, p.a.q16, p.a.ldq, p.a.bt.M, p.a.nkv, p.a.G, HD, p.T);
    if (rc) return rc;
    e = b2::launch_pdl(attn_long_kernel<HD>, dim3(p.a.long_ctas), dim3(kThreads), smem, s, tq, tk, tv, p);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace

int b2_paged_attention_long(b2p::AttnParams& a, const B2PagedKV* kv, int hd, int dev, int sms, cudaStream_t s) {
    LongParams p{a, kLongRows / a.G, 1};
    // entries of the line's prefix: tile pairs, or groups of neighbouring ones
    const long long pairs = (a.bt.M + 2ll * p.T - 1) / (2 * p.T) + a.bt.n_seqs;
    while ((pairs + p.group - 1) / p.group + a.bt.n_seqs > kMaxItems) p.group++;
    const long long cap = ((long long)kv->max_pages * kv->page_size + kBlk - 1) / kBlk;
    if (pairs * a.nkv * cap >= (1ll << 31) - 65536)
        return b2_set_error(B2_ERR_INVALID_ARG, "b2_attention_paged: %lld blocks of work in one call", pairs * a.nkv * cap);
    a.long_ctas = p.a.long_ctas = sms < kMaxLongCtas ? sms : kMaxLongCtas;
    return hd == 128 ? launch_long<128>(p, kv, dev, sms, s) : launch_long<64>(p, kv, dev, sms, s);
}
