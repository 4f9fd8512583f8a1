// Attention of chunks of new rows over a paged KV cache: the part of
// b2_attention_paged for sequences that bring many rows (prompts, drafted
// tokens of wide GQA groups), on the 5th-generation tensor cores.
//
// A tile is 128 rows of one kv head: T = 128 / G tokens times the G q heads of
// its group, so K and V are read once for the whole group.  A CTA works on a
// pair of tiles (2 T tokens) against blocks of 128 slots:
//
//   warp 8      producer: Q tiles, then K and V blocks by TMA through the page
//               table into a ring of shared-memory stages; unmapped pages and
//               pages past kv_len are fetched from outside the tensor, which
//               fills zeros;
//   warp 9      one thread issues tcgen05.mma: S_t = Q_t K^T (128 x 128, FP32 in
//               tensor memory) and O_t += P_t V with P_t read from tensor memory;
//   warps 0-3, 4-7   the softmax of tile 0 and of tile 1, one row per thread:
//               maximum, exponentials, sum, P_t as FP16 over S_t's columns.
//
// While one tile's softmax runs, the tensor cores work on the other tile.  O_t is
// rescaled only when a row's maximum has grown by more than 2^8 since the last
// time: until then the weights are taken relative to the older maximum, which
// changes no result (the sum carries the same factor).
//
// Bound by the two products (4 hd FLOP per row and slot) and, at hd 128 just as
// much, by the exponentials: 16 per clock and SM.
//
// The work of the call is one line of blocks, cut into equal stretches for the
// CTAs; pairs that a cut divides leave pieces (maximum, sum, unnormalised O) in
// the workspace, which the kernel launched behind this one merges.
#include "b2_tc.cuh"

namespace {

using namespace b2p;

constexpr int kBlk = 128;
// Three warpgroups; the third's last two warps only fill it up.  Launched with 168
// registers a thread; the softmax warpgroups, which hold a row of 128 scores, go to
// 208 and the third gives them up: 208 + 208 + 88 = 3 x 168.
constexpr int kThreads = 384;
constexpr int kMaxItems = 2048;  // entries of the line's prefix in shared memory
constexpr int kMinBlocks = 2;    // shortest stretch of a CTA
constexpr float kLazy = 8.f;     // growth of the maximum (log2) that O tolerates without rescaling
// Weights are 2^(s - m + kUp) <= 2^(kLazy + kUp) = 2^15 in FP16; kUp keeps small
// ones out of FP16's subnormals down to 2^-21 of the reference.
constexpr float kUp = 7.f;

template <int HD>
struct Cfg {
    static constexpr int kHalves = HD / 64;
    static constexpr int kTile = 128 * HD * 2;  // one Q tile, K block or V block, bytes
    static constexpr int kStages = HD == 128 ? 4 : 8;
    static constexpr uint32_t kS = 0, kO = 256;  // tensor-memory columns: S_t at 128 t, O_t at 256 + HD t
};

template <int HD>
struct Smem {
    alignas(1024) unsigned char q[2][Cfg<HD>::kTile];
    alignas(1024) unsigned char ring[Cfg<HD>::kStages][Cfg<HD>::kTile];
    uint64_t full[Cfg<HD>::kStages], empty[Cfg<HD>::kStages];
    uint64_t q_full, q_empty;
    uint64_t s_full[2], p_ready[2][2], o_done[2], o_free[2], drain;  // p_ready: [tile][half of the slots]
    uint32_t tmem;
    int failed;
    int mapped[8];  // bit w of entry (block count % 8): slots 16 w .. 16 w + 15 are mapped
    int pre_seq[B2_PAGED_MAX_SEQS + 1];
    int pre[kMaxItems + 1];
};

// A stretch's part of one tile pair: blocks [b0, b1) of its nb.
struct Seg {
    int s, g, i0;
    int tok[2];   // tokens of each tile
    int live[2];  // end of the stretch's blocks that some row of the tile sees
    int b0, b1, nb, x0;
    Seq sq;
    __device__ __forceinline__ int end() const { return max(live[0], live[1]); }
};

struct LongParams {
    AttnParams a;
    int T;      // tokens of one tile
    int group;  // tile pairs of one entry of the line's prefix
};

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
#pragma unroll
    for (int t = 0; t < 2; t++) {
        r.tok[t] = max(0, min(p.T, rest - t * p.T));
        const int end = r.tok[t] ? min(r.sq.len, max(0, r.sq.base + r.i0 + t * p.T + r.tok[t])) : 0;
        r.live[t] = min(r.b1, cdiv(end, kBlk));
    }
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
    volatile int* failed = &sm.failed;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 1);
        }
        mbar_init(&sm.q_full, 1);
        mbar_init(&sm.q_empty, 1);
        mbar_init(&sm.drain, 1);
        for (int t = 0; t < 2; t++) {
            mbar_init(&sm.s_full[t], 1);
            mbar_init(&sm.p_ready[t][0], 128);
            mbar_init(&sm.p_ready[t][1], 128);
            mbar_init(&sm.o_done[t], 1);
            mbar_init(&sm.o_free[t], 128);
        }
        sm.failed = 0;
        mbar_init_fence();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tq) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
    }
    if (warp == 9) tmem_alloc512(&sm.tmem);
    b2::pdl_wait();
    // The kernel behind this one works on other rows and waits for this grid before
    // it merges, but it does not wait for the kernels before this one: let it start
    // only now that they are done.
    b2::pdl_trigger();
    prefix_work(sm.pre_seq, bt.n_seqs, [&](int s) { return cdiv(pairs_of(p, bt.seq(s)), p.group); });
    const int items = sm.pre_seq[bt.n_seqs];
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
    const int x0 = (int)min((long long)W, (long long)blockIdx.x * per), x1 = min(W, x0 + per);
    bool ok = true;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;" ::: "memory");
        if (warp == 8) {
            // ── producer ──
            const int page_rows = 1 << bt.page_shift, box_rows = min(page_rows, kBlk), boxes = kBlk / box_rows;
            const int box = lane / C::kHalves, half = lane % C::kHalves;
            int k = 0, n = 0, seg = 0;  // ring entries, blocks, segments with work
            for (int x = x0; x < x1 && ok;) {
                const Seg g = find_seg<HD>(p, sm, items, x, x1);
                x += g.b1 - g.b0;
                if (g.end() <= g.b0) continue;
                if (seg && !mbar_wait(&sm.q_empty, (seg - 1) & 1, failed)) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int tiles = g.tok[1] ? 2 : 1, rows = p.T * p.a.G;
                if (lane == 0) mbar_expect_tx(&sm.q_full, tiles * rows * HD * 2);
                __syncwarp();
                if (lane < tiles * C::kHalves) {
                    const int t = lane / C::kHalves;
                    // (64 dims, q heads of the group, tokens, halves, kv heads): rows land as token * G + head
                    tma_load_5d(sm.q[t] + half * 16384, &tq, 0, 0, g.sq.row0 + g.i0 + t * p.T, half, g.g, &sm.q_full);
                }
                seg++;
                for (int b = g.b0; b < g.end() && ok; b++, n++) {
                    const int j = b * kBlk + box * box_rows;
                    const int page = box < boxes && j < g.sq.len ? bt.page(g.s, j) : -1;
                    const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
#pragma unroll
                    for (int kv = 0; kv < 2; kv++, k++) {
                        const int st = k % C::kStages;
                        if (k >= C::kStages && !mbar_wait(&sm.empty[st], (k / C::kStages - 1) & 1, failed)) ok = false;
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) {
                            if (kv == 0) {
                                int bits = 0;
                                for (int w = 0; w < 8; w++) bits |= (have >> (w * 16 / box_rows * C::kHalves) & 1) << w;
                                sm.mapped[n & 7] = bits;
                            }
                            mbar_expect_tx(&sm.full[st], C::kTile);
                        }
                        __syncwarp();
                        if (box < boxes)
                            tma_load_5d(sm.ring[st] + half * 16384 + box * box_rows * 128, kv ? &tv : &tk, 0, j & (page_rows - 1),
                                        half, g.g, page >= 0 ? page : bt.n_pages, &sm.full[st]);
                    }
                }
            }
            if (!ok && lane == 0)  // let the copies in flight land (bounded) before the CTA ends
                for (int i = max(0, k - C::kStages); i < k; i++)
                    for (long long it = 0; it <= kWaitLimit; it++)
                        if (mbar_try_wait(&sm.full[i % C::kStages], (i / C::kStages) & 1)) break;
            if (!ok && lane == 0 && seg)
                for (long long it = 0; it <= kWaitLimit; it++)
                    if (mbar_try_wait(&sm.q_full, (seg - 1) & 1)) break;
        } else if (warp == 9) {
            // ── tensor cores ──
            constexpr uint32_t id_s = idesc_f16(128, 128, false), id_o = idesc_f16(128, HD, true);
            const uint32_t lead = lane == 0, tm = (uint32_t)uniform((int)tmem);
            int k = 0, seg = 0;
            int np0 = 0, np1 = 0;  // P tiles consumed of either tile
            int no0 = 0, no1 = 0;  // segments whose O the tile has summed
            auto wait = [&](uint64_t* bar, int parity) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, failed));
                tc_fence_after();
                return ok;
            };
            // descriptors of the first element; later ones add to the 14-bit address field
            const uint64_t dq = sw128_desc(smem_u32(sm.q[0]), 16), dk = sw128_desc(smem_u32(sm.ring[0]), 16),
                           dv = sw128_desc(smem_u32(sm.ring[0]), 16384);
            auto mma_s = [&](int t, int st) {
                const uint64_t a = dq + t * (C::kTile >> 4), b = dk + st * (C::kTile >> 4);
#pragma unroll
                for (int i = 0; i < HD / 16; i++) {
                    const uint32_t o = ((i >> 2) * 16384 + (i & 3) * 32) >> 4;
                    umma_ss(tm + C::kS + 128 * t, a + o, b + o, id_s, i != 0, lead);
                }
                umma_commit(&sm.s_full[t], lead);
            };
            // O_t += P_t V for one block; first: the segment's first, once the segment before's O has been read
            auto mma_o = [&](int t, int st, bool first, int& np, int& no) {
                if (first && no++ && !wait(&sm.o_free[t], no & 1)) return false;
                const uint64_t v = dv + st * (C::kTile >> 4);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (!wait(&sm.p_ready[t][h], np & 1)) return false;
#pragma unroll
                    for (int i = 4 * h; i < 4 * h + 4; i++)
                        umma_ts(tm + C::kO + HD * t, tm + C::kS + 128 * t + 8 * i, v + i * (2048 >> 4), id_o,
                                !first || i > 0, lead);
                }
                np++;
                umma_commit(&sm.o_done[t], lead);
                return true;
            };
            for (int x = x0; x < x1 && ok;) {
                const Seg g = find_seg<HD>(p, sm, items, x, x1);
                x = uniform(x + g.b1 - g.b0);
                const int b0 = uniform(g.b0), live0 = uniform(g.live[0]), live1 = uniform(g.live[1]);
                const int e = max(live0, live1);
                if (e <= b0) continue;
                if (!wait(&sm.q_full, seg & 1)) break;
                seg++;
                if (!wait(&sm.full[k % C::kStages], (k / C::kStages) & 1)) break;
                if (b0 < live0) mma_s(0, k % C::kStages);
                if (b0 < live1) mma_s(1, k % C::kStages);
                umma_commit(&sm.empty[k % C::kStages], lead);
                if (b0 + 1 == e) umma_commit(&sm.q_empty, lead);
                for (int b = b0; b < e; b++, k += 2) {
                    const int sv = (k + 1) % C::kStages, sk = (k + 2) % C::kStages;
                    if (!wait(&sm.full[sv], ((k + 1) / C::kStages) & 1)) break;
                    if (b < live0 && !mma_o(0, sv, b == b0, np0, no0)) break;
                    if (b + 1 < e && !wait(&sm.full[sk], ((k + 2) / C::kStages) & 1)) break;
                    if (b + 1 < live0) mma_s(0, sk);
                    if (b < live1 && !mma_o(1, sv, b == b0, np1, no1)) break;
                    umma_commit(&sm.empty[sv], lead);
                    if (b + 1 < live1) mma_s(1, sk);
                    if (b + 1 < e) umma_commit(&sm.empty[sk], lead);
                    if (b + 2 == e) umma_commit(&sm.q_empty, lead);
                }
            }
            if (!ok) {  // nothing of the tensor cores may be left running
                umma_commit(&sm.drain, lead);
                for (long long it = 0; it <= kWaitLimit; it++)
                    if (mbar_try_wait(&sm.drain, 0)) break;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;" ::: "memory");
        // ── softmax of tile t: thread = row ──
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + C::kS + 128 * t, to = tmem + lanes + C::kO + HD * t;
        const float scale = kLog2e / sqrtf((float)HD);
        int nblk = 0;  // blocks of all segments so far (the producer's count)
        int ns = 0;    // of them this tile's
        bool owns = false;
        for (int x = x0; x < x1 && ok;) {
            const Seg g = find_seg<HD>(p, sm, items, x, x1);
            x += g.b1 - g.b0;
            const int tok = r / p.a.G, first = g.b0;
            const bool live = tok < g.tok[t];
            const int lim = live ? min(g.sq.len - 1, g.sq.base + g.i0 + t * p.T + tok) : -1;
            float m = -INFINITY;
            uint64_t l2[2] = {pack_f2(0.f, 0.f), pack_f2(0.f, 0.f)};  // sums, two slots at a time
            for (int b = first; b < g.live[t]; b++, ns++) {
                const int j0 = b * kBlk, n = nblk + (b - first);
                ok = mbar_wait(&sm.s_full[t], ns & 1, failed);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc_fence_after();
                uint32_t sv[128];
                tmem_ld32<0>(ts, sv);
                tmem_ld32<32>(ts + 32, sv);
                tmem_wait_ld();
                tmem_ld32<64>(ts + 64, sv);
                tmem_ld32<96>(ts + 96, sv);
                const int bits = *(volatile int*)&sm.mapped[n & 7];
                const bool masked = bits != 0xff || __any_sync(0xffffffffu, live && lim < j0 + kBlk - 1);
                auto mask = [&](int c0) {
#pragma unroll
                    for (int c = c0; c < c0 + 64; c++)
                        if (j0 + c > lim || !(bits >> (c >> 4) & 1)) sv[c] = 0xff800000u;  // -inf
                };
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto top = [&](int c0) {
#pragma unroll
                    for (int c = c0; c < c0 + 64; c += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            mx4[e] = max3(mx4[e], __uint_as_float(sv[c + 2 * e]), __uint_as_float(sv[c + 2 * e + 1]));
                };
                if (masked) mask(0);
                top(0);
                tmem_wait_ld();
                if (masked) mask(64);
                top(64);
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale;
                // a new reference for rows that outgrew theirs
                const bool grow = live && (mx > m + kLazy || (m == -INFINITY && mx > m));
                if (b == first) {
                    m = mx;
                } else if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? ex2(m - mx) : 1.f;
                    ok = mbar_wait(&sm.o_done[t], (ns - 1) & 1, failed);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t ov[32];
                        tmem_ld32<0>(to + c, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
                        tmem_st32(to + c, ov);
                    }
                    l2[0] = fma_f2(l2[0], pack_f2(f, f), pack_f2(0.f, 0.f));
                    l2[1] = fma_f2(l2[1], pack_f2(f, f), pack_f2(0.f, 0.f));
                    if (grow) m = mx;
                }
                if (g.sq.len < j0 + kBlk) {
                    // V rows past kv_len may hold anything: zero them (their P is zero, and 0 x inf is not)
                    const int kvn = 2 * n + 1;
                    ok = mbar_wait(&sm.full[kvn % C::kStages], (kvn / C::kStages) & 1, failed);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    unsigned char* v = sm.ring[kvn % C::kStages];
                    for (int i = r; i < (j0 + kBlk - g.sq.len) * (HD / 8); i += 128) {
                        const int row = g.sq.len - j0 + i / (HD / 8), c = i % (HD / 8);
                        *reinterpret_cast<uint4*>(v + (c >> 3) * 16384 + row * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                const float bias = m == -INFINITY ? 0.f : kUp - m;
                const uint64_t scale2 = pack_f2(scale, scale), bias2 = pack_f2(bias, bias);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const int c = 64 * h + 2 * i;
                        float x, y;
                        unpack_f2(fma_f2(pack_f2(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])), scale2, bias2), x, y);
                        x = ex2(x);
                        y = ex2(y);
                        l2[i & 1] = add_f2(l2[i & 1], pack_f2(x, y));
                        pk[i] = pack_h2(x, y);
                    }
                    tmem_st32(ts + 32 * h, pk);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&sm.p_ready[t][h]);
                }
            }
            if (!ok) break;
            nblk += max(0, g.end() - first);
            // the pair's result, or this stretch's piece of it
            const bool whole = g.b0 == 0 && g.b1 == g.nb, any = g.live[t] > first;
            if (any) {
                ok = mbar_wait(&sm.o_done[t], (ns - 1) & 1, failed);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc_fence_after();
            }
            float la, lb;
            unpack_f2(add_f2(l2[0], l2[1]), la, lb);
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
            if (any) mbar_arrive(&sm.o_free[t]);
            if (!whole && g.b0 == 0) {
                owns = true;
                if (threadIdx.x == 0)
                    p.a.cuts[blockIdx.x] =
                        Cut{(g.x0 + g.nb - 1) / per - (int)blockIdx.x + 1, g.sq.row0 + g.i0, g.tok[0] + g.tok[1], g.g};
            }
        }
        if (threadIdx.x == 0 && !owns) p.a.cuts[blockIdx.x] = Cut{0, 0, 0, 0};
    }
    if (!ok && lane == 0) atomicExch(p.a.err, 1);
    tc_fence_before();
    __syncthreads();
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
    int rc = b2_paged_map(&tk, kv->k_pages, kv, p.a.nkv, HD, box, 1);
    if (!rc) rc = b2_paged_map(&tv, kv->v_pages, kv, p.a.nkv, HD, box, 1);
    if (!rc) rc = q_map(&tq, p.a.q16, p.a.ldq, p.a.bt.M, p.a.nkv, p.a.G, HD, p.T);
    if (rc) return rc;
    e = b2::launch_pdl(attn_long_kernel<HD>, dim3(sms), dim3(kThreads), smem, s, tq, tk, tv, p);
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
    a.long_ctas = p.a.long_ctas = sms;
    return hd == 128 ? launch_long<128>(p, kv, dev, sms, s) : launch_long<64>(p, kv, dev, sms, s);
}
