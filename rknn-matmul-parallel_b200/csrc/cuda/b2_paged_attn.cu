// Attention of a batch's new rows over a paged KV cache (b2_attention_paged).
//
//   s_ij = q_i . k_j / sqrt(hd)   for the mapped slots j up to row i's own,
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,   lse_i = m_i + ln l_i,
// with the running maximum m and sum l of one pass over the slots (the online
// softmax): a new maximum rescales what was summed before it.
#include <algorithm>

#include "b2_paged.cuh"

namespace {

using namespace b2p;

// The weights are formed as 2^(s - m + kUp) with s and m in units of log2: the
// FP16 copy that the product with V takes then keeps 11 bits down to 2^-28 of
// the row's largest weight, where weights of a long row lie.  Sums carry the
// same factor, which the division by l takes out.
constexpr float kUp = 14.f;

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// ─── few rows per sequence: decode steps, drafted tokens ───
//
// Bound by reading K and V once from HBM.  A tile is T tokens x the G q heads
// of one kv head, at most R = 8 NT rows.  The work of the call is one line of
// blocks of 64 slots: sequences, then tiles and kv heads, then the tile's
// blocks.  Every CTA takes an equal stretch of that line, so sequences of any
// mix of lengths load the SMs evenly; a tile that a stretch boundary cuts is
// summed in pieces, which the last CTA to arrive merges in the line's order.
// A boundary near a tile's end moves there.
//
// One step of 64 sequences of up to 4096 slots, 8 kv heads, hd 128: 55 us, 0.80
// of the measured copy rate (50 without computing and merging); one step of a
// context of 200 thousand slots, 2 kv heads: 45 us, 0.70, of which two levels of
// merging 148 pieces of a head take 9.
//
// A producer warp walks the stretch: for each tile it copies the Q rows, then
// the K and V blocks through the page table into a ring of stages, across tile
// boundaries.  Four warps compute, each on 16 slots of a stage:
//   S^T = K Q^T    mma m16n8k16: slots are the M rows, the tile's rows the N
//                  columns;
//   O^T += V^T P^T the head dims are M, the slots K; P^T moves from the
//                  accumulator to the B-operand layout with movmatrix.
constexpr int kBlk = 64;
constexpr int kThreads = 160;  // four computing warps, one producer
constexpr int kMinBlocks = 2;  // shortest stretch of a CTA
constexpr int kFan = 16;       // pieces that one CTA merges; more are merged in two levels

// A stretch's part of one tile: blocks [b0, b1) of the tile's nb.
struct Seg {
    int g, i0, rows_t;  // kv head, first token, tokens
    int b0, b1, live;   // live: end of the blocks that some row of the tile sees
    int nb, x0;         // the tile's blocks, and where it starts on the line
    int s;
    Seq sq;
};

template <int HD, int NT>
struct Short {
    static constexpr int R = 8 * NT;
    static constexpr int kStage = kBlk * HD * 4;  // K and V, bytes
    static constexpr int kStages = HD == 128 ? 3 : 6;
    static constexpr int kQ = NT == 1 || HD == 64 ? 2 : 1;  // Q tiles ahead: what two CTAs per SM leave room for
    static constexpr int kLdQ = HD + 8;           // row of a Q tile (halves): eight rows hit distinct banks
    // Row of the merge buffer: + 4 lets the four lane columns hit distinct banks,
    // where two CTAs per SM leave room for it.
    static constexpr int kLd = HD + (NT == 1 || HD == 64 ? 4 : 0);
    // Floats of one partial tile: o[R][HD], (m, l)[R], (m, l)[R] of a first merge.
    static constexpr int kTile = R * (HD + 4);
    static constexpr int kFrag = HD / 16 * 32 * 4;  // floats of one warp's O for one column group
    static constexpr int kMerge = 2 * kFrag > R * kLd ? 2 * kFrag : R * kLd;
};

template <int HD, int NT>
struct ShortSmem {
    alignas(1024) unsigned char ring[Short<HD, NT>::kStages * Short<HD, NT>::kStage];
    float o[Short<HD, NT>::kMerge];
    alignas(16) __half q[Short<HD, NT>::kQ][Short<HD, NT>::R * Short<HD, NT>::kLdQ];
    float m[4][Short<HD, NT>::R], l[4][Short<HD, NT>::R];
    uint64_t full[Short<HD, NT>::kStages], empty[Short<HD, NT>::kStages];
    uint64_t q_full[Short<HD, NT>::kQ], q_empty[Short<HD, NT>::kQ];
    Seg seg[Short<HD, NT>::kQ];
    int mapped[Short<HD, NT>::kStages];  // bit w: the 16 slots of warp w are mapped
    volatile int failed[2];  // some warp's wait ran out; polls after which one does
    volatile int copied, q_copied;  // blocks and Q tiles that the producer has asked for
    int last;
    int pre[B2_PAGED_MAX_SEQS + 1];
};

// Where the stretch of CTA c begins.  T: tokens of one tile.
__device__ __forceinline__ int stretch_start(const AttnParams& p, const int* pre, int W, int per, int c) {
    const long long at = (long long)c * per;
    if (at >= W) return W;
    const int x = (int)at, s = prefix_find(pre, p.bt.n_seqs, x);
    const int nb = max(1, cdiv(p.bt.seq(s).len, kBlk));
    return snap_to(x, (x - pre[s]) % nb, nb, per);
}

__device__ __forceinline__ Seg find_seg(const AttnParams& p, int T, const int* pre, int x, int x1) {
    Seg r;
    r.s = prefix_find(pre, p.bt.n_seqs, x);
    r.sq = p.bt.seq(r.s);
    r.nb = max(1, cdiv(r.sq.len, kBlk));
    const int off = x - pre[r.s], item = off / r.nb;
    r.b0 = off - item * r.nb;
    r.b1 = min(r.nb, r.b0 + (x1 - x));
    r.x0 = x - r.b0;
    r.g = item % p.nkv;
    r.i0 = item / p.nkv * T;
    r.rows_t = min(T, min(r.sq.Q, p.max_q) - r.i0);
    const int end = min(r.sq.len, max(0, r.sq.base + r.i0 + r.rows_t));
    r.live = min(r.b1, cdiv(end, kBlk));
    return r;
}

// The rows of a tile from pieces of CTAs first, first + step, ... (n of them, own
// the one that begins the tile): to the outputs, or to the slot of `first`.
template <int HD, int NT>
__device__ __forceinline__ void merge_pieces(const AttnParams& p, const Seg& sg, int own, int first, int step, int n,
                                             bool final) {
    using C = Short<HD, NT>;
    constexpr int kWide = 16;
    const int rows = sg.rows_t * p.G, ml0 = C::R * (HD + (step > 1 ? 2 : 0));
    auto slot = [&](int i) {
        const int c = first + i * step;
        return p.part + (size_t)(2 * c + (c == own)) * C::kTile;
    };
    const int all = rows * (HD / 4);
    for (int i0 = threadIdx.x; i0 < (all + 31) / 32 * 32; i0 += 128) {
        const int i = min(i0, all - 1), r = i / (HD / 4), c = i % (HD / 4) * 4;
        float M = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        // kWide pieces in flight: the loads' latency is what a merge costs
        for (int j0 = 0; j0 < n; j0 += kWide) {
            float2 ml[kWide];
            float4 o[kWide];
#pragma unroll
            for (int j = 0; j < kWide; j++) {
                const float* q = slot(min(j0 + j, n - 1));
                ml[j] = ld_cg2(q + ml0 + 2 * r);
                o[j] = ld_cg4(q + r * HD + c);
            }
            // No load moves behind this: left alone the compiler puts each load in front of its use,
            // and a merge of 16 pieces waits 16 times (8.5 instead of 2.9 us).
            __syncwarp();
            float top = M;
#pragma unroll
            for (int j = 0; j < kWide; j++) top = fmaxf(top, ml[j].x);
            const float f = piece_weight(M, top);
            M = top;
            l *= f;
            acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
#pragma unroll
            for (int j = 0; j < kWide; j++) {
                if (j0 + j >= n) break;
                const float w = piece_weight(ml[j].x, M);
                l = fmaf(ml[j].y, w, l);
                acc.x = fmaf(o[j].x, w, acc.x);
                acc.y = fmaf(o[j].y, w, acc.y);
                acc.z = fmaf(o[j].z, w, acc.z);
                acc.w = fmaf(o[j].w, w, acc.w);
            }
        }
        if (i0 >= all) continue;
        if (final) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const size_t row = (size_t)(sg.sq.row0 + sg.i0 + r / p.G);
            const int h = sg.g * p.G + r % p.G;
            uint2 u;
            u.x = pack_h2(acc.x * inv, acc.y * inv);
            u.y = pack_h2(acc.z * inv, acc.w * inv);
            *reinterpret_cast<uint2*>(p.out16 + (row * p.nq + h) * HD + c) = u;
            if (c == 0 && p.lse) p.lse[row * p.nq + h] = l == 0.f ? -INFINITY : (M - kUp) * kLn2 + logf(l);
        } else {
            *reinterpret_cast<float4*>(slot(0) + r * HD + c) = acc;
            if (c == 0) *reinterpret_cast<float2*>(slot(0) + C::R * (HD + 2) + 2 * r) = make_float2(M, l);
        }
    }
}

// ─── the long kernel's pieces ───
//
// Tile pairs that it left in pieces, by the four computing warps, one row per
// thread.  A task is CC chunks of four dims of one tile; the tasks of all pairs
// go round the CTAs.  NB pieces are in flight at a time: bound by reading them.
template <int HD, int CC, int NB>
__device__ __forceinline__ void merge_task(const AttnParams& p, int owner, const Cut& cut, int t, int c0) {
    const int r = threadIdx.x, T = kLongRows / p.G, tok = r / p.G;
    const bool live = tok < min(T, cut.tokens - t * T);
    if (!__any_sync(0xffffffffu, live)) return;
    const int ml0 = 2 * kLongRows * HD + 2 * (t * kLongRows + r), o0 = (t * (HD / 4) + c0) * kLongRows * 4 + 4 * r;
    float M = -INFINITY, l = 0.f;
    float4 acc[CC];
#pragma unroll
    for (int c = 0; c < CC; c++) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < cut.pieces; j0 += NB) {
        float2 ml[NB];
        float4 o[NB][CC];
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int i = min(j0 + j, cut.pieces - 1);
            const float* q = p.long_part + (size_t)(2 * (owner + i) + (i == 0)) * long_piece_floats(HD);
            ml[j] = ld_cg2(q + ml0);
#pragma unroll
            for (int c = 0; c < CC; c++) o[j][c] = ld_cg4(q + o0 + c * kLongRows * 4);
        }
        __syncwarp();  // no load moves behind this
        float top = M;
#pragma unroll
        for (int j = 0; j < NB; j++) top = fmaxf(top, ml[j].x);
        const float f = piece_weight(M, top);
        M = top;
        l *= f;
#pragma unroll
        for (int c = 0; c < CC; c++) acc[c].x *= f, acc[c].y *= f, acc[c].z *= f, acc[c].w *= f;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            if (j0 + j >= cut.pieces) break;
            const float w = piece_weight(ml[j].x, M);
            l = fmaf(ml[j].y, w, l);
#pragma unroll
            for (int c = 0; c < CC; c++) {
                acc[c].x = fmaf(o[j][c].x, w, acc[c].x);
                acc[c].y = fmaf(o[j][c].y, w, acc[c].y);
                acc[c].z = fmaf(o[j][c].z, w, acc[c].z);
                acc[c].w = fmaf(o[j][c].w, w, acc[c].w);
            }
        }
    }
    if (!live) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t row = (size_t)(cut.row0 + t * T + tok);
    const int h = cut.g * p.G + r % p.G;
    __half* dst = p.out16 + (row * p.nq + h) * HD + 4 * c0;
#pragma unroll
    for (int c = 0; c < CC; c++) {
        uint2 u;
        u.x = pack_h2(acc[c].x * inv, acc[c].y * inv);
        u.y = pack_h2(acc[c].z * inv, acc[c].w * inv);
        *reinterpret_cast<uint2*>(dst + 4 * c) = u;
    }
    if (c0 == 0 && p.lse) p.lse[row * p.nq + h] = l == 0.f ? -INFINITY : M * kLn2 + logf(l);
}

// scratch: kMergeInts ints that only the four computing warps touch.
constexpr int kMergeInts = kMaxLongCtas + 1 + 4;
template <int HD>
__device__ __forceinline__ void merge_long(const AttnParams& p, int* scratch) {
    constexpr int kMaxCuts = kMaxLongCtas;
    static_assert(kMaxCuts == 2 * 128, "two cuts per thread");
    constexpr int kFew = 16;  // pieces up to which a task takes four chunks; more pieces, more tasks
    int* before = scratch;    // tasks of the cuts before each
    int* sums = scratch + kMaxCuts + 1;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto tasks_of = [&](const Cut& c) {
        if (c.pieces == 0) return 0;
        const int tiles = c.tokens > kLongRows / p.G ? 2 : 1;
        return tiles * (c.pieces <= kFew ? HD / 16 : HD / 4);
    };
    auto cut_at = [&](int i) {
        const int4 v = i < p.long_ctas ? __ldcg(reinterpret_cast<const int4*>(p.cuts + i)) : make_int4(0, 0, 0, 0);
        return Cut{v.x, v.y, v.z, v.w};
    };
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int a = tasks_of(cut_at(2 * tid)), b = tasks_of(cut_at(2 * tid + 1));
    int incl = a + b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    if (lane == 31) sums[warp] = incl;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int w = 0; w < warp; w++) incl += sums[w];
    before[2 * tid] = incl - a - b;
    before[2 * tid + 1] = incl - b;
    if (tid == 127) before[kMaxCuts] = incl;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int total = before[kMaxCuts];
    for (int k = blockIdx.x; k < total; k += gridDim.x) {
        const int i = prefix_find(before, kMaxCuts, k), rest = k - before[i];
        const Cut cut = cut_at(i);
        const bool few = cut.pieces <= kFew;
        const int per_tile = few ? HD / 16 : HD / 4;
        if (few) merge_task<HD, 4, 4>(p, i, cut, rest / per_tile, rest % per_tile * 4);
        else merge_task<HD, 1, 16>(p, i, cut, rest / per_tile, rest % per_tile);
    }
}

template <int HD, int NT>
__global__ void __launch_bounds__(kThreads, 2) attn_short_kernel(const __grid_constant__ CUtensorMap tk,
                                                                 const __grid_constant__ CUtensorMap tv,
                                                                 const AttnParams p) {
    using C = Short<HD, NT>;
    constexpr int R = C::R;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    ShortSmem<HD, NT>& sm = *reinterpret_cast<ShortSmem<HD, NT>*>(smem_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 4);
        }
        for (int i = 0; i < C::kQ; i++) {
            mbar_init(&sm.q_full[i], 1);
            mbar_init(&sm.q_empty[i], 4);
        }
        sm.failed[0] = 0;
        sm.failed[1] = p.limit;
        sm.copied = sm.q_copied = 0;
        mbar_init_fence();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
    }
    b2::pdl_trigger();
    // Behind the long kernel this grid begins on the SMs whose long CTA is done (no SM has
    // shared memory for both) and waits for the others only before it merges.
    int before = 0;
    if (!p.long_ctas) {
        b2::pdl_wait();
    } else {
        if (threadIdx.x == 0) sm.last = was_told(p);
        __syncthreads();
        if (!sm.last) b2::pdl_wait();
        if (threadIdx.x == 0) before = atomicAdd(waited_word(p), 1);
        // what the kernels before wrote, for the copies too
        asm volatile("fence.proxy.async.global;" ::: "memory");
    }
    const int T = R / p.G;
    prefix_work(sm.pre, p.bt.n_seqs, [&](int s) {
        const Seq q = p.bt.seq(s);
        const int n = min(q.Q, p.max_q);
        return n * p.G > p.short_rows ? 0 : cdiv(n, T) * p.nkv * max(1, cdiv(q.len, kBlk));
    });
    if (before == kWaited + (int)gridDim.x - 1) *waited_word(p) = 0;  // (only where a long kernel ran)
    const int W = sm.pre[p.bt.n_seqs];
    const int per = max(kMinBlocks, cdiv(W, gridDim.x));
    const int x0 = stretch_start(p, sm.pre, W, per, blockIdx.x), x1 = stretch_start(p, sm.pre, W, per, blockIdx.x + 1);
    const int page_rows = 1 << p.bt.page_shift, box_rows = min(page_rows, kBlk);
    volatile int* failed = sm.failed;

    if (warp == 4) {  // producer: lane i copies the i-th box of a stage and the i-th row of a Q tile
        const int boxes = kBlk / box_rows, box_bytes = box_rows * HD * 2;
        int k = 0, n = 0;
        bool ok = true;
        for (int x = x0; x < x1 && ok; n++) {
            const Seg g = find_seg(p, T, sm.pre, x, x1);
            x += g.b1 - g.b0;
            const int qb = n % C::kQ, rows = g.rows_t * p.G;
            // page ids of the next 32 boxes, one per lane
            int ids_from = g.b0, id = -1;
            auto load_ids = [&]() {
                const int j = ids_from * kBlk + lane * box_rows;
                id = j < g.sq.len && ids_from + lane / boxes < g.live ? p.bt.page(g.s, j) : -1;
            };
            load_ids();
            if (n >= C::kQ) ok = warp_wait(&sm.q_empty[qb], (n / C::kQ - 1) & 1, failed);
            if (!ok) break;
            if (lane == 0) {
                sm.seg[qb] = g;
                sm.q_copied = n + 1;
                mbar_expect_tx(&sm.q_full[qb], rows * HD * 2);
            }
            __syncwarp();
            if (lane < rows)
                bulk_copy(sm.q[qb] + lane * C::kLdQ,
                          p.q16 + (size_t)(g.sq.row0 + g.i0 + lane / p.G) * p.ldq + (size_t)(g.g * p.G + lane % p.G) * HD,
                          HD * 2, &sm.q_full[qb]);
            for (int b = g.b0; b < g.live; b++, k++) {
                const int st = k % C::kStages, j = b * kBlk + lane * box_rows;
                if ((b - ids_from + 1) * boxes > 32) {
                    ids_from = b;
                    load_ids();
                }
                const int mine = __shfl_sync(0xffffffffu, id, ((b - ids_from) * boxes + lane) & 31);
                const int page = lane < boxes ? mine : -1;
                if (k >= C::kStages) ok = warp_wait(&sm.empty[st], (k / C::kStages - 1) & 1, failed);
                if (!ok) break;
                const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
                if (lane == 0) {
                    int bits = 0;
                    for (int w = 0; w < 4; w++) bits |= (have >> (w * 16 / box_rows) & 1) << w;
                    sm.mapped[st] = bits;
                    sm.copied = k + 1;
                    mbar_expect_tx(&sm.full[st], __popc(have) * 2 * box_bytes);
                }
                __syncwarp();
                if (page >= 0) {
                    unsigned char* dst = sm.ring + st * C::kStage + lane * box_bytes;
                    const int row = j & (page_rows - 1);
                    tma_load_5d(dst, &tk, 0, row, 0, g.g, page, &sm.full[st]);
                    tma_load_5d(dst + C::kStage / 2, &tv, 0, row, 0, g.g, page, &sm.full[st]);
                }
            }
        }
        __syncthreads();  // no warp waits for copies any more
        if (*failed && lane == 0) {
            // some warp may have given up with copies in flight, which the CTA must not end before
            atomicExch(p.err, 1);
            copies_land(sm.full, C::kStages, sm.copied);
            copies_land(sm.q_full, C::kQ, sm.q_copied);
        }
        return;
    }

    const float scale = kLog2e / sqrtf((float)HD);  // to log2 units
    const int pw = warp * 16;
    const int bshift = box_rows == 16 ? 4 : box_rows == 32 ? 5 : 6;
    const int tid = threadIdx.x;
    auto sync4 = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    int k = 0, n = 0;
    bool ok = true;
    for (int x = x0; x < x1; n++) {
        const int qi = n % C::kQ;
        ok = warp_wait(&sm.q_full[qi], (n / C::kQ) & 1, failed);
        const Seg sg = sm.seg[qi];
        x += sg.b1 - sg.b0;
        const int rows = sg.rows_t * p.G;  // rows of the tile: token i0 + r / G, q head g G + r % G
        uint32_t qb[HD / 16][NT][2];
        int lim[NT][2];  // last slot that this lane's two columns see
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const __half* qp = sm.q[qi] + (8 * t + (lane >> 2)) * C::kLdQ + 2 * (lane & 3);
#pragma unroll
            for (int i = 0; i < HD / 16; i++) {
                qb[i][t][0] = *reinterpret_cast<const uint32_t*>(qp + 16 * i);
                qb[i][t][1] = *reinterpret_cast<const uint32_t*>(qp + 16 * i + 8);
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int c = 8 * t + 2 * (lane & 3) + j;
                lim[t][j] = c < rows ? min(sg.sq.len - 1, sg.sq.base + sg.i0 + c / p.G) : -1;
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_empty[qi]);
        float o[HD / 16][NT][4], mx[NT][2], ls[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int i = 0; i < HD / 16; i++) o[i][t][0] = o[i][t][1] = o[i][t][2] = o[i][t][3] = 0.f;
            mx[t][0] = mx[t][1] = -INFINITY;
            ls[t][0] = ls[t][1] = 0.f;
        }
        for (int b = sg.b0; b < sg.live && ok; b++, k++) {
            const int st = k % C::kStages;
            ok = warp_wait(&sm.full[st], (k / C::kStages) & 1, failed);
            if (!ok) break;
            unsigned char* stage = sm.ring + st * C::kStage;
            const int j0 = b * kBlk + pw, np = sg.sq.len - j0;  // np: cached slots from this warp's first
            if ((sm.mapped[st] >> warp & 1) && np > 0) {
                // this warp's 16 rows within their box: [dims 0-63, 64-127][box_rows][128 bytes]
                const uint32_t bo = (pw >> bshift) * box_rows * HD * 2 + (pw & (box_rows - 1)) * 128;
                const uint32_t half = box_rows * 128;
                const uint32_t ka = smem_u32(stage) + bo, va = ka + C::kStage / 2;
                if (np < 16) {
                    // V rows past kv_len may hold anything: zero them (their P is zero, and 0 x inf is not)
                    for (int r = np + (lane >> 4); r < 16; r += 2) {
                        const int c = lane & 15;
                        if (c < HD / 8)
                            *reinterpret_cast<uint4*>(stage + C::kStage / 2 + bo + (c >> 3) * half + r * 128 +
                                                      (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    // ordered before the next copy into this stage
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                float sc[NT][4];
#pragma unroll
                for (int t = 0; t < NT; t++) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
                for (int i = 0; i < HD / 16; i++) {
                    // K rows (+8 for odd lane groups), dims 16 i (+8 for the upper two groups)
                    const int r = (lane & 7) + ((lane >> 3) & 1) * 8, d = 16 * i + (lane >> 4) * 8;
                    uint32_t a[4];
                    ldsm_x4(ka + (d >> 6) * half + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4), a);
#pragma unroll
                    for (int t = 0; t < NT; t++) mma16816(sc[t], a, qb[i][t][0], qb[i][t][1]);
                }
                const int ja = j0 + (lane >> 2), jb = ja + 8;
                uint32_t pb[NT][2];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float pr[4], corr[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float sa = ja <= lim[t][j] ? sc[t][j] * scale : -INFINITY;
                        const float sb = jb <= lim[t][j] ? sc[t][j + 2] * scale : -INFINITY;
                        float cm = fmaxf(sa, sb);
                        cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, 4));
                        cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, 8));
                        cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, 16));
                        const float mn = fmaxf(mx[t][j], cm);
                        const float ref = mn == -INFINITY ? 0.f : mn - kUp;
                        corr[j] = mn == -INFINITY ? 1.f : ex2(mx[t][j] - mn);
                        pr[j] = ex2(sa - ref);
                        pr[j + 2] = ex2(sb - ref);
                        ls[t][j] = fmaf(ls[t][j], corr[j], pr[j] + pr[j + 2]);  // this lane's slots only
                        mx[t][j] = mn;
                    }
#pragma unroll
                    for (int i = 0; i < HD / 16; i++) {
                        o[i][t][0] *= corr[0];
                        o[i][t][1] *= corr[1];
                        o[i][t][2] *= corr[0];
                        o[i][t][3] *= corr[1];
                    }
                    pb[t][0] = movm_t(pack_h2(pr[0], pr[1]));
                    pb[t][1] = movm_t(pack_h2(pr[2], pr[3]));
                }
                // An infinite or NaN V at a slot that some row does not see would reach that row too
                // (0 x inf): added to the rows that see it, whose weight changes nothing in it, and zeroed.
                if (B2_RARE(min(j0 + 15, sg.sq.len - 1) > sg.sq.base + sg.i0)) {
                    unsigned char* v = stage + C::kStage / 2 + bo;
                    bool bad = false;
                    for (int i = lane; i < 16 * (HD / 8); i += 32)
                        bad |= non_finite8(*reinterpret_cast<const uint4*>(v + (i % (HD / 8) >> 3) * half +
                                                                           i / (HD / 8) * 128 + (i & 7) * 16));
                    if (__any_sync(0xffffffffu, bad)) {
                        auto at = [&](int r, int d) {
                            return reinterpret_cast<__half*>(v + (d >> 6) * half + r * 128 +
                                                             ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 7) * 2);
                        };
#pragma unroll 1
                        for (int r = 0; r < 16; r++) {
#pragma unroll
                            for (int i = 0; i < HD / 16; i++)
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const float x = __half2float(*at(r, 16 * i + (lane >> 2) + (e >> 1) * 8));
#pragma unroll
                                    for (int t = 0; t < NT; t++)
                                        if (!isfinite(x) && j0 + r <= lim[t][e & 1]) o[i][t][e] += x;
                                }
                        }
                        __syncwarp();
#pragma unroll 1
                        for (int i = lane; i < 16 * HD; i += 32)
                            if (!isfinite(__half2float(*at(i / HD, i % HD)))) *at(i / HD, i % HD) = __float2half(0.f);
                        // ordered before the next copy into this stage
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                }
#pragma unroll
                for (int i = 0; i < HD / 16; i++) {
                    // V^T: dims 16 i (+8 for odd lane groups), slots (+8 for the upper two groups)
                    const int r = (lane & 7) + (lane >> 4) * 8, d = 16 * i + ((lane >> 3) & 1) * 8;
                    uint32_t a[4];
                    ldsm_x4_t(va + (d >> 6) * half + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4), a);
#pragma unroll
                    for (int t = 0; t < NT; t++) mma16816(o[i][t], a, pb[t][0], pb[t][1]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[st]);
        }
        // Merge the four warps' states: 2 into 0 and 3 into 1, then 1 into 0.
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                ls[t][j] += __shfl_xor_sync(0xffffffffu, ls[t][j], 4);
                ls[t][j] += __shfl_xor_sync(0xffffffffu, ls[t][j], 8);
                ls[t][j] += __shfl_xor_sync(0xffffffffu, ls[t][j], 16);
            }
        }
        auto give = [&](int t, float* to) {
            if (lane < 4) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    sm.m[warp][8 * t + 2 * lane + j] = mx[t][j];
                    sm.l[warp][8 * t + 2 * lane + j] = ls[t][j];
                }
            }
#pragma unroll
            for (int i = 0; i < HD / 16; i++)
                *reinterpret_cast<float4*>(to + (i * 32 + lane) * 4) = make_float4(o[i][t][0], o[i][t][1], o[i][t][2], o[i][t][3]);
        };
        auto take = [&](int t, const float* from, int w) {
            float fa[2], fb[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int c = 8 * t + 2 * (lane & 3) + j;
                const float m2 = sm.m[w][c], l2 = sm.l[w][c], M = fmaxf(mx[t][j], m2);
                fa[j] = piece_weight(mx[t][j], M);
                fb[j] = piece_weight(m2, M);
                ls[t][j] = ls[t][j] * fa[j] + l2 * fb[j];
                mx[t][j] = M;
            }
#pragma unroll
            for (int i = 0; i < HD / 16; i++) {
                const float4 v = *reinterpret_cast<const float4*>(from + (i * 32 + lane) * 4);
                o[i][t][0] = o[i][t][0] * fa[0] + v.x * fb[0];
                o[i][t][1] = o[i][t][1] * fa[1] + v.y * fb[1];
                o[i][t][2] = o[i][t][2] * fa[0] + v.z * fb[0];
                o[i][t][3] = o[i][t][3] * fa[1] + v.w * fb[1];
            }
        };
        int bad = 0;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (warp >= 2) give(t, sm.o + (warp - 2) * C::kFrag);
            if (t == 0) {
                // one decision for the four warps: a failed wait ends the stretch
                asm volatile(
                    "{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.s32 "
                    "%0, 1, 0, q;\n}\n"
                    : "=r"(bad)
                    : "r"(ok ? 0 : 1)
                    : "memory");
                if (bad) break;
            } else {
                sync4();
            }
            if (warp < 2) take(t, sm.o + warp * C::kFrag, warp + 2);
            if (warp == 1) give(t, sm.o + C::kFrag);
            sync4();
            if (warp == 0) take(t, sm.o + C::kFrag, 1);
            if (t + 1 < NT) sync4();
        }
        if (bad) {
            ok = false;
            break;
        }
        // Warp 0 has the sum: through shared memory to rows.
        if (warp == 0) {
            __syncwarp();
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int c = 8 * t + 2 * (lane & 3);
#pragma unroll
                for (int i = 0; i < HD / 16; i++) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        sm.o[(c + (e & 1)) * C::kLd + 16 * i + (lane >> 2) + (e >> 1) * 8] = o[i][t][e];
                }
                if (lane < 4) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        sm.m[0][c + j] = mx[t][j];
                        sm.l[0][c + j] = ls[t][j];
                    }
                }
            }
        }
        sync4();
        int own, last;  // CTAs of the tile's pieces
        cut_of(sg.x0, sg.nb, per, own, last);
        const bool whole = own >= last;
        float* part = p.part + (size_t)(2 * blockIdx.x + (sg.b0 == 0 ? 1 : 0)) * C::kTile;
        for (int i = tid; i < rows * (HD / 8); i += 128) {
            const int r = i / (HD / 8), c = i % (HD / 8) * 8;
            const float M = sm.m[0][r], l = sm.l[0][r];
            const float4 u = *reinterpret_cast<const float4*>(&sm.o[r * C::kLd + c]);
            const float4 v = *reinterpret_cast<const float4*>(&sm.o[r * C::kLd + c + 4]);
            if (whole) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const size_t row = (size_t)(sg.sq.row0 + sg.i0 + r / p.G);
                const int h = sg.g * p.G + r % p.G;
                uint4 w;
                w.x = pack_h2(u.x * inv, u.y * inv);
                w.y = pack_h2(u.z * inv, u.w * inv);
                w.z = pack_h2(v.x * inv, v.y * inv);
                w.w = pack_h2(v.z * inv, v.w * inv);
                *reinterpret_cast<uint4*>(p.out16 + (row * p.nq + h) * HD + c) = w;
                if (c == 0 && p.lse) p.lse[row * p.nq + h] = l == 0.f ? -INFINITY : (M - kUp) * kLn2 + logf(l);
            } else {
                *reinterpret_cast<float4*>(part + r * HD + c) = u;
                *reinterpret_cast<float4*>(part + r * HD + c + 4) = v;
                if (c == 0) *reinterpret_cast<float2*>(part + R * HD + 2 * r) = make_float2(M, l);
            }
        }
        if (!whole) {
            // true for the CTA that finds the other n - 1 arrivals counted (and resets the count)
            auto last_of = [&](int* count, int all) {
                // One thread's release behind the barrier covers the CTA's stores, and its acquire
                // the loads behind the next one.
                sync4();
                if (tid == 0) {
                    int was;
                    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(was) : "l"(count) : "memory");
                    sm.last = was == all - 1;
                    if (was == all - 1) *count = 0;
                }
                sync4();
                return sm.last != 0;
            };
            const int pieces = last - own + 1, me = (int)blockIdx.x;
            if (pieces <= kFan) {
                if (last_of(p.counters + 2 * own + 1, pieces)) merge_pieces<HD, NT>(p, sg, own, own, 1, pieces, true);
            } else {
                const int first = own + (me - own) / kFan * kFan, some = min(kFan, last - first + 1);
                if (last_of(p.counters + 2 * first + (first == own), some)) {
                    merge_pieces<HD, NT>(p, sg, own, first, 1, some, false);
                    if (last_of(p.counters + 2 * gridDim.x + own, cdiv(pieces, kFan)))
                        merge_pieces<HD, NT>(p, sg, own, own, kFan, cdiv(pieces, kFan), true);
                }
            }
        }
        sync4();  // the merge area is free for the next tile
    }
    __syncthreads();
    if (p.long_ctas) {
        b2::pdl_wait();
        // (not over sm.pre: nothing orders a CTA without a tile behind its producer's reads of that)
        static_assert(sizeof(sm.o) >= kMergeInts * sizeof(int), "scratch of the merge");
        merge_long<HD>(p, reinterpret_cast<int*>(sm.o));
    }
}

constexpr int kMaxGroup = 16;
// (token, head) rows of a kv head up to which this file's kernel takes a sequence: one
// tile, so that K and V are read once.  Two q heads each, 8 kv heads, hd 128, 128 to
// 4096 slots: 8 tokens, 16 rows, take 83 us for 64 sequences (30 for 8, 205 for 200)
// here and 137 (39, 370) in the chunk kernel; 9 tokens, as two tiles, 138 (32, 382) here
// and 138 (38, 371) there, 16 tokens 144 (32, 393) and 142 (38, 372).
constexpr int kShortRows = 16;
constexpr size_t kCounterBytes = kCounters * sizeof(int), kCutBytes = kMaxLongCtas * sizeof(Cut);

// CTAs of a launch: one or two per SM.
template <int HD, int NT>
int short_grid(int dev, int sms) {
    static std::atomic<int> per[64];
    std::atomic<int>& c = per[dev & 63];
    int n = c.load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attn_short_kernel<HD, NT>, kThreads,
                                                          sizeof(ShortSmem<HD, NT>)) != cudaSuccess || n < 1)
            n = 1;
        n = n < 2 ? n : 2;
        c.store(n, std::memory_order_relaxed);
    }
    return n * sms;
}

template <int HD, int NT>
int launch_short(const AttnParams& p, const B2PagedKV* kv, int dev, int sms, long long blocks, cudaStream_t s) {
    static std::atomic<unsigned long long> done{0};
    constexpr size_t smem = sizeof(ShortSmem<HD, NT>);
    static_assert(smem <= 115712, "two CTAs per SM");
    cudaError_t e = allow_smem(attn_short_kernel<HD, NT>, smem, done, dev);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged smem: %s", cudaGetErrorString(e));
    CUtensorMap tk, tv;
    const int box = kv->page_size < kBlk ? kv->page_size : kBlk;
    int rc = b2_paged_map(&tk, kv->k_pages, kv, p.nkv, HD, box, HD / 64);
    if (!rc) rc = b2_paged_map(&tv, kv->v_pages, kv, p.nkv, HD, box, HD / 64);
    if (rc) return rc;
    long long grid = std::min<long long>(short_grid<HD, NT>(dev, sms), (kCounters - 1) / 3);
    if (!p.long_ctas && grid > (blocks + kMinBlocks - 1) / kMinBlocks) grid = (blocks + kMinBlocks - 1) / kMinBlocks;
    e = b2::launch_pdl(attn_short_kernel<HD, NT>, dim3((unsigned)grid), dim3(kThreads), smem, s, tk, tv, p);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged: %s", cudaGetErrorString(e));
    return 0;
}

int device_sms(int* dev) {
    int sms = 148;
    *dev = 0;
    cudaGetDevice(dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, *dev);
    return sms;
}

// Workspace: counters, cuts, the short kernel's pieces (two of up to 16 rows for
// each of at most two CTAs per SM), the long kernel's (two per SM).
size_t short_part_bytes(int sms, int hd) { return (size_t)sms * 2 * 2 * kShortRows * (hd + 4) * sizeof(float); }

}  // namespace

extern "C" size_t b2_attention_paged_workspace(int n_seqs, int max_q, int nq, int nkv, int hd) {
    int dev;
    const int sms = device_sms(&dev);
    const bool any_long = n_seqs > 0 && nkv > 0 && (long long)max_q * nq > (long long)kShortRows * nkv;
    return kCounterBytes + kCutBytes + short_part_bytes(sms, hd) +
           (any_long ? (size_t)sms * 2 * long_piece_floats(hd) * sizeof(float) : 0);
}

extern "C" int b2_attention_paged(uint16_t* out16, float* lse, const uint16_t* q16, int ldq, int M, int max_q, int nq,
                                  int nkv, int hd, const B2PagedKV* kv, void* work, int* err, b2_stream_t s) {
    int rc = b2_paged_check("b2_attention_paged", kv, nkv, hd, true);
    if (rc) return rc;
    if ((M > 0 && (!out16 || !q16)) || !work || !err || M < 0 || max_q < 0 || nq <= 0 || nq % nkv || nq / nkv > kMaxGroup)
        return b2_set_error(B2_ERR_INVALID_ARG, "b2_attention_paged: bad arguments (nq a multiple of nkv, at most %d)",
                            kMaxGroup);
    if (ldq < (long long)nq * hd || ldq % 8 || (reinterpret_cast<uintptr_t>(q16) & 15) || (reinterpret_cast<uintptr_t>(out16) & 15) ||
        (reinterpret_cast<uintptr_t>(work) & 15))
        return b2_set_error(B2_ERR_INVALID_ARG,
                            "b2_attention_paged: q16, out16 and work must be 16-byte aligned, ldq a multiple of 8 that "
                            "holds every head");
    if (M == 0 || kv->n_seqs == 0 || max_q == 0) return 0;
    if (max_q > M) max_q = M;
    int dev;
    const int sms = device_sms(&dev);
    const int G = nq / nkv;
    const long long rows = (long long)max_q * G;
    unsigned char* w = reinterpret_cast<unsigned char*>(work);
    AttnParams p{make_batch(kv, M), reinterpret_cast<const __half*>(q16), ldq, reinterpret_cast<__half*>(out16), lse, max_q,
                 nq, nkv, G, kShortRows, reinterpret_cast<int*>(w),
                 reinterpret_cast<float*>(w + kCounterBytes + kCutBytes), reinterpret_cast<Cut*>(w + kCounterBytes),
                 reinterpret_cast<float*>(w + kCounterBytes + kCutBytes + short_part_bytes(sms, hd)), 0, err, wait_limit()};
    // the line's length when every sequence fills its table: what the kernel's 32-bit places must hold
    const long long cap = ((long long)kv->max_pages * kv->page_size + kBlk - 1) / kBlk;
    const long long tiles = (long long)kv->n_seqs * kShortRows;
    const long long blocks = (tiles < M + 0ll ? tiles : (long long)M) * nkv * cap;
    if (blocks >= (1ll << 31) - 65536)
        return b2_set_error(B2_ERR_INVALID_ARG, "b2_attention_paged: %lld blocks of work in one call", blocks);
    cudaStream_t st = (cudaStream_t)s;
    if (rows > kShortRows) {
        rc = b2_paged_attention_long(p, kv, hd, dev, sms, st);
        if (rc) return rc;
    }
    if (rows <= 8) return hd == 128 ? launch_short<128, 1>(p, kv, dev, sms, blocks, st) : launch_short<64, 1>(p, kv, dev, sms, blocks, st);
    return hd == 128 ? launch_short<128, 2>(p, kv, dev, sms, blocks, st) : launch_short<64, 2>(p, kv, dev, sms, blocks, st);
}
