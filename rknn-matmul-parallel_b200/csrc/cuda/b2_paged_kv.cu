// Writing a paged KV cache: new rows (b2_qk_rope_kv_paged) and eviction by
// accumulated attention weight (b2_kv_evict_paged).
#include "b2_paged.cuh"

// (No pointer of these kernels is __restrict__: they may start while the kernel before
// them still writes what they read behind their wait, and the compiler would take the
// read-only path, which no wait orders.)

int b2_paged_check(const char* who, const B2PagedKV* kv, int nkv, int hd, bool rows) {
    if (!kv || !kv->k_pages || !kv->v_pages ||
        (kv->n_seqs > 0 && (!kv->page_table || !kv->kv_len || (rows && !kv->q_start))))
        return b2_set_error(B2_ERR_INVALID_ARG, "%s: null pointer in the cache description", who);
    if (hd != 64 && hd != 128) return b2_set_error(B2_ERR_INVALID_ARG, "%s: head_dim %d not in {64, 128}", who, hd);
    if (kv->page_size != 16 && kv->page_size != 32 && kv->page_size != 64 && kv->page_size != 128)
        return b2_set_error(B2_ERR_INVALID_ARG, "%s: page_size %d not in {16, 32, 64, 128}", who, kv->page_size);
    if (kv->n_pages <= 0 || kv->max_pages <= 0 || kv->n_seqs < 0 || kv->n_seqs > B2_PAGED_MAX_SEQS || nkv <= 0 ||
        (long long)kv->max_pages * kv->page_size > 0x7fffff00ll)
        return b2_set_error(B2_ERR_INVALID_ARG, "%s: bad counts (pages %d, table row %d, sequences %d of at most %d)",
                            who, kv->n_pages, kv->max_pages, kv->n_seqs, B2_PAGED_MAX_SEQS);
    const long long lim = 1ll << 39;
    if ((reinterpret_cast<uintptr_t>(kv->k_pages) & 15) || (reinterpret_cast<uintptr_t>(kv->v_pages) & 15) ||
        kv->page_stride % 8 || kv->head_stride % 8 || kv->row_stride % 8 || kv->page_stride <= 0 ||
        kv->head_stride <= 0 || kv->row_stride < hd || kv->page_stride >= lim || kv->head_stride >= lim ||
        kv->row_stride >= lim)
        return b2_set_error(B2_ERR_INVALID_ARG,
                            "%s: pages must be 16-byte aligned with positive strides that are multiples of 8", who);
    return 0;
}

int b2_paged_map(CUtensorMap* map, const uint16_t* base, const B2PagedKV* kv, int nkv, int hd, int box_rows,
                 int box_halves) {
    const uint64_t dims[5] = {64, (uint64_t)kv->page_size, (uint64_t)hd / 64, (uint64_t)nkv, (uint64_t)kv->n_pages};
    const uint64_t strides[4] = {(uint64_t)kv->row_stride * 2, 128, (uint64_t)kv->head_stride * 2,
                                 (uint64_t)kv->page_stride * 2};
    const uint32_t box[5] = {64, (uint32_t)box_rows, (uint32_t)box_halves, 1, 1};
    return b2_tensor_map_f16_5d(map, base, dims, strides, box);
}

namespace {

struct PageStrides {
    uint16_t *k, *v;
    long long page, head, row;
};

// ─── b2_qk_rope_kv_paged ───
//
// x = one head of one row; for q and k (with norm weights)
//     n = (x / sqrt(mean(x^2) + eps)) * w
// then the rotation of pairs (2i, 2i + 1) or (i, i + hd / 2) by the angle of
// the row's position, and the rounding to FP16: q for the tensor cores of the
// attention, K and V as the cache keeps them.  FP32 throughout, the sum of
// squares across the warp.  Bound by HBM: 4 bytes read and 2 written per
// element.  A warp takes `steps` times kHeads heads of one row, kHeads at a time
// and the next ones on their way: with many rows a whole row, so that its place
// and angles are looked up once, with few rows kHeads, so that there are warps.  7467 rows of 32
// heads, hd 128: 35.7 us at 1.78 GHz (33.7 at best), 0.80 of the measured copy rate; 64 rows: 3.9.
constexpr int kAppendThreads = 128;
constexpr int kHeads = 4;

template <int E>
__device__ __forceinline__ void load_vec(float (&v)[E], const float* p, bool aligned) {
    if (!aligned) {
#pragma unroll
        for (int j = 0; j < E; j++) v[j] = p[j];
    } else if constexpr (E == 4) {
        const float4 u = *reinterpret_cast<const float4*>(p);
        v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
    } else {
        const float2 u = *reinterpret_cast<const float2*>(p);
        v[0] = u.x, v[1] = u.y;
    }
}

// (volatile: not kept in registers over a loop)
template <int E>
__device__ __forceinline__ void load_shared(float (&v)[E], const float* p) {
    if constexpr (E == 4)
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(b2p::smem_u32(p)));
    else
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(b2p::smem_u32(p)));
}

// The four heads' sums together: two exchanges halve what a lane adds for, so that
// eight lanes each end with one head, and take its root once.  (One by one: 0.3 us more
// of 4.3 with 64 rows, 0.5 of 40 with 7467.)
template <int HD>
__device__ __forceinline__ void four_norms(const float (&x)[kHeads][HD / 32], float eps, int lane, float (&norm)[kHeads]) {
    static_assert(kHeads == 4, "two exchanges");
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 32; j++) s[i] = fmaf(x[i][j], x[i][j], s[i]);
    }
    const bool up = lane & 16, odd = lane & 8;
    const float a = (up ? s[2] : s[0]) + __shfl_xor_sync(0xffffffffu, up ? s[0] : s[2], 16);
    const float b = (up ? s[3] : s[1]) + __shfl_xor_sync(0xffffffffu, up ? s[1] : s[3], 16);
    float t = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    t = 1.0f / sqrtf(t / (float)HD + eps);
#pragma unroll
    for (int i = 0; i < 4; i++) norm[i] = __shfl_sync(0xffffffffu, t, 8 * i);
}

// aligned: the angle tables allow 16-byte loads.  Seven CTAs per SM: 34.7 us, 35.8
// with eight, 39.9 with nine, whose registers hold fewer loads ahead.
template <int HD>
__global__ void __launch_bounds__(kAppendThreads, 7) append_kernel(
    __half* q16, int ldq, const float* qkv, int ldqkv, int nq, int nkv,
    const float* q_norm_w, const float* k_norm_w, float eps, const float* cos_tab,
    const float* sin_tab, int max_pos, int rope_style, const int* pos_of, b2p::Batch bt,
    PageStrides pg, bool aligned, int steps) {
    constexpr int E = HD / 32;  // elements per lane
    b2::pdl_trigger();
    b2::pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = nq + 2 * nkv, per_row = (heads + kHeads * steps - 1) / (kHeads * steps);
    const long long job = (long long)blockIdx.x * (kAppendThreads / 32) + warp;
    const int m = (int)(job / per_row);
    int h0 = (int)(job % per_row) * kHeads * steps;
    const int h_end = min(heads, h0 + kHeads * steps);
    // The norm weights wait in shared memory: in eight registers of every thread they
    // cost the loads ahead their room (7467 rows: 39.5 us so, 35.8 here).
    __shared__ alignas(16) float nw[2][HD];
    static_assert(kAppendThreads >= HD, "one element per thread");
    if (threadIdx.x < HD) {
        if (q_norm_w) nw[0][threadIdx.x] = q_norm_w[threadIdx.x];
        if (k_norm_w) nw[1][threadIdx.x] = k_norm_w[threadIdx.x];
    }
    // The first heads' elements are asked for before it is known where the row belongs.
    float x[kHeads][E];
    const float* src = qkv + (size_t)min(m, bt.M - 1) * ldqkv + lane * E;
#pragma unroll
    for (int i = 0; i < kHeads; i++) load_vec(x[i], src + (size_t)min(h0 + i, heads - 1) * HD, true);
    __syncthreads();
    if (m >= bt.M || m >= bt.q_start[bt.n_seqs] || m < bt.q_start[0]) return;
    int pos = pos_of ? pos_of[m] : 0;
    // largest s with q_start[s] <= m: every lane tests one splitter per round, and in the
    // last one has the sequence's entries at hand (what a row waits for is this chain of loads)
    int lo = 0, hi = bt.n_seqs;
    b2p::Seq sq;
    for (bool found = false; !found;) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const bool in = at < hi;
        found = step == 1;
        const int start = in ? bt.q_start[at] : 0;
        const int end = in && found ? bt.q_start[at + 1] : 0, cached = in && found ? bt.kv_len[at] : 0;
        const int f = 31 - __clz(__ballot_sync(0xffffffffu, in && start <= m));
        lo += f * step;
        hi = min(hi, lo + step);
        sq = bt.seq_of(__shfl_sync(0xffffffffu, start, f), __shfl_sync(0xffffffffu, end, f),
                       __shfl_sync(0xffffffffu, cached, f));
    }
    const int slot = sq.base + (m - sq.row0);
    if (!pos_of) pos = slot;
    if (pos < 0 || pos >= max_pos || m - sq.row0 >= sq.Q) return;
    const int page = slot >= 0 && slot < sq.len ? bt.page(lo, slot) : -1;
    const long long at = page >= 0 ? page * pg.page + (slot & ((1 << bt.page_shift) - 1)) * pg.row : 0;

    // angle of element j: that of the pair (2i, 2i+1), or (i, i + HD/2)
    float c[E], sn[E];
    const float *ct = cos_tab + (size_t)pos * (HD / 2), *st = sin_tab + (size_t)pos * (HD / 2);
    if (rope_style == 0) {
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            c[j] = c[j + 1] = ct[(lane * E + j) >> 1];
            sn[j] = sn[j + 1] = st[(lane * E + j) >> 1];
        }
    } else {
        load_vec(c, ct + (lane * E & (HD / 2 - 1)), aligned);
        load_vec(sn, st + (lane * E & (HD / 2 - 1)), aligned);
    }
    for (; h0 < h_end; h0 += kHeads) {
        float nx[kHeads][E];  // the heads after these
        if (h0 + kHeads < h_end) {
#pragma unroll
            for (int i = 0; i < kHeads; i++) load_vec(nx[i], src + (size_t)min(h0 + kHeads + i, heads - 1) * HD, true);
        }
        float norm[kHeads];  // 1 / sqrt(mean of squares + eps) of each head
        if (q_norm_w || k_norm_w) four_norms<HD>(x, eps, lane, norm);
#pragma unroll
        for (int i = 0; i < kHeads; i++) {
            const int h = h0 + i;
            if (h >= h_end) break;
            const bool is_q = h < nq, is_v = h >= nq + nkv;
            if (!is_v) {
                if (is_q ? q_norm_w : k_norm_w) {
                    float w[E];
                    load_shared(w, &nw[is_q ? 0 : 1][lane * E]);
#pragma unroll
                    for (int j = 0; j < E; j++) x[i][j] = (x[i][j] * norm[i]) * w[j];
                }
                if (rope_style == 0) {
#pragma unroll
                    for (int j = 0; j < E; j += 2) {
                        const float a = x[i][j], b = x[i][j + 1];
                        x[i][j] = a * c[j] - b * sn[j];
                        x[i][j + 1] = b * c[j] + a * sn[j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < E; j++) {
                        const float o = __shfl_xor_sync(0xffffffffu, x[i][j], 16);
                        x[i][j] = lane < 16 ? x[i][j] * c[j] - o * sn[j] : x[i][j] * c[j] + o * sn[j];
                    }
                }
            }
            __half* dst;
            if (is_q) {
                dst = q16 + (size_t)m * ldq + (size_t)h * HD;
            } else {
                if (page < 0) continue;
                const int g = is_v ? h - nq - nkv : h - nq;
                dst = reinterpret_cast<__half*>(is_v ? pg.v : pg.k) + at + g * pg.head;
            }
            if constexpr (E == 4) {
                uint2 u;
                u.x = b2p::pack_h2(x[i][0], x[i][1]);
                u.y = b2p::pack_h2(x[i][2], x[i][3]);
                *reinterpret_cast<uint2*>(dst + lane * E) = u;
            } else {
                *reinterpret_cast<uint32_t*>(dst + lane * E) = b2p::pack_h2(x[i][0], x[i][1]);
            }
        }
#pragma unroll
        for (int i = 0; i < kHeads; i++)
#pragma unroll
            for (int j = 0; j < E; j++) x[i][j] = nx[i][j];
    }
}

// ─── b2_kv_evict_paged ───
//
// Selection: a cluster of S CTAs per (sequence, kv head), each with an S-th of
// the slots.  A slot becomes a key that orders as the contract does (0: not
// mapped, the largest: always kept, else the weight's order), held in shared
// memory, and the k-th largest key is found 8 bits at a time from histograms that
// the CTAs add up through distributed shared memory (one cluster barrier a digit).
// Slots above it are kept, and as many of those equal to it as are missing,
// lowest first.  A warp owns a contiguous run of its CTA's slots, 32 at a time, so
// ballots give the places in slot order and one scan over the warps joins them.
// The search ends early once all slots that share the digits so far are kept.
// Bound by latency: 100 thousand slots of 8 heads take 24 us (the keys and the first
// digit 8, each other digit 3, the places 7), 4096 slots of 128 (sequence, head)
// pairs 11.
constexpr int kBatch = 8;  // groups of 32 slots whose loads a warp has in flight
constexpr int kMaxKeys = 48 * 1024;  // keys a CTA holds; more are formed again for every digit
constexpr int kMaxSplit = 8;

// Key of slot j from its page entry and weight.
__device__ __forceinline__ uint32_t evict_key(int page, int n_pages, float w, bool always) {
    if (page < 0 || page >= n_pages) return 0u;
    if (always) return 0xFFFFFFFFu;
    // + 0 turns -0 into 0, so that the two are equal here too
    return min(max(b2::float_order(w + 0.f), 1u), 0xFFFFFFFEu);
}

__device__ __forceinline__ int ld_rank(const int* p, int rank) {
    uint32_t a;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(b2p::smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sync_cluster(int S) {
    if (S > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    else __syncthreads();
}

// S = gridDim.x.
template <int kSelThreads>
__global__ void __launch_bounds__(kSelThreads, 1024 / kSelThreads) evict_select_kernel(b2p::Batch bt, const float* weights,
                                                                   long long ldw, int nkv, int budget, int sink,
                                                                   int recent, int held, int* kept,
                                                                   float* dst_weights,
                                                                   int* new_len) {
    constexpr int kSelWarps = kSelThreads / 32;
    extern __shared__ uint32_t keys[];
    __shared__ int hist[2][257];  // [digit parity]; [256]: unmapped slots
    __shared__ int sum[256];
    __shared__ int counts[2];     // slots above the k-th key, and equal to it
    __shared__ int warp_gt[kSelWarps], warp_eq[kSelWarps];
    __shared__ int found[3], before[2], unmapped;
    const int S = gridDim.x, rank = blockIdx.x, g = blockIdx.y, s = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    b2::pdl_trigger();
    b2::pdl_wait();
    const int n = max(bt.kv_len[s], 0);
    const long long cap = (long long)bt.max_pages << bt.page_shift;
    const int len = (int)((long long)n < cap ? n : cap);
    // this CTA's slots, and this warp's: whole groups of 32
    const int groups = b2p::cdiv(len, 32), cta_g = b2p::cdiv(groups, S), warp_g = b2p::cdiv(cta_g, kSelWarps);
    const int g0 = min(groups, rank * cta_g), g1 = min(groups, g0 + cta_g);
    const int w0 = min(g1, g0 + warp * warp_g), w1 = min(g1, w0 + warp_g);
    const bool cached = cta_g * 32 <= held;
    const float* w = weights + ((size_t)s * nkv + g) * ldw;
    const int* table = bt.page_table + (size_t)s * bt.max_pages;
    // kBatch groups' page entries and weights, all requested before any is used
    auto make_keys = [&](int q0, uint32_t (&key)[kBatch]) {
        int pg[kBatch];
        float wv[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; e++) {
            const int j = (q0 + e) * 32 + lane;
            const bool in = q0 + e < w1 && j < len;
            pg[e] = in ? table[j >> bt.page_shift] : -1;
            wv[e] = in && j < ldw ? w[j] : 0.f;
        }
        __syncwarp();  // no load moves behind this
#pragma unroll
        for (int e = 0; e < kBatch; e++) {
            const int j = (q0 + e) * 32 + lane;
            key[e] = evict_key(pg[e], bt.n_pages, wv[e], j < sink || j >= len - recent);
        }
    };
    auto get_keys = [&](int q0, uint32_t (&key)[kBatch]) {
        if (cached) {
#pragma unroll
            for (int e = 0; e < kBatch; e++) key[e] = q0 + e < w1 ? keys[(q0 + e - g0) * 32 + lane] : 0u;
        } else {
            make_keys(q0, key);
        }
    };
    for (int i = tid; i < 2 * 257; i += kSelThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    uint32_t prefix = 0;  // the digits found so far of the k-th largest key
    int need = 0, k = 0;  // slots still to take among those that share them; slots kept
    bool whole = false;
    for (int d = 0; d < 4; d++) {
        const int shift = 24 - 8 * d;
        int* h = hist[d & 1];
        int none = 0;
        for (int q = w0; q < w1; q += kBatch) {
            uint32_t keyv[kBatch];
            if (d == 0) {
                make_keys(q, keyv);
#pragma unroll
                for (int e = 0; e < kBatch; e++) {
                    const uint32_t key = keyv[e];
                    if (cached && q + e < w1) keys[(q + e - g0) * 32 + lane] = key;
                    none += q + e < w1 && (q + e) * 32 + lane < len && key == 0;
                    // one addition per distinct digit of the warp: weights share exponents
                    const unsigned same = __match_any_sync(0xffffffffu, key ? key >> 24 : 256u);
                    if (key && lane == __ffs(same) - 1) atomicAdd(&h[key >> 24], __popc(same));
                }
            } else {
                get_keys(q, keyv);
#pragma unroll
                for (int e = 0; e < kBatch; e++) {
                    const uint32_t key = keyv[e];
                    const bool in = (key >> (shift + 8)) == (prefix >> (shift + 8)) && key != 0;
                    const unsigned who = __ballot_sync(0xffffffffu, in);
                    if (who == 0) continue;
                    // few slots share a prefix, and their digits differ, unless their weights are equal:
                    // one addition for the first one's digit, others by themselves
                    const unsigned dig = (key >> shift) & 255;
                    const int first = __ffs(who) - 1;
                    const unsigned lead = __shfl_sync(0xffffffffu, dig, first);
                    const unsigned same = __ballot_sync(0xffffffffu, in && dig == lead);
                    if (lane == first) atomicAdd(&h[dig], __popc(same));
                    else if (in && !(same >> lane & 1)) atomicAdd(&h[dig], 1);
                }
            }
        }
        if (d == 0) {
            none = __reduce_add_sync(0xffffffffu, none);
            if (lane == 0 && none) atomicAdd(&h[256], none);
        }
        sync_cluster(S);
        if (tid < 256 || (d == 0 && tid == 256)) {
            int v[kMaxSplit];  // every CTA's asked for before any is used
#pragma unroll
            for (int r = 0; r < kMaxSplit; r++) v[r] = S == 1 ? (r == 0 ? h[tid] : 0) : r < S ? ld_rank(&h[tid], r) : 0;
            int all = 0;
#pragma unroll
            for (int r = 0; r < kMaxSplit; r++) all += v[r];
            (tid < 256 ? sum[tid] : unmapped) = all;
        }
        __syncthreads();
        if (d == 0) {
            k = min(len - unmapped, budget);
            need = k;
            if (k == 0 || k == len - unmapped) break;  // nothing to choose
        }
        if (warp == 0) {
            // from the top: lane l has bins 255 - 8 l - 7 .. 255 - 8 l
            int c[8], t = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) t += c[e] = sum[255 - 8 * lane - e];
            int incl = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += u;
            }
            int over = incl - t;  // slots in higher bins
            if (over < need && incl >= need) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (over < need && over + c[e] >= need) {
                        found[0] = 255 - 8 * lane - e;
                        found[1] = need - over;
                        found[2] = need - over == c[e];
                    }
                    over += c[e];
                }
            }
        }
        // the other parity's bins were read behind the barrier before this one
        if (d > 0)
            for (int i = tid; i < 256; i += kSelThreads) hist[(d + 1) & 1][i] = 0;
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift;
        need = found[1];
        if (found[2]) {  // every slot that shares these digits is kept: the rest of them does not matter
            whole = true;
            break;
        }
    }
    if (rank == 0 && g == 0 && tid == 0) new_len[s] = k;
    // kept: keys above `bar`, and unless that is all `need` of those equal to it
    const bool every = whole || k == len - unmapped;
    const uint32_t bar = !every ? prefix : whole && prefix > 0 ? prefix - 1 : 0u;
    if (k > 0) {  // the same for every CTA of the cluster
        int gt = 0, eq = 0;
        for (int q = w0; q < w1; q += kBatch) {
            uint32_t key[kBatch];
            get_keys(q, key);
#pragma unroll
            for (int e = 0; e < kBatch; e++) {
                gt += key[e] > bar;
                eq += key[e] == bar && !every;
            }
        }
        gt = __reduce_add_sync(0xffffffffu, gt);
        eq = __reduce_add_sync(0xffffffffu, eq);
        if (lane == 0) {
            warp_gt[warp] = gt;
            warp_eq[warp] = eq;
        }
        __syncthreads();
        if (warp == 0) {  // exclusive sums over the warps
            int a = lane < kSelWarps ? warp_gt[lane] : 0, b = lane < kSelWarps ? warp_eq[lane] : 0;
            const int a0 = a, b0 = b;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, a, o), v = __shfl_up_sync(0xffffffffu, b, o);
                if (lane >= o) a += u, b += v;
            }
            if (lane < kSelWarps) {
                warp_gt[lane] = a - a0;
                warp_eq[lane] = b - b0;
            }
            if (lane == 31) counts[0] = a, counts[1] = b;
        }
        sync_cluster(S);
        if (warp == 0) {
            const int a = __reduce_add_sync(0xffffffffu, lane < rank ? ld_rank(&counts[0], lane) : 0);
            const int b = __reduce_add_sync(0xffffffffu, lane < rank ? ld_rank(&counts[1], lane) : 0);
            if (lane == 0) before[0] = a, before[1] = b;
        }
        __syncthreads();
        int above = before[0] + warp_gt[warp], equal = before[1] + warp_eq[warp];  // in slots before this group
        const size_t o0 = ((size_t)s * nkv + g) * budget;
        const unsigned below = (1u << lane) - 1;
        for (int q = w0; q < w1; q += kBatch) {
            uint32_t keyv[kBatch];
            float wv[kBatch];
            get_keys(q, keyv);
#pragma unroll
            for (int e = 0; e < kBatch; e++) {
                const int j = (q + e) * 32 + lane;
                wv[e] = dst_weights && keyv[e] != 0 && keyv[e] >= bar && j < ldw ? w[j] : 0.f;
            }
            __syncwarp();  // no load moves behind this
#pragma unroll
            for (int e = 0; e < kBatch; e++) {
                const uint32_t key = keyv[e];
                const bool is_gt = key > bar, is_eq = key == bar && !every;
                const unsigned bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq);
                const int eq_rank = equal + __popc(be & below);
                if (is_gt || (is_eq && eq_rank < need)) {
                    const int at = above + __popc(bg & below) + (every ? 0 : min(eq_rank, need));
                    kept[o0 + at] = (q + e) * 32 + lane;
                    if (dst_weights) dst_weights[o0 + at] = wv[e];
                }
                above += __popc(bg);
                equal += __popc(be);
            }
        }
    }
    if (S > 1) sync_cluster(S);  // the others may still read this CTA's counts
}

// Moves the kept rows: 16 bytes per thread, K and V of a row by neighbouring
// threads, four rows in flight per thread.  Bound by HBM: 16 x 8 heads of 1024 rows
// take 24 us (134 MB moved: 0.85 of the measured copy rate), one context of 20
// thousand rows 30 (164 MB, 0.84).  Two or eight rows per thread: 1 us more.
constexpr int kMoveThreads = 128;
constexpr int kMoveRows = 4;

template <int HD>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(b2p::Batch bt, PageStrides pg, int budget,
                                                                  const int* dst_table, int dst_max_pages,
                                                                  const int* kept,
                                                                  const int* new_len) {
    constexpr int C = HD / 8;  // 16-byte chunks of a row
    constexpr int kRows = kMoveThreads / (2 * C);
    b2::pdl_trigger();
    b2::pdl_wait();
    const int s = blockIdx.z, g = blockIdx.y, nkv = gridDim.y;
    const unsigned n = new_len[s];  // (unsigned: a place past it, by up to a stride of the grid, may pass 2^31)
    const int c = threadIdx.x % C, which = threadIdx.x / C % 2;
    uint16_t* pool = (which ? pg.v : pg.k) + g * pg.head + c * 8;
    const int mask = (1 << bt.page_shift) - 1;
    const int* from_of = kept + ((size_t)s * nkv + g) * budget;
    for (unsigned j0 = blockIdx.x * kRows * kMoveRows + threadIdx.x / (2 * C); j0 < n; j0 += gridDim.x * kRows * kMoveRows) {
        int from[kMoveRows], to[kMoveRows], page[kMoveRows];
        uint4 v[kMoveRows];
#pragma unroll
        for (int i = 0; i < kMoveRows; i++) {
            const unsigned j = j0 + i * kRows, dp = j >> bt.page_shift;
            from[i] = j < n ? from_of[j] : -1;
            to[i] = j < n && dp < (unsigned)dst_max_pages ? dst_table[(size_t)s * dst_max_pages + dp] : -1;
        }
#pragma unroll
        for (int i = 0; i < kMoveRows; i++)
            page[i] = from[i] >= 0 && to[i] >= 0 && to[i] < bt.n_pages ? bt.page(s, from[i]) : -1;
#pragma unroll
        for (int i = 0; i < kMoveRows; i++)
            if (page[i] >= 0)
                v[i] = *reinterpret_cast<const uint4*>(pool + page[i] * pg.page + (from[i] & mask) * pg.row);
#pragma unroll
        for (int i = 0; i < kMoveRows; i++)
            if (page[i] >= 0) __stcs(reinterpret_cast<uint4*>(pool + to[i] * pg.page + ((j0 + i * kRows) & mask) * pg.row), v[i]);
    }
}

}  // namespace

extern "C" int b2_qk_rope_kv_paged(uint16_t* q16, int ldq, const float* qkv, int ldqkv, int M, int nq, int nkv, int hd,
                                   const float* q_norm_w, const float* k_norm_w, float eps, const float* cos_tab,
                                   const float* sin_tab, int max_pos, int rope_style, const int* pos,
                                   const B2PagedKV* kv, b2_stream_t s) {
    int rc = b2_paged_check("b2_qk_rope_kv_paged", kv, nkv, hd, true);
    if (rc) return rc;
    if ((M > 0 && (!q16 || !qkv)) || !cos_tab || !sin_tab || M < 0 || nq <= 0 || max_pos <= 0 || (rope_style != 0 && rope_style != 1))
        return b2_set_error(B2_ERR_INVALID_ARG, "b2_qk_rope_kv_paged: bad arguments");
    if (ldqkv < (nq + 2ll * nkv) * hd || ldq < (long long)nq * hd || ldqkv % 4 || ldq % 4 ||
        (reinterpret_cast<uintptr_t>(qkv) & 15) || (reinterpret_cast<uintptr_t>(q16) & 7))
        return b2_set_error(B2_ERR_INVALID_ARG,
                            "b2_qk_rope_kv_paged: rows must be aligned (qkv 16 bytes, ldqkv %% 4; q16 8 bytes, ldq %% 4) "
                            "and hold every head");
    if (M == 0 || kv->n_seqs == 0) return 0;
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    // Whole rows once there are more jobs of four heads than warps that the SMs can hold.  32 heads of
    // 128: 600 rows take 13.3 us as jobs of four heads and 16.4 as rows, 900 15.2 and 16.4, 1200 18.3
    // and 16.4, 2000 23.2 and 18.4, 7500 58.3 and 41.0 (launch by launch, inputs not in L2).
    const int all = (nq + 2 * nkv + kHeads - 1) / kHeads;
    const int steps = (long long)M * all > 64ll * sms ? all : 1;
    const long long jobs = (long long)M * ((all + steps - 1) / steps);
    const long long grid = (jobs + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
    if (grid > 0x7fffffffll) return b2_set_error(B2_ERR_INVALID_ARG, "b2_qk_rope_kv_paged: too many rows");
    const PageStrides pg{kv->k_pages, kv->v_pages, kv->page_stride, kv->head_stride, kv->row_stride};
    const bool aligned = ((reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab)) & 15) == 0;
    const cudaError_t e =
        b2::launch_pdl(hd == 128 ? append_kernel<128> : append_kernel<64>, dim3((unsigned)grid), dim3(kAppendThreads), 0,
                       (cudaStream_t)s, reinterpret_cast<__half*>(q16), ldq, qkv, ldqkv, nq, nkv, q_norm_w, k_norm_w,
                       eps, cos_tab, sin_tab, max_pos, rope_style, pos, b2p::make_batch(kv, M), pg, aligned, steps);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_qk_rope_kv_paged: %s", cudaGetErrorString(e));
    return 0;
}

extern "C" int b2_kv_evict_paged(const B2PagedKV* kv, int nkv, int hd, const float* weights, long long ldw, int budget,
                                 int sink, int recent, const int* dst_table, int dst_max_pages, int* kept,
                                 float* dst_weights, int* new_len, b2_stream_t s) {
    int rc = b2_paged_check("b2_kv_evict_paged", kv, nkv, hd, false);
    if (rc) return rc;
    if ((kv->n_seqs > 0 && (!weights || !new_len)) || ldw < 0 || budget < 0 || sink < 0 || recent < 0 ||
        (budget > 0 && (!dst_table || !kept || dst_max_pages <= 0)) || (long long)sink + recent > budget || nkv > 65535)
        return b2_set_error(B2_ERR_INVALID_ARG, "b2_kv_evict_paged: bad arguments (sink + recent <= budget)");
    if (kv->n_seqs == 0) return 0;
    // One head's CTAs store while others still read: nothing that is written may be among what is read.
    const long long n = kv->n_seqs, rows = n * nkv, row = ldw < (1ll << 34) ? ldw : 1ll << 34;
    const struct {
        const void* p;
        long long count;
    } out[3] = {{kept, rows * budget}, {dst_weights, rows * budget}, {new_len, n}},
      in[4] = {{weights, rows * row}, {kv->page_table, n * kv->max_pages}, {kv->kv_len, n}, {dst_table, n * dst_max_pages}};
    for (int i = 0; i < 3; i++) {
        bool bad = false;
        for (int j = 0; j < 4; j++) bad |= b2_paged_overlap(out[i].p, out[i].count, in[j].p, in[j].count);
        for (int j = 0; j < i; j++) bad |= b2_paged_overlap(out[i].p, out[i].count, out[j].p, out[j].count);
        if (bad)
            return b2_set_error(B2_ERR_INVALID_ARG, "b2_kv_evict_paged: %s overlaps another array of the call",
                                i == 0 ? "kept" : i == 1 ? "dst_weights" : "new_len");
    }
    const b2p::Batch bt = b2p::make_batch(kv, 0);
    const PageStrides pg{kv->k_pages, kv->v_pages, kv->page_stride, kv->head_stride, kv->row_stride};
    cudaStream_t st = (cudaStream_t)s;
    // CTAs per (sequence, kv head): as many as have 4096 slots each when the table is
    // full, and as two per SM have room for.  (4096 slots of 128 pairs: 35 us with
    // one, 37 with two; 100 thousand slots of 8 heads: 233 us with one, 54 with eight.)
    const long long cap = (long long)kv->max_pages * kv->page_size, heads = (long long)kv->n_seqs * nkv;
    int dev = 0, sms = 148, S = 1;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    while (S < kMaxSplit && cap > 4096ll * S && heads * S * 2 <= 2 * sms) S *= 2;
    long long held = ((cap + 31) / 32 + S - 1) / S * 32;
    if (held > kMaxKeys) held = kMaxKeys;
    // Twice the threads where a CTA has an SM to itself and slots for them.
    const bool wide = held > 2048 && heads * S <= sms;
    static std::atomic<unsigned long long> allowed[2];
    cudaError_t e = wide ? b2p::allow_smem(evict_select_kernel<1024>, kMaxKeys * 4, allowed[1], dev)
                         : b2p::allow_smem(evict_select_kernel<512>, kMaxKeys * 4, allowed[0], dev);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_kv_evict_paged smem: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S, nkv, kv->n_seqs);
    cfg.blockDim = dim3(wide ? 1024 : 512);
    cfg.dynamicSmemBytes = (size_t)held * 4;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = S;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = S > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, wide ? evict_select_kernel<1024> : evict_select_kernel<512>, bt, weights, ldw, nkv, budget, sink, recent, (int)held, kept,
                           dst_weights, new_len);
    if (e == cudaSuccess && budget > 0) {
        const int rows = kMoveThreads / (2 * (hd / 8)) * kMoveRows;
        const long long want = ((long long)budget + rows - 1) / rows;
        const dim3 grid((unsigned)(want < 4096 ? want : 4096), nkv, kv->n_seqs);
        e = b2::launch_pdl(hd == 128 ? evict_move_kernel<128> : evict_move_kernel<64>, grid, dim3(kMoveThreads), 0, st, bt,
                           pg, budget, dst_table, dst_max_pages, (const int*)kept, (const int*)new_len);
    }
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_kv_evict_paged: %s", cudaGetErrorString(e));
    return 0;
}
