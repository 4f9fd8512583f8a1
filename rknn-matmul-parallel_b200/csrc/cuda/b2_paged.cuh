// Shared pieces of the paged-cache kernels (b2_paged_kv.cu, b2_paged_attn.cu,
// b2_paged_weights.cu): argument checks, the per-sequence view of a batch and
// the barrier / copy wrappers.
#pragma once
#include <cuda.h>  // CUtensorMap
#include <math.h>
#include <stdlib.h>

#include <atomic>

#include "b2_common.cuh"

// 5-D FP16 tensor map with the 128-byte swizzle; strides in bytes of dimensions
// 1..4.  Defined in b2_gemm.cu.
int b2_tensor_map_f16_5d(void* map, const void* base, const uint64_t (&dims)[5], const uint64_t (&strides)[4],
                         const uint32_t (&box)[5]);

// Host checks shared by the entry points; 0 or an error code with its message.
int b2_paged_check(const char* who, const B2PagedKV* kv, int nkv, int hd, bool rows);
// Whether two arrays of so many 4-byte entries share any.
inline bool b2_paged_overlap(const void* a, long long na, const void* b, long long nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && na > 0 && nb > 0 && (x < y ? y - x < 4ull * na : x - y < 4ull * nb);
}
// Tensor map of K or V pages: dimensions (64 dims, rows of a page, head_dim / 64,
// kv heads, pages), boxes of box_rows rows and box_halves times 64 dims: a box
// lands as [box_halves][box_rows][128 bytes], each 128-byte row swizzled.
int b2_paged_map(CUtensorMap* map, const uint16_t* base, const B2PagedKV* kv, int nkv, int hd, int box_rows,
                 int box_halves);

// A branch seldom taken: its code goes out of line, so that a hot loop stays in a
// few lines of the instruction cache.
#define B2_RARE(x) __builtin_expect(!!(x), 0)

namespace b2p {

// A sequence of the batch, with the caller's device values bounded so that no
// index computed from them leaves its array.
struct Seq {
    int row0;  // its first row
    int Q;     // its rows
    int len;   // cached positions, at most the table's capacity
    int base;  // slot of row 0 (negative when kv_len < Q: those rows see nothing)
};

struct Batch {
    const int* page_table;
    const int* kv_len;
    const int* q_start;
    int n_seqs, max_pages, n_pages, page_shift, M;

    __device__ __forceinline__ Seq seq(int s) const { return seq_of(q_start[s], q_start[s + 1], kv_len[s]); }
    // From the sequence's entries.
    __device__ __forceinline__ Seq seq_of(int start, int end, int cached) const {
        Seq x;
        const int a = min(max(start, 0), M), b = min(max(end, a), M), n = max(cached, 0);
        x.row0 = a;
        x.Q = b - a;
        x.base = n - x.Q;
        const long long cap = (long long)max_pages << page_shift;
        x.len = (int)((long long)n < cap ? n : cap);
        return x;
    }
    // Page of slot j, or -1 where none is mapped.
    __device__ __forceinline__ int page(int s, int j) const {
        const int p = page_table[(size_t)s * max_pages + (j >> page_shift)];
        return p >= 0 && p < n_pages ? p : -1;
    }
};

inline Batch make_batch(const B2PagedKV* kv, int M) {
    Batch b{kv->page_table, kv->kv_len, kv->q_start, kv->n_seqs, kv->max_pages, kv->n_pages, 0, M};
    while ((1 << b.page_shift) < kv->page_size) b.page_shift++;
    return b;
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Polls after which a wait gives up (a poll takes 1.5 us: six seconds).  The variable is for tests.
constexpr int kWaitLimit = 1 << 22;
inline int wait_limit() {
    const char* e = getenv("B2_PAGED_POLL_LIMIT");
    return e ? atoi(e) : kWaitLimit;
}
// Bounded wait of a whole warp: false, with the CTA's failure flag failed[0] set, after
// failed[1] polls or once another warp has given up.  The warp polls as one: behind
// a loop that its lanes might leave one by one it would have to gather them again.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
    for (int it = 0; B2_RARE(!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))); it++) {
        if (B2_RARE(__any_sync(0xffffffffu, it > failed[1] || failed[0]))) {
            failed[0] = 1;
            return false;
        }
    }
    return true;
}
// For one thread of a CTA that gave up: the last `depth` of `count` copies (or of groups of
// them) into a ring of so many barriers have landed.  Bounded again, by the usual limit.
__device__ __forceinline__ void copies_land(uint64_t* bars, int depth, int count) {
    for (int i = max(0, count - depth); i < count; i++)
        for (int it = 0; it <= kWaitLimit && !mbar_try_wait(&bars[i % depth], (i / depth) & 1); it++) {}
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int x, int row, int half, int head,
                                            int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(row), "r"(half), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

// Untiled copy: addresses and size multiples of 16 bytes.
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

// Eight FP16 values, one of them infinite or NaN.
__device__ __forceinline__ bool non_finite8(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) bad |= ((w[i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    return bad != 0;
}

// Loads past L1 of what other CTAs wrote.
__device__ __forceinline__ float2 ld_cg2(const float* p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cg4(const float* p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}

// 2^x (ex2.approx: 2 ulp; subnormal results flush to zero).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Work of each sequence -> exclusive prefix pre[0..n] (shared memory, n + 1
// ints), by all threads of the CTA.  The sums stop at kMaxWork, which the host
// checks for sequences that share no rows: with any q_start the prefix rises, and
// a place below pre[n] lies in the work of the sequence that prefix_find gives.
constexpr unsigned kMaxWork = (1u << 31) - 65536;
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) {
    return a + b < a ? ~0u : a + b;
}
template <typename F>
__device__ __forceinline__ void prefix_work(int* pre, int n, F work) {
    for (int s = threadIdx.x; s < n; s += blockDim.x) pre[s + 1] = work(s);
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        unsigned carry = 0;
        for (int b = 0; b < n; b += 32) {
            unsigned v = b + lane < n ? (unsigned)pre[b + lane + 1] : 0u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned t = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v = add_sat(v, t);
            }
            v = min(add_sat(carry, v), kMaxWork);
            if (b + lane < n) pre[b + lane + 1] = (int)v;
            carry = __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) pre[0] = 0;
    }
    __syncthreads();
}
// Largest s in [0, n) with pre[s] <= x (x < pre[n]).
__device__ __forceinline__ int prefix_find(const int* pre, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// What both attention kernels of a call take.
struct AttnParams {
    Batch bt;
    const __half* q16;
    int ldq;
    __half* out16;
    float* lse;
    int max_q, nq, nkv, G;
    int short_rows;  // sequences with at most this many (token, head) rows per kv head are the short kernel's
    int* counters;   // kCounters of them, zero between calls
    float* part;     // the short kernel's partial tiles
    struct Cut* cuts;       // [long CTAs] tiles that the long kernel left in pieces
    float* long_part;       // their pieces
    int long_ctas;          // CTAs of the long kernel (0: none launched)
    int* err;
    int limit;              // polls of a wait
};

// The short kernel's CTAs begin beside the long kernel, which their own wait would
// have to see complete.  What the kernels before the two wrote they see through the
// last counter: a CTA of the long kernel adds kWaited there (release) behind its own
// wait, before it lets the short kernel start, and the short kernel's CTAs acquire
// that.  Each then adds one, and the last of them makes the counter zero again.
constexpr int kCounters = 1024;
constexpr int kWaited = 1 << 16;
__device__ __forceinline__ int* waited_word(const AttnParams& p) { return p.counters + kCounters - 1; }
__device__ __forceinline__ void tell_waited(const AttnParams& p) {
    asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(waited_word(p)), "r"(kWaited) : "memory");
}
// True with what the telling CTA saw visible.  The word is there before the short kernel
// starts; should it not be seen at once, the caller waits for the long kernel instead.
__device__ __forceinline__ bool was_told(const AttnParams& p) {
    int v = 0;
    for (int it = 0; it < 64 && v < kWaited; it++)
        asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(waited_word(p)) : "memory");
    return v >= kWaited;
}

// A tile pair that the long kernel's CTA c (its owner) began and later CTAs
// finished: pieces c, c + 1, ... wait for the merge.
struct Cut {
    int pieces;  // 0: none
    int row0;    // first token row
    int tokens;
    int g;
};
// Floats of one piece: for each of two tiles o[hd / 4][128 rows][4], then
// (maximum, sum)[2][128].  CTA c's slot 2 c holds a piece that continues a
// pair, slot 2 c + 1 one that begins it.
constexpr int kLongRows = 128;
constexpr int kMaxLongCtas = 256;
__host__ __device__ constexpr int long_piece_floats(int hd) { return 2 * kLongRows * (hd + 2); }

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;

// Factor of a piece with maximum m (log2 units) in a sum whose maximum is M.  A
// piece that saw no slot has m = -inf and sums of 0; one that saw only NaN has
// NaN sums, which the factor 1 keeps.
__device__ __forceinline__ float piece_weight(float m, float M) { return m == -INFINITY ? 1.f : ex2(m - M); }

__host__ __device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }

// The line of work and its cuts.  CTA c's stretch begins at place c per, or at the
// near end of the tile there (nb blocks, the place being b into it) when that is
// within snap_of blocks: a piece costs about as much as six blocks of 64 slots, so
// short stretches rather take a tile of up to 16 blocks whole, and long ones stay
// even.
__device__ __forceinline__ int snap_of(int per) { return per <= 8 ? 8 : min(8, max(3, per / 8)); }
__device__ __forceinline__ int snap_to(int x, int b, int nb, int per) {
    const int snap = snap_of(per);
    return b <= snap && b <= nb - b ? x - b : nb - b <= snap ? x - b + nb : x;
}
// The CTAs own .. last whose stretches share the tile of nb blocks at place x0: it
// is whole where own >= last.
__device__ __forceinline__ void cut_of(int x0, int nb, int per, int& own, int& last) {
    const int snap = snap_of(per);
    own = (x0 + snap) / per;
    last = cdiv(x0 + nb - snap, per) - 1;
}

// Host: dynamic shared memory opt-in, once per kernel and device.
template <typename K>
inline cudaError_t allow_smem(K kern, size_t bytes, std::atomic<unsigned long long>& done, int dev) {
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

}  // namespace b2p

// The long kernel (b2_paged_chunk.cu): launches it for the sequences with more
// than p.short_rows rows and sets p.long_ctas.
int b2_paged_attention_long(b2p::AttnParams& p, const B2PagedKV* kv, int hd, int dev, int sms, cudaStream_t s);
