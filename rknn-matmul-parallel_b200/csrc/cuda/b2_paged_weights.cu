// Attention weight per cached slot (b2_attention_paged_weights):
//
//   weights[g][j] = prev[g][j] + sum_{i, h in g} exp(s_ijh - lse_ih)
//
// over the new rows i that see slot j, from q, K and the row sums that the
// attention left.  Every slot belongs to one warp, which adds its rows in
// their order: no atomics, and the result does not depend on timing.
#include "b2_paged.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct WeightParams {
    b2p::Batch bt;
    const uint16_t* k;
    long long page_stride, head_stride, row_stride;
    const __half* q16;
    int ldq;
    const float* lse;
    int max_q, nq, nkv, G;
    float* weights;
    const float* prev;
    long long ldw;
};

// ─── few rows per sequence ───
//
// Bound by reading K once.  A warp owns 16 slots: S = K Q^T on mma m16n8k16
// with the slots as M rows and eight (token, head) rows as N columns.  The dims
// of the sum may go in any order as long as K and Q agree, so a lane takes 16
// consecutive bytes of its row for two k steps and the fragments come straight
// from global memory, a row's four lanes reading 64 consecutive bytes.
constexpr int kThreads = 128;
constexpr int kBlk = 64;

template <int HD>
__global__ void __launch_bounds__(kThreads) weights_short_kernel(const WeightParams p) {
    __shared__ int pre[B2_PAGED_MAX_SEQS + 1];
    b2::pdl_trigger();
    b2::pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c4 = lane & 3;
    b2p::prefix_work(pre, p.bt.n_seqs, [&](int s) { return (p.bt.seq(s).len + kBlk - 1) / kBlk * p.nkv; });
    const int W = pre[p.bt.n_seqs];
    const float scale = kLog2e / sqrtf((float)HD);
    for (int x = blockIdx.x; x < W; x += gridDim.x) {
        const int s = b2p::prefix_find(pre, p.bt.n_seqs, x);
        const b2p::Seq sq = p.bt.seq(s);
        const int nb = (sq.len + kBlk - 1) / kBlk, g = (x - pre[s]) / nb, j0 = (x - pre[s]) % nb * kBlk + warp * 16;
        if (j0 >= sq.len) continue;
        const int page = p.bt.page(s, j0);
        const int rows = min(sq.Q, p.max_q) * p.G;
        const int ja = j0 + n, jb = ja + 8;
        float acc[2] = {0.f, 0.f};
        // first row that may see a slot of this warp, down to a column tile's start
        const int r_first = max(0, j0 - sq.base) * p.G / 8 * 8;
        if (page >= 0 && r_first < rows) {
            const uint16_t* kp = p.k + page * p.page_stride + g * p.head_stride +
                                 (long long)((j0 & ((1 << p.bt.page_shift) - 1)) + n) * p.row_stride + 8 * c4;
            uint4 a[2][HD / 32];
#pragma unroll
            for (int u = 0; u < HD / 32; u++) {
                a[0][u] = b2::ld_stream16(kp + 32 * u);
                a[1][u] = b2::ld_stream16(kp + 8 * p.row_stride + 32 * u);
            }
            for (int r0 = r_first; r0 < rows; r0 += 8) {
                const int rq = r0 + n;
                uint4 b[HD / 32];
                const __half* qp = p.q16 + (size_t)(sq.row0 + rq / p.G) * p.ldq + (size_t)(g * p.G + rq % p.G) * HD + 8 * c4;
#pragma unroll
                for (int u = 0; u < HD / 32; u++)
                    b[u] = rq < rows ? *reinterpret_cast<const uint4*>(qp + 32 * u) : make_uint4(0, 0, 0, 0);
                float l2[2];
                int lim[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = r0 + 2 * c4 + e;
                    const float l = r < rows ? p.lse[(size_t)(sq.row0 + r / p.G) * p.nq + g * p.G + r % p.G] : -INFINITY;
                    lim[e] = l == -INFINITY ? -1 : min(sq.len - 1, sq.base + r / p.G);
                    l2[e] = l * kLog2e;
                }
                float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < HD / 32; u++) {
                    const uint32_t f0[4] = {a[0][u].x, a[1][u].x, a[0][u].y, a[1][u].y};
                    const uint32_t f1[4] = {a[0][u].z, a[1][u].z, a[0][u].w, a[1][u].w};
                    b2p::mma16816(sc, f0, b[u].x, b[u].y);
                    b2p::mma16816(sc, f1, b[u].z, b[u].w);
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if (ja <= lim[e]) acc[0] += b2p::ex2(fmaf(sc[e], scale, -l2[e]));
                    if (jb <= lim[e]) acc[1] += b2p::ex2(fmaf(sc[e + 2], scale, -l2[e]));
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 1);
            acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 2);
        }
        const int j = c4 == 0 ? ja : jb;
        if (c4 < 2 && j < sq.len && j < p.ldw) {
            const size_t o = ((size_t)s * p.nkv + g) * p.ldw + j;
            p.weights[o] = (p.prev ? p.prev[o] : 0.f) + (c4 == 0 ? acc[0] : acc[1]);
        }
    }
}

}  // namespace

extern "C" int b2_attention_paged_weights(float* weights, const float* prev, long long ldw, const uint16_t* q16, int ldq,
                                          const float* lse, int M, int max_q, int nq, int nkv, int hd,
                                          const B2PagedKV* kv, int* err, b2_stream_t s) {
    int rc = b2_paged_check("b2_attention_paged_weights", kv, nkv, hd, true);
    if (rc) return rc;
    if (!weights || !q16 || !lse || !err || ldw < 0 || M < 0 || max_q < 0 || nq <= 0 || nq % nkv || nq / nkv > 16)
        return b2_set_error(B2_ERR_INVALID_ARG,
                            "b2_attention_paged_weights: bad arguments (nq a multiple of nkv, at most 16)");
    if (ldq < nq * hd || ldq % 8 || (reinterpret_cast<uintptr_t>(q16) & 15))
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
    const WeightParams p{b2p::make_batch(kv, M), kv->k_pages, kv->page_stride, kv->head_stride, kv->row_stride,
                         reinterpret_cast<const __half*>(q16), ldq, lse, max_q, nq, nkv, nq / nkv, weights, prev, ldw};
    const long long grid = blocks < sms * 8 ? blocks : sms * 8;
    const cudaError_t e = b2::launch_pdl(hd == 128 ? weights_short_kernel<128> : weights_short_kernel<64>,
                                         dim3((unsigned)grid), dim3(kThreads), 0, (cudaStream_t)s, p);
    if (e != cudaSuccess) return b2_set_error(B2_ERR_CUDA, "b2_attention_paged_weights: %s", cudaGetErrorString(e));
    return 0;
}
