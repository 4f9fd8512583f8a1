// tcgen05 wrappers shared by the paged-cache kernels.
#pragma once
#include "b2_paged.cuh"

namespace b2p {

__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc512(uint32_t* to) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(to)), "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free512(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}
// The issuing warp runs converged and `lead` (one lane, always the same) issues:
// with a divergent branch around them every operand would go through a vector
// register first (4096 new rows after 12288: 555 us with it, 534 without).
__device__ __forceinline__ void umma_commit(uint64_t* bar, uint32_t lead) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q "
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
        "r"(lead)
        : "memory");
}
// A value that is the same in every lane, said so to the compiler.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
// Operand in 128-byte rows with the 128-byte swizzle, eight-row groups 1024 bytes
// apart.  K-major (Q, K): a row is 64 consecutive k.  Also the form of V, whose
// rows are k and whose 64-wide column chunks lie `lead` bytes apart.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)((lead >> 4) & 0x3FFF) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16: FP16 operands, FP32 accumulator; bit 16: B's rows are k (MN-major).
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
    return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q "
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
// A from tensor memory.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q "
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
#define B2_R32(v, o)                                                                                                  \
    "=r"(v[o + 0]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]),   \
        "=r"(v[o + 7]), "=r"(v[o + 8]), "=r"(v[o + 9]), "=r"(v[o + 10]), "=r"(v[o + 11]), "=r"(v[o + 12]),            \
        "=r"(v[o + 13]), "=r"(v[o + 14]), "=r"(v[o + 15]), "=r"(v[o + 16]), "=r"(v[o + 17]), "=r"(v[o + 18]),         \
        "=r"(v[o + 19]), "=r"(v[o + 20]), "=r"(v[o + 21]), "=r"(v[o + 22]), "=r"(v[o + 23]), "=r"(v[o + 24]),         \
        "=r"(v[o + 25]), "=r"(v[o + 26]), "=r"(v[o + 27]), "=r"(v[o + 28]), "=r"(v[o + 29]), "=r"(v[o + 30]),         \
        "=r"(v[o + 31])
// 32 columns of this warp's lanes into v[O..O+31] (no wait).
template <int O, int N>
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[N]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : B2_R32(v, O)
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define B2_I32(v)                                                                                                \
    "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), \
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),          \
        "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),          \
        "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        B2_I32(v)
        : "memory");
}

// Pairs of FP32 values in one instruction.
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// (2^x, 2^y) without the exponential unit: x = n + f with n whole and |f| <= 1/2
// (adding 1.5 2^23 rounds to whole numbers), 2^f by the polynomial of degree 5 of
// least relative error (7.5e-8 before rounding, 2.1e-7 with FP32 arithmetic; fitted
// by the Remez exchange), and 2^n from its exponent field,
// which is 0 from n = -127 down and infinity from 128 up.  NaN gives NaN.
__device__ __forceinline__ uint64_t ex2_f2(float x, float y) {
    asm("{max.NaN.f32 %0, %0, %2; max.NaN.f32 %1, %1, %2; min.NaN.f32 %0, %0, %3; min.NaN.f32 %1, %1, %3;}"
        : "+f"(x), "+f"(y)
        : "f"(-127.f), "f"(128.f));
    const uint64_t v = pack_f2(x, y), magic = pack_f2(12582912.f, 12582912.f);
    const uint64_t r = add_f2(v, magic), n = add_f2(r, pack_f2(-12582912.f, -12582912.f));
    const uint64_t f = fma_f2(n, pack_f2(-1.f, -1.f), v);
    auto both = [](float c) { return pack_f2(c, c); };
    uint64_t p = fma_f2(both(0x1.5c08e6p-10f), f, both(0x1.3d0c52p-7f));
    p = fma_f2(p, f, both(0x1.c6b6e4p-5f));
    p = fma_f2(p, f, both(0x1.ebf918p-3f));
    p = fma_f2(p, f, both(0x1.62e428p-1f));
    p = fma_f2(p, f, both(0x1.000002p+0f));
    float a, b;
    unpack_f2(r, a, b);
    return mul_f2(p, pack_f2(__uint_as_float((__float_as_uint(a) << 23) + 0x3f800000u),
                             __uint_as_float((__float_as_uint(b) << 23) + 0x3f800000u)));
}
// One column of a warp's 32 lanes.
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t addr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// max of three (a NaN loses).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Tensor map of the q16 rows: (64 dims, q heads of a group, tokens, head_dim / 64,
// kv heads); a box is `tokens` x the whole group, so a tile's rows land as token *
// G + head, each 64-dim half [rows][128 bytes].
inline int q_map(CUtensorMap* map, const void* q16, int ldq, int M, int nkv, int G, int hd, int tokens) {
    const uint64_t dims[5] = {64, (uint64_t)G, (uint64_t)M, (uint64_t)hd / 64, (uint64_t)nkv};
    const uint64_t strides[4] = {(uint64_t)hd * 2, (uint64_t)ldq * 2, 128, (uint64_t)G * hd * 2};
    const uint32_t box[5] = {64, (uint32_t)G, (uint32_t)tokens, 1, 1};
    return b2_tensor_map_f16_5d(map, q16, dims, strides, box);
}

}  // namespace b2p
