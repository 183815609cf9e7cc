// Helpers of the 4-bit float operators (quant_fp4.cu, gemm_fp4.cu): conversion, scale places, scaled MMAs.
#pragma once
#include "text.cuh"

namespace yk {

constexpr int kFp4Block = 512;       // bytes of 128 rows x 4 groups of scales
static inline int fp4_group(int format) { return format == YK_NVFP4 ? 16 : 32; }
// Scale blocks along a row of `cols` columns.
static inline int fp4_blocks(int cols, int format) { return (int)(((long long)cols + 4 * fp4_group(format) - 1) / (4 * fp4_group(format))); }
static inline bool fp4_format(int f) { return f == YK_NVFP4 || f == YK_MXFP4; }

// Eight floats to e2m1 codes, the first in the lowest 4 bits; round to nearest even, saturating at +-6.
__device__ __forceinline__ uint32_t floats_to_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight codes as half2 pairs; exact.  (A byte register has to be the low one of its word: the upper ones of an unpacked
// word read as the low one.)
__device__ __forceinline__ void e2m1x8_to_half2x4(uint32_t codes, uint32_t (&h)[4]) {
#pragma unroll
  for (int e = 0; e < 4; e++)
    asm("{\n\t.reg .b8 a, b;\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tmov.b16 {a, b}, lo;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}"
        : "=r"(h[e]) : "r"(codes >> (8 * e)));
}
// Packed 16-bit maximum of |a| and |b|; a NaN stays.
template <bool BF16>
__device__ __forceinline__ uint32_t amax_nan_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
  return r;
}

// D[tmem] (+)= A[smem] * B[smem]^T over 64 columns of e2m1 codes with scales in TMEM, fp32 sums.
template <bool NV>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                           uint32_t accumulate) {
  if (NV)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
// The same over the shared memory of a CTA pair, M = 256.
template <bool NV>
__device__ __forceinline__ void tc_mma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                                uint32_t accumulate) {
  if (NV)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
// Instruction descriptor: e2m1 A and B, both K-major, M = m (128, a pair 256), N = n; the scales are e4m3 or powers of
// two.  The latter come two a step: `half` says which two of the four in a TMEM word.
template <bool NV>
__host__ __device__ constexpr uint32_t idesc_fp4(int m, int n, int half = 0) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (NV ? 0u : 1u << 23) | ((uint32_t)(m >> 7) << 27) |
         (uint32_t)(2 * half) << 4 | (uint32_t)(2 * half) << 29;
}

// One lane of the warp, the same at each call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Arrive on another CTA's barrier, for accesses to TMEM that tcgen05.wait and tcgen05.fence have ordered.  A release at
// cluster scope would wait for the thread's own stores too (1200 cycles beside the loads of a product).
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// mbar_wait for a phase that is due: tries a while before it reads the clock and the limit of the wait, as the load of the
// limit from memory alone takes longer than four MMAs.
__device__ __forceinline__ bool mbar_wait_due(uint32_t bar, uint32_t parity, int code) {
#pragma unroll 1
  for (int i = 0; i < 256; i++)
    if (mbar_try(bar, parity)) return true;
  return mbar_wait(bar, parity, code);
}

// Bytes from global to shared memory, completing on the mbarrier; 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar) : "memory");
}

}  // namespace yk
