// Helpers shared by the text-decoder operators (kv.cu, attn8.cu, norm8.cu, gemv4.cu, rotate.cu,
// quant_fp4.cu, gemm_fp4.cu, sample.cu): e4m3 conversion, 16-bit type selection, refusals with a reason.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace yk {

constexpr float kE4m3Max = 448.f;              // 1.75 * 2^8
constexpr float kMinScale = 1.17549435e-38f;   // 2^-126, the smallest normal float: 1 / scale is finite

// Reason of a refusal, read through yk_last_cuda_error(); returns `code`.
static int refuse(int code, const char* what) {
  snprintf(g_cuda_err, sizeof g_cuda_err, "%s", what);
  return code;
}
// SMs of the current device.
static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
}
static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Two e4m3 codes (low and high byte) as a half2; exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
// Four codes: bytes 0, 1 and bytes 2, 3.
__device__ __forceinline__ void e4m3x4_to_half2x2(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t codes) {
  const uint32_t h = e4m3x2_to_half2(codes & 0xffffu);
  return __half22float2(*(const __half2*)&h);
}
// Two floats to e4m3 codes, round to nearest even, saturating at +-448 (infinities too); NaN
// stays NaN.
__device__ __forceinline__ uint32_t float2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t float4_to_e4m3x4(float a, float b, float c, float d) {
  return float2_to_e4m3x2(a, b) | (float2_to_e4m3x2(c, d) << 16);
}

// 16-bit element pairs as floats and back.
template <bool BF16>
__device__ __forceinline__ float2 pair_to_float2(uint32_t u) {
  if (BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  return __half22float2(*(const __half2*)&u);
}
template <bool BF16>
__device__ __forceinline__ uint32_t float2_to_pair(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&v;
  }
  return pack_half2(a, b);
}
template <bool BF16>
__device__ __forceinline__ float elem_to_float(uint16_t u) {
  if (BF16) return __uint_as_float((uint32_t)u << 16);
  return __half2float(__ushort_as_half(u));
}
template <bool BF16>
__device__ __forceinline__ uint16_t float_to_elem(float a) {
  if (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(a));
  return __half_as_ushort(__float2half_rn(a));
}

// |v| of a finite v, 0 of an infinity or NaN.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}

// 1 / v to within one unit in the last place, for normal v with a normal inverse.
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Both products, rounded each; the sign of a zero stays (mul2 adds 0 to it).
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return ffma2(a, b, make_float2(0.f, 0.f)); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return ffma2(a, make_float2(1.f, 1.f), b); }
// Packed 16-bit maximum of m and |v|; a NaN in v is left out.
template <bool BF16>
__device__ __forceinline__ uint32_t amax_pair(uint32_t m, uint32_t v) {
  v &= 0x7fff7fffu;
  uint32_t r;
  if (BF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(v));
  else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(v));
  return r;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// cp.async of B bytes (16 or 8); without `ok`, zeros and no read.
template <int B>
__device__ __forceinline__ void cp_async_at(uint32_t dst, const void* src, bool ok) {
  if (B == 16) cp_async16(dst, src, ok ? 16 : 0);
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
}
template <int B>
__device__ __forceinline__ void cp_async_at(uint32_t dst, const void* src) {
  if (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

static inline int check_cache(const YkKvCache* c) {
  if (!c || !c->k || !c->v || !c->kscale || !c->vscale) return refuse(YK_EINVAL, "kv cache: null pointer");
  if (c->tokens != 16 && c->tokens != 32 && c->tokens != 64 && c->tokens != 128)
    return refuse(YK_EUNSUP, "kv cache: tokens of a block must be 16, 32, 64 or 128");
  if (c->dim != 64 && c->dim != 128 && c->dim != 256)
    return refuse(YK_EUNSUP, "kv cache: dim must be 64, 128 or 256");
  if (c->blocks < 1 || c->heads < 1 || (long long)c->blocks * c->tokens > 0x7fffffffll)
    return refuse(YK_EINVAL, "kv cache: blocks and heads must be positive, blocks * tokens below 2^31");
  if (!aligned16(c->k) || !aligned16(c->v) || c->block_stride % 16 ||
      c->block_stride < (long long)c->heads * c->tokens * c->dim || c->scale_stride < c->heads)
    return refuse(YK_EINVAL, "kv cache: codes need 16-byte alignment, strides at least one block's size");
  return YK_OK;
}

}  // namespace yk
