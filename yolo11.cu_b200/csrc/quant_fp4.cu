// Rows to 4-bit floats with a scale for each group of columns (yk_quant_fp4).
#include <math.h>

#include "fp4.cuh"

namespace yk {

struct QuantFp4Args {
  YkQuantFp4 p;
  int blocks;        // scale blocks along a row
  int x_align, v_align;   // 16 where rows of x, of values allow such accesses, else 2
  int exact;         // the matrix's scale is a power of two
  float six, over_six, over_scale;     // 6 scale, 1 / (6 scale), 1 / scale
};

// HBM bound: x is read once, everything else written once.  A CTA has 32 rows of 256 columns: a warp takes four rows'
// 256 at once, a lane 8 of each, so that a group is 2 or 4 neighbouring lanes and its maximum one or two shuffles.
// The rows are 8 behind one another and the ones 32, 64 and 96 further on, as their scales lie together
// (128 bytes of each block): they meet in shared memory, as a group's own byte would be a 32-byte sector of its own.
// The arithmetic would take longer than the memory if it divided:
//  * a / b is a * r with r = 1 / b rounded, then one correction by the remainder a - q b (Markstein, 1990): it rounds as
//    a / b does, so that values halfway between two codes go the way that the definition says.
//  * r comes from the 8 fractions that an e4m3 scale can have, times the matrix's scale, in a table; powers of two
//    move its exponent.  Where S is a power of two, the product alone is exact.
// Groups with infinities or NaN, tiny or clamped scales divide plainly; groups of zeros, which edges are full of, do not (460 x 429
// MXFP4: 10.9 -> 5.2 us).
// 12000 x 5120 to codes, scales and values: 53 us back to back, 5.2 TB/s, 57 with inputs that change (63 with a division and a
// byte store for each group; the same loads and stores without arithmetic 42.5, without that of the values 49; 4 or 6 CTAs
// an SM instead of 5 take 2 us more).
// Codes and scales alone, as the decoder has them: 42 us (NVFP4 45) of 24 that the bytes take; the instructions of the codes bound it.
// 16 x 4096: 2.8 us, the launch.
constexpr int kQuantCols = 256, kQuantThreads = 256;

// Eight 16-bit elements (two where there are fewer columns) at any even address, as pairs.
__device__ __forceinline__ uint4 quant_load8(const uint16_t* x, int align, int cols, bool first) {
  uint4 v = make_uint4(0, 0, 0, 0);
  uint32_t* u = (uint32_t*)&v;
  if (cols >= 8 && align == 16) return __ldcs((const uint4*)x);
  if (cols >= 8 && ((uintptr_t)x & 2) == 0) {
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = ((const uint32_t*)x)[e];
  } else if (cols >= 9 && !first) {
    // the pairs around them, from the element before to the one behind
    const uint32_t* w = (const uint32_t*)(x - 1);
    uint32_t last = w[0];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t next = w[e + 1];
      u[e] = __byte_perm(last, next, 0x5432);
      last = next;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < cols) u[e >> 1] |= (uint32_t)x[e] << (16 * (e & 1));
  }
  return v;
}
__device__ __forceinline__ void quant_store8(uint16_t* y, int align, int cols, const uint32_t (&o)[4]) {
  if (cols >= 8 && align == 16) {
    __stcs((uint4*)y, make_uint4(o[0], o[1], o[2], o[3]));
  } else if (cols >= 8 && ((uintptr_t)y & 2) == 0) {
#pragma unroll
    for (int e = 0; e < 4; e++) ((uint32_t*)y)[e] = o[e];
  } else if (cols >= 8) {
    y[0] = (uint16_t)o[0];
#pragma unroll
    for (int e = 0; e < 3; e++) ((uint32_t*)(y + 1))[e] = __byte_perm(o[e], o[e + 1], 0x5432);
    y[7] = (uint16_t)(o[3] >> 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < cols) y[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
  }
}

// The rare cases, out of line so that the others' code stays together: the largest finite |x| of a group's eight, and the
// codes (without signs) by division, 0 in a group with a NaN.
template <bool BF16>
__device__ __noinline__ float quant_finite_max(uint4 raw) {
  const uint32_t* u = (const uint32_t*)&raw;
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float2 v = pair_to_float2<BF16>(u[e]);
    m = fmaxf(m, fmaxf(finite_abs(v.x), finite_abs(v.y)));
  }
  return m;
}
template <bool BF16>
__device__ __noinline__ uint32_t quant_plain(uint4 raw, float S, bool nan) {
  const uint32_t* u = (const uint32_t*)&raw;
  float q[8];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float2 v = pair_to_float2<BF16>(u[e]);
    q[2 * e] = nan ? 0.f : fminf(fmaxf(v.x / S, -6.f), 6.f);
    q[2 * e + 1] = nan ? 0.f : fminf(fmaxf(v.y / S, -6.f), 6.f);
  }
  return floats_to_e2m1x8(q);
}

template <bool BF16, bool NV>
__global__ void __launch_bounds__(kQuantThreads, 5) quant_fp4_kernel(const __grid_constant__ QuantFp4Args a) {
  constexpr int kLanes = NV ? 2 : 4;                 // of a group
  constexpr int kBlocks = NV ? 4 : 2;                // scale blocks of 256 columns
  constexpr int kRows = 4;                           // of a warp
  __shared__ __align__(16) uint8_t sc[kBlocks * 128];
  __shared__ float2 fraction[8];                     // scale * (1 + i / 8), and 1 / that
  const YkQuantFp4& p = a.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = blockIdx.y & 3, row0 = (blockIdx.y >> 2) * 128;  // rows part * 8 + warp, and 32, 64, 96 on
  const int c = blockIdx.x * kQuantCols + lane * 8;
  const int rows = min(128, p.rows - row0), cols = p.cols - c;      // columns from the lane's first on
  if (threadIdx.x < kBlocks * 32) ((uint32_t*)sc)[threadIdx.x] = 0;
  if (NV && threadIdx.x >= 128 && threadIdx.x < 136) {
    const float m = p.scale * (1.f + 0.125f * (threadIdx.x - 128));
    fraction[threadIdx.x - 128] = make_float2(m, 1.f / m);
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int g = lane / kLanes;                       // group of the CTA's columns
  uint8_t* const sc_at = sc + g / 4 * 128 + warp * 16 + g % 4;
  {
    const int r0 = part * 8 + warp;
    uint4 raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int r = r0 + 32 * i;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (r < rows && cols > 0) raw[i] = quant_load8((const uint16_t*)p.x + (long long)(row0 + r) * p.x_row + c, a.x_align, cols, c == 0);
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int r = r0 + 32 * i;
      if (r >= rows) break;                          // (the whole warp)
      const uint32_t* u = (const uint32_t*)&raw[i];
      // largest |x|, NaN above infinity
      uint32_t top = amax_nan_pair<BF16>(amax_nan_pair<BF16>(u[0], u[1]), amax_nan_pair<BF16>(u[2], u[3]));
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) top = amax_nan_pair<BF16>(top, __shfl_xor_sync(~0u, top, o));
      top = amax_nan_pair<BF16>(top, top >> 16);
      float amax = elem_to_float<BF16>((uint16_t)top);
      const bool odd = !(amax < INFINITY), nan = amax != amax;
      if (__any_sync(~0u, odd)) {                    // rare: finite values only
        float m = quant_finite_max<BF16>(raw[i]);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        amax = m;
      }
      float S, inv;                                  // the group's scale * the matrix's, and its inverse
      uint32_t byte;
      bool plain = odd;
      if (NV) {
        const float q = amax * a.over_six, t = q < 512.f ? fmaf(fmaf(-q, a.six, amax), a.over_six, q) : q;   // (clamped beyond)
        byte = float2_to_e4m3x2(fminf(fmaxf(t, 0.001953125f), 448.f), 0.f) & 0xffu;
        plain |= !(t <= 448.f);
        const uint32_t s = __float_as_uint(e4m3x2_to_float2(byte).x), power = (s & 0x7f800000u) - 0x3f800000u;
        const float2 f = fraction[(s >> 20) & 7];
        S = __uint_as_float(__float_as_uint(f.x) + power);
        inv = __uint_as_float(__float_as_uint(f.y) - power);
      } else {
        // the smallest power of two >= amax / (6 scale): difference of the exponents, and one more if the fraction is larger
        const int e = ((int)(__float_as_uint(amax) - __float_as_uint(a.six)) + 0x7fffff) >> 23, k = min(max(e, -96), 96);
        plain |= e > 96;
        byte = k + 127;
        S = __uint_as_float(__float_as_uint(p.scale) + k * 0x800000);
        inv = __uint_as_float(__float_as_uint(a.over_scale) - k * 0x800000);
      }
      if (nan) byte = NV ? 0x7fu : 0xffu;
      plain |= S < 8.6736174e-19f && amax > 0.f;     // 2^-60: the remainder below would lose bits
      uint32_t codes;
      if (plain) {
        codes = quant_plain<BF16>(raw[i], S, nan);
      } else {
        float q[8];
        const float2 r2 = make_float2(inv, inv), s2 = make_float2(-S, -S);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 v = pair_to_float2<BF16>(u[e]);
          float2 d = fmul2(v, r2);
          if (NV || !a.exact) d = ffma2(ffma2(d, s2, v), r2, d);
          q[2 * e] = d.x;
          q[2 * e + 1] = d.y;
        }
        codes = floats_to_e2m1x8(q);
      }
      // signs come from x itself: those of zeros and of quotients that underflow would be lost
      const uint32_t s01 = __byte_perm(u[0], u[1], 0x7531), s23 = __byte_perm(u[2], u[3], 0x7531);
      const uint32_t signs = (__byte_perm(s01, s23, 0x6420) & 0x80808080u) >> 4 | (__byte_perm(s01, s23, 0x7531) & 0x80808080u);
      codes |= nan ? 0u : signs;
      if (lane % kLanes == 0 && cols > 0) sc_at[i * 4] = (uint8_t)byte;
      if (cols <= 0) continue;
      *(uint32_t*)((uint8_t*)p.codes + (long long)(row0 + r) * p.codes_row + c / 2) = codes;
      if (p.values) {
        uint32_t h[4], o[4];
        e2m1x8_to_half2x4(codes, h);
        const float f = nan ? __uint_as_float(0x7fc00000u) : S;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 w = fmul2(__half22float2(*(const __half2*)&h[e]), make_float2(f, f));
          o[e] = float2_to_pair<BF16>(w.x, w.y);
        }
        quant_store8((uint16_t*)p.values + (long long)(row0 + r) * p.values_row + c, a.v_align, cols, o);
      }
    }
  }
  __syncthreads();
  // this CTA's part of its blocks, which lie behind one another
  const int b0 = blockIdx.x * kBlocks, nb = min(kBlocks, a.blocks - b0);
  uint8_t* to = (uint8_t*)p.scales + ((long long)(blockIdx.y >> 2) * a.blocks + b0) * kFp4Block + part * 128;
  if (threadIdx.x < nb * 8) ((uint4*)(to + threadIdx.x / 8 * kFp4Block))[threadIdx.x % 8] = ((const uint4*)sc)[threadIdx.x];
}

}  // namespace yk

using namespace yk;

extern "C" size_t yk_fp4_scale_bytes(int rows, int cols, int format) {
  if (rows < 1 || cols < 1 || !fp4_format(format)) return 0;
  return (size_t)((rows + 127ll) / 128) * fp4_blocks(cols, format) * kFp4Block;
}

extern "C" int yk_quant_fp4(const YkQuantFp4* p, yk_stream_t st) {
  if (!p || !p->x || !p->codes || !p->scales) return refuse(YK_EINVAL, "quant_fp4: null pointer");
  if (!fp4_format(p->format)) return refuse(YK_EUNSUP, "quant_fp4: format must be YK_NVFP4 or YK_MXFP4");
  if (p->dtype != YK_F16 && p->dtype != YK_BF16) return refuse(YK_EUNSUP, "quant_fp4: dtype must be fp16 or bf16");
  if (p->rows < 0 || p->cols < 1) return refuse(YK_EINVAL, "quant_fp4: bad rows or cols");
  if (p->rows > 1 << 20 || p->cols > 1 << 30) return refuse(YK_EUNSUP, "quant_fp4: at most 2^20 rows and 2^30 columns");
  if (p->scale != 0.f && !(p->scale >= 9.3132257e-10f && p->scale <= 1073741824.f))
    return refuse(YK_EINVAL, "quant_fp4: scale must be 0 or between 2^-30 and 2^30");
  if (!aligned16(p->codes) || !aligned16(p->scales) || p->codes_row % 16 || p->codes_row < (p->cols + 1ll) / 2)
    return refuse(YK_EINVAL, "quant_fp4: codes and scales need 16-byte alignment, codes_row a multiple of 16 that holds a row");
  if (p->x_row < 0 || (p->values && p->values_row < p->cols))
    return refuse(YK_EINVAL, "quant_fp4: a row stride is negative or below its row");
  if (((uintptr_t)p->x | (uintptr_t)p->values) & 1) return refuse(YK_EINVAL, "quant_fp4: x and values need the alignment of their type");
  if (p->rows == 0) return YK_OK;
  QuantFp4Args a{*p};
  if (a.p.scale == 0.f) a.p.scale = 1.f;
  a.six = 6.f * a.p.scale;
  a.over_six = 1.f / a.six;
  a.over_scale = 1.f / a.p.scale;
  int power;
  a.exact = frexpf(a.p.scale, &power) == 0.5f;
  a.blocks = fp4_blocks(p->cols, p->format);
  a.x_align = aligned16(p->x) && p->x_row % 8 == 0 ? 16 : 2;
  a.v_align = aligned16(p->values) && p->values_row % 8 == 0 ? 16 : 2;
  const bool bf = p->dtype == YK_BF16, nv = p->format == YK_NVFP4;
  const auto kern = nv ? bf ? quant_fp4_kernel<true, true> : quant_fp4_kernel<false, true>
                       : bf ? quant_fp4_kernel<true, false> : quant_fp4_kernel<false, false>;
  launch_k(kern, dim3((unsigned)((p->cols + (long long)kQuantCols - 1) / kQuantCols), (unsigned)((p->rows + 127) / 128 * 4)),
           kQuantThreads, 0, (cudaStream_t)st, a);
  note_launch();
  return check_launch("quant_fp4");
}
