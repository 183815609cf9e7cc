// Rows to 4-bit floats with a scale for each group of columns (yk_quant_fp4).
#include "fp4.cuh"

namespace yk {

struct QuantFp4Args {
  YkQuantFp4 p;
  int blocks;       // scale blocks along a row
  int x_vec, v_vec; // x, values allow 16-byte accesses
};

// HBM bound: x is read once, everything else written once.  A CTA has 128 rows (a scale block's) of 256
// columns: a warp takes a row's 256 at a time, a lane 8 of them, so that a group is 2 or 4 neighbouring
// lanes and its maximum one or two shuffles; four rows are in flight.  Scales meet in shared memory and
// leave as whole blocks, as a group's own byte would be a 32-byte sector of its own.
// The division is x * r with r = 1 / S rounded, then one correction by the remainder x - q S (Markstein,
// 1990): it rounds as x / S does, so that values halfway between two codes go the way that the definition says, at two
// packed FMAs for two columns.  Groups with infinities or NaN, tiny or clamped scales divide plainly.
constexpr int kQuantCols = 256, kQuantThreads = 256;

template <bool BF16, bool NV>
__global__ void __launch_bounds__(kQuantThreads) quant_fp4_kernel(const __grid_constant__ QuantFp4Args a) {
  constexpr int kLanes = NV ? 2 : 4;                 // of a group
  constexpr int kBlocks = NV ? 4 : 2;                // scale blocks of 256 columns
  constexpr int kRows = 4;                           // of a warp in flight
  __shared__ __align__(16) uint8_t sc[kBlocks * kFp4Block];
  const YkQuantFp4& p = a.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.y * 128, c = blockIdx.x * kQuantCols + lane * 8;
  const int rows = min(128, p.rows - row0), cols = p.cols - c;      // columns from the lane's first on
  for (int i = threadIdx.x; i < kBlocks * kFp4Block / 4; i += kQuantThreads) ((uint32_t*)sc)[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int g = lane / kLanes;                       // group of the CTA's columns
  uint8_t* const sc_at = sc + g / 4 * kFp4Block + g % 4;
  for (int r0 = warp; r0 < rows; r0 += 8 * kRows) {
    uint4 raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int r = r0 + 8 * i;
      const uint16_t* x = (const uint16_t*)p.x + (long long)(row0 + r) * p.x_row + c;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (r >= rows || cols <= 0) continue;
      if (a.x_vec && cols >= 8) {
        raw[i] = __ldcs((const uint4*)x);
      } else {
        uint32_t* u = (uint32_t*)&raw[i];
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (e < cols) u[e >> 1] |= (uint32_t)x[e] << (16 * (e & 1));
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int r = r0 + 8 * i;
      if (r >= rows) break;                          // (the whole warp)
      const uint32_t* u = (const uint32_t*)&raw[i];
      float2 v[4];
      uint32_t top = 0;                              // largest |x| as bits: a NaN is above infinity
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[e] = pair_to_float2<BF16>(u[e]);
        top = max(top, max(__float_as_uint(v[e].x) & 0x7fffffffu, __float_as_uint(v[e].y) & 0x7fffffffu));
      }
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
      const bool nan = top > 0x7f800000u;
      float amax = __uint_as_float(top);
      if (__any_sync(~0u, top >= 0x7f800000u)) {     // rare: finite values only
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) m = fmaxf(m, fmaxf(finite_abs(v[e].x), finite_abs(v[e].y)));
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        amax = m;
      }
      const float t = amax / (6.f * p.scale);
      float s;
      uint32_t byte;
      bool plain = top >= 0x7f800000u;
      if (NV) {
        byte = float2_to_e4m3x2(fminf(fmaxf(t, 0.001953125f), 448.f), 0.f) & 0xffu;
        s = e4m3x2_to_float2(byte).x;
        plain |= t > 448.f;
      } else {
        // the exponent of the smallest power of two >= t, as a float's biased one
        const uint32_t b = __float_as_uint(t);
        byte = min(max((b >> 23) + ((b & 0x7fffffu) != 0), 127u - 96u), 127u + 96u);
        s = __uint_as_float(byte << 23);
        plain |= t > 7.9228162514264338e28f;         // 2^96
      }
      const float S = s * p.scale;
      plain |= S < 8.6736174e-19f;                   // 2^-60: the remainder below would lose bits
      if (nan) byte = NV ? 0x7fu : 0xffu;
      float q[8];
      if (plain) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float d = (e & 1 ? v[e >> 1].y : v[e >> 1].x) / S;
          q[e] = nan ? 0.f : fminf(fmaxf(d, -6.f), 6.f);
        }
      } else {
        const float inv = 1.f / S;
        const float2 r2 = make_float2(inv, inv), s2 = make_float2(-S, -S);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 q0 = mul2(v[e], r2), d = ffma2(ffma2(q0, s2, v[e]), r2, q0);
          q[2 * e] = d.x;
          q[2 * e + 1] = d.y;
        }
      }
      // signs come from x itself: those of zeros and of quotients that underflow would be lost
      const uint32_t s01 = __byte_perm(u[0], u[1], 0x7531), s23 = __byte_perm(u[2], u[3], 0x7531);
      const uint32_t signs = (__byte_perm(s01, s23, 0x6420) & 0x80808080u) >> 4 | (__byte_perm(s01, s23, 0x7531) & 0x80808080u);
      const uint32_t codes = floats_to_e2m1x8(q) | (nan ? 0u : signs);
      if (lane % kLanes == 0 && cols > 0) sc_at[r % 32 * 16 + r / 32 * 4] = (uint8_t)byte;
      if (cols <= 0) continue;
      *(uint32_t*)((uint8_t*)p.codes + (long long)(row0 + r) * p.codes_row + c / 2) = codes;
      if (p.values) {
        uint32_t h[4], o[4];
        e2m1x8_to_half2x4(codes, h);
        const float f = nan ? __uint_as_float(0x7fc00000u) : S;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 w = mul2(mul2(__half22float2(*(const __half2*)&h[e]), make_float2(16384.f, 16384.f)), make_float2(f, f));
          o[e] = float2_to_pair<BF16>(w.x, w.y);
        }
        uint16_t* to = (uint16_t*)p.values + (long long)(row0 + r) * p.values_row + c;
        if (a.v_vec && cols >= 8) {
          *(uint4*)to = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (e < cols) to[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
  __syncthreads();
  // this CTA's blocks lie behind one another
  const int b0 = blockIdx.x * kBlocks, nb = min(kBlocks, a.blocks - b0);
  uint4* to = (uint4*)((uint8_t*)p.scales + ((long long)blockIdx.y * a.blocks + b0) * kFp4Block);
  for (int i = threadIdx.x; i < nb * kFp4Block / 16; i += kQuantThreads) to[i] = ((const uint4*)sc)[i];
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
  if (p->rows > 65535 * 128 || p->cols > 1 << 30) return refuse(YK_EUNSUP, "quant_fp4: at most 8388480 rows and 2^30 columns");
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
  a.blocks = fp4_blocks(p->cols, p->format);
  a.x_vec = aligned16(p->x) && p->x_row % 8 == 0;
  a.v_vec = aligned16(p->values) && p->values_row % 8 == 0;
  const bool bf = p->dtype == YK_BF16, nv = p->format == YK_NVFP4;
  const auto kern = nv ? bf ? quant_fp4_kernel<true, true> : quant_fp4_kernel<false, true>
                       : bf ? quant_fp4_kernel<true, false> : quant_fp4_kernel<false, false>;
  launch_k(kern, dim3((unsigned)((p->cols + (long long)kQuantCols - 1) / kQuantCols), (unsigned)((p->rows + 127) / 128)),
           kQuantThreads, 0, (cudaStream_t)st, a);
  note_launch();
  return check_launch("quant_fp4");
}
