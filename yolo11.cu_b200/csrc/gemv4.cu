// Products of a few rows with a 4-bit weight matrix (yk_gemv4).
#include "text.cuh"

namespace yk {

// HBM bound for a few rows: n * k / 2 bytes of codes against 2 * rows * n * k operations.  The
// codes go through the warp MMA (m16n8k16, fp32 sums) as its A operand, 16 outputs a tile, and
// rows of x as the B operand, 8 a tile: a code costs about one instruction to become a 16-bit
// integer (bit masks into the mantissa of 1024 or 128, one packed subtraction of the zero point,
// all exact), where scalar products would cost three a row.  Scales multiply the fp32 sums at each
// group's end.
//  * A chunk is 16 outputs x 128 columns (1 KB).  cp.async brings it by 16-byte pieces into the
//    warp's own ring, piece (output, 32-column block) at block * 256 + output * 16, so that lane
//    (g, t) reads its word t of outputs g and g + 8 of a block without bank conflicts; the block's
//    32 columns are two MMAs, in an order of columns that x follows.
//  * Scales and zero points of the chunk travel in the same stage, as the aligned words that hold
//    them.
//  * The CTA's 8 warps are WN along the outputs times WK along the columns; each warp takes R
//    output tiles, which share the x operand.  The WK partial sums meet in shared memory.
struct Gemv4Args {
  YkGemv4 p;
  int x_vec;       // x rows allow 16-byte (e4m3: 8-byte) loads
  int zero;        // there are zero points
  int bf16;        // type of scales and y
  int xgroup;      // columns of a scale of e4m3 x; 0: one a row, or none
};
constexpr int kGemvWarps = 8;

template <bool F16>
__device__ __forceinline__ void mma_gemv(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16) {
    mma16816(d, a, b0, b1);
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*(const __half2*)&a, *(const __half2*)&b);
  return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*(const __half2*)&a, *(const __half2*)&b, *(const __half2*)&c);
  return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t bsub2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
  return *(const uint32_t*)&r;
}
// The 8 codes of a word minus the zero point z: pairs (0, 4), (1, 5), (2, 6), (3, 7).
// fp16: 1024 + q in the low nibble's place; 1024 + 16 q a nibble higher, times 1/16.
template <bool F16>
__device__ __forceinline__ void codes8(uint32_t w, uint32_t z, uint32_t (&o)[4]) {
  if (F16) {
    const uint32_t z0 = 0x64006400u | z * 0x10001u, z1 = 0xd400d400u + z * 0x100010u;   // 1024 + z, -(64 + z)
    o[0] = hsub2((w & 0x000f000fu) | 0x64006400u, z0);
    o[1] = hfma2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, z1);
    w >>= 8;
    o[2] = hsub2((w & 0x000f000fu) | 0x64006400u, z0);
    o[3] = hfma2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, z1);
  } else {
    const uint32_t z0 = 0x43004300u | z * 0x10001u;                                     // 128 + z
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = bsub2(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u, z0);
  }
}

template <int NT, int R>
struct Gemv {
  static constexpr int kStages = R == 1 ? 5 : 4;
  static constexpr int kTile = 1024 + 256 + 256;     // codes, scales, zero points of 16 outputs
  static constexpr int kStage = R * kTile;
  static constexpr int kRing = kGemvWarps * kStages * kStage, kMeet = kGemvWarps * R * NT * 512;
  static constexpr int kSmem = kRing > kMeet ? kRing : kMeet;
};

// XT: type of x; the MMA is bf16 for bf16 rows and fp16 otherwise (e4m3 converts exactly).
template <int XT, int NT, int R, int WN>
__global__ void __launch_bounds__(32 * kGemvWarps, NT == 8 ? 1 : 2) gemv4_kernel(const __grid_constant__ Gemv4Args ga) {
  using S = Gemv<NT, R>;
  constexpr bool X8 = XT == YK_E4M3, F16 = XT != YK_BF16;
  constexpr int WK = kGemvWarps / WN, kStages = S::kStages, kStage = S::kStage, kTile = S::kTile;
  extern __shared__ __align__(16) uint8_t gemv_sm[];
  uint8_t* const sm = gemv_sm;
  const YkGemv4& p = ga.p;
  const bool zero = ga.zero;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int wn = warp % WN, wk = warp / WN;
  const int n0 = (blockIdx.x * WN + wn) * R * 16;   // this warp's first output
  const int K = p.k, G = p.group, chunks = (K + 127) / 128;
  const int count = n0 < p.n && chunks > wk ? (chunks - wk + WK - 1) / WK : 0;
  const uint32_t ring = smem_u32(sm) + warp * kStages * kStage;

  const uint8_t* wrow[R][2];
  const uint8_t *srow[R][2], *zrow[R][2];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const long long n = min(n0 + r * 16 + g + 8 * i, p.n - 1);
      wrow[r][i] = (const uint8_t*)p.w + n * p.w_row + t * 16;
      srow[r][i] = (const uint8_t*)p.wscale + n * p.group_row * 2;
      zrow[r][i] = zero ? (const uint8_t*)p.wzero + n * p.group_row : nullptr;
    }
  const uint8_t* s_end = (const uint8_t*)p.wscale + ((long long)(p.n - 1) * p.group_row + K / G) * 2;
  const uint8_t* z_end = zero ? (const uint8_t*)p.wzero + (long long)(p.n - 1) * p.group_row + K / G : nullptr;
  const int t_group = t * 32 / G;                    // group of block t in its chunk
  // the aligned word around `a`, up to the array's end
  const auto word = [&](uint32_t dst, const uint8_t* a, const uint8_t* end, bool ok) {
    const uint8_t* w = (const uint8_t*)((uintptr_t)a & ~(uintptr_t)3);
    const int bytes = ok ? (int)min((long long)4, (long long)(end - w)) : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(w), "r"(bytes) : "memory");
  };
  uint32_t fill = ring;
  const auto issue = [&](int i) {
    if (i < count) {
      const int c = wk + i * WK;
      const bool ok = c * 128 + t * 32 < K;
      const int gi = c * (128 / G) + t_group;
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t at = fill + r * kTile;
          cp_async16(at + t * 256 + (g + 8 * h) * 16, wrow[r][h] + (ok ? c * 64ll : 0), ok ? 16 : 0);
          word(at + 1024 + h * 128 + lane * 4, srow[r][h] + (ok ? gi * 2 : 0), s_end, ok);
          if (zero) word(at + 1280 + h * 128 + lane * 4, zrow[r][h] + (ok ? gi : 0), z_end, ok);
        }
      fill = fill + kStage == ring + kStages * kStage ? ring : fill + kStage;
    }
    cp_async_commit();
  };
  pdl_wait();
  pdl_trigger();
#pragma unroll
  for (int i = 0; i < kStages - 1; i++) issue(i);

  float tot[R][NT][4];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < NT; j++) tot[r][j][0] = tot[r][j][1] = tot[r][j][2] = tot[r][j][3] = 0.f;
  // x of row j * 8 + g, columns k .. k + 7 (k < K): pairs (0, 4), (1, 5), (2, 6), (3, 7)
  const auto load_x = [&](int j, int k, uint32_t (&o)[4]) {
    const int m = j * 8 + g;
    if (m >= p.rows || k >= K) {
      o[0] = o[1] = o[2] = o[3] = 0;
      return;
    }
    const long long at = (long long)m * p.x_row + k;
    if (X8) {
      const uint8_t* x = (const uint8_t*)p.x + at;
      uint2 v;
      if (ga.x_vec) {
        v = *(const uint2*)x;
      } else {
        v.x = x[0] | x[1] << 8 | x[2] << 16 | (uint32_t)x[3] << 24;
        v.y = x[4] | x[5] << 8 | x[6] << 16 | (uint32_t)x[7] << 24;
      }
      e4m3x4_to_half2x2(__byte_perm(v.x, v.y, 0x5140), o[0], o[1]);
      e4m3x4_to_half2x2(__byte_perm(v.x, v.y, 0x7362), o[2], o[3]);
    } else {
      const uint16_t* x = (const uint16_t*)p.x + at;
      uint4 v;
      if (ga.x_vec) {
        v = *(const uint4*)x;
      } else {
        v = make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16,
                       x[6] | (uint32_t)x[7] << 16);
      }
      o[0] = __byte_perm(v.x, v.z, 0x5410);
      o[1] = __byte_perm(v.x, v.z, 0x7632);
      o[2] = __byte_perm(v.y, v.w, 0x5410);
      o[3] = __byte_perm(v.y, v.w, 0x7632);
    }
  };

  uint32_t src = ring;
#pragma unroll 1
  for (int i = 0; i < count; i++) {
    issue(i + kStages - 1);
    cp_async_wait<kStages - 1>();
    __syncwarp();                 // every lane's pieces of this stage are there
    const int c = wk + i * WK;
    float acc[R][NT][4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const bool starts = b * 32 % G == 0, ends = (b + 1) * 32 % G == 0;   // of a group of scales
      uint32_t x[NT][4];
#pragma unroll
      for (int j = 0; j < NT; j++) load_x(j, c * 128 + b * 32 + t * 8, x[j]);
#pragma unroll
      for (int r = 0; r < R; r++) {
        if (starts) {
#pragma unroll
          for (int j = 0; j < NT; j++) acc[r][j][0] = acc[r][j][1] = acc[r][j][2] = acc[r][j][3] = 0.f;
        }
        const uint32_t at = src + r * kTile;
        uint32_t q[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t z = 8;
          if (zero) {
            const uint32_t low = (uint32_t)(uintptr_t)(zrow[r][h] + c * (128 / G) + b * 32 / G) & 3;
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(z) : "r"(at + 1280 + h * 128 + (g * 4 + b) * 4 + low));
          }
          uint32_t w;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at + b * 256 + (g + 8 * h) * 16 + t * 4));
          codes8<F16>(w, z, q[h]);
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t a[4] = {q[0][2 * e], q[1][2 * e], q[0][2 * e + 1], q[1][2 * e + 1]};
#pragma unroll
          for (int j = 0; j < NT; j++) mma_gemv<F16>(acc[r][j], a, x[j][2 * e], x[j][2 * e + 1]);
        }
        if (ends) {
          float s[2];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t low = (uint32_t)(uintptr_t)(srow[r][h] + (c * (128 / G) + b * 32 / G) * 2) & 2;
            uint16_t u;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(at + 1024 + h * 128 + (g * 4 + b) * 4 + low));
            s[h] = XT == YK_BF16 || (X8 && ga.bf16) ? elem_to_float<true>(u) : elem_to_float<false>(u);
          }
#pragma unroll
          for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float xs = 1.f;
              if (X8 && ga.xgroup) {
                const int m = min(j * 8 + 2 * t + e, p.rows - 1);
                xs = p.xscale[m * p.xscale_row + min(c * 128 + b * 32, K - 1) / ga.xgroup];
              }
              tot[r][j][e] = fmaf(acc[r][j][e], s[0] * xs, tot[r][j][e]);
              tot[r][j][2 + e] = fmaf(acc[r][j][2 + e], s[1] * xs, tot[r][j][2 + e]);
            }
        }
      }
    }
    __syncwarp();                 // every lane has read the stage
    src = src + kStage == ring + kStages * kStage ? ring : src + kStage;
  }
  cp_async_wait<0>();
  __syncthreads();
  // sums of the WK warps along the columns: [warp][tile][row of x][output]
  float* meet = (float*)sm;
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        meet[((warp * R + r) * NT * 8 + j * 8 + 2 * t + (e & 1)) * 16 + g + (e >> 1) * 8] = tot[r][j][e];
  __syncthreads();
  constexpr int kOut = WN * R * 16;
  for (int i = tid; i < kOut * p.rows; i += 32 * kGemvWarps) {
    const int m = i / kOut, j = i % kOut, n = blockIdx.x * kOut + j;
    if (n >= p.n) continue;
    const int w = j / (R * 16), r = j / 16 % R;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WK; k++) v += meet[(((k * WN + w) * R + r) * NT * 8 + m) * 16 + j % 16];
    if (X8 && !ga.xgroup) v *= p.xscale[m * p.xscale_row];
    if (p.bias) v += p.bias[n];
    ((uint16_t*)p.y)[m * p.y_row + n] = ga.bf16 ? float_to_elem<true>(v) : float_to_elem<false>(v);
  }
}

template <int XT, int NT, int R, int WN>
static int launch_gemv4(const Gemv4Args& a, cudaStream_t st) {
  const auto kern = gemv4_kernel<XT, NT, R, WN>;
  if (smem_attr(kern, Gemv<NT, R>::kSmem) != cudaSuccess) return check_launch("gemv4 attr");
  constexpr int outputs = WN * R * 16;
  launch_k(kern, (a.p.n + outputs - 1) / outputs, 32 * kGemvWarps, Gemv<NT, R>::kSmem, st, a);
  note_launch();
  return check_launch("gemv4");
}
template <int XT>
static int launch_gemv4(const Gemv4Args& a, cudaStream_t st) {
  const int m = a.p.rows, n = a.p.n;
  if (m <= 8) return launch_gemv4<XT, 1, 1, 1>(a, st);
  if (m <= 16) return n >= 64 * 148 ? launch_gemv4<XT, 2, 2, 2>(a, st) : launch_gemv4<XT, 2, 1, 1>(a, st);
  if (m <= 32) return launch_gemv4<XT, 4, 1, 2>(a, st);
  return launch_gemv4<XT, 8, 1, 2>(a, st);
}

}  // namespace yk

using namespace yk;

extern "C" int yk_gemv4(const YkGemv4* p, yk_stream_t st) {
  if (!p || !p->x || !p->w || !p->wscale || !p->y) return refuse(YK_EINVAL, "gemv4: null pointer");
  if (p->dtype != YK_F16 && p->dtype != YK_BF16) return refuse(YK_EUNSUP, "gemv4: dtype must be fp16 or bf16");
  if (p->xtype != p->dtype && p->xtype != YK_E4M3)
    return refuse(YK_EUNSUP, "gemv4: xtype must be dtype or e4m3");
  if (p->rows < 1 || p->n < 1 || p->k < 1) return refuse(YK_EINVAL, "gemv4: rows, n and k must be positive");
  if (p->rows > 64) return refuse(YK_EUNSUP, "gemv4: at most 64 rows");
  if (p->group != 32 && p->group != 64 && p->group != 128)
    return refuse(YK_EUNSUP, "gemv4: group must be 32, 64 or 128");
  if (p->k % p->group) return refuse(YK_EINVAL, "gemv4: k must be a multiple of group");
  const bool x8 = p->xtype == YK_E4M3;
  if (x8 && (!p->xscale || p->xgroup < 0 || p->xgroup % p->group))
    return refuse(YK_EINVAL, "gemv4: e4m3 rows need scales, and an xgroup that is a multiple of group");
  if (!aligned16(p->w) || p->w_row % 16 || p->w_row < p->k / 2 || p->group_row < p->k / p->group ||
      p->x_row < 0 || p->y_row < p->n)
    return refuse(YK_EINVAL, "gemv4: weights need 16-byte alignment, strides at least a row");
  if (x8 && p->xscale_row < (p->xgroup ? (p->k + p->xgroup - 1) / p->xgroup : 1))
    return refuse(YK_EINVAL, "gemv4: xscale stride below its row");
  const uintptr_t at = (uintptr_t)p->x | (uintptr_t)(x8 ? p->x_row : p->x_row * 2);
  const Gemv4Args a{*p, at % (x8 ? 8 : 16) == 0, p->wzero != nullptr, p->dtype == YK_BF16, x8 ? p->xgroup : 0};
  cudaStream_t s = (cudaStream_t)st;
  return x8 ? launch_gemv4<YK_E4M3>(a, s) : a.bf16 ? launch_gemv4<YK_BF16>(a, s) : launch_gemv4<YK_F16>(a, s);
}
