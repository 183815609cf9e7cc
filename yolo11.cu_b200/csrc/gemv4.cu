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
//  * Lane (g, t) reads the scales and zero points of block t of its outputs one chunk ahead; they
//    reach the other lanes by shuffles.  (In the ring, by aligned words, they cost as many L2
//    sectors as the codes.)
//  * The CTA's 8 warps are WN along the outputs times WK along the columns.  The WK partial sums meet
//    in shared memory.
// Measured (fp16 x, groups of 128): 1 x 4096 x 4096 6.7 us (of which a launch is about 2.5), 1 x 28672 x 8192 58 us,
// 2.0 TB/s: bound by the instructions around the MMAs (275 a KB of codes).  With one row 1 or 2 warps
// along the outputs (WN) are within 5 % there; small products want WN = 1 (512 outputs: 4.6 us, else 6.5 and
// more).
struct Gemv4Args {
  YkGemv4 p;
  int x_vec;       // x rows allow 16-byte (e4m3: 8-byte) loads
  int zero;        // there are zero points
  int s_vec;       // scales and zero points allow loads of 8 groups
  int bf16;        // type of scales and y
  int xgroup;      // columns of a scale of e4m3 x; 0: one a row, or none
  int x_shift;     // its logarithm, -1: not a power of two
  int x_inside;    // it may change inside a chunk of 128 columns
};
constexpr int kGemvWarps = 8;
// Which kernel, for more than 8 rows.  A round of this one's CTAs (two an SM of 16 or of 32 outputs, or one of
// 32) covers 1, 2, 1 times kGemvRound outputs for 9 - 16, 17 - 32, 33 - 64 rows.  The tcgen05 kernel
// (gemv4_tc.cuh) has 128 outputs a CTA, so one of its rounds covers four times that, at a higher price: it is
// taken where this one would need a fourth, a second, a second round.  Measured, us here | there, fp16 rows, 4096
// columns in groups of 64: 16 rows: 9472 outputs 18.5 | 26.3, 14208: 26.4 | 26.8, 18944: 34.1 | 27.6; 32 rows:
// 9472: 24.8 | 26.0, 9600: 41.3 | 26.0; 64 rows: 4096: 36.3 | 40.4, 4800: 66.2 | 40.4, 28672: 221 | 80 (512
// columns: 4800: 11.9 | 12.7).  1 and 8 rows of 28672 x 8192: 58 | 70, 67 | 70.
// e4m3 rows cost this kernel twice as much at 33 - 64 rows: 4096 x 4096, 64 rows 81 | 53, 33 rows 59 | 50 (512
// columns: 13.6 | 17.6, 9.6 | 15.1; groups of 32: 82 | 77, 61 | 73).  So there tcgen05 takes any number of outputs
// from kGemvLong columns on, except in groups of 32.
constexpr int kGemvRound = 32 * 148, kGemvLong = 2048;

// d = a * b + (first ? 0 : d)
template <bool F16>
__device__ __forceinline__ void mma_gemv(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  const float c0 = first ? 0.f : d[0], c1 = first ? 0.f : d[1], c2 = first ? 0.f : d[2], c3 = first ? 0.f : d[3];
  if (F16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
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
// A zero point z as the packed operands that codes8 takes.
struct Zero {
  uint32_t a, b;
};
template <bool F16>
__device__ __forceinline__ Zero zero_of(uint32_t z) {
  if (F16) return {0x64006400u + z * 0x10001u, 0xd400d400u + z * 0x100010u};   // 1024 + z, -(64 + z)
  return {0x43004300u + z * 0x10001u, 0};                                      // 128 + z
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {   // (a & b) | c
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// The 8 codes of a word minus the zero point: pairs (0, 4), (1, 5), (2, 6), (3, 7).  A known conversion: small
// integers put into the low mantissa bits of a power of two are that power plus the integer.
// fp16: 1024 + q in the low nibble's place; 1024 + 16 q a nibble higher, times 1/16.
template <bool F16>
__device__ __forceinline__ void codes8(uint32_t w, const Zero& z, uint32_t (&o)[4]) {
  if (F16) {
    o[0] = hsub2(and_or(w, 0x000f000fu, 0x64006400u), z.a);
    o[1] = hfma2(and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, z.b);
    w >>= 8;
    o[2] = hsub2(and_or(w, 0x000f000fu, 0x64006400u), z.a);
    o[3] = hfma2(and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, z.b);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = bsub2(and_or(w >> (4 * i), 0x000f000fu, 0x43004300u), z.a);
  }
}
template <int NT>
struct Gemv {
  static constexpr int kStages = 5;
  // codes of 16 outputs: four blocks, 32 bytes more than 256 apart so that the pieces a warp
  // writes at once fall into different banks
  static constexpr int kBlock = 256 + 32, kTile = 4 * kBlock;
  static constexpr int kRing = kGemvWarps * kStages * kTile, kMeet = kGemvWarps * NT * 512;
  static constexpr int kSmem = kRing > kMeet ? kRing : kMeet;
};

// XT: type of x; the MMA is bf16 for bf16 rows and fp16 otherwise (e4m3 converts exactly).
// GB: blocks (32 columns) of a group of w.
template <int XT, int GB, int NT, int WN>
__global__ void __launch_bounds__(32 * kGemvWarps, NT == 8 ? 1 : 2) gemv4_kernel(const __grid_constant__ Gemv4Args ga) {
  using S = Gemv<NT>;
  constexpr bool X8 = XT == YK_E4M3, F16 = XT != YK_BF16;
  constexpr int WK = kGemvWarps / WN, kStages = S::kStages, kTile = S::kTile;
  extern __shared__ __align__(16) uint8_t gemv_sm[];
  uint8_t* const sm = gemv_sm;
  const YkGemv4& p = ga.p;
  const bool zero = ga.zero;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int wn = warp % WN, wk = warp / WN;
  const int n0 = (blockIdx.x * WN + wn) * 16;   // this warp's first output
  const int K = p.k, chunks = (K + 127) / 128;
  const int count = n0 < p.n && chunks > wk ? (chunks - wk + WK - 1) / WK : 0;
  const uint32_t ring = smem_u32(sm) + warp * kStages * kTile;
  const uint8_t* const ring_p = sm + warp * kStages * kTile;

  // first codes, scales and zero points of this lane's outputs g, g + 8
  const uint8_t *wrow[2], *zrow[2];
  const uint16_t* srow[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const long long n = min(n0 + g + 8 * h, p.n - 1);
    wrow[h] = (const uint8_t*)p.w + n * p.w_row + t * 16;
    srow[h] = (const uint16_t*)p.wscale + n * p.group_row + t / GB;
    zrow[h] = (const uint8_t*)p.wzero + n * p.group_row + t / GB;
  }
  constexpr int kPer = 4 / GB;       // groups of a chunk
  const auto x_group = [&](int k) { return ga.x_shift >= 0 ? k >> ga.x_shift : k / ga.xgroup; };
  uint32_t fill = ring;
  const uint32_t piece = t * S::kBlock + g * 16;
  const auto issue = [&](int i) {
    if (i < count) {
      const int c = wk + i * WK;
      const bool ok = c * 128 + t * 32 < K;
#pragma unroll
      for (int h = 0; h < 2; h++) cp_async_at<16>(fill + piece + h * 128, wrow[h] + c * 64, ok);
      fill = fill + kTile == ring + kStages * kTile ? ring : fill + kTile;
    }
    cp_async_commit();
  };
  pdl_wait();
  pdl_trigger();
#pragma unroll
  for (int i = 0; i < kStages - 1; i++) issue(i);

  float tot[NT][4];
#pragma unroll
  for (int j = 0; j < NT; j++) tot[j][0] = tot[j][1] = tot[j][2] = tot[j][3] = 0.f;

  // x of rows j * 8 + g (past the last row that row again: its sums are not written): this lane's
  // 8 columns of a block
  constexpr int kSize = X8 ? 1 : 2;
  const uint8_t* xp[NT];
#pragma unroll
  for (int j = 0; j < NT; j++)
    xp[j] = (const uint8_t*)p.x + ((long long)min(j * 8 + g, p.rows - 1) * p.x_row + t * 8) * kSize;
  const auto raw_x = [&](int j, int k, uint32_t (&v)[2 * kSize]) {     // columns k + 8 t ..
    const bool ok = k < K;
    const uint8_t* x = xp[j] + k * kSize;
    if (ga.x_vec) {
      if (X8) {
        const uint2 u = ok ? *(const uint2*)x : make_uint2(0, 0);
        v[0] = u.x; v[1] = u.y;
      } else {
        const uint4 u = ok ? *(const uint4*)x : make_uint4(0, 0, 0, 0);
        v[0] = u.x; v[1] = u.y; v[2 * kSize - 2] = u.z; v[2 * kSize - 1] = u.w;
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < 2 * kSize; i++) {
        uint32_t u = 0;
        if (ok)
          u = X8 ? x[4 * i] | x[4 * i + 1] << 8 | x[4 * i + 2] << 16 | (uint32_t)x[4 * i + 3] << 24
                 : ((const uint16_t*)x)[2 * i] | (uint32_t)((const uint16_t*)x)[2 * i + 1] << 16;
#pragma unroll
        for (int e = 0; e < 2 * kSize; e++) v[e] = e == i ? u : v[e];
      }
    }
  };
  // as the B operand: pairs (0, 4), (1, 5), (2, 6), (3, 7)
  const auto pairs_x = [&](const uint32_t (&v)[2 * kSize], uint32_t (&o)[4]) {
    if (X8) {
      e4m3x4_to_half2x2(__byte_perm(v[0], v[1], 0x5140), o[0], o[1]);
      e4m3x4_to_half2x2(__byte_perm(v[0], v[1], 0x7362), o[2], o[3]);
    } else {
      o[0] = __byte_perm(v[0], v[2 * kSize - 2], 0x5410);
      o[1] = __byte_perm(v[0], v[2 * kSize - 2], 0x7632);
      o[2] = __byte_perm(v[1], v[2 * kSize - 1], 0x5410);
      o[3] = __byte_perm(v[1], v[2 * kSize - 1], 0x7632);
    }
  };
  const float* xs_row[NT][2];        // scales of the rows whose sums this lane holds
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int e = 0; e < 2; e++)
      xs_row[j][e] = X8 ? p.xscale + min(j * 8 + 2 * t + e, p.rows - 1) * p.xscale_row : nullptr;

  // scales and zero points of the next chunk's block t
  uint32_t s_next[2], z_next[2];
  const auto load_scales = [&](int i) {
    const int c = wk + i * WK;
    const bool ok = i < count && c * 128 + t * 32 < K;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s_next[h] = ok ? srow[h][c * kPer] : 0;
      z_next[h] = zero && ok ? zrow[h][c * kPer] : 8;
    }
  };
  load_scales(0);

  const uint8_t* src = ring_p + g * 16 + t * 4;      // this lane's word of output g
  constexpr int kAhead = NT <= 2 ? 4 : 1;     // blocks of x read before they are used
#pragma unroll 1
  for (int i = 0; i < count; i++) {
    const int c = wk + i * WK;
    uint32_t raw[kAhead][NT][2 * kSize];
    if (kAhead == 4) {
#pragma unroll
      for (int b = 0; b < kAhead; b++)
#pragma unroll
        for (int j = 0; j < NT; j++) raw_x(j, c * 128 + b * 32, raw[b][j]);
    }
    float xs[NT][2];
    const int xg = X8 && ga.xgroup ? x_group(c * 128) : 0;
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int e = 0; e < 2; e++) xs[j][e] = X8 && ga.xgroup ? xs_row[j][e][xg] : 1.f;
    float sw[2];                  // of block t
    uint32_t zw[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      sw[h] = XT == YK_BF16 || (X8 && ga.bf16) ? elem_to_float<true>(s_next[h]) : elem_to_float<false>(s_next[h]);
      zw[h] = z_next[h];
    }
    issue(i + kStages - 1);
    load_scales(i + 1);
    cp_async_wait<kStages - 1>();
    __syncwarp();                 // every lane's pieces of this stage are there
    float acc[NT][4];
    Zero zp[2];
#pragma unroll
    for (int b = 0; b < 4; b++) {
      uint32_t x[NT][4];
#pragma unroll
      for (int j = 0; j < NT; j++) {
        if (kAhead != 4) raw_x(j, c * 128 + b * 32, raw[0][j]);
        pairs_x(raw[kAhead == 4 ? b : 0][j], x[j]);
      }
      if (X8 && b && ga.x_inside && c * 128 + b * 32 < K) {
        const int xb = x_group(c * 128 + b * 32);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) xs[j][e] = xs_row[j][e][xb];
      }
      const uint8_t* at = src + b * S::kBlock;
      if (b % GB == 0) {
#pragma unroll
        for (int h = 0; h < 2; h++)
          zp[h] = zero_of<F16>(zero ? __shfl_sync(~0u, zw[h], (lane & ~3) + b) : 8);
      }
      uint32_t q[2][4];
#pragma unroll
      for (int h = 0; h < 2; h++) codes8<F16>(*(const uint32_t*)(at + 128 * h), zp[h], q[h]);
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const uint32_t a[4] = {q[0][2 * e], q[1][2 * e], q[0][2 * e + 1], q[1][2 * e + 1]};
#pragma unroll
        for (int j = 0; j < NT; j++) mma_gemv<F16>(acc[j], a, x[j][2 * e], x[j][2 * e + 1], b % GB == 0 && e == 0);
      }
      if (b % GB == GB - 1) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float f = GB == 4 ? sw[h] : __shfl_sync(~0u, sw[h], (lane & ~3) + b);
#pragma unroll
          for (int j = 0; j < NT; j++) {
            const float2 both = X8 ? ffma2(make_float2(f, f), make_float2(xs[j][0], xs[j][1]), make_float2(0.f, 0.f))
                                   : make_float2(f, f);
            const float2 v = ffma2(make_float2(acc[j][2 * h], acc[j][2 * h + 1]), both,
                                   make_float2(tot[j][2 * h], tot[j][2 * h + 1]));
            tot[j][2 * h] = v.x;
            tot[j][2 * h + 1] = v.y;
          }
        }
      }
    }
    __syncwarp();                 // every lane has read the stage
    src += kTile;
    if (src >= ring_p + kStages * kTile) src -= kStages * kTile;
  }
  cp_async_wait<0>();
  __syncthreads();
  // sums of the WK warps along the columns: [warp][row of x][output]
  float* meet = (float*)sm;
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int e = 0; e < 4; e++)
      meet[(warp * NT * 8 + j * 8 + 2 * t + (e & 1)) * 16 + g + (e >> 1) * 8] = tot[j][e];
  __syncthreads();
  constexpr int kOut = WN * 16;
  for (int i = tid; i < kOut * p.rows; i += 32 * kGemvWarps) {
    const int m = i / kOut, j = i % kOut, n = blockIdx.x * kOut + j;
    if (n >= p.n) continue;
    const int w = j / 16;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WK; k++) v += meet[((k * WN + w) * NT * 8 + m) * 16 + j % 16];
    if (X8 && !ga.xgroup) v *= p.xscale[m * p.xscale_row];
    if (p.bias) v += p.bias[n];
    ((uint16_t*)p.y)[m * p.y_row + n] = ga.bf16 ? float_to_elem<true>(v) : float_to_elem<false>(v);
  }
}

#include "gemv4_tc.cuh"

template <int XT, int GB, int NT, int WN>
static int launch_gemv4(const Gemv4Args& a, cudaStream_t st) {
  const auto kern = gemv4_kernel<XT, GB, NT, WN>;
  if (smem_attr(kern, Gemv<NT>::kSmem) != cudaSuccess) return check_launch("gemv4 attr");
  constexpr int outputs = WN * 16;
  launch_k(kern, (a.p.n + outputs - 1) / outputs, 32 * kGemvWarps, Gemv<NT>::kSmem, st, a);
  note_launch();
  return check_launch("gemv4");
}
template <int XT, int GB>
static int launch_gemv4(const Gemv4Args& a, cudaStream_t st) {
  const int m = a.p.rows, n = a.p.n;
  const bool many = n > kGemvRound * (m <= 16 ? 3 : m <= 32 ? 2 : 1);
  const bool dear = XT == YK_E4M3 && GB > 1 && m > 32 && a.p.k >= kGemvLong;
  if (m > 8 && (many || dear) && (!a.xgroup || !a.x_inside)) {
    if (m <= 16) return launch_gemv4_tc<XT, GB, 16>(a, st);
    if (m <= 32) return launch_gemv4_tc<XT, GB, 32>(a, st);
    return launch_gemv4_tc<XT, GB, 64>(a, st);
  }
  if (m <= 8) return launch_gemv4<XT, GB, 1, 1>(a, st);
  if (m <= 16) return launch_gemv4<XT, GB, 2, 1>(a, st);
  if (m <= 32) return launch_gemv4<XT, GB, 4, 2>(a, st);
  return launch_gemv4<XT, GB, 8, 2>(a, st);
}
template <int XT>
static int launch_gemv4(const Gemv4Args& a, cudaStream_t st) {
  switch (a.p.group) {
    case 32: return launch_gemv4<XT, 1>(a, st);
    case 64: return launch_gemv4<XT, 2>(a, st);
    default: return launch_gemv4<XT, 4>(a, st);
  }
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
  Gemv4Args a{*p};
  a.x_vec = at % (x8 ? 8 : 16) == 0;
  a.zero = p->wzero != nullptr;
  a.s_vec = aligned16(p->wscale) && p->group_row % 8 == 0 && p->k / p->group % 8 == 0 && (uintptr_t)p->wzero % 8 == 0;
  a.bf16 = p->dtype == YK_BF16;
  a.xgroup = x8 ? p->xgroup : 0;
  a.x_shift = a.xgroup && !(a.xgroup & (a.xgroup - 1)) ? __builtin_ctz(a.xgroup) : -1;
  a.x_inside = a.xgroup % 128 != 0;
  cudaStream_t s = (cudaStream_t)st;
  return x8 ? launch_gemv4<YK_E4M3>(a, s) : a.bf16 ? launch_gemv4<YK_BF16>(a, s) : launch_gemv4<YK_F16>(a, s);
}
