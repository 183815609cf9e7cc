// Products of 4-bit float matrices with group scales (yk_gemm_fp4).
#include "fp4.cuh"

namespace yk {

struct GemmFp4Args {
  YkGemmFp4 p;
  int blocks;              // scale blocks along a row
  int chunks;              // of 256 columns
  int tiles_m, tiles_n;    // of the tile kernel
  int y_vec;               // y allows 16-byte stores
  int y_pair;              // y allows 4-byte stores
};

constexpr int kFp4Cols = 256;              // columns of a stage: 128 bytes of codes a row, four MMAs
constexpr int kFp4Codes = 128 * 128;       // codes of 128 rows
constexpr int kFp4Threads = 192;           // loads, MMAs, four warps of sums
template <bool NV>
constexpr int kFp4Bpc = NV ? 4 : 2;        // scale blocks of 256 columns

// ---------------- many rows: 128 x 256 tiles ----------------
// y tiles of 128 rows x 256 outputs (gated: 128 of g and the 128 of the other factor), persistent CTAs, one an SM.
//  * warp 0: codes by tensor copies (128-byte swizzle, zeros past the edges), scales by plain bulk copies of
//    whole blocks, one ring of stages of 256 columns.
//  * warp 1: copies a stage's scales into TMEM, issues its four MMAs.  Scales have two places there, by
//    turns, so that a stage's copies do not wait for the last stage's MMAs.
//  * warps 2-5: sums out of TMEM, factor, bias or gate, rounding, through shared memory to rows of 64 bytes.
// TMEM: two accumulators of 256 columns and two scale places of 48 are 96 columns too many.  So the
// accumulators share 96 columns (0-255 and 160-415): a tile's shared ones are drained first, and the next tile
// may begin.
template <bool NV>
struct Fp4Tile {
  static constexpr int kStages = 4;
  static constexpr int kSa = kFp4Bpc<NV> * kFp4Block;
  static constexpr int kStage = 3 * kFp4Codes + 3 * 2048;
  static constexpr int kStaging = 4 * 32 * 64;
  static constexpr int kSmem = kStages * kStage + kStaging + 1024;
  static constexpr int kD1 = 160, kSf = 416, kSfSet = 48;
};

__device__ __forceinline__ void fp4_tile_at(const GemmFp4Args& a, int t, int& tm, int& tn) {
  // bands of 16 row tiles, so that a band's rows and the outputs in work stay in L2
  const int band = t / (16 * a.tiles_n), in = t - band * 16 * a.tiles_n, high = min(16, a.tiles_m - band * 16);
  tn = in / high;
  tm = band * 16 + in - tn * high;
}

template <bool NV, bool GATED, bool BF16>
__global__ void __launch_bounds__(kFp4Threads, 1)
gemm_fp4_tile_kernel(const __grid_constant__ GemmFp4Args a, const __grid_constant__ CUtensorMap tx,
                     const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tw2) {
  using S = Fp4Tile<NV>;
  extern __shared__ uint8_t fp4_raw[];
  __shared__ __align__(8) uint64_t bars[2 * S::kStages + 2];
  __shared__ uint32_t tslot;
  __shared__ volatile int abort_flag;
  const YkGemmFp4& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(fp4_raw) + 1023) & ~1023u;
  const uint32_t full = smem_u32(&bars[0]), empty = smem_u32(&bars[S::kStages]),
                 done = smem_u32(&bars[2 * S::kStages]), shared_free = done + 8;
  if (tid == 0) {
    for (int i = 0; i < S::kStages; i++) {
      mbar_init(full + i * 8, 1);
      mbar_init(empty + i * 8, 1);
    }
    mbar_init(done, 1);
    mbar_init(shared_free, 4);
    abort_flag = 0;
    mbar_fence_init();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 1) {
    tmem_alloc(smem_u32(&tslot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  const int tiles = a.tiles_m * a.tiles_n;
  constexpr int kBpc = kFp4Bpc<NV>, kOut = GATED ? 128 : 256;   // outputs of a tile

  if (warp == 0) {
    if (lane == 0) {
      uint32_t g = 0;
      for (int t = blockIdx.x; t < tiles && !abort_flag; t += gridDim.x) {
        int tm, tn;
        fp4_tile_at(a, t, tm, tn);
        const int m0 = tm * 128, n0 = tn * kOut;
        const bool second = GATED || n0 + 128 < p.n;
        const uint8_t* sx = (const uint8_t*)p.xscale + (long long)tm * a.blocks * kFp4Block;
        const uint8_t* sw = (const uint8_t*)p.wscale + (long long)(n0 / 128) * a.blocks * kFp4Block;
        const uint8_t* sw2 = GATED ? (const uint8_t*)p.w2scale + (long long)(n0 / 128) * a.blocks * kFp4Block
                                   : sw + (long long)a.blocks * kFp4Block;
        for (int c = 0; c < a.chunks; c++, g++) {
          const int s = g % S::kStages;
          if (g >= S::kStages && !mbar_wait(empty + s * 8, (g / S::kStages - 1) & 1, 0x611)) { abort_flag = 1; break; }
          const uint32_t at = base + s * S::kStage, sc = at + 3 * kFp4Codes, bar = full + s * 8;
          const uint32_t bytes = min(kBpc, a.blocks - c * kBpc) * kFp4Block;
          mbar_expect_tx(bar, 2 * (kFp4Codes + bytes) + (second ? kFp4Codes + bytes : 0));
          tma_load_2d(at, &tx, bar, c * 128, m0);
          tma_load_2d(at + kFp4Codes, &tw, bar, c * 128, n0);
          bulk_load(sc, sx + c * (kBpc * kFp4Block), bytes, bar);
          bulk_load(sc + 2048, sw + c * (kBpc * kFp4Block), bytes, bar);
          if (second) {
            tma_load_2d(at + 2 * kFp4Codes, GATED ? &tw2 : &tw, bar, c * 128, GATED ? n0 : n0 + 128);
            bulk_load(sc + 4096, sw2 + c * (kBpc * kFp4Block), bytes, bar);
          }
        }
      }
      if (abort_flag)                // copies in flight land before the CTA ends
        for (uint32_t i = g > S::kStages ? g - S::kStages : 0; i < g; i++) mbar_wait(full + i % S::kStages * 8, (i / S::kStages) & 1, 0x612);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t g = 0, li = 0;
      const uint64_t x_desc = sw128_desc(base), w_desc = sw128_desc(base + kFp4Codes), s_desc = scales_desc(base + 3 * kFp4Codes);
      for (int t = blockIdx.x; t < tiles && !abort_flag; t += gridDim.x, li++) {
        if (li && !mbar_wait(shared_free, (li - 1) & 1, 0x613)) { abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t d = tmem + (li & 1) * S::kD1;
        for (int c = 0; c < a.chunks; c++, g++) {
          const int s = g % S::kStages;
          if (!mbar_wait(full + s * 8, (g / S::kStages) & 1, 0x614)) { abort_flag = 1; break; }
          // the MMAs that read this place of the scales are those of two stages ago
          if (g >= 2 && !mbar_wait(empty + (g - 2) % S::kStages * 8, ((g - 2) / S::kStages) & 1, 0x615)) { abort_flag = 1; break; }
          tc_fence_after();
          const uint32_t sf = tmem + S::kSf + (g & 1) * S::kSfSet;
          const uint64_t step = (uint64_t)(s * S::kStage) >> 4;
          const int blocks = min(kBpc, a.blocks - c * kBpc);
#pragma unroll
          for (int b = 0; b < kBpc; b++) {
            if (b >= blocks) break;
            tmem_cp_scales(sf + b * 4, s_desc + step + b * (kFp4Block >> 4));
            tmem_cp_scales(sf + 16 + b * 8, s_desc + step + ((2048 + b * kFp4Block) >> 4));
            tmem_cp_scales(sf + 20 + b * 8, s_desc + step + ((4096 + b * kFp4Block) >> 4));
          }
          const int steps = min(4, (p.k - c * kFp4Cols + 63) / 64);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            if (k >= steps) break;
            const int b = NV ? k : k >> 1;
            tc_mma_fp4<NV>(d, x_desc + step + k * 2, w_desc + step + k * 2, idesc_fp4_m128<NV>(256, NV ? 0 : k & 1),
                           sf + b * 4, sf + 16 + b * 8, (c | k) != 0);
          }
          tc_commit(empty + s * 8);
        }
        if (!abort_flag) tc_commit(done);
      }
    }
  } else {
    const int sub = warp & 3;
    const uint32_t lanes = (uint32_t)(sub * 32) << 16;
    const uint32_t stage = base + S::kStages * S::kStage + sub * 2048;
    const uint8_t* stage_p = fp4_raw + (stage - smem_u32(fp4_raw));
    const float alpha = p.alpha, alpha2 = p.alpha2;
    uint32_t li = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, li++) {
      if (!mbar_wait(done, li & 1, 0x616)) { abort_flag = 1; break; }
      tc_fence_after();
      int tm, tn;
      fp4_tile_at(a, t, tm, tn);
      const int m0 = tm * 128 + sub * 32, n0 = tn * kOut;
      const uint32_t d = tmem + (li & 1) * S::kD1 + lanes;
      constexpr int kUnits = kOut / 32, kFirst = 3;   // units that hold the shared columns
#pragma unroll 1
      for (int i = 0; i < kUnits; i++) {
        const int u = (li & 1) ? i : (i + kUnits - kFirst) % kUnits;
        uint32_t r[32], o[16];
        tmem_ld16p(d + u * 32, r);
        tmem_ld16p(d + u * 32 + 16, r + 16);
        if (GATED) {
          uint32_t r2[32];
          tmem_ld16p(d + 128 + u * 32, r2);
          tmem_ld16p(d + 128 + u * 32 + 16, r2 + 16);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e++) {
            const float v = __uint_as_float(r[e]) * alpha;
            r[e] = __float_as_uint(v / (1.f + __expf(-v)) * (__uint_as_float(r2[e]) * alpha2));
          }
        } else {
          tmem_ld_wait();
        }
        if (i == kFirst - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(shared_free);
        }
        const int c0 = n0 + u * 32;
        if (c0 >= p.n) continue;
        if (!GATED) {
          const float bias = p.bias && c0 + lane < p.n ? p.bias[c0 + lane] : 0.f;
#pragma unroll
          for (int e = 0; e < 32; e++)
            r[e] = __float_as_uint(fmaf(__uint_as_float(r[e]), alpha, p.bias ? __shfl_sync(~0u, bias, e) : 0.f));
        }
#pragma unroll
        for (int e = 0; e < 16; e++) o[e] = float2_to_pair<BF16>(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 4; h++)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((h ^ ((lane >> 1) & 3)) << 4)),
                       "r"(o[4 * h]), "r"(o[4 * h + 1]), "r"(o[4 * h + 2]), "r"(o[4 * h + 3]) : "memory");
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int row = j * 8 + (lane >> 2), h = lane & 3, c = c0 + h * 8;
          if (m0 + row >= p.rows || c >= p.n) continue;
          const uint4 v = *(const uint4*)(stage_p + row * 64 + ((h ^ ((row >> 1) & 3)) << 4));
          uint16_t* y = (uint16_t*)p.y + (long long)(m0 + row) * p.y_row + c;
          if (a.y_vec && c + 8 <= p.n) {
            *(uint4*)y = v;
          } else {
            const uint32_t* w = (const uint32_t*)&v;
#pragma unroll
            for (int e = 0; e < 8; e++)
              if (c + e < p.n) y[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------- few rows or few tiles: columns split over a cluster ----------------
// The weights are the left-hand operand (128 outputs a tile), NT rows of x the right-hand one, and a
// cluster's CTAs take a share of the columns each: a stream of weights over all SMs.  Their sums meet in
// distributed shared memory, in the order of the CTAs, so that a result does not depend on timing.
template <bool NV, bool GATED, int NT>
struct Fp4Split {
  static constexpr int kA = GATED ? 2 : 1;                       // weight matrices
  static constexpr int kX = NT * 128;
  static constexpr int kStage = kA * kFp4Codes + kX + (kA + 1) * 2048;
  static constexpr int kCtas = GATED ? 1 : 2;                    // an SM
  static constexpr int kStages = GATED ? (NT == 32 ? 5 : 4) : (NT == 32 ? 4 : 3);
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr int kSf = kA * NT, kSfSet = 16 * (kA + 1);    // TMEM: sums, then two places of scales
  static constexpr int kNeed = kSf + 2 * kSfSet;
  static constexpr int kTmem = kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
  static_assert(kA * NT * 512 <= kStages * kStage, "sums fit the ring");
  static_assert(kCtas * kTmem <= 512 && kCtas * (kSmem + 1024) <= 228 * 1024, "CTAs of an SM");
};

template <bool NV, bool GATED, int NT>
__global__ void __launch_bounds__(kFp4Threads)
gemm_fp4_split_kernel(const __grid_constant__ GemmFp4Args a, const __grid_constant__ CUtensorMap tx,
                      const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tw2, int split) {
  using S = Fp4Split<NV, GATED, NT>;
  extern __shared__ uint8_t fp4_raw[];
  __shared__ __align__(8) uint64_t bars[2 * S::kStages + 1];
  __shared__ uint32_t tslot;
  __shared__ volatile int abort_flag;
  const YkGemmFp4& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(fp4_raw) + 1023) & ~1023u;
  const uint32_t full = smem_u32(&bars[0]), empty = smem_u32(&bars[S::kStages]), done = smem_u32(&bars[2 * S::kStages]);
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int n0 = blockIdx.x / split * 128, m0 = blockIdx.y * NT;
  const int c_first = (int)((long long)a.chunks * rank / split), c_end = (int)((long long)a.chunks * (rank + 1) / split);
  if (tid == 0) {
    for (int i = 0; i < S::kStages; i++) {
      mbar_init(full + i * 8, 1);
      mbar_init(empty + i * 8, 1);
    }
    mbar_init(done, 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 1) {
    tmem_alloc(smem_u32(&tslot), S::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  constexpr int kBpc = kFp4Bpc<NV>;
  constexpr int kScales = S::kA * kFp4Codes + S::kX;            // of a stage: weights', second weights', x's

  if (warp == 0) {
    if (lane == 0) {
      uint32_t g = 0;
      const long long wb = (long long)(n0 / 128) * a.blocks * kFp4Block, xb = (long long)(m0 / 128) * a.blocks * kFp4Block;
      for (int c = c_first; c < c_end; c++, g++) {
        const int s = g % S::kStages;
        if (g >= S::kStages && !mbar_wait(empty + s * 8, (g / S::kStages - 1) & 1, 0x621)) { abort_flag = 1; break; }
        const uint32_t at = base + s * S::kStage, sc = at + kScales, bar = full + s * 8;
        const uint32_t bytes = min(kBpc, a.blocks - c * kBpc) * kFp4Block;
        const long long off = (long long)c * (kBpc * kFp4Block);
        mbar_expect_tx(bar, S::kA * (kFp4Codes + bytes) + S::kX + bytes);
        tma_load_2d(at, &tw, bar, c * 128, n0);
        if (GATED) tma_load_2d(at + kFp4Codes, &tw2, bar, c * 128, n0);
        tma_load_2d(at + S::kA * kFp4Codes, &tx, bar, c * 128, m0);
        bulk_load(sc, (const uint8_t*)p.wscale + wb + off, bytes, bar);
        if (GATED) bulk_load(sc + 2048, (const uint8_t*)p.w2scale + wb + off, bytes, bar);
        bulk_load(sc + S::kA * 2048, (const uint8_t*)p.xscale + xb + off, bytes, bar);
      }
      if (abort_flag)
        for (uint32_t i = g > S::kStages ? g - S::kStages : 0; i < g; i++) mbar_wait(full + i % S::kStages * 8, (i / S::kStages) & 1, 0x622);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint64_t w_desc = sw128_desc(base), x_desc = sw128_desc(base + S::kA * kFp4Codes), s_desc = scales_desc(base + kScales);
      uint32_t g = 0;
      for (int c = c_first; c < c_end; c++, g++) {
        const int s = g % S::kStages;
        if (!mbar_wait(full + s * 8, (g / S::kStages) & 1, 0x623)) { abort_flag = 1; break; }
        if (g >= 2 && !mbar_wait(empty + (g - 2) % S::kStages * 8, ((g - 2) / S::kStages) & 1, 0x624)) { abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t sf = tmem + S::kSf + (g & 1) * S::kSfSet;
        const uint64_t step = (uint64_t)(s * S::kStage) >> 4;
        const int blocks = min(kBpc, a.blocks - c * kBpc);
#pragma unroll
        for (int b = 0; b < kBpc; b++) {
          if (b >= blocks) break;
#pragma unroll
          for (int x = 0; x <= S::kA; x++) tmem_cp_scales(sf + x * 16 + b * 4, s_desc + step + ((x * 2048 + b * kFp4Block) >> 4));
        }
        const int steps = min(4, (p.k - c * kFp4Cols + 63) / 64);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if (k >= steps) break;
          const int b = NV ? k : k >> 1;
#pragma unroll
          for (int x = 0; x < S::kA; x++)
            tc_mma_fp4<NV>(tmem + x * NT, w_desc + step + x * (kFp4Codes >> 4) + k * 2, x_desc + step + k * 2,
                           idesc_fp4_m128<NV>(NT, NV ? 0 : k & 1), sf + x * 16 + b * 4, sf + S::kA * 16 + b * 4, (c - c_first) | k);
        }
        tc_commit(empty + s * 8);
      }
      if (!abort_flag) tc_commit(done);
    }
  }
  const int rows = min(NT, p.rows - m0);
  float* const part = (float*)(fp4_raw + (base - smem_u32(fp4_raw)));     // [matrix][row][128 outputs], in the ring
  if (warp >= 2) {
    const int sub = warp & 3;
    if (mbar_wait(done, 0, 0x625)) {
      tc_fence_after();
#pragma unroll 1
      for (int x = 0; x < S::kA; x++) {
#pragma unroll 1
        for (int m = 0; m < rows; m += 16) {
          uint32_t r[16];
          tmem_ld16p(tmem + ((uint32_t)(sub * 32) << 16) + x * NT + m, r);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; e++) part[(x * NT + m + e) * 128 + sub * 32 + lane] = __uint_as_float(r[e]);
        }
      }
    } else {
      abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncwarp();
  if (split > 1) cluster_barrier();
  else __syncthreads();
  const uint32_t part_sm = smem_u32(part);
  // two outputs a thread and turn; rows rank, rank + split, ..
  for (int i = tid; i < ((rows - rank + split - 1) / split) * 64; i += kFp4Threads) {
    const int m = rank + i / 64 * split, j = i % 64 * 2;
    if (n0 + j >= p.n) continue;
    float v[S::kA][2];
#pragma unroll
    for (int x = 0; x < S::kA; x++) {
      v[x][0] = v[x][1] = 0.f;
      const uint32_t at = part_sm + ((x * NT + m) * 128 + j) * 4;
      for (int q = 0; q < split; q++) {
        float b0, b1;
        if (split > 1)
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(b0), "=f"(b1) : "r"(cluster_map(at, q)) : "memory");
        else
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(b0), "=f"(b1) : "r"(at) : "memory");
        v[x][0] += b0;
        v[x][1] += b1;
      }
    }
    float o[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      o[e] = v[0][e] * p.alpha;
      if (GATED) o[e] = o[e] / (1.f + __expf(-o[e])) * (v[S::kA - 1][e] * p.alpha2);
      else if (p.bias && n0 + j + e < p.n) o[e] = fmaf(v[0][e], p.alpha, p.bias[n0 + j + e]);
    }
    uint16_t* y = (uint16_t*)p.y + (long long)(m0 + m) * p.y_row + n0 + j;
    const uint32_t w = p.dtype == YK_BF16 ? float2_to_pair<true>(o[0], o[1]) : float2_to_pair<false>(o[0], o[1]);
    if (a.y_pair && n0 + j + 1 < p.n) {
      *(uint32_t*)y = w;
    } else {
      y[0] = (uint16_t)w;
      if (n0 + j + 1 < p.n) y[1] = (uint16_t)(w >> 16);
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
  if (split > 1) {
    __syncwarp();
    cluster_barrier();       // no CTA leaves while others read its sums
  }
}

static PFN_cuTensorMapEncodeTiled tensor_map_encode() {
  static const PFN_cuTensorMapEncodeTiled encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
           q == cudaDriverEntryPointSuccess ? (PFN_cuTensorMapEncodeTiled)fn : nullptr;
  }();
  return encode;
}

// Codes as bytes: columns past the row's end read as zero.
static bool encode_fp4(CUtensorMap* m, const void* base, int rows, int k, long long row_bytes, int box_rows) {
  const PFN_cuTensorMapEncodeTiled encode = tensor_map_encode();
  if (!encode) return false;
  const cuuint64_t dims[2] = {((cuuint64_t)k + 1) / 2, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)row_bytes};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int fp4_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
}

template <bool NV, bool GATED, bool BF16>
static int launch_fp4_tile(const GemmFp4Args& a, cudaStream_t st) {
  using S = Fp4Tile<NV>;
  const auto kern = gemm_fp4_tile_kernel<NV, GATED, BF16>;
  const YkGemmFp4& p = a.p;
  CUtensorMap tx, tw, tw2;
  if (!encode_fp4(&tx, p.x, p.rows, p.k, p.x_row, 128) || !encode_fp4(&tw, p.w, p.n, p.k, p.w_row, 128) ||
      !encode_fp4(&tw2, GATED ? p.w2 : p.w, p.n, p.k, p.w_row, 128))
    return refuse(YK_EUNSUP, "gemm_fp4: no tensor map for these sizes");
  if (smem_attr(kern, S::kSmem) != cudaSuccess) return check_launch("gemm_fp4 attr");
  const int tiles = a.tiles_m * a.tiles_n, sms = fp4_sms();
  launch_k(kern, tiles < sms ? tiles : sms, kFp4Threads, S::kSmem, st, a, tx, tw, tw2);
  note_launch();
  return check_launch("gemm_fp4");
}

template <bool NV, bool GATED, int NT>
static int launch_fp4_split(const GemmFp4Args& a, int split, cudaStream_t st) {
  using S = Fp4Split<NV, GATED, NT>;
  const auto kern = gemm_fp4_split_kernel<NV, GATED, NT>;
  const YkGemmFp4& p = a.p;
  CUtensorMap tx, tw, tw2;
  if (!encode_fp4(&tx, p.x, p.rows, p.k, p.x_row, NT) || !encode_fp4(&tw, p.w, p.n, p.k, p.w_row, 128) ||
      !encode_fp4(&tw2, GATED ? p.w2 : p.w, p.n, p.k, p.w_row, 128))
    return refuse(YK_EUNSUP, "gemm_fp4: no tensor map for these sizes");
  if (smem_attr(kern, S::kSmem) != cudaSuccess) return check_launch("gemm_fp4 attr");
  launch_kc(kern, dim3((unsigned)((p.n + 127) / 128 * split), (unsigned)((p.rows + NT - 1) / NT)), kFp4Threads, S::kSmem, split, st,
            a, tx, tw, tw2, split);
  note_launch();
  return check_launch("gemm_fp4");
}

static int g_fp4_kernel = 0, g_fp4_split = 0;

template <bool NV, bool GATED>
static int launch_fp4(GemmFp4Args& a, cudaStream_t st) {
  const YkGemmFp4& p = a.p;
  const int sms = fp4_sms();
  a.tiles_m = (p.rows + 127) / 128;
  a.tiles_n = (p.n + (GATED ? 127 : 255)) / (GATED ? 128 : 256);
  const long long tiles = (long long)a.tiles_m * a.tiles_n;
  if (tiles > 0x7fffffffll) return refuse(YK_EUNSUP, "gemm_fp4: rows * n too large");
  const int nt = p.rows <= 32 ? 32 : 128;
  const long long small = (long long)((p.n + 127) / 128) * ((p.rows + nt - 1) / nt);
  int split = 1;
  while (split < 8 && small * split * 2 <= sms * (GATED ? 1 : 2) && a.chunks >= 2 * split) split *= 2;
  if (g_fp4_split && g_fp4_split <= a.chunks) split = g_fp4_split;
  if (g_fp4_kernel ? g_fp4_kernel == 1 : p.rows > 128 && tiles * 2 >= sms)
    return p.dtype == YK_BF16 ? launch_fp4_tile<NV, GATED, true>(a, st) : launch_fp4_tile<NV, GATED, false>(a, st);
  if ((p.rows + nt - 1) / nt > 65535 || small * split > 0x7fffffffll) return refuse(YK_EUNSUP, "gemm_fp4: rows * n too large");
  return nt == 32 ? launch_fp4_split<NV, GATED, 32>(a, split, st) : launch_fp4_split<NV, GATED, 128>(a, split, st);
}

}  // namespace yk

using namespace yk;

extern "C" int yk_gemm_fp4(const YkGemmFp4* p, yk_stream_t st) {
  if (!p || !p->x || !p->xscale || !p->w || !p->wscale || !p->y) return refuse(YK_EINVAL, "gemm_fp4: null pointer");
  if (!p->w2 != !p->w2scale) return refuse(YK_EINVAL, "gemm_fp4: w2 and w2scale go together");
  if (p->w2 && p->bias) return refuse(YK_EINVAL, "gemm_fp4: no bias with w2");
  if (!fp4_format(p->format)) return refuse(YK_EUNSUP, "gemm_fp4: format must be YK_NVFP4 or YK_MXFP4");
  if (p->dtype != YK_F16 && p->dtype != YK_BF16) return refuse(YK_EUNSUP, "gemm_fp4: dtype must be fp16 or bf16");
  if (p->rows < 0 || p->n < 1 || p->k < 1) return refuse(YK_EINVAL, "gemm_fp4: n and k must be positive, rows not negative");
  if (p->k > 1 << 30 || p->rows > 1 << 30 || p->n > 1 << 30) return refuse(YK_EUNSUP, "gemm_fp4: rows, n and k up to 2^30");
  const long long bytes = (p->k + 1ll) / 2;
  if (p->x_row % 16 || p->w_row % 16 || p->x_row < bytes || p->w_row < bytes || p->y_row < p->n ||
      p->x_row >= 1ll << 40 || p->w_row >= 1ll << 40)
    return refuse(YK_EINVAL, "gemm_fp4: x_row and w_row are multiples of 16 that hold a row, y_row at least n");
  if (!aligned16(p->x) || !aligned16(p->w) || !aligned16(p->w2) || !aligned16(p->xscale) || !aligned16(p->wscale) || !aligned16(p->w2scale))
    return refuse(YK_EINVAL, "gemm_fp4: codes and scales need 16-byte alignment");
  if ((uintptr_t)p->y & 1 || (uintptr_t)p->bias & 3) return refuse(YK_EINVAL, "gemm_fp4: y and bias need the alignment of their type");
  if (p->alpha != p->alpha || p->alpha2 != p->alpha2) return refuse(YK_EINVAL, "gemm_fp4: alpha is not a number");
  if (p->rows == 0) return YK_OK;
  GemmFp4Args a{*p};
  if (a.p.alpha == 0.f) a.p.alpha = 1.f;
  if (a.p.alpha2 == 0.f) a.p.alpha2 = 1.f;
  a.blocks = fp4_blocks(p->k, p->format);
  a.chunks = (p->k + kFp4Cols - 1) / kFp4Cols;
  a.y_vec = aligned16(p->y) && p->y_row % 8 == 0;
  a.y_pair = (uintptr_t)p->y % 4 == 0 && p->y_row % 2 == 0;
  cudaStream_t s = (cudaStream_t)st;
  if (p->format == YK_NVFP4) return p->w2 ? launch_fp4<true, true>(a, s) : launch_fp4<true, false>(a, s);
  return p->w2 ? launch_fp4<false, true>(a, s) : launch_fp4<false, false>(a, s);
}

extern "C" int yk_test_gemm_fp4(int kernel, int split) {
  if (kernel < 0 || kernel > 2 || split < 0 || split > 8 || (split & (split - 1))) return YK_EINVAL;
  g_fp4_kernel = kernel;
  g_fp4_split = split;
  return YK_OK;
}
