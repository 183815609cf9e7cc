// Products of 4-bit float matrices with group scales (yk_gemm_fp4).
#include "fp4.cuh"

namespace yk {

struct GemmFp4Args {
  YkGemmFp4 p;
  int blocks;              // scale blocks along a row
  int chunks;              // of 256 columns
  int tiles_m, tiles_n;    // of the pair kernel
  int y_vec;               // y allows 16-byte stores
  int y_pair;              // y allows 4-byte stores
};

constexpr int kFp4Cols = 256;              // columns of a stage: 128 bytes of codes a row, four MMAs
constexpr int kFp4Codes = 128 * 128;       // codes of 128 rows
constexpr int kFp4Threads = 256;           // of a split product: loads, MMAs, four warps for scales and sums, two that join them
template <bool NV>
constexpr int kFp4Bpc = NV ? 4 : 2;        // scale blocks of 256 columns

// v / (1 + exp(-v)), within 2^-20 + |v| 2^-23 of itself
__device__ __forceinline__ float fp4_silu(float v) { return __fdividef(v, 1.f + __expf(-v)); }

// Scales go from shared memory to TMEM through registers: row r's four scales of a 512-byte block belong in lane r % 32,
// column r / 32, so a lane's 16 bytes of the block are four columns.  All four warps of a group do the same for their
// lanes, as the MMA wants them.  Copies by the tensor pipe itself (tcgen05.cp) take 45 of its cycles each, beside 128 for an MMA.
__device__ __forceinline__ void fp4_get_scales(uint32_t* v, uint32_t sm, int lane) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(sm + lane * 16) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  tmem_ld16p(taddr, r);
  tmem_ld16p(taddr + 16, r + 16);
}
template <int N>
__device__ __forceinline__ void fp4_put_scales(uint32_t taddr, const uint32_t* v) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr + i), "r"(v[i]), "r"(v[i + 1]),
                 "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7]) : "memory");
}

// ---------------- many rows: 256 x 256 tiles of CTA pairs ----------------
// One MMA of 256 rows x 256 outputs (gated: 128 of g and the 128 of the other factor) over the shared memory of two SMs: each
// CTA holds 128 rows of x and 128 of w, so that it takes in 64 bytes a cycle at the full rate, where an SM by itself would
// need 96.  An MMA of 64 columns takes 128 cycles whatever its outputs, so only full tiles reach the rate.
//  * warp 0: codes by tensor copies (128-byte swizzle, zeros past the edges) onto the leader's barrier, scales by plain
//    bulk copies of whole blocks onto the CTA's own; one ring of stages of 256 columns.
//  * warps 2-5 and 6-9: scales from shared memory to TMEM (x's of the CTA's own rows, w's of all) for every other stage,
//    each four warps with a place of their own there.
//  * warp 1 of the leader: the MMAs.
//  * warps 10-17: sums out of TMEM, factor, bias or gate, rounding, through shared memory to rows of 64 bytes; of the two
//    warps that can read a lane each takes every other unit.
// TMEM: two accumulators of 256 columns and two places of 48 for scales are 96 columns too many.  So the
// accumulators share 96 columns (0-255 and 160-415): a tile's shared ones are drained first, and the next tile
// may begin.
// 2048 x 8192 x 8192: 55 us in a burst (5.0 PFLOP/s; 66 us back to back for long, at the power limit's clocks).  The MMAs
// take 550 of at least 512 cycles a stage; 256 tiles on 74 pairs are 3.5 rounds, of which the last half runs on half the
// SMs, and one epilogue stands alone.  Gated 1024 x 9472 x 4096: 31 us (5.1 PFLOP/s); 777 x 11000 x 4000: 45 us, as rows of
// 2000 bytes put each 128-byte piece of a row into two L2 lines (37 us for 4096 columns) and 9 rows take a quarter of the tiles.
constexpr int kFp4PairThreads = 576;
template <bool NV>
struct Fp4Pair {
  static constexpr int kStages = 5;
  static constexpr int kStage = 2 * kFp4Codes + 3 * 2048;
  static constexpr int kStaging = 8 * 32 * 64;
  static constexpr int kSmem = kStages * kStage + kStaging + 1024;
  static constexpr int kD1 = 160, kSf = 416, kSfSet = 48;
};

__device__ __forceinline__ void fp4_tile_at(const GemmFp4Args& a, int t, int& tm, int& tn) {
  // bands of 8 row tiles, so that a band's rows and the outputs in work stay in L2
  const int band = t / (8 * a.tiles_n), in = t - band * 8 * a.tiles_n, high = min(8, a.tiles_m - band * 8);
  tn = in / high;
  tm = band * 8 + in - tn * high;
}

template <bool NV, bool GATED, bool BF16>
__global__ void __launch_bounds__(kFp4PairThreads, 1)
gemm_fp4_pair_kernel(const __grid_constant__ GemmFp4Args a, const __grid_constant__ CUtensorMap tx,
                     const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tw2) {
  using S = Fp4Pair<NV>;
  extern __shared__ uint8_t fp4_raw[];
  __shared__ __align__(8) uint64_t bars[3 * S::kStages + 4];
  __shared__ uint32_t tslot;
  const YkGemmFp4& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0);
  const uint32_t base = (smem_u32(fp4_raw) + 1023) & ~1023u;
  // codes of both CTAs (leader's), the CTA's scales; a stage is free; scales in TMEM of both CTAs (leader's); a tile's
  // sums are complete; the shared columns are drained in both CTAs (leader's)
  const uint32_t full = smem_u32(&bars[0]), sfull = full + 8 * S::kStages, empty = sfull + 8 * S::kStages,
                 sready = empty + 8 * S::kStages, done = sready + 16, shared_free = done + 8;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (tid == 0) {
    for (int i = 0; i < S::kStages; i++) {
      mbar_init(full + i * 8, 1);
      mbar_init(sfull + i * 8, 1);
      mbar_init(empty + i * 8, 1);
    }
    mbar_init(sready, 8);
    mbar_init(sready + 8, 8);
    mbar_init(done, 1);
    mbar_init(shared_free, 16);
    mbar_fence_init();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tslot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncwarp();
  cluster_barrier();                 // barriers and TMEM of both CTAs
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, tslot, 0);
  const int tiles = a.tiles_m * a.tiles_n;
  constexpr int kBpc = kFp4Bpc<NV>, kOut = GATED ? 128 : 256;   // outputs of a tile
  bool ok = true;                    // a wait that ran out ends the warp's part (the others' waits run out then too)

  if (warp == 0) {
    // (the whole warp takes part and one lane issues, here and below: operands then stay in uniform registers)
    const bool issuer = elect_one();
    const uint32_t lead_full = cluster_map(full, 0);
    uint32_t g = 0, s = 0, phase = 1;                // of the stage's last use
    for (int t = pair; t < tiles && ok; t += pairs) {
      int tm, tn;
      fp4_tile_at(a, t, tm, tn);
      const int m0 = tm * 256 + (int)rank * 128, n0 = tn * kOut, w0 = n0 + (int)rank * (GATED ? 64 : 128);
      const bool rows_there = m0 < p.rows, second = GATED || n0 + 128 < p.n;
      const uint8_t* sx = (const uint8_t*)p.xscale + (long long)(m0 / 128) * a.blocks * kFp4Block;
      const uint8_t* sw = (const uint8_t*)p.wscale + (long long)(n0 / 128) * a.blocks * kFp4Block;
      const uint8_t* sw2 = GATED ? (const uint8_t*)p.w2scale + (long long)(n0 / 128) * a.blocks * kFp4Block
                                 : sw + (long long)a.blocks * kFp4Block;
      for (int c = 0; c < a.chunks; c++) {
        if (g >= S::kStages && !__all_sync(~0u, mbar_wait_due(empty + s * 8, phase, 0x611))) { ok = false; break; }
        if (issuer) {
          const uint32_t at = base + s * S::kStage, sc = at + 2 * kFp4Codes, bar = sfull + s * 8, lead_bar = lead_full + s * 8;
          const uint32_t bytes = min(kBpc, a.blocks - c * kBpc) * kFp4Block;
          const long long off = (long long)c * (kBpc * kFp4Block);
          if (rank == 0) mbar_expect_tx(full + s * 8, 4 * kFp4Codes);
          tma_pair_2d(at, &tx, lead_bar, c * 128, m0);
          tma_pair_2d(at + kFp4Codes, &tw, lead_bar, c * 128, w0);
          if (GATED) tma_pair_2d(at + kFp4Codes + kFp4Codes / 2, &tw2, lead_bar, c * 128, w0);   // (64 rows of each)
          mbar_expect_tx(bar, bytes * (1 + rows_there + second));
          if (rows_there) bulk_load(sc, sx + off, bytes, bar);
          bulk_load(sc + 2048, sw + off, bytes, bar);
          if (second) bulk_load(sc + 4096, sw2 + off, bytes, bar);
        }
        __syncwarp();
        g++;
        if (++s == S::kStages) { s = 0; phase ^= 1; }
      }
    }
    if (!ok)                  // copies in flight land before the CTA ends
      for (uint32_t i = g > S::kStages ? g - S::kStages : 0; i < g; i++) {
        mbar_wait(sfull + i % S::kStages * 8, (i / S::kStages) & 1, 0x612);
        if (rank == 0) mbar_wait(full + i % S::kStages * 8, (i / S::kStages) & 1, 0x612);
      }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool issuer = elect_one();
      const uint32_t peer_empty = cluster_map(empty, 1), peer_done = cluster_map(done, 1);
      uint32_t s = 0, phase = 0, set = 0, set_phase = 0, li = 0;
      for (int t = pair; t < tiles && ok; t += pairs, li++) {
        if (li && !__all_sync(~0u, mbar_wait_due(shared_free, (li - 1) & 1, 0x613))) { ok = false; break; }
        const uint32_t d = tmem + (li & 1) * S::kD1;
        int c = 0;
        for (; c < a.chunks; c++) {
          if (!__all_sync(~0u, mbar_wait_due(full + s * 8, phase, 0x614) && mbar_wait_due(sready + set * 8, set_phase, 0x615))) { ok = false; break; }
          tc_fence_after();
          if (issuer) {
            const uint32_t sf = tmem + S::kSf + set * S::kSfSet, at = base + s * S::kStage;
            const uint64_t x_desc = sw128_desc(at), w_desc = sw128_desc(at + kFp4Codes);
            const int steps = (p.k - c * kFp4Cols + 63) / 64;
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const int b = NV ? k : k >> 1;
              if (k == 0 || k < steps)
                tc_mma_fp4_pair<NV>(d, x_desc + k * 2, w_desc + k * 2, idesc_fp4<NV>(256, 256, NV ? 0 : k & 1),
                                    sf + b * 4, sf + 4 * kBpc + b * 8, (c | k) != 0);
            }
            tc_commit_pair(empty + s * 8);
            tc_commit_pair(peer_empty + s * 8);
          }
          __syncwarp();
          if (++s == S::kStages) { s = 0; phase ^= 1; }
          set ^= 1;
          set_phase ^= set == 0;
        }
        if (issuer && c == a.chunks) {
          tc_commit_pair(done);
          tc_commit_pair(peer_done);
        }
        __syncwarp();
      }
    }
  } else if (warp < 10) {
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, lead_ready = cluster_map(sready, 0);
    const uint32_t sc0 = base + 2 * kFp4Codes;
    constexpr int kWords = 12 * kBpc;                // x's 4 a block, then w's 8 a block
    const uint32_t total = (uint32_t)((tiles - pair + pairs - 1) / pairs) * a.chunks;   // (the launch has no pair without a tile)
    const uint32_t set = warp >= 6, place = tmem + lanes + S::kSf + set * S::kSfSet;
    for (uint32_t g = set; g < total; g += 2) {
      const uint32_t s = g % S::kStages;
      uint32_t v[kWords];
      if (!__all_sync(~0u, mbar_wait_due(sfull + s * 8, (g / S::kStages) & 1, 0x616))) { ok = false; break; }
#pragma unroll
      for (int b = 0; b < kBpc; b++) {
        const uint32_t sc = sc0 + s * S::kStage + b * kFp4Block;
        fp4_get_scales(v + 4 * b, sc, lane);
        uint32_t w[8];
        fp4_get_scales(w, sc + 2048, lane);
        fp4_get_scales(w + 4, sc + 4096, lane);
#pragma unroll
        for (int i = 0; i < 8; i++) v[4 * kBpc + 8 * b + i] = GATED ? w[(i & 2) * 2 + (i >> 2) * 2 + (i & 1)] : w[i];
      }
      // the MMAs that read this place are those of two stages ago
      if (g >= 2 && !__all_sync(~0u, mbar_wait_due(empty + (g - 2) % S::kStages * 8, ((g - 2) / S::kStages) & 1, 0x617))) { ok = false; break; }
      tc_fence_after();
      fp4_put_scales<kWords>(place, v);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(lead_ready + set * 8);
    }
  } else {
    const int sub = warp & 3;
    const uint32_t lanes = (uint32_t)(sub * 32) << 16, lead_free = cluster_map(shared_free, 0);
    const int half = warp >= 14;
    const uint32_t stage = base + S::kStages * S::kStage + (warp - 10) * 2048;
    const uint8_t* stage_p = fp4_raw + (stage - smem_u32(fp4_raw));
    const float alpha = p.alpha, alpha2 = p.alpha2;
    // 32 outputs of the warp's 32 rows, from column c0 on: rounded ..
    const auto finish = [&](const uint32_t* r, const uint32_t* r2, int c0, uint32_t (&o)[16]) {
      float v[32];
      if (GATED) {
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = fp4_silu(__uint_as_float(r[e]) * alpha) * (__uint_as_float(r2[e]) * alpha2);
      } else {
        const float bias = p.bias && c0 + lane < p.n ? p.bias[c0 + lane] : 0.f;
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = fmaf(__uint_as_float(r[e]), alpha, p.bias ? __shfl_sync(~0u, bias, e) : 0.f);
      }
#pragma unroll
      for (int e = 0; e < 16; e++) o[e] = float2_to_pair<BF16>(v[2 * e], v[2 * e + 1]);
    };
    // .. and stored
    const auto emit = [&](uint32_t (&o)[16], int m0, int c0) {
      if (c0 >= p.n || m0 >= p.rows) return;
      const bool wide = a.y_vec && c0 + 32 <= p.n;
      uint16_t* const y = (uint16_t*)p.y + (long long)m0 * p.y_row + c0;
      uint16_t* const mine = y + lane * p.y_row;
      const bool odd = ((uintptr_t)mine & 2) != 0;   // the row starts between two words: pairs from its second element on
      if (!wide && odd) {
        if (m0 + lane < p.rows) mine[0] = (uint16_t)o[0];
#pragma unroll
        for (int e = 0; e < 15; e++) o[e] = __byte_perm(o[e], o[e + 1], 0x5432);
        o[15] >>= 16;
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 4; h++)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((h ^ ((lane >> 1) & 3)) << 4)),
                     "r"(o[4 * h]), "r"(o[4 * h + 1]), "r"(o[4 * h + 2]), "r"(o[4 * h + 3]) : "memory");
      __syncwarp();
      if (wide) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int row = j * 8 + (lane >> 2), h = lane & 3;
          v[j] = *(const uint4*)(stage_p + row * 64 + ((h ^ ((row >> 1) & 3)) << 4));
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int row = j * 8 + (lane >> 2);
          if (m0 + row < p.rows) *(uint4*)(y + row * p.y_row + (lane & 3) * 8) = v[j];
        }
      } else {
        // two rows at once, a pair a lane (every other row starts alike); what is left of a row at its end by the row's own
        // lane.  (With shifts and choices at each store 1775 x 21393 x 377 took 68 us, now 39; 29 with aligned rows.)
        const int left = min(32, p.n - c0), here = p.rows - m0;
        const int q = lane & 15, r0 = lane >> 4;
        uint16_t* to = y + r0 * p.y_row + 2 * q;
        const int shift = ((uintptr_t)to & 2) != 0, pairs_to = 2 * q + shift + 1 < left ? here : 0;
        to += shift;
#pragma unroll
        for (int j0 = 0; j0 < 16; j0 += 8) {
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const int row = (j0 + j) * 2 + r0;
            w[j] = *(const uint32_t*)(stage_p + row * 64 + (((q >> 2) ^ ((row >> 1) & 3)) << 4) + (q & 3) * 4);
          }
#pragma unroll
          for (int j = 0; j < 8; j++) {
            if ((j0 + j) * 2 + r0 < pairs_to) *(uint32_t*)to = w[j];
            to += 2 * p.y_row;
          }
        }
        const int last = left - 1 - odd;             // from the first pair on
        if (last >= 0 && last % 2 == 0 && lane < here)
          mine[left - 1] = *(const uint16_t*)(stage_p + lane * 64 + (((last >> 3) ^ ((lane >> 1) & 3)) << 4) + (last & 7) * 2);
      }
    };
    uint32_t li = 0;
    for (int t = pair; t < tiles && ok; t += pairs, li++) {
      if (!__all_sync(~0u, mbar_wait_due(done, li & 1, 0x618))) { ok = false; break; }
      tc_fence_after();
      int tm, tn;
      fp4_tile_at(a, t, tm, tn);
      const int m0 = tm * 256 + (int)rank * 128 + sub * 32, n0 = tn * kOut;
      const uint32_t d = tmem + (li & 1) * S::kD1 + lanes;
      // 32 outputs are a unit of 32 columns (gated: and as many 64 further on, for the other factor).  The ones that hold shared columns
      // (three; gated two) first and together (a load takes 600 cycles beside the MMAs, however much it brings); then the
      // next tile may begin.  (Not unrolled: the code of all units would be fetched once a tile.)
      constexpr int kUnits = kOut / 32, kFirst = GATED ? 2 : 3, kOnce = GATED ? 1 : 2, kCols = GATED ? 64 : 32;
      const auto unit = [&](int i) { return (li & 1) ? i : (i + kUnits - kFirst) % kUnits; };
#pragma unroll 1
      for (int i0 = half; i0 < kUnits; i0 += 2 * kOnce) {
        uint32_t r[kOnce][kCols], o[16];
#pragma unroll
        for (int i = 0; i < kOnce; i++) {
          const int u = unit(i0 + 2 * i), at = GATED ? (u >> 1) * 128 + (u & 1) * 32 : u * 32;
          tmem_ld32(d + at, r[i]);
          if (GATED) tmem_ld32(d + at + 64, r[i] + 32);
        }
        tmem_ld_wait();
        if (i0 == half) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(lead_free);
        }
#pragma unroll
        for (int i = 0; i < kOnce; i++) {
          finish(r[i], r[i] + (GATED ? 32 : 0), n0 + unit(i0 + 2 * i) * 32, o);
          emit(o, m0, n0 + unit(i0 + 2 * i) * 32);
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_barrier();                 // no remote arrivals or MMAs into the other CTA remain
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---------------- few rows or few tiles: columns split over a cluster ----------------
// The weights are the left-hand operand (128 outputs a tile), NT rows of x the right-hand one, and a
// cluster's CTAs take a share of the columns each: a stream of weights over all SMs.  Their sums meet in
// distributed shared memory, in the order of the CTAs, so that a result does not depend on timing.
// Bound by the weights' bytes: 16 x 28672 x 8192 25 us, 5.3 TB/s; 1 x 4096 x 4096 5.2 us, of which 1.4 are bytes and the rest
// launch, the first loads, the last MMAs and the meeting of the cluster.
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
  __shared__ __align__(8) uint64_t bars[2 * S::kStages + 3];
  __shared__ uint32_t tslot;
  const YkGemmFp4& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0);
  const uint32_t base = (smem_u32(fp4_raw) + 1023) & ~1023u;
  const uint32_t full = smem_u32(&bars[0]), empty = smem_u32(&bars[S::kStages]), done = smem_u32(&bars[2 * S::kStages]),
                 sready = done + 8;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int n0 = blockIdx.x / split * 128, m0 = blockIdx.y * NT;
  const int c_first = (int)((long long)a.chunks * rank / split), c_end = (int)((long long)a.chunks * (rank + 1) / split);
  if (tid == 0) {
    for (int i = 0; i < S::kStages; i++) {
      mbar_init(full + i * 8, 1);
      mbar_init(empty + i * 8, 1);
    }
    mbar_init(done, 1);
    mbar_init(sready, 4);
    mbar_init(sready + 8, 4);
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
  const uint32_t tmem = __shfl_sync(~0u, tslot, 0);
  constexpr int kBpc = kFp4Bpc<NV>;
  constexpr int kScales = S::kA * kFp4Codes + S::kX;            // of a stage: weights', second weights', x's
  bool ok = true;                    // a wait that ran out ends the warp's part (the others' waits run out then too)

  if (warp == 0) {
    const bool issuer = elect_one();
    const long long wb = (long long)(n0 / 128) * a.blocks * kFp4Block, xb = (long long)(m0 / 128) * a.blocks * kFp4Block;
    uint32_t g = 0, s = 0, phase = 1;                // of the stage's last use
    for (int c = c_first; c < c_end; c++) {
      if (g >= S::kStages && !__all_sync(~0u, mbar_wait_due(empty + s * 8, phase, 0x621))) { ok = false; break; }
      if (issuer) {
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
      __syncwarp();
      g++;
      if (++s == S::kStages) { s = 0; phase ^= 1; }
    }
    if (!ok)
      for (uint32_t i = g > S::kStages ? g - S::kStages : 0; i < g; i++) mbar_wait(full + i % S::kStages * 8, (i / S::kStages) & 1, 0x622);
  } else if (warp == 1) {
    const bool issuer = elect_one();
    uint32_t s = 0, phase = 0, set = 0, set_phase = 0;
    int c = c_first;
    for (; c < c_end; c++) {
      if (!__all_sync(~0u, mbar_wait_due(full + s * 8, phase, 0x623) && mbar_wait_due(sready + set * 8, set_phase, 0x624))) { ok = false; break; }
      tc_fence_after();
      if (issuer) {
        const uint32_t sf = tmem + S::kSf + set * S::kSfSet, at = base + s * S::kStage;
        const uint64_t w_desc = sw128_desc(at), x_desc = sw128_desc(at + S::kA * kFp4Codes);
        const int steps = (p.k - c * kFp4Cols + 63) / 64;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int b = NV ? k : k >> 1;
#pragma unroll
          for (int x = 0; x < S::kA; x++)
            if (k == 0 || k < steps)
              tc_mma_fp4<NV>(tmem + x * NT, w_desc + x * (kFp4Codes >> 4) + k * 2, x_desc + k * 2, idesc_fp4<NV>(128, NT, NV ? 0 : k & 1),
                             sf + (x * kBpc + b) * 4, sf + (S::kA * kBpc + b) * 4, (c - c_first) | k);
        }
        tc_commit(empty + s * 8);
      }
      __syncwarp();
      if (++s == S::kStages) { s = 0; phase ^= 1; }
      set ^= 1;
      set_phase ^= set == 0;
    }
    if (issuer && c == c_end) tc_commit(done);
    __syncwarp();
  }
  const int rows = min(NT, p.rows - m0);
  float* const part = (float*)(fp4_raw + (base - smem_u32(fp4_raw)));     // [matrix][row][128 outputs], in the ring
  if (warp >= 2 && warp < 6) {
    const int sub = warp & 3;
    const uint32_t lanes = (uint32_t)(sub * 32) << 16;
    constexpr int kWords = 4 * kBpc * (S::kA + 1);   // weights', second weights', x's
    uint32_t g = 0;
    for (int c = c_first; c < c_end; c++, g++) {
      const int s = g % S::kStages;
      uint32_t v[kWords];
      if (!__all_sync(~0u, mbar_wait_due(full + s * 8, (g / S::kStages) & 1, 0x626))) { ok = false; break; }
#pragma unroll
      for (int x = 0; x <= S::kA; x++)
#pragma unroll
        for (int b = 0; b < kBpc; b++)
          fp4_get_scales(v + (x * kBpc + b) * 4, base + s * S::kStage + kScales + x * 2048 + b * kFp4Block, lane);
      // the MMAs that read this place of the scales are those of two stages ago
      if (g >= 2 && !__all_sync(~0u, mbar_wait_due(empty + (g - 2) % S::kStages * 8, ((g - 2) / S::kStages) & 1, 0x627))) { ok = false; break; }
      tc_fence_after();
      fp4_put_scales<kWords>(tmem + lanes + S::kSf + (g & 1) * S::kSfSet, v);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sready + (g & 1) * 8);
    }
    if (ok && __all_sync(~0u, mbar_wait_due(done, 0, 0x625))) {
      tc_fence_after();
#pragma unroll 1
      for (int x = 0; x < S::kA; x++) {
#pragma unroll 1
        for (int m = 0; m < rows; m += 32) {
          uint32_t r[32];
          tmem_ld32(tmem + lanes + x * NT + m, r);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e++) part[(x * NT + m + e) * 128 + sub * 32 + lane] = __uint_as_float(r[e]);
        }
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  if (split > 1) cluster_barrier();
  else __syncthreads();
  const uint32_t part_sm = smem_u32(part);
  // two outputs a thread, four rows a turn, of rows rank, rank + split, ..
  const int j = tid % 64 * 2, step = kFp4Threads / 64 * split;
  if (n0 + j < p.n) {
    const bool two = n0 + j + 1 < p.n;
    const float bias0 = p.bias ? p.bias[n0 + j] : 0.f, bias1 = p.bias && two ? p.bias[n0 + j + 1] : 0.f;
#pragma unroll 1
    for (int m = rank + tid / 64 * split; m < rows; m += 4 * step) {
      float2 v[S::kA][4];
#pragma unroll
      for (int x = 0; x < S::kA; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) v[x][i] = make_float2(0.f, 0.f);
      // four CTAs' at a time, added in the CTAs' order
#pragma unroll 1
      for (int q0 = 0; q0 < split; q0 += 4) {
        float2 b[4][S::kA][4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const uint32_t from = split > 1 ? cluster_map(part_sm, min(q0 + q, split - 1)) : part_sm;
#pragma unroll
          for (int x = 0; x < S::kA; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              b[q][x][i] = make_float2(0.f, 0.f);
              if (q0 + q < split && m + i * step < rows) {
                const uint32_t at = from + ((x * NT + m + i * step) * 128 + j) * 4;
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(b[q][x][i].x), "=f"(b[q][x][i].y) : "r"(at) : "memory");
              }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int x = 0; x < S::kA; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              v[x][i].x += b[q][x][i].x;
              v[x][i].y += b[q][x][i].y;
            }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (m + i * step >= rows) break;
        float2 o = make_float2(fmaf(v[0][i].x, p.alpha, bias0), fmaf(v[0][i].y, p.alpha, bias1));
        if (GATED) {
          const float2 u = v[S::kA - 1][i];
          o = make_float2(fp4_silu(o.x) * (u.x * p.alpha2), fp4_silu(o.y) * (u.y * p.alpha2));
        }
        uint16_t* y = (uint16_t*)p.y + (long long)(m0 + m + i * step) * p.y_row + n0 + j;
        const uint32_t w = p.dtype == YK_BF16 ? float2_to_pair<true>(o.x, o.y) : float2_to_pair<false>(o.x, o.y);
        if (a.y_pair && two) {
          *(uint32_t*)y = w;
        } else {
          y[0] = (uint16_t)w;
          if (two) y[1] = (uint16_t)(w >> 16);
        }
      }
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

template <bool NV, bool GATED, bool BF16>
static int launch_fp4_pair(const GemmFp4Args& a, cudaStream_t st) {
  using S = Fp4Pair<NV>;
  const auto kern = gemm_fp4_pair_kernel<NV, GATED, BF16>;
  const YkGemmFp4& p = a.p;
  CUtensorMap tx, tw, tw2;
  if (!encode_fp4(&tx, p.x, p.rows, p.k, p.x_row, 128) || !encode_fp4(&tw, p.w, p.n, p.k, p.w_row, GATED ? 64 : 128) ||
      !encode_fp4(&tw2, GATED ? p.w2 : p.w, p.n, p.k, p.w_row, GATED ? 64 : 128))
    return refuse(YK_EUNSUP, "gemm_fp4: no tensor map for these sizes");
  if (smem_attr(kern, S::kSmem) != cudaSuccess) return check_launch("gemm_fp4 attr");
  const int tiles = a.tiles_m * a.tiles_n, pairs = sm_count() / 2;
  launch_kc(kern, 2 * (tiles < pairs ? tiles : pairs), kFp4PairThreads, S::kSmem, 2, st, a, tx, tw, tw2);
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
  const int sms = sm_count();
  a.tiles_m = (p.rows + 255) / 256;
  a.tiles_n = (p.n + (GATED ? 127 : 255)) / (GATED ? 128 : 256);
  const long long tiles = (long long)a.tiles_m * a.tiles_n;
  if (tiles > 0x7fffffffll) return refuse(YK_EUNSUP, "gemm_fp4: rows * n too large");
  // One round of CTAs, with at least two stages of columns each: as many CTAs share a tile's columns as the SMs have room
  // for (measured, 16 x 4096 outputs x 8192 columns: 1, 2, 4, 8 give 12.3, 8.9, 6.5, 7.9 us; 16 x 12000 x 4096: 8.0,
  // 8.4, 10.7, 16.8; 16 x 2000 x 2000, 8 stages: 5.6, 5.2, 4.7, 5.6).
  const int nt = p.rows <= 32 ? 32 : 128;
  const long long small = (long long)((p.n + 127) / 128) * ((p.rows + nt - 1) / nt);
  int split = 1;
  while (split < 8 && small * split * 2 <= sms && a.chunks >= 4 * split) split *= 2;
  if (g_fp4_split && g_fp4_split <= a.chunks) split = g_fp4_split;
  // Pairs beyond that round: their tiles are four times as large (measured, split by the rule against pairs: 400 x 4096 x
  // 8192, 128 tiles, 18.2 and 18.6 us; 400 x 12000 x 4096, 376 tiles, 25.0 and 21.3; 800 x 12000 x 4096 40.9 and 28.6).  Gated
  // tiles leave room for one CTA an SM and take twice the work: half a round (800 x 2000 x 2000, 112 tiles, 17.0 and 11.3 us;
  // 100 x 12000 x 1000 12.7 and 11.2; 400 x 2000 x 2000, 64 tiles, 11.8 and 11.0).
  if (g_fp4_kernel ? g_fp4_kernel == 1 : p.rows > (GATED ? 64 : 128) && small > (GATED ? sms / 2 : sms))
    return p.dtype == YK_BF16 ? launch_fp4_pair<NV, GATED, true>(a, st) : launch_fp4_pair<NV, GATED, false>(a, st);
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
