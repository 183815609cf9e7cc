// Attention over the paged 8-bit key/value cache (yk_attn_kv8).
#include "text.cuh"

namespace yk {

struct Attn8Args {
  YkKvCache c;
  YkAttnKv8 a;
  float scale_log2;   // a.scale * log2(e): weights are powers of two
  int min_part;       // granules a CTA takes at least
};

// ---------------- few rows: split along the keys ----------------
// The rows of a request that share a key head (its q tokens x the heads of the group) fill
// 16-row tiles of warp MMAs (m16n8k16, fp16 in, fp32 sums); e4m3 codes convert to fp16 exactly,
// bf16 queries are scaled by a power of two a row to fp16 (exact but for parts below 2^-28 of
// the row's largest).  HBM bound: each code is read once, straight into the lane that feeds it
// to the MMA.
//  * Keys: lane (g, t) of a warp (g = lane / 4, t = lane % 4) needs, as the B operand, channels of
//    token g; any order of the channels serves if q has the same, so it takes 16 consecutive
//    ones with one 16-byte load.
//  * Values: as the B operand it needs pairs of tokens (2t, 2t + 1) of one channel; it loads 16
//    channels of both and interleaves their bytes (one byte permute per two channels), so
//    nothing is transposed through shared memory.
//  Every lane therefore copies (cp.async) and reads back only its own bytes: the ring of stages
//  needs no barrier at all, and each warp runs over its own 16-token subtiles with its own
//  running maximum.  The warps' states meet in shared memory once a segment.
//  * The work of all (request, key head, row tile) items is one list of granules (64 tokens);
//    each CTA takes an equal run of it, whatever the lengths.  An item that spans several CTAs
//    leaves partial sums in the workspace and the CTA that arrives last joins them in CTA order
//    (so the result does not depend on the order of arrival).
//  * One scale a (block, head): the key scale multiplies the scores; the value scale multiplies
//    the weights, whose 16-bit form is taken relative to the largest weight * scale so far (M
//    below, kept beside the softmax's m), so blocks of very different loudness keep their bits.
constexpr int kDecWarps = 4;
constexpr int kDecGran = 16 * kDecWarps;   // tokens of a granule
constexpr int kDecCtas = 148 * 2;

template <int D>
struct Dec {
  static constexpr int kStage = 32 * D;                      // bytes of a warp's stage (K and V)
  static constexpr int kStages = D == 64 ? 8 : D == 128 ? 5 : 3;
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kSmem = kDecWarps * kWarpBytes;
  static constexpr int kKC = D / 64;                         // 16-byte key chunks a lane and token
  static constexpr int kVC = D == 256 ? 2 : 1;               // value chunks a lane and token
  static constexpr int kVB = D == 64 ? 8 : 16;               // bytes of a value chunk
  static constexpr int kRow = D + 8;                         // floats of a row when states meet
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <int B>
__device__ __forceinline__ void cp_async_lane(uint32_t dst, const void* src, bool ok) {
  if (B == 16) {
    cp_async16(dst, src, ok ? 16 : 0);
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
  }
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// o += p (16 rows x 16 tokens) * v: words v[j] hold 4 channels a word of the lane's token j (of
// 2t, 2t + 1, 2t + 8, 2t + 9); bytes of a token pair interleave into the B operand.
template <int W>
__device__ __forceinline__ void pv_mma(float (*o)[4], const uint32_t (&pa)[4], const uint32_t (&v)[4][W]) {
#pragma unroll
  for (int w = 0; w < W; w++) {
    const uint32_t lo01 = __byte_perm(v[0][w], v[1][w], 0x5140), lo23 = __byte_perm(v[0][w], v[1][w], 0x7362);
    const uint32_t hi01 = __byte_perm(v[2][w], v[3][w], 0x5140), hi23 = __byte_perm(v[2][w], v[3][w], 0x7362);
    mma16816(o[4 * w], pa, e4m3x2_to_half2(lo01), e4m3x2_to_half2(hi01));
    mma16816(o[4 * w + 1], pa, e4m3x2_to_half2(lo01 >> 16), e4m3x2_to_half2(hi01 >> 16));
    mma16816(o[4 * w + 2], pa, e4m3x2_to_half2(lo23), e4m3x2_to_half2(hi23));
    mma16816(o[4 * w + 3], pa, e4m3x2_to_half2(lo23 >> 16), e4m3x2_to_half2(hi23 >> 16));
  }
}

// The first key that a row at position `pos` sees.
__device__ __forceinline__ int first_key(int pos, int window) {
  return window ? (int)max(0ll, (long long)pos - window + 1) : 0;
}

// A request's rows and keys, with whatever the arrays hold brought into range.
struct Req {
  int q0, q, kv, lo;   // first row, rows, keys, first key that any row sees
};
__device__ __forceinline__ Req attn_req(const YkKvCache& c, const YkAttnKv8& a, int r) {
  Req o;
  o.q0 = min(max(a.cu[r], 0), a.rows);
  o.q = min(max(a.cu[r + 1], o.q0), a.rows) - o.q0;
  o.kv = (int)min((long long)max(a.kv_lens[r], 0), (long long)a.max_blocks * c.tokens);
  o.lo = a.causal ? min(o.kv, first_key(o.kv - o.q, a.window)) : 0;
  return o;
}

template <bool BF16, int D>
__global__ void __launch_bounds__(32 * kDecWarps, 2) attn8_split_kernel(const __grid_constant__ Attn8Args p) {
  pdl_wait();
  pdl_trigger();
  using L = Dec<D>;
  extern __shared__ __align__(128) uint8_t dec_sm[];
  __shared__ long long part[32], pre[32 * kDecWarps];
  __shared__ float wm[kDecWarps][16], wl[kDecWarps][16];
  __shared__ uint4 qsm[D == 256 ? D / 16 : 1][32];   // q fragments (registers below 256 channels)
  __shared__ int arrived;
  const YkAttnKv8& a = p.a;
  const YkKvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int G = a.heads / c.heads, T = c.tokens;

  // granules of a request: (items) x (granules of an item, at least one: empty rows are written)
  const auto item_gran = [&](const Req& q) { return max(1, (q.kv - (q.lo & ~15) + kDecGran - 1) / kDecGran); };
  const auto row_tiles = [&](const Req& q) { return (int)(((long long)q.q * G + 15) / 16); };
  const auto req_gran = [&](const Req& q) { return q.q ? (long long)item_gran(q) * row_tiles(q) * c.heads : 0ll; };
  const int per_thread = (a.requests + 32 * kDecWarps - 1) / (32 * kDecWarps);
  long long sum = 0, total;
  for (int r = tid * per_thread; r < min(a.requests, (tid + 1) * per_thread); r++) sum += req_gran(attn_req(c, a, r));
  pre[tid] = block_exclusive(sum, part, &total);
  __syncthreads();
  const long long per = max((total + gridDim.x - 1) / gridDim.x, (long long)p.min_part);
  long long f = blockIdx.x * per;
  const long long f_end = min(total, f + per);
  if (f >= f_end) return;
  int lo = 0, hi = 32 * kDecWarps;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= f) lo = m; else hi = m;
  }
  int r = lo * per_thread;
  long long base = pre[lo];        // granules before request r
  Req q = attn_req(c, a, r);
  long long rg = req_gran(q);

  const uint32_t ring = smem_u32(dec_sm) + warp * L::kWarpBytes;
  while (f < f_end) {
    while (f >= base + rg) {       // f < total: some later request holds it
      base += rg;
      q = attn_req(c, a, ++r);
      rg = req_gran(q);
    }
    const int n = item_gran(q);
    const long long item = (f - base) / n;
    const int g0 = (int)(f - base - item * n);
    const int g1 = (int)min((long long)n, g0 + (f_end - f));
    const int tiles = row_tiles(q), kh = (int)(item / tiles), tile = (int)(item - (long long)kh * tiles);

    // rows g and g + 8 of this lane: row in a.q, head, and the keys it sees [first, last]
    int row_tok[2], row_head[2], first[2], last[2];
    const int row_n = min(16, q.q * G - tile * 16);
    int tile_lo = q.kv, tile_hi = 0;      // keys that any row of the tile sees
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int rr = tile * 16 + min(g + 8 * i, row_n - 1);
      row_tok[i] = rr / G;
      row_head[i] = kh * G + rr - row_tok[i] * G;
      last[i] = a.causal ? min(q.kv - 1, q.kv - q.q + row_tok[i]) : q.kv - 1;
      first[i] = a.causal ? first_key(q.kv - q.q + row_tok[i], a.window) : 0;
    }
    {
      const int t0 = tile * 16 / G, t1 = (tile * 16 + row_n - 1) / G;   // the tile's tokens
      tile_hi = a.causal ? max(0, q.kv - q.q + t1 + 1) : q.kv;
      tile_lo = a.causal ? first_key(q.kv - q.q + t0, a.window) : 0;
    }
    // 16-token subtiles of the segment that the tile needs
    const int s_base = (q.lo >> 4);
    const int s_lo = max(s_base + g0 * kDecWarps, tile_lo >> 4);
    const int s_hi = min(s_base + g1 * kDecWarps, (tile_hi + 15) >> 4);
    const int count = s_hi > s_lo + warp ? (s_hi - s_lo - warp + kDecWarps - 1) / kDecWarps : 0;

    // ---- the ring: block ids and scales of 32 subtiles at a time, one a lane ----
    const int* table = a.table + r * a.table_stride;
    const auto block_at = [&](int i) -> int {   // of this warp's i-th subtile; -1: none
      if (i >= count) return -1;
      const int b = table[(s_lo + warp + i * kDecWarps) * 16 / T];
      return (unsigned)b < (unsigned)c.blocks ? b : -1;
    };
    int id_i = -1, id_n = block_at(lane), id_c = -1;
    float ks_i = 0.f, vs_i = 0.f, ks_c = 0.f, vs_c = 0.f;
    const uint8_t* kcodes = (const uint8_t*)c.k + (long long)kh * T * D;
    const uint8_t* vcodes = (const uint8_t*)c.v + (long long)kh * T * D;
    const auto issue = [&](int i) {
      if ((i & 31) == 0) {
        id_i = id_n;
        if (id_i >= 0) {
          ks_i = c.kscale[id_i * c.scale_stride + kh];
          vs_i = c.vscale[id_i * c.scale_stride + kh];
        }
        id_n = block_at(i + 32 + lane);
      }
      const int id = __shfl_sync(~0u, id_i, i & 31);
      const int tok0 = (s_lo + warp + i * kDecWarps) * 16;
      const long long at = max(id, 0) * c.block_stride + (long long)(tok0 & (T - 1)) * D;
      const uint32_t dst = ring + (i % L::kStages) * L::kStage;
      const int left = id < 0 ? 0 : tile_hi - tok0;   // tokens past what the tile sees read as zero
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int h = 0; h < L::kKC; h++)
          cp_async_lane<16>(dst + (j * L::kKC + h) * 512 + lane * 16,
                            kcodes + at + (8 * j + g) * D + (t + 4 * h) * 16, 8 * j + g < left);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int tok = 2 * t + (j & 1) + 8 * (j >> 1);
#pragma unroll
        for (int h = 0; h < L::kVC; h++)
          cp_async_lane<L::kVB>(dst + 2 * L::kKC * 512 + (j * L::kVC + h) * (32 * L::kVB) + lane * L::kVB,
                                vcodes + at + tok * D + h * 128 + g * L::kVB, tok < left);
      }
    };
#pragma unroll
    for (int i = 0; i < L::kStages - 1; i++) {
      if (i < count) issue(i);
      cp_async_commit();
    }

    // ---- q fragments: chunk h, part i: channels (t + 4 h) * 16 + 4 i + {0, 1 | 2, 3} ----
    uint32_t qf[D == 256 ? 1 : D / 16][4];
    float fac[2];      // score factor of the row: scale * log2 e * the power of two taken out of q
    {
      const uint16_t* qp[2];
#pragma unroll
      for (int i = 0; i < 2; i++)
        qp[i] = (const uint16_t*)a.q + (long long)(q.q0 + row_tok[i]) * a.q_row + (long long)row_head[i] * D;
      float up[2] = {1.f, 1.f};
      fac[0] = fac[1] = p.scale_log2;
      if (BF16) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float m = 0.f;
#pragma unroll
          for (int h = 0; h < 2 * L::kKC; h++) {
            const uint4 v = *(const uint4*)(qp[i] + (t + 4 * (h >> 1)) * 16 + (h & 1) * 8);
            const uint32_t* u = (const uint32_t*)&v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float2 x = pair_to_float2<true>(u[e]);
              m = fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
          }
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
          int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;   // m in [2^e, 2^(e+1))
          e = m > 0.f ? max(-110, min(e, 120)) : 13;
          up[i] = __uint_as_float((uint32_t)(127 + 13 - e) << 23);     // the largest becomes 2^13 .. 2^14
          fac[i] = p.scale_log2 * __uint_as_float((uint32_t)(127 - 13 + e) << 23);
        }
      }
#pragma unroll
      for (int h = 0; h < L::kKC; h++) {
        uint4 v[2][2];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int e = 0; e < 2; e++) v[i][e] = *(const uint4*)(qp[i] + (t + 4 * h) * 16 + e * 8);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {   // rows g, g + 8 of channels 0, 1; then of 2, 3
            const uint32_t u = ((const uint32_t*)&v[e & 1][i >> 1])[(i & 1) * 2 + (e >> 1)];
            if (BF16) {
              const float2 x = pair_to_float2<true>(u);
              w[e] = pack_half2(x.x * up[e & 1], x.y * up[e & 1]);
            } else {
              w[e] = u;
            }
          }
          if (D == 256) {
            if (warp == 0) qsm[h * 4 + i][lane] = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) qf[h * 4 + i][e] = w[e];
          }
        }
      }
      if (D == 256) __syncthreads();
    }

    // ---- the subtiles ----
    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, M[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll 1
    for (int i = 0; i < count; i++) {
      if (i + L::kStages - 1 < count) issue(i + L::kStages - 1);
      cp_async_commit();
      cp_async_wait<L::kStages - 1>();
      if ((i & 31) == 0) { id_c = id_i; ks_c = ks_i; vs_c = vs_i; }   // issue() is in the same 32
      const int id = __shfl_sync(~0u, id_c, i & 31);
      const float ks = __shfl_sync(~0u, ks_c, i & 31), vs = __shfl_sync(~0u, vs_c, i & 31);
      if (id < 0) continue;
      const int tok0 = (s_lo + warp + i * kDecWarps) * 16;
      const uint32_t src = ring + (i % L::kStages) * L::kStage;
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int h = 0; h < L::kKC; h++) {
          const uint4 kw = lds128(src + (j * L::kKC + h) * 512 + lane * 16);
          const uint32_t* w = (const uint32_t*)&kw;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t b0 = e4m3x2_to_half2(w[e]), b1 = e4m3x2_to_half2(w[e] >> 16);
            if (D == 256) {
              const uint4 qv = qsm[h * 4 + e][lane];
              const uint32_t qa[4] = {qv.x, qv.y, qv.z, qv.w};
              mma16816(s[j], qa, b0, b1);
            } else {
              mma16816(s[j], qf[D == 256 ? 0 : h * 4 + e], b0, b1);
            }
          }
        }
      }
      const float lv = __log2f(vs);
      const bool edge = tok0 < first[0] || tok0 < first[1] || tok0 + 15 > last[0] || tok0 + 15 > last[1];
      const bool any_edge = __any_sync(~0u, edge);
      float corr[2], corr_o[2], f_v[2];
#pragma unroll
      for (int i2 = 0; i2 < 2; i2++) {
        const float k = ks * fac[i2];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float& x = s[j][2 * i2 + e];
            x *= k;
            if (any_edge) {
              const int tok = tok0 + 8 * j + 2 * t + e;
              if (tok < first[i2] || tok > last[i2]) x = -INFINITY;
            }
            top = fmaxf(top, x);
          }
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        const float mn = fmaxf(m[i2], top);
        const float ref = mn == -INFINITY ? 0.f : mn;
        corr[i2] = ex2(m[i2] - ref);
        m[i2] = mn;
        const float Mn = fmaxf(M[i2], top + lv);
        const float Mref = Mn == -INFINITY ? 0.f : Mn;
        corr_o[i2] = exp2f(M[i2] - Mref);
        M[i2] = Mn;
        f_v[i2] = Mn == -INFINITY || lv == -INFINITY ? 0.f : vs * exp2f(ref - Mref);
        l[i2] *= corr[i2];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float& x = s[j][2 * i2 + e];
            x = ex2(x - ref);
            l[i2] += x;
            x *= f_v[i2];
          }
      }
      if (__any_sync(~0u, corr_o[0] != 1.f || corr_o[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < D / 8; j++) {
          o[j][0] *= corr_o[0];
          o[j][1] *= corr_o[0];
          o[j][2] *= corr_o[1];
          o[j][3] *= corr_o[1];
        }
      }
      const uint32_t pa[4] = {pack_half2(s[0][0], s[0][1]), pack_half2(s[0][2], s[0][3]),
                              pack_half2(s[1][0], s[1][1]), pack_half2(s[1][2], s[1][3])};
#pragma unroll
      for (int h = 0; h < L::kVC; h++) {
        uint32_t v[4][L::kVB / 4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t at = src + 2 * L::kKC * 512 + (j * L::kVC + h) * (32 * L::kVB) + lane * L::kVB;
          if (L::kVB == 16) {
            const uint4 x = lds128(at);
            v[j][0] = x.x; v[j][1] = x.y; v[j][L::kVB / 4 - 2] = x.z; v[j][L::kVB / 4 - 1] = x.w;
          } else {
            const uint2 x = lds64(at);
            v[j][0] = x.x; v[j][1] = x.y;
          }
        }
        // 0 * NaN: a NaN code that only some rows of the tile see must not reach the others, so
        // each row then goes through the MMA by itself, without the tokens that it does not see
        bool nan = false;
        if (any_edge) {
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int w = 0; w < L::kVB / 4; w++) nan |= (((v[j][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
          nan = __any_sync(~0u, nan);
        }
        if (!nan) {
          pv_mma<L::kVB / 4>(o + h * 16, pa, v);
        } else {
#pragma unroll 1
          for (int i2 = 0; i2 < 16; i2++) {
            const int src_lane = (i2 & 7) * 4;
            const int f0 = __shfl_sync(~0u, first[0], src_lane), f1 = __shfl_sync(~0u, first[1], src_lane);
            const int l0 = __shfl_sync(~0u, last[0], src_lane), l1 = __shfl_sync(~0u, last[1], src_lane);
            uint32_t seen[4][L::kVB / 4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int tok = tok0 + 2 * t + (j & 1) + 8 * (j >> 1);
              const bool see = tok >= (i2 < 8 ? f0 : f1) && tok <= (i2 < 8 ? l0 : l1);
#pragma unroll
              for (int w = 0; w < L::kVB / 4; w++) seen[j][w] = see ? v[j][w] : 0;
            }
            float one[L::kVB][4];
#pragma unroll
            for (int j = 0; j < L::kVB; j++) one[j][0] = one[j][1] = one[j][2] = one[j][3] = 0.f;
            pv_mma<L::kVB / 4>(one, pa, seen);
#pragma unroll
            for (int j = 0; j < L::kVB; j++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (g == (i2 & 7) && (e >> 1) == (i2 >> 3)) o[h * 16 + j][e] += one[j][e];
          }
        }
      }
    }
    cp_async_wait<0>();

    // ---- the warps' states meet: o relative to the common m ----
#pragma unroll
    for (int i = 0; i < 2; i++) {
      l[i] += __shfl_xor_sync(~0u, l[i], 1);
      l[i] += __shfl_xor_sync(~0u, l[i], 2);
      if (t == 0) { wm[warp][g + 8 * i] = m[i]; wl[warp][g + 8 * i] = l[i]; }
    }
    __syncthreads();
    float* mine = (float*)(dec_sm + warp * L::kWarpBytes);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float top = wm[0][g + 8 * i];
#pragma unroll
      for (int w = 1; w < kDecWarps; w++) top = fmaxf(top, wm[w][g + 8 * i]);
      const float k = M[i] == -INFINITY ? 0.f : exp2f(M[i] - top);
#pragma unroll
      for (int j = 0; j < D / 8; j++)
        *(float2*)(mine + (g + 8 * i) * L::kRow + j * 8 + 2 * t) = make_float2(o[j][2 * i] * k, o[j][2 * i + 1] * k);
    }
    __syncthreads();
    // thread (row, column n of the MMA tiles): channels n * kVB .. of each 128 (64)
    const int row = tid >> 3, col = tid & 7;
    float top = wm[0][row], lsum = 0.f;
#pragma unroll
    for (int w = 1; w < kDecWarps; w++) top = fmaxf(top, wm[w][row]);
#pragma unroll
    for (int w = 0; w < kDecWarps; w++) lsum = fmaf(wl[w][row], wm[w][row] == -INFINITY ? 0.f : exp2f(wm[w][row] - top), lsum);
    float acc[D / 8];
#pragma unroll
    for (int j = 0; j < D / 8; j++) {
      acc[j] = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWarps; w++)
        acc[j] += ((const float*)(dec_sm + w * L::kWarpBytes))[row * L::kRow + j * 8 + col];
    }
    // ---- a whole item is written out; a part goes to the workspace ----
    bool write = true;
    if (g0 > 0 || g1 < n) {
      const long long fs = f - g0;
      const int ca = (int)(fs / per), cb = (int)((fs + n - 1) / per);   // the CTAs of this item
      float* ws = (float*)((uint8_t*)a.ws + kDecCtas * sizeof(int));
      constexpr int kPart = 16 * D + 32;     // floats of a part: o, then m and l of each row
      int* counter = (int*)a.ws + ca;
      const bool starts = (int)blockIdx.x == ca;
      float* slot = ws + ((long long)blockIdx.x * 2 + (starts ? 1 : 0)) * kPart;
      if (row < row_n) {
#pragma unroll
        for (int j = 0; j < D / 8; j += 4)
          *(float4*)(slot + (row * 8 + col) * (D / 8) + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        if (col == 0) { slot[16 * D + row] = top; slot[16 * D + 16 + row] = lsum; }
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) arrived = atomicAdd(counter, 1);
      __syncthreads();
      write = arrived == cb - ca;
      if (write) {
        __threadfence();
        if (tid == 0) *counter = 0;          // as the next call expects it
        if (row < row_n) {
          const auto part_of = [&](int b) { return ws + ((long long)b * 2 + (b == ca ? 1 : 0)) * kPart; };
          top = -INFINITY;
          for (int b = ca; b <= cb; b++) top = fmaxf(top, __ldcg(part_of(b) + 16 * D + row));
          lsum = 0.f;
#pragma unroll
          for (int j = 0; j < D / 8; j++) acc[j] = 0.f;
          for (int b = ca; b <= cb; b++) {
            const float* s = part_of(b);
            const float pm = __ldcg(s + 16 * D + row);
            const float k = pm == -INFINITY ? 0.f : exp2f(pm - top);
            lsum = fmaf(k, __ldcg(s + 16 * D + 16 + row), lsum);
#pragma unroll
            for (int j = 0; j < D / 8; j += 4) {
              const float4 v = __ldcg((const float4*)(s + (row * 8 + col) * (D / 8) + j));
              acc[j] = fmaf(k, v.x, acc[j]);
              acc[j + 1] = fmaf(k, v.y, acc[j + 1]);
              acc[j + 2] = fmaf(k, v.z, acc[j + 2]);
              acc[j + 3] = fmaf(k, v.w, acc[j + 3]);
            }
          }
        }
      }
    }
    if (write && row < row_n) {
      const int rr = tile * 16 + row, tok = rr / G, head = kh * G + rr - tok * G;
      const float inv = lsum > 0.f ? 1.f / lsum : 0.f;
      uint16_t* op = (uint16_t*)a.out + (long long)(q.q0 + tok) * a.out_row + (long long)head * D;
#pragma unroll
      for (int h = 0; h < L::kVC; h++)
#pragma unroll
        for (int j = 0; j < L::kVB; j += 8) {
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; e++)
            u[e] = float2_to_pair<BF16>(acc[h * 16 + j + 2 * e] * inv, acc[h * 16 + j + 2 * e + 1] * inv);
          *(uint4*)(op + h * 128 + col * L::kVB + j) = make_uint4(u[0], u[1], u[2], u[3]);
        }
      if (a.lse && col == 0)
        a.lse[(long long)(q.q0 + tok) * a.heads + head] =
            lsum == 0.f ? -INFINITY : (top + log2f(lsum)) * 0.6931471805599453f;
    }
    __syncthreads();      // the ring and the small arrays are used again
    f += g1 - g0;
  }
}

}  // namespace yk

using namespace yk;

extern "C" size_t yk_attn_kv8_workspace_bytes(int requests, int rows, int heads, int kv_heads, int dim) {
  // a counter and two parts (o, m, l of 16 rows) for each CTA, whatever the lengths
  (void)requests; (void)rows; (void)heads; (void)kv_heads;
  return kDecCtas * (sizeof(int) + 2 * (16 * (size_t)std::max(dim, 0) + 32) * sizeof(float));
}

template <bool BF16, int D>
static int launch_attn8_split(const Attn8Args& p, cudaStream_t st) {
  const auto kern = attn8_split_kernel<BF16, D>;
  if (smem_attr(kern, Dec<D>::kSmem) != cudaSuccess) return check_launch("attn_kv8 attr");
  launch_k(kern, kDecCtas, 32 * kDecWarps, Dec<D>::kSmem, st, p);
  note_launch();
  return check_launch("attn_kv8");
}

extern "C" int yk_attn_kv8(const YkKvCache* c, const YkAttnKv8* a, yk_stream_t st) {
  const int bad = check_cache(c);
  if (bad) return bad;
  if (!a || !a->cu || !a->kv_lens || !a->table || !a->ws) return refuse(YK_EINVAL, "attn_kv8: null pointer");
  if (a->dtype != YK_F16 && a->dtype != YK_BF16) return refuse(YK_EUNSUP, "attn_kv8: dtype must be fp16 or bf16");
  if (a->requests < 1 || a->rows < 0 || a->heads < 1 || a->heads % c->heads || a->max_blocks < 1 ||
      a->table_stride < a->max_blocks || a->window < 0 || !(a->scale >= 0.f))
    return refuse(YK_EINVAL, "attn_kv8: bad requests, rows, heads, table, window or scale");
  if (a->requests > 16384) return refuse(YK_EUNSUP, "attn_kv8: at most 16384 requests");
  if (a->window && !a->causal) return refuse(YK_EINVAL, "attn_kv8: a window needs causal");
  if (a->rows == 0) return YK_OK;
  if (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out) || a->q_row % 8 || a->out_row % 8 ||
      a->out_row < (long long)a->heads * c->dim || a->q_row < 0)
    return refuse(YK_EINVAL, "attn_kv8: q and out need 16-byte alignment and row strides that are multiples of 8");
  if (!aligned16(a->ws) || a->ws_bytes < yk_attn_kv8_workspace_bytes(a->requests, a->rows, a->heads, c->heads, c->dim))
    return refuse(YK_EINVAL, "attn_kv8: workspace too small or not 16-byte aligned");
  Attn8Args p{*c, *a, 0.f, 1};
  if (p.a.scale == 0.f) p.a.scale = 1.f / sqrtf((float)c->dim);
  p.scale_log2 = p.a.scale * 1.4426950408889634f;
  const bool bf = a->dtype == YK_BF16;
  cudaStream_t s = (cudaStream_t)st;
  switch (c->dim) {
    case 64: return bf ? launch_attn8_split<true, 64>(p, s) : launch_attn8_split<false, 64>(p, s);
    case 128: return bf ? launch_attn8_split<true, 128>(p, s) : launch_attn8_split<false, 128>(p, s);
    default: return bf ? launch_attn8_split<true, 256>(p, s) : launch_attn8_split<false, 256>(p, s);
  }
}
