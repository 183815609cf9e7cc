// Attention over the paged 8-bit key/value cache (yk_attn_kv8).
#include "text.cuh"

namespace yk {

struct Attn8Args {
  YkKvCache c;
  YkAttnKv8 a;
  float scale_log2;   // a.scale * log2(e): weights are powers of two
  int lead;           // cost of starting an item, in granules
  int min_part;       // cost that a CTA takes on at least
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
//  * The work of all (request, key head, row tile) items is one list of granules (128 tokens), with a
//    lead for each item's start and end; each CTA takes an equal run of it, whatever the lengths.  An item that spans several CTAs
//    leaves partial sums in the workspace and the CTA that arrives last joins them in CTA order
//    (so the result does not depend on the order of arrival).
//  * One scale a (block, head): the key scale multiplies the scores; the value scale multiplies
//    the weights, whose 16-bit form is taken relative to the largest weight * scale so far (M
//    below, kept beside the softmax's m), so blocks of very different loudness keep their bits.
//  * Weights enter the second product as fp16 (11 bits, where bf16 has 8); their sum l stays in fp32.  The
//    largest lies at 2^9 .. 2^15 (kLift, kSlack), so a weight keeps its bits down to 2^-23 of the largest, times
//    scale, and is lost below 2^-34: a long flat tail behind one loud key still counts.  One rounding makes
//    an fp16 output 1.27 - 1.42 times as far from 64 bits as its own rounding alone; up to 8 rows a tile, the other 8
//    rows carry the rest of the weights for nothing (1.00 times).  For more rows the rest would need MMAs of
//    its own (64 requests of 4 rows 68.8 -> 74.0 us), so they round once, like bf16 outputs, where it does not show.
//  * References that move only when the maximum passes them by a slack are a known variant of the one-pass softmax.
// Measured: 2 requests over 283,000 keys (8 query heads a key head, 128 channels, 145 MB) 50 us, 2.9 TB/s:
// the keys themselves pass at 5.3 TB/s (28 us), 5 us go before the first of them (lengths, table, block,
// codes: four loads in a row), the rest into meeting and joining 74 parts an item; 64 requests of 64 to
// 8192 keys (221 MB) 64 us, 3.5 TB/s; one request of 431 keys 8.4 us.
constexpr int kDecWarps = 4;
constexpr int kDecSub = 2 * kDecWarps;     // 16-token subtiles of a granule: two for each warp
constexpr int kDecGran = 16 * kDecSub;     // tokens of a granule
// Cost of starting an item and the least share of a CTA, in granules (measured, 64 requests of 64
// to 8192 keys, 32 / 8 heads of 128: lead 0, 1, 2, 3, 4 give 93, 75, 64, 65, 68 us; one request of
// 431 keys: least share 3, 6 give 10.0, 8.5 us).
constexpr int kDecLead = 2, kDecMin = 6;
constexpr int kDecCtas = 148 * 2;
// References of the weights, both kernels: m of 2^(score - m), M of the 16-bit weight * value scale.  Both
// follow the running maximum only when it passes them by more than 2^kSlack, so the sums are rescaled a
// few times a segment; M lies 2^kLift below its maximum, so the 16-bit weights stay below 2^(kLift + kSlack)
// (fp16 holds 2^15), and no more than 2^126 below m, so that 2^(m - M) is finite.
constexpr float kNone = -1e30f, kSlack = 6.f, kLift = 9.f;
__device__ __forceinline__ float lifted(float M, float top_v, float m) {
  return fmaxf(M, fmaxf(top_v - kLift, m - 126.f));
}
// Value scale * 2^(m - M), by which weights become their 16-bit form.  It passes 2^128 only for a block whose
// scores lie 2^113 and more below the row's (a block of zero values has scale 2^-126, so M can lie that far
// below m); its weights 0 .. 2^-113 then count for less, but not as 0 * inf.
__device__ __forceinline__ float weight_factor(float scale, float gain) { return fminf(scale * gain, 3.402823466e38f); }
// Which kernel: the tcgen05 tiles take whole rows of keys, so they need enough tiles to fill the SMs; the
// split list fills them with anything but does 16 rows at a time.  Measured, 16 / 4 heads, rows a request and
// key head -> us on the split list | on tiles: 8 requests of 2000 keys, 128 channels: 16: 24 | 50, 64: 26 | 50,
// 128: 38 | 51, 256: 60 | 52; 64 requests of 500 keys: 16: 17 | 32, 32: 37 | 33, 64: 54 | 33; 1 request of 8000
// keys: 256: 44 | 162; 256 channels, 8 of 2000: 16: 32 | 64, 64: 66 | 66, 128: 94 | 69.  So tiles from kProTiles
// 16-row tiles on, or that many for every round of CTAs; and only for several new tokens a request, since a
// decode batch's lengths may differ by any factor, which only the split evens out.
constexpr int kProTokens = 8;              // new tokens a request, on average
template <int D>
constexpr int kProTiles = D == 256 ? 150 : 430;
static std::atomic<int> g_attn_kernel{0};  // test hook: 1 split list, 2 tiles, 0 the rule
constexpr int kAtOnce = 8;                 // parts that a join reads at a time

template <int D>
struct Dec {
  static constexpr int kStage = 32 * D;                      // bytes of a warp's stage (K and V)
  static constexpr int kStages = D == 64 ? 8 : 4;
  static constexpr int kPairs = kStages / 2;                 // a warp's iteration takes two stages
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kKC = D / 64;                         // 16-byte key chunks a lane and token
  static constexpr int kVC = D == 256 ? 2 : 1;               // value chunks a lane and token
  static constexpr int kVB = D == 64 ? 8 : 16;               // bytes of a value chunk
  static constexpr int kCol = D / 8 + 1, kRow = 8 * kCol;    // floats of an MMA column, of a row, when states meet
  static constexpr int kMeet = D == 256 ? 1 : 2;
  static constexpr int kQRow = 2 * D + 16, kQBytes = 16 * kQRow;
  static constexpr int kSmem = kDecWarps * kWarpBytes + 2 * kQBytes + kMeet * 16 * kRow * (int)sizeof(float);
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// o += p (16 rows x 16 tokens) * v for two subtiles: words v[u][j] hold 4 channels a word of the
// lane's token j (of 2t, 2t + 1, 2t + 8, 2t + 9); bytes of a token pair interleave into the B operand.
template <int W>
__device__ __forceinline__ void pv_mma(float (*o)[4], const uint32_t (&pa)[2][4], const uint32_t (&v)[2][4][W]) {
#pragma unroll
  for (int w = 0; w < W; w++)
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t sel = half ? 0x7362 : 0x5140;
        uint32_t a0, a1, b0, b1;
        e4m3x4_to_half2x2(__byte_perm(v[u][0][w], v[u][1][w], sel), a0, a1);
        e4m3x4_to_half2x2(__byte_perm(v[u][2][w], v[u][3][w], sel), b0, b1);
        mma16816(o[4 * w + 2 * half], pa[u], a0, b0);
        mma16816(o[4 * w + 2 * half + 1], pa[u], a1, b1);
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
  // (a little below 2^31, so that sums with a tile's size stay in 32 bits)
  o.kv = (int)min((long long)min(max(a.kv_lens[r], 0), 0x7fff0000), (long long)a.max_blocks * c.tokens);
  o.lo = a.causal ? min(o.kv, first_key(o.kv - o.q, a.window)) : 0;
  return o;
}

// What a CTA does next: granules g0 .. g1 of the n of item (key head kh, row tile) of request r.
struct Seg {
  int r, kh, tile, row_n;        // row_n: rows of the tile
  int q0, q, kv;                 // the request's first row, rows, keys
  int g0, g1, n, cost;           // none (g0 == g1) where the CTA's share ends in the item's lead
  int s_lo, s_hi;                // 16-token subtiles [s_lo, s_hi) that the tile needs of them
  int tile_hi;                   // keys that any of its rows sees end here
};

template <bool BF16, int D>
__global__ void __launch_bounds__(32 * kDecWarps, D == 256 ? 1 : 2) attn8_split_kernel(const __grid_constant__ Attn8Args p) {
  using L = Dec<D>;
  extern __shared__ __align__(128) uint8_t dec_sm[];    // rings, then q rows (two), then meeting rows
  __shared__ Sums part[32];
  __shared__ long long pre[32 * kDecWarps];
  __shared__ float wm[kDecWarps][16], wl[kDecWarps][16], row_m[16], row_l[16];
  __shared__ uint4 qsm[D == 256 ? D / 16 : 1][32];   // q fragments (registers below 256 channels)
  __shared__ int arrived;
  const YkAttnKv8& a = p.a;
  const YkKvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int G = a.heads / c.heads, T = c.tokens, lead = p.lead;
  pdl_wait();
  pdl_trigger();

  // granules of a request: (items) x (granules of an item, at least one: empty rows are written)
  const auto item_gran = [&](const Req& q) { return max(1, (q.kv - (q.lo & ~15) + kDecGran - 1) / kDecGran); };
  const auto row_tiles = [&](const Req& q) { return (int)(((long long)q.q * G + 15) / 16); };
  const auto req_cost = [&](const Req& q) { return q.q ? (long long)(item_gran(q) + lead) * row_tiles(q) * c.heads : 0ll; };
  const int per_thread = (a.requests + 32 * kDecWarps - 1) / (32 * kDecWarps);
  Sums sum = {0, 0}, total2;
  for (int r = tid * per_thread; r < min(a.requests, (tid + 1) * per_thread); r++) sum.a += req_cost(attn_req(c, a, r));
  pre[tid] = block_exclusive2(sum, part, &total2).a;
  const long long total = total2.a;
  __syncthreads();
  const long long per = max((total + gridDim.x - 1) / gridDim.x, (long long)p.min_part);
  long long f = blockIdx.x * per;
  const long long f_end = min(total, f + per);
  if (f >= f_end) return;
  int at_r;
  long long base;                  // granules before request at_r
  {
    int lo = 0, hi = 32 * kDecWarps;
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (pre[m] <= f) lo = m; else hi = m;
    }
    at_r = lo * per_thread;
    base = pre[lo];
  }
  Req rq = attn_req(c, a, at_r);
  long long rg = req_cost(rq);
  // the segment at f, of which there is one; moves the cursor (at_r, base, rq, rg) to its request
  const auto segment_at = [&](long long f) -> Seg {
    while (f >= base + rg) {
      base += rg;
      rq = attn_req(c, a, ++at_r);
      rg = req_cost(rq);
    }
    Seg s;
    s.r = at_r; s.q0 = rq.q0; s.q = rq.q; s.kv = rq.kv;
    s.n = item_gran(rq);
    const long long item = (f - base) / (s.n + lead);
    const int at = (int)(f - base - item * (s.n + lead));
    s.cost = (int)min((long long)(s.n + lead - at), f_end - f);
    s.g0 = max(0, at - lead);
    s.g1 = max(0, at + s.cost - lead);
    const int tiles = row_tiles(rq);
    s.kh = (int)(item / tiles);
    s.tile = (int)(item - (long long)s.kh * tiles);
    s.row_n = min(16, rq.q * G - s.tile * 16);
    const int t0 = s.tile * 16 / G, t1 = (s.tile * 16 + s.row_n - 1) / G;   // the tile's tokens
    s.tile_hi = a.causal ? max(0, rq.kv - rq.q + t1 + 1) : rq.kv;
    const int tile_lo = a.causal ? first_key(rq.kv - rq.q + t0, a.window) : 0;
    s.s_lo = max((rq.lo >> 4) + s.g0 * kDecSub, tile_lo >> 4);
    s.s_hi = min((rq.lo >> 4) + s.g1 * kDecSub, (s.tile_hi + 15) >> 4);
    return s;
  };

  const uint32_t ring = smem_u32(dec_sm) + warp * L::kWarpBytes;
  uint8_t* const q_sm = dec_sm + kDecWarps * L::kWarpBytes;
  float* const meet = (float*)(q_sm + 2 * L::kQBytes);
  // Twin tiles: with at most 8 rows, rows 8 .. 15 of an fp16 tile are the same rows again, and hold what the
  // 16-bit rounding of the weights leaves (bf16 outputs are too coarse to show it).
  const auto twins = [&](const Seg& s) { return !BF16 && s.row_n <= 8; };
  // rows of a segment's q into buffer b (each thread its own 16-byte chunks)
  const auto load_q = [&](const Seg& s, int b) {
    for (int i = tid; i < 16 * D / 8; i += 32 * kDecWarps) {
      const int rr = s.tile * 16 + min(i / (D / 8) & (twins(s) ? 7 : 15), s.row_n - 1), tok = rr / G;
      cp_async_at<16>(smem_u32(q_sm) + b * L::kQBytes + i / (D / 8) * L::kQRow + i % (D / 8) * 16,
                        (const uint16_t*)a.q + (long long)(s.q0 + tok) * a.q_row + (long long)(s.kh * G + rr - tok * G) * D + i % (D / 8) * 8);
    }
  };

  // ---- the ring: block ids and scales of 32 subtiles at a time, one a lane ----
  int count;                               // subtiles of this warp
  const int* table;
  const uint8_t *kcodes, *vcodes;
  int s_first, tile_hi;
  const auto sub_at = [&](int i) { return s_first + (i >> 1) * kDecSub + (i & 1); };   // this warp's i-th subtile
  const auto block_at = [&](int i) -> int {   // of this warp's i-th subtile; -1: none
    if (i >= count) return -1;
    const int b = table[sub_at(i) * 16 / T];
    return (unsigned)b < (unsigned)c.blocks ? b : -1;
  };
  int id_i = -1, id_n = -1, kh_i = 0;
  float ks_i = 0.f, vs_i = 0.f;
  uint32_t fill = ring;                       // the stage that the next copy fills
  const auto open = [&](const Seg& s) {       // from here on issue() copies segment s
    s_first = s.s_lo + 2 * warp;
    const int left = max(0, s.s_hi - s_first);
    count = left / kDecSub * 2 + min(2, left % kDecSub);
    table = a.table + s.r * a.table_stride;
    kh_i = s.kh;
    tile_hi = s.tile_hi;
    kcodes = (const uint8_t*)c.k + (long long)kh_i * T * D + g * D + t * 16;
    vcodes = (const uint8_t*)c.v + (long long)kh_i * T * D + 2 * t * D + g * L::kVB;
    id_n = block_at(lane);
  };
  const auto issue = [&](int i) {
    if ((i & 31) == 0) {
      id_i = id_n;
      ks_i = id_i < 0 ? 0.f : c.kscale[id_i * c.scale_stride + kh_i];
      vs_i = id_i < 0 ? 0.f : c.vscale[id_i * c.scale_stride + kh_i];
      id_n = block_at(i + 32 + lane);
    }
    const int id = __shfl_sync(~0u, id_i, i & 31);
    const int tok0 = sub_at(i) * 16;
    const long long at = max(id, 0) * c.block_stride + (tok0 & (T - 1)) * D;
    const uint8_t *kp = kcodes + at, *vp = vcodes + at;
    const uint32_t kd = fill + lane * 16, vd = fill + 2 * L::kKC * 512 + lane * L::kVB;
    const int left = id < 0 ? 0 : tile_hi - tok0;   // tokens past what the tile sees read as zero
    if (left >= 16) {
#pragma unroll
      for (int j = 0; j < 2 * L::kKC; j++)
        cp_async_at<16>(kd + j * 512, kp + 8 * (j / L::kKC) * D + (j % L::kKC) * 64);
#pragma unroll
      for (int j = 0; j < 4 * L::kVC; j++)
        cp_async_at<L::kVB>(vd + j * 32 * L::kVB, vp + ((j / L::kVC & 1) + 8 * (j / L::kVC >> 1)) * D + (j % L::kVC) * 128);
    } else {
#pragma unroll
      for (int j = 0; j < 2 * L::kKC; j++)
        cp_async_at<16>(kd + j * 512, kp + 8 * (j / L::kKC) * D + (j % L::kKC) * 64, 8 * (j / L::kKC) + g < left);
#pragma unroll
      for (int j = 0; j < 4 * L::kVC; j++) {
        const int tok = (j / L::kVC & 1) + 8 * (j / L::kVC >> 1);
        cp_async_at<L::kVB>(vd + j * 32 * L::kVB, vp + tok * D + (j % L::kVC) * 128, 2 * t + tok < left);
      }
    }
    fill += L::kStage;
    if (fill == ring + L::kWarpBytes) fill = ring;
  };
  // Subtiles go in pairs (a warp's iteration), each pair a group of its own; one past the end
  // reads as zero.
  const auto issue_pair = [&](int i) {
    if (i < count) {
      issue(i);
      issue(i + 1);
    }
    cp_async_commit();
  };
  const auto prologue = [&] {
#pragma unroll
    for (int i = 0; i < L::kPairs - 1; i++) issue_pair(2 * i);
  };

  // The next segment's q rows are copied, and its first block ids read, while this one runs; its
  // first stages are under way while the warps' states of this one meet.
  Seg cur = segment_at(f);
  if (cur.g0 == cur.g1) return;
  load_q(cur, 0);
  cp_async_commit();
  open(cur);
  prologue();
  const uint8_t* const ring_p = dec_sm + warp * L::kWarpBytes;
  const uint8_t* src = ring_p;
  cp_async_wait<L::kPairs - 1>();
  __syncthreads();                 // q is there
  for (int turn = 0;; turn ^= 1) {
    const long long f_next = f + cur.cost;

    const bool twin = twins(cur);
    // rows g and g + 8 of this lane: the keys they see, [first, last]
    int first[2], last[2], all_lo = 0, all_hi = cur.kv;    // [all_lo, all_hi): keys that every row sees
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int pos = cur.kv - cur.q + (cur.tile * 16 + min(g + (twin ? 0 : 8 * i), cur.row_n - 1)) / G;
      last[i] = a.causal ? min(cur.kv - 1, pos) : cur.kv - 1;
      first[i] = a.causal ? first_key(pos, a.window) : 0;
    }
    if (a.causal) {
      all_hi = cur.kv - cur.q + cur.tile * 16 / G + 1;
      all_lo = first_key(cur.kv - cur.q + (cur.tile * 16 + cur.row_n - 1) / G, a.window);
    }

    // ---- q fragments: chunk h, part i: channels (t + 4 h) * 16 + 4 i + {0, 1 | 2, 3} ----
    uint32_t qf[D == 256 ? 1 : D / 16][4];
    float fac[2];      // score factor of the row: scale * log2 e * the power of two taken out of q
    {
      const uint8_t* qp[2] = {q_sm + turn * L::kQBytes + g * L::kQRow, q_sm + turn * L::kQBytes + (g + 8) * L::kQRow};
      float up[2] = {1.f, 1.f};
      fac[0] = fac[1] = p.scale_log2;
      if (BF16) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float m = 0.f;
#pragma unroll
          for (int h = 0; h < 2 * L::kKC; h++) {
            const uint4 v = *(const uint4*)(qp[i] + (t + 4 * (h >> 1)) * 32 + (h & 1) * 16);
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
          for (int e = 0; e < 2; e++) v[i][e] = *(const uint4*)(qp[i] + (t + 4 * h) * 32 + e * 16);
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
    Seg next = cur;
    bool more = f_next < f_end;
    if (more) {
      next = segment_at(f_next);
      more = next.g0 < next.g1;
      if (more) load_q(next, turn ^ 1);      // joins the next group that is committed
    }

    // ---- the subtiles ----
    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    // references and sums of rows g, g + 8; gain = 2^(m - M)
    float m[2] = {kNone, kNone}, M[2] = {kNone, kNone}, gain[2] = {1.f, 1.f}, l[2] = {0.f, 0.f};
    int tok0 = s_first * 16, id_c = -1;
    float ks_c = 0.f, vs_c = 0.f;
#pragma unroll 1
    for (int i = 0; i < count; i += 2, tok0 += kDecGran, src = src + 2 * L::kStage == ring_p + L::kWarpBytes ? ring_p : src + 2 * L::kStage) {
      const uint8_t *src_k = src + lane * 16, *src_v = src + 2 * L::kKC * 512 + lane * L::kVB;
      issue_pair(i + 2 * (L::kPairs - 1));
      cp_async_wait<L::kPairs - 1>();
      if ((i & 31) == 0) { id_c = id_i; ks_c = ks_i; vs_c = vs_i; }   // issue() is in the same 32
      float s[2][2][4];          // of subtile u, token octet j
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int j = 0; j < 2; j++) s[u][j][0] = s[u][j][1] = s[u][j][2] = s[u][j][3] = 0.f;
#pragma unroll
      for (int h = 0; h < L::kKC; h++) {
        uint4 kw[2][2];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int j = 0; j < 2; j++) kw[u][j] = *(const uint4*)(src_k + u * L::kStage + (j * L::kKC + h) * 512);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t qa[4];
          if (D == 256) {
            const uint4 qv = qsm[h * 4 + e][lane];
            qa[0] = qv.x; qa[1] = qv.y; qa[2] = qv.z; qa[3] = qv.w;
          } else {
#pragma unroll
            for (int x = 0; x < 4; x++) qa[x] = qf[D == 256 ? 0 : h * 4 + e][x];
          }
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
              uint32_t b0, b1;
              e4m3x4_to_half2x2(((const uint32_t*)&kw[u][j])[e], b0, b1);
              mma16816(s[u][j], qa, b0, b1);
            }
        }
      }
      float k[2][2], vs[2], lv[2], top[2] = {-INFINITY, -INFINITY}, top_v[2] = {-INFINITY, -INFINITY};
      bool edge[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int id = __shfl_sync(~0u, id_c, (i & 31) + u);
        const float ks = __shfl_sync(~0u, ks_c, (i & 31) + u);
        vs[u] = __shfl_sync(~0u, vs_c, (i & 31) + u);
        lv[u] = __log2f(vs[u]);
        const int at = tok0 + 16 * u;
        edge[u] = id < 0 || at < all_lo || at + 16 > all_hi;   // some row does not see some token
#pragma unroll
        for (int r2 = 0; r2 < 2; r2++) {
          k[u][r2] = fmaxf(ks * fac[r2], 1e-38f);   // above 0: masked scores stay -inf
          if (edge[u]) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const int tok = at + 8 * j + 2 * t + e;
                if (id < 0 || tok < first[r2] || tok > last[r2]) s[u][j][2 * r2 + e] = -INFINITY;
              }
          }
          const float x = fmaxf(fmaxf(s[u][0][2 * r2], s[u][0][2 * r2 + 1]), fmaxf(s[u][1][2 * r2], s[u][1][2 * r2 + 1])) * k[u][r2];
          top[r2] = fmaxf(top[r2], x);
          top_v[r2] = fmaxf(top_v[r2], x + lv[u]);
        }
      }
      if (twin) {                // one reference for both
        top[1] = top[0];
        top_v[1] = top_v[0];
      }
      const bool grew = top[0] > m[0] + kSlack || top[1] > m[1] + kSlack ||
                        top_v[0] > M[0] + (kSlack + kLift) || top_v[1] > M[1] + (kSlack + kLift);
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int r2 = 0; r2 < 2; r2++) {
          float x = top[r2], y = top_v[r2];
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 2));
          y = fmaxf(y, __shfl_xor_sync(~0u, y, 1));
          y = fmaxf(y, __shfl_xor_sync(~0u, y, 2));
          const float mn = fmaxf(m[r2], x), Mn = lifted(M[r2], y, mn);
          l[r2] *= ex2(m[r2] - mn);
          const float corr = ex2(M[r2] - Mn);
          m[r2] = mn;
          M[r2] = Mn;
          gain[r2] = ex2(mn - Mn);
#pragma unroll
          for (int j = 0; j < D / 8; j++) {
            o[j][2 * r2] *= corr;
            o[j][2 * r2 + 1] *= corr;
          }
        }
      }
      uint32_t pa[2][4];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const auto weights = [&](int r2, int j) {
          const float x0 = ex2(fmaf(s[u][j][2 * r2], k[u][r2], -m[r2]));
          const float x1 = ex2(fmaf(s[u][j][2 * r2 + 1], k[u][r2], -m[r2]));
          l[r2] += x0 + x1;
          const float f_v = weight_factor(vs[u], gain[r2]);
          return make_float2(x0 * f_v, x1 * f_v);
        };
        if (twin) {
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const float2 x = weights(0, j);
            pa[u][2 * j] = pack_half2(x.x, x.y);
            const float2 is = pair_to_float2<false>(pa[u][2 * j]);
            pa[u][2 * j + 1] = pack_half2(x.x - is.x, x.y - is.y);
          }
        } else {
#pragma unroll
          for (int r2 = 0; r2 < 2; r2++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const float2 x = weights(r2, j);
              pa[u][2 * j + r2] = pack_half2(x.x, x.y);
            }
        }
      }
#pragma unroll
      for (int h = 0; h < L::kVC; h++) {
        uint32_t v[2][4][L::kVB / 4];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint8_t* at = src_v + u * L::kStage + (j * L::kVC + h) * (32 * L::kVB);
            if (L::kVB == 16) {
              const uint4 x = *(const uint4*)at;
              v[u][j][0] = x.x; v[u][j][1] = x.y; v[u][j][L::kVB / 4 - 2] = x.z; v[u][j][L::kVB / 4 - 1] = x.w;
            } else {
              const uint2 x = *(const uint2*)at;
              v[u][j][0] = x.x; v[u][j][1] = x.y;
            }
          }
        // 0 * NaN: a NaN code that only some rows of the tile see must not reach the others, so
        // each row then goes through the MMA by itself, without the tokens that it does not see
        bool nan = false;
        if (edge[0] || edge[1]) {
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int w = 0; w < L::kVB / 4; w++) nan |= (((v[u][j][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
          nan = __any_sync(~0u, nan);
        }
        if (!nan) {
          pv_mma<L::kVB / 4>(o + h * 16, pa, v);
        } else {
#pragma unroll 1
          for (int r16 = 0; r16 < 16; r16++) {
            const int src_lane = (r16 & 7) * 4;
            const int f0 = __shfl_sync(~0u, first[0], src_lane), f1 = __shfl_sync(~0u, first[1], src_lane);
            const int l0 = __shfl_sync(~0u, last[0], src_lane), l1 = __shfl_sync(~0u, last[1], src_lane);
            uint32_t seen[2][4][L::kVB / 4];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const int tok = tok0 + 16 * u + 2 * t + (j & 1) + 8 * (j >> 1);
                const bool see = tok >= (r16 < 8 ? f0 : f1) && tok <= (r16 < 8 ? l0 : l1);
#pragma unroll
                for (int w = 0; w < L::kVB / 4; w++) seen[u][j][w] = see ? v[u][j][w] : 0;
              }
            float one[L::kVB][4];
#pragma unroll
            for (int j = 0; j < L::kVB; j++) one[j][0] = one[j][1] = one[j][2] = one[j][3] = 0.f;
            pv_mma<L::kVB / 4>(one, pa, seen);
#pragma unroll
            for (int j = 0; j < L::kVB; j++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (g == (r16 & 7) && (e >> 1) == (r16 >> 3)) o[h * 16 + j][e] += one[j][e];
          }
        }
      }
    }

    if (twin) {
#pragma unroll
      for (int j = 0; j < D / 8; j++) {
        o[j][0] += o[j][2];
        o[j][1] += o[j][3];
      }
    }

    // ---- the next segment's first stages ----
    cp_async_commit();
    cp_async_wait<0>();            // the next q too
    if (more) {
      open(next);
      fill = ring;
      src = ring_p;
      prologue();
    }

    // ---- the warps' states meet: o relative to the common m ----
    // kMeet warps at a time leave their rows in shared memory or add them to what is there.
#pragma unroll
    for (int i = 0; i < 2; i++) {
      l[i] += __shfl_xor_sync(~0u, l[i], 1);
      l[i] += __shfl_xor_sync(~0u, l[i], 2);
      if (m[i] == kNone) m[i] = -INFINITY;
      if (t == 0) { wm[warp][g + 8 * i] = m[i]; wl[warp][g + 8 * i] = l[i]; }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float top = wm[0][g + 8 * i], sum = 0.f;
#pragma unroll
      for (int w = 1; w < kDecWarps; w++) top = fmaxf(top, wm[w][g + 8 * i]);
#pragma unroll
      for (int w = 0; w < kDecWarps; w++)
        sum = fmaf(wl[w][g + 8 * i], wm[w][g + 8 * i] == -INFINITY ? 0.f : ex2(wm[w][g + 8 * i] - top), sum);
      if (warp == 0 && t == 0) { row_m[g + 8 * i] = top; row_l[g + 8 * i] = sum; }
      const float k = m[i] == -INFINITY ? 0.f : ex2(M[i] - top);
#pragma unroll
      for (int j = 0; j < D / 8; j++) {
        o[j][2 * i] *= k;
        o[j][2 * i + 1] *= k;
      }
    }
    float* mine = meet + warp % L::kMeet * (16 * L::kRow) + g * L::kRow + 2 * t * L::kCol;
#pragma unroll
    for (int round = 0; round < kDecWarps / L::kMeet; round++) {
      if (warp / L::kMeet == round) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int j = 0; j < D / 8; j++) {
            float *p0 = mine + 8 * i * L::kRow + j, *p1 = p0 + L::kCol;
            *p0 = (round ? *p0 : 0.f) + o[j][2 * i];
            *p1 = (round ? *p1 : 0.f) + o[j][2 * i + 1];
          }
      }
      __syncthreads();
    }
    // From here on thread `tid` holds the quads tid, tid + 128, ... of the rows x D outputs: quad
    // e is row e / (D / 4), MMA column (e / (D / 32)) % 8, four of its D / 8 channels.
    constexpr int kQuads = D / 32;
    const int quads = cur.row_n * (D / 4);
    float4 acc[kQuads];
    float row_top[kQuads], row_sum[kQuads];     // m and l of the quads' rows
#pragma unroll
    for (int x = 0; x < kQuads; x++) {
      const int e = tid + x * 32 * kDecWarps;
      const float* p4 = meet + e / (D / 4) * L::kRow + e / kQuads % 8 * L::kCol + e % kQuads * 4;
      acc[x] = make_float4(p4[0], p4[1], p4[2], p4[3]);
      if (L::kMeet == 2) {
        const float* p5 = p4 + 16 * L::kRow;
        acc[x] = make_float4(acc[x].x + p5[0], acc[x].y + p5[1], acc[x].z + p5[2], acc[x].w + p5[3]);
      }
      row_top[x] = row_m[e / (D / 4)];
      row_sum[x] = row_l[e / (D / 4)];
    }
    // ---- a whole item is written out; a part goes to the workspace ----
    // Parts join in two steps, groups of 8 (16 from 129 parts on) first, so that no CTA has many to
    // read; the last to arrive does it, in the order of the parts.
    bool write = true;
    if (cur.g0 > 0 || cur.g1 < cur.n) {
      const long long f0 = f + cur.cost - cur.g1;       // the item's first granule
      const int ca = (int)(f0 / per), cb = (int)((f0 + cur.n - 1) / per);   // the CTAs of this item
      const int parts = cb - ca + 1;
      const int size = parts <= 16 * kAtOnce ? kAtOnce : 2 * kAtOnce;
      const int me = (int)blockIdx.x - ca, head_g = me - me % size, count_g = min(size, parts - head_g);
      // counters and parts of CTA b: 1 where an item begins that goes on, 0 where one continues
      const auto at_of = [&](int i) { return (ca + i) * 2 + (i == 0 ? 1 : 0); };
      int* counters = (int*)a.ws;
      const auto part_of = [&](int i) {
        return (float*)((uint8_t*)a.ws + kDecCtas * 3 * sizeof(int)) + (long long)at_of(i) * (16 * D + 32);
      };
      const auto put = [&](float* slot) {
#pragma unroll
        for (int x = 0; x < kQuads; x++) {
          const int e = tid + x * 32 * kDecWarps;
          if (e < quads) {
            __stcg((float4*)slot + e, acc[x]);
            if (e % (D / 4) == 0) __stcg((float2*)(slot + 16 * D) + e / (D / 4), make_float2(row_top[x], row_sum[x]));
          }
        }
      };
      const auto last_of = [&](int* counter, int n_parts) {
        __syncthreads();                                  // every thread's part is written
        if (tid == 0) {
          __threadfence();
          arrived = atomicAdd(counter, 1);
          if (arrived == n_parts - 1) *counter = 0;      // as the next call expects it
          __threadfence();
        }
        __syncthreads();
        return arrived == n_parts - 1;
      };
      const auto join = [&](int from, int step, int n_parts) {   // parts from, from + step, ...
#pragma unroll
        for (int x0 = 0; x0 < kQuads; x0 += 2) {        // two quads of up to kAtOnce parts in flight
          if (tid + x0 * 32 * kDecWarps >= quads) break;
          float4 sum4[2] = {};
          float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll 1
          for (int i0 = 0; i0 < n_parts; i0 += kAtOnce) {
            float4 v[kAtOnce][2];
            float2 ml[kAtOnce][2];
#pragma unroll
            for (int i = 0; i < kAtOnce; i++)
#pragma unroll
              for (int x = 0; x < 2; x++) {
                const int e = min(tid + (x0 + x) * 32 * kDecWarps, quads - 1);
                const float* s = part_of(from + min(i0 + i, n_parts - 1) * step);
                v[i][x] = __ldcg((const float4*)s + e);
                ml[i][x] = __ldcg((const float2*)(s + 16 * D) + e / (D / 4));
              }
#pragma unroll
            for (int x = 0; x < 2; x++) {
              float mn = top[x];
#pragma unroll
              for (int i = 0; i < kAtOnce; i++) {
                if (i0 + i >= n_parts) ml[i][x] = make_float2(-INFINITY, 0.f);
                mn = fmaxf(mn, ml[i][x].x);
              }
              const float k0 = top[x] == -INFINITY ? 0.f : ex2(top[x] - mn);
              top[x] = mn;
              sum[x] *= k0;
              sum4[x].x *= k0;
              sum4[x].y *= k0;
              sum4[x].z *= k0;
              sum4[x].w *= k0;
#pragma unroll
              for (int i = 0; i < kAtOnce; i++) {
                if (i0 + i >= n_parts) break;
                const float k = ml[i][x].x == -INFINITY ? 0.f : ex2(ml[i][x].x - mn);
                sum[x] = fmaf(k, ml[i][x].y, sum[x]);
                sum4[x].x = fmaf(k, v[i][x].x, sum4[x].x);
                sum4[x].y = fmaf(k, v[i][x].y, sum4[x].y);
                sum4[x].z = fmaf(k, v[i][x].z, sum4[x].z);
                sum4[x].w = fmaf(k, v[i][x].w, sum4[x].w);
              }
            }
          }
#pragma unroll
          for (int x = 0; x < 2; x++) {
            acc[x0 + x] = sum4[x];
            row_top[x0 + x] = top[x];
            row_sum[x0 + x] = sum[x];
          }
        }
      };
      put(part_of(me));
      write = last_of(counters + at_of(head_g), count_g);
      if (write) {
        join(head_g, 1, count_g);
        if (parts > size) {
          __syncthreads();       // all of the group's parts are read: its sum takes the first one's place
          put(part_of(head_g));
          const int groups = (parts + size - 1) / size;
          write = last_of(counters + 2 * kDecCtas + ca, groups);
          if (write) join(0, size, groups);
        }
      }
    }
    if (write) {
#pragma unroll
      for (int x = 0; x < kQuads; x++) {
        const int e = tid + x * 32 * kDecWarps;
        if (e >= quads) break;
        const int row = e / (D / 4), col = e / kQuads % 8, j = e % kQuads * 4;
        const int rr = cur.tile * 16 + row, tok = rr / G, head = cur.kh * G + rr - tok * G;
        const float inv = row_sum[x] > 0.f ? 1.f / row_sum[x] : 0.f;
        uint16_t* op = (uint16_t*)a.out + (long long)(cur.q0 + tok) * a.out_row + (long long)head * D;
        *(uint2*)(op + (j / L::kVB) * 128 + col * L::kVB + j % L::kVB) =
            make_uint2(float2_to_pair<BF16>(acc[x].x * inv, acc[x].y * inv),
                       float2_to_pair<BF16>(acc[x].z * inv, acc[x].w * inv));
        if (a.lse && e % (D / 4) == 0)
          a.lse[(long long)(cur.q0 + tok) * a.heads + head] =
              row_sum[x] == 0.f ? -INFINITY : (row_top[x] + log2f(row_sum[x])) * 0.6931471805599453f;
      }
    }
    if (!more) break;
    f = f_next;
    cur = next;
    __syncthreads();      // the next q is there; the small arrays are used again
  }
}

#include "attn8_prompt.cuh"

}  // namespace yk

using namespace yk;

extern "C" int yk_test_attn_kv8(int kernel) {
  if (kernel < 0 || kernel > 2) return refuse(YK_EINVAL, "test_attn_kv8: 0, 1 or 2");
  g_attn_kernel = kernel;
  return YK_OK;
}

extern "C" size_t yk_attn_kv8_workspace_bytes(int requests, int rows, int heads, int kv_heads, int dim) {
  // three counters and two parts (o, m, l of 16 rows) for each CTA, whatever the lengths
  (void)requests; (void)rows; (void)heads; (void)kv_heads;
  return kDecCtas * (3 * sizeof(int) + 2 * (16 * (size_t)std::max(dim, 0) + 32) * sizeof(float));
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
  if ((long long)a->rows * a->heads > 0x7fffffffll) return refuse(YK_EUNSUP, "attn_kv8: rows * heads must be below 2^31");
  if (a->window && !a->causal) return refuse(YK_EINVAL, "attn_kv8: a window needs causal");
  if (a->rows == 0) return YK_OK;
  if (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out) || a->q_row % 8 || a->out_row % 8 ||
      a->out_row < (long long)a->heads * c->dim || a->q_row < 0)
    return refuse(YK_EINVAL, "attn_kv8: q and out need 16-byte alignment and row strides that are multiples of 8");
  if (!aligned16(a->ws) || a->ws_bytes < yk_attn_kv8_workspace_bytes(a->requests, a->rows, a->heads, c->heads, c->dim))
    return refuse(YK_EINVAL, "attn_kv8: workspace too small or not 16-byte aligned");
  Attn8Args p{*c, *a, 0.f, kDecLead, kDecMin};
  if (p.a.scale == 0.f) p.a.scale = 1.f / sqrtf((float)c->dim);
  p.scale_log2 = p.a.scale * 1.4426950408889634f;
  const bool bf = a->dtype == YK_BF16;
  cudaStream_t s = (cudaStream_t)st;
  const long long G = a->heads / c->heads, tiles16 = (long long)a->rows * a->heads / 16;
  const long long ctas = (a->rows * G / 128 + a->requests) * c->heads, slots = c->dim == 256 ? 148 : 296;
  const int least = c->dim == 256 ? kProTiles<256> : kProTiles<128>, force = g_attn_kernel.load();
  if (force ? force == 2
            : a->rows >= (long long)kProTokens * a->requests && tiles16 * slots >= least * std::max(slots, ctas)) {
    switch (c->dim) {
      case 64: return bf ? launch_attn8_prompt<true, 64>(p, s) : launch_attn8_prompt<false, 64>(p, s);
      case 128: return bf ? launch_attn8_prompt<true, 128>(p, s) : launch_attn8_prompt<false, 128>(p, s);
      default: return bf ? launch_attn8_prompt<true, 256>(p, s) : launch_attn8_prompt<false, 256>(p, s);
    }
  }
  switch (c->dim) {
    case 64: return bf ? launch_attn8_split<true, 64>(p, s) : launch_attn8_split<false, 64>(p, s);
    case 128: return bf ? launch_attn8_split<true, 128>(p, s) : launch_attn8_split<false, 128>(p, s);
    default: return bf ? launch_attn8_split<true, 256>(p, s) : launch_attn8_split<false, 256>(p, s);
  }
}
