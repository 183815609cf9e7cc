// Attention over the paged 8-bit cache, many rows: the rows of a request that share a key head
// fill 128-row tiles of tcgen05 MMAs (included by attn8.cu).
//
// Tensor and exponential bound.  One CTA a (128-row tile, key head); per 64 keys S = Q K^T (fp32 in
// TMEM), softmax, O += P V (O in TMEM, fp16 operands).  Roles:
//  * warps 0-3, softmax: a thread owns a row (a TMEM lane), so maxima and sums need no shuffles.
//    Weights are taken relative to a reference that follows the row's maximum only when that passes
//    it by 2^6, so a tile is read once: if its maximum stays below, the weights stand; else (seldom)
//    the reference moves, O is rescaled, and the tile is done again.  P goes as fp16 over the columns of
//    its S: it is the A operand straight from TMEM.  (One rounding: fp16 outputs 1.39 - 1.42 times as far from 64 bits as
//    their own rounding alone; a second part would double the PV products and half of the weights' work again.)
//  * warps 4-7 read the codes of the next tile into registers while this one's are in use, convert them
//    (exactly) to fp16 and write them into 128-byte-swizzled tiles [slab of 64 channels][token][64], which
//    the MMA reads as a K-major operand for the keys and as an MN-major one for the values.
//  * one thread of warp 8 issues the MMAs.  Everything comes twice (S and P, keys, values), so QK of
//    tile j + 1 is done before the softmax of tile j is, and PV of tile j runs beside the softmax of
//    tile j + 1.
// Two CTAs an SM up to 128 channels.
// Measured: 8 ragged requests, 5616 rows of 16 heads over up to 3832 keys (67.6 GFLOP) 139 us, 0.49 PFLOP/s, 29 %
// of the measured burst rate (the warp-MMA tiles of the split kernel: 650 us).  A CTA spends about 2800
// cycles a tile: 1200 in the weights (64 exponentials a row, shared with the other CTA), the rest in
// waits for S and in the chain P -> PV -> QK; longest tiles first leave an SM within 10 % of the mean.
constexpr int kProThreads = 288;
constexpr int kProSort = 128;          // requests up to which tiles are ordered by their length

template <int D>
struct Pro {
  static constexpr int kTile = 64 * D * 2;              // fp16 bytes of 64 keys
  static constexpr int kSmem = 6 * kTile + 1024;        // q (128 rows), two of keys, two of values; alignment
  static constexpr int kCols = D == 256 ? 512 : 256;    // TMEM columns: S twice 64, O D
  static constexpr int kK = 2 * (D / 64);               // 16-byte code chunks of a converting thread
};

// D[tmem] (+)= A[tmem] * B[smem desc]^T, fp16 inputs, fp32 accumulate.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t dtmem, uint32_t atmem, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(dtmem),
      "r"(atmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Shared-memory descriptor of an MN-major operand in the 128-byte swizzle layout: slabs of 64 elements
// (128-byte rows, one for each k) `slab` bytes apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t slab) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(slab >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint32_t kBMnMajor = 1u << 16;       // instruction descriptor: B is MN-major
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
      "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// 16-byte chunk `ch` (of 64 columns: 8 a row) of row `row` of a swizzled slab of 128-byte rows
__device__ __forceinline__ uint32_t swz_at(int row, int ch) { return row * 128 + ((ch ^ (row & 7)) << 4); }

template <bool BF16, int D>
__global__ void __launch_bounds__(kProThreads, D == 256 ? 1 : 2) attn8_prompt_kernel(const __grid_constant__ Attn8Args p) {
  using L = Pro<D>;
  extern __shared__ uint8_t pro_raw[];
  __shared__ __align__(8) uint64_t bars[10];
  __shared__ uint32_t tslot;
  __shared__ int found_r, found_tile;
  __shared__ int nan_lo, nan_hi;                  // tiles of keys where a NaN value was taken out
  // scales of the 16-token groups of tile j at j % 4, with the logarithm of the value scale; ks < 0: not there
  __shared__ __align__(16) float ks_sm[4][4], vs_sm[4][4], lv_sm[4][4];
  const YkAttnKv8& a = p.a;
  const YkKvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.heads / c.heads, T = c.tokens;
  pdl_wait();
  pdl_trigger();

  const int kh = blockIdx.x % c.heads, index = blockIdx.x / c.heads;
  int r = 0;
  long long tile = -1;
  if (a.requests <= kProSort && warp == 0) {
    // Tiles in descending order of the keys they see, in tiles of 64 (then of request and tile), so
    // that the longest start first.  A request's tiles see more and more: those of length >= n start
    // at tile `from`.  One warp finds tile `index`, its lanes sharing the requests out.
    const auto all_tiles = [&](const Req& q) { return (int)(((long long)q.q * G + 127) / 128); };
    const auto from = [&](const Req& q, int n) {
      const long long key = (n - 1) * 64ll;                    // the first key past n - 1 tiles is seen
      if (n <= 0) return 0;
      if (!a.causal) return q.kv > key ? 0 : all_tiles(q);
      const long long t = key - q.kv + q.q;                    // from this token on
      return t >= q.q ? all_tiles(q) : t <= 0 ? 0 : (int)(t * G / 128);
    };
    const auto longer = [&](int n) {                           // tiles of length >= n, over all requests
      int sum = 0;
      for (int i = lane; i < a.requests; i += 32) {
        const Req q = attn_req(c, a, i);
        sum += all_tiles(q) - from(q, n);
      }
      return (int)__reduce_add_sync(~0u, (unsigned)sum);
    };
    int n = 0, most = 0;
    for (int i = lane; i < a.requests; i += 32) most = max(most, attn_req(c, a, i).kv);
    for (int hi = __reduce_max_sync(~0u, most) / 64 + 2; hi - n > 1;) {     // longer(n) > index >= longer(hi)
      const int m = (n + hi) >> 1;
      if (longer(m) > index) n = m; else hi = m;
    }
    int rank = index - longer(n + 1);                          // among the tiles of length n
    const int end = index < longer(0) ? a.requests : 0;
    for (int i0 = 0; i0 < end && tile < 0; i0 += 32) {
      int mine = 0, first = 0;
      if (i0 + lane < a.requests) {
        const Req q = attn_req(c, a, i0 + lane);
        first = from(q, n);
        mine = from(q, n + 1) - first;
      }
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned past = __ballot_sync(~0u, upto > rank);
      if (past) {
        const int l = __ffs(past) - 1;
        r = i0 + l;
        tile = __shfl_sync(~0u, first + rank - (upto - mine), l);
      }
      rank -= __shfl_sync(~0u, upto, 31);
    }
    if (lane == 0) {
      found_r = r;
      found_tile = (int)tile;
    }
  }
  if (a.requests <= kProSort) {
    __syncthreads();
    r = found_r;
    tile = found_tile;
  } else {
    // Request r owns the tile numbers from rows_before * G / 128 + r on: at least as many as it has
    // tiles.  High numbers go first.
    const long long number = gridDim.x / c.heads - 1 - index;
    const auto first_number = [&](int r) { return (long long)min(max(a.cu[r], 0), a.rows) * G / 128 + r; };
    for (int hi = a.requests; hi - r > 1;) {
      const int m = (r + hi) >> 1;
      if (first_number(m) <= number) r = m; else hi = m;
    }
    tile = number - first_number(r);
  }
  if (tile < 0) return;
  const Req rq = attn_req(c, a, r);
  if (tile * 128 >= (long long)rq.q * G) return;
  const int row0 = (int)tile * 128, row_n = min(128, rq.q * G - row0);
  const int t0 = row0 / G, t1 = (row0 + row_n - 1) / G;              // the tile's tokens
  const int hi_key = a.causal ? max(0, rq.kv - rq.q + t1 + 1) : rq.kv;   // keys that some row sees: [lo_key, hi_key)
  const int lo_key = a.causal ? first_key(rq.kv - rq.q + t0, a.window) : 0;
  const int all_hi = a.causal ? rq.kv - rq.q + t0 + 1 : rq.kv;          // that every row sees: [all_lo, all_hi)
  const int all_lo = a.causal ? first_key(rq.kv - rq.q + t1, a.window) : 0;
  const int j0 = lo_key / 64, j1 = (hi_key + 63) / 64;                // tiles of 64 keys

  // this thread's row (softmax warps; rows past row_n follow the last one and are not written)
  const int rr = row0 + min(tid & 127, row_n - 1), tok = rr / G, head = kh * G + rr - tok * G;
  const long long out_row = rq.q0 + tok;
  if (j1 <= j0) {                       // no keys at all
    if (tid < row_n) {
      for (int d = 0; d < D; d += 8) *(uint4*)((uint16_t*)a.out + out_row * a.out_row + (long long)head * D + d) = make_uint4(0, 0, 0, 0);
      if (a.lse) a.lse[out_row * a.heads + head] = -INFINITY;
    }
    return;
  }

  const uint32_t base = (smem_u32(pro_raw) + 1023) & ~1023u;
  const uint32_t q_sm = base, k_sm = base + 2 * L::kTile, v_sm = base + 4 * L::kTile;
  // two of each, for even and odd tiles
  const uint32_t k_full = smem_u32(&bars[0]), v_full = smem_u32(&bars[2]), s_full = smem_u32(&bars[4]),
                 p_full = smem_u32(&bars[6]), o_done = smem_u32(&bars[8]);
  if (tid == 0) {
    for (int i = 0; i < 16; i += 8) {
      mbar_init(k_full + i, 128);
      mbar_init(v_full + i, 128);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
      mbar_init(o_done + i, 1);
    }
    mbar_fence_init();
    nan_lo = 0x7fffffff;
    nan_hi = -1;
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&tslot), L::kCols);
    tmem_relinquish();
  }
  // q: a thread its row, bf16 scaled by a power of two to fp16
  float fac = p.scale_log2;             // score factor of the row: scale * log2 e * the power of two taken out of q
  if (warp < 4) {
    const uint4* qp = (const uint4*)((const uint16_t*)a.q + out_row * a.q_row + (long long)head * D);
    float up = 1.f;
    if (BF16) {
      uint32_t m2 = 0;
#pragma unroll 4
      for (int i = 0; i < D / 8; i++) {
        const uint4 v = qp[i];
        m2 = amax_pair<true>(amax_pair<true>(m2, v.x), v.y);
        m2 = amax_pair<true>(amax_pair<true>(m2, v.z), v.w);
      }
      const float2 f = pair_to_float2<true>(m2);
      const float m = fmaxf(f.x, f.y);
      int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;   // m in [2^e, 2^(e+1))
      e = m > 0.f ? max(-110, min(e, 120)) : 13;
      up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);     // the largest becomes 2^13 .. 2^14
      fac = p.scale_log2 * __uint_as_float((uint32_t)(127 - 13 + e) << 23);
    }
#pragma unroll 4
    for (int i = 0; i < D / 8; i++) {
      uint4 v = qp[i];
      if (BF16) {
        uint32_t* u = (uint32_t*)&v;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 x = pair_to_float2<true>(u[e]);
          u[e] = pack_half2(x.x * up, x.y * up);
        }
      }
      sts128(q_sm + (i >> 3) * 16384 + swz_at(tid, i & 7), v.x, v.y, v.z, v.w);
    }
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot, s_tm = tmem, o_tm = tmem + 128;
  const int tiles = j1 - j0;

  if (warp < 4) {
    // ---------------- softmax ----------------
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int pos = rq.kv - rq.q + tok;
    const int last = a.causal ? min(rq.kv - 1, pos) : rq.kv - 1, first = a.causal ? first_key(pos, a.window) : 0;
    float m = kNone, M = kNone, gain = 1.f, l = 0.f;
    bool ok = true;
    for (int j = 0; j < tiles; j++) {
      const int buf = j & 1, turn = (j >> 1) & 1;
      const uint32_t s_at = s_tm + lanes + buf * 64;
      if (!mbar_wait(s_full + buf * 8, turn, 0x503)) { ok = false; break; }
      tc_fence_after();
      const int key0 = (j0 + j) * 64;
      __align__(16) float kk[4], vs[4], lv[4];
      bool gone = false;
      *(float4*)kk = *(const float4*)ks_sm[j & 3];
      *(float4*)vs = *(const float4*)vs_sm[j & 3];
      *(float4*)lv = *(const float4*)lv_sm[j & 3];
#pragma unroll
      for (int g = 0; g < 4; g++) {
        gone |= kk[g] < 0.f;
        kk[g] = fmaxf(kk[g] * fac, 1e-38f);      // above 0: masked scores stay -inf
      }
      const bool edge = gone || key0 < all_lo || key0 + 64 > all_hi;
      const int c_lo = first - key0, c_hi = last - key0;       // columns that this row sees
      const auto load_s = [&](uint32_t (&s)[32], int c0) {
        tmem_ld16p(s_at + c0, s);
        tmem_ld16p(s_at + c0 + 16, s + 16);
        tmem_ld_wait();
        if (edge) {
#pragma unroll
          for (int i = 0; i < 32; i++)
            if (c0 + i < c_lo || c0 + i > c_hi) s[i] = 0xff800000u;
          if (gone) {
#pragma unroll
            for (int g = 0; g < 2; g++)
              if (ks_sm[j & 3][c0 / 16 + g] < 0.f) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[16 * g + i] = 0xff800000u;
              }
          }
        }
      };
      uint32_t w[32];
      float2 sum;
      bool move = j == 0;
      while (true) {
        if (move) {              // the reference moves up to this tile's maximum
          float top = -INFINITY, top_v = -INFINITY;
#pragma unroll 1
          for (int c0 = 0; c0 < 64; c0 += 32) {
            uint32_t s[32];
            load_s(s, c0);
#pragma unroll
            for (int g = 0; g < 2; g++) {
              float x = __uint_as_float(s[16 * g]);
#pragma unroll
              for (int i = 1; i < 16; i++) x = fmaxf(x, __uint_as_float(s[16 * g + i]));
              x *= c0 ? kk[2 + g] : kk[g];
              top = fmaxf(top, x);
              top_v = fmaxf(top_v, x + (c0 ? lv[2 + g] : lv[g]));
            }
          }
          const float mn = fmaxf(m, top), Mn = lifted(M, top_v, mn);
          l *= ex2(m - mn);
          const float corr = ex2(M - Mn);
          m = mn;
          M = Mn;
          gain = ex2(mn - Mn);
          if (j > 0) {
            if (!mbar_wait(o_done + (buf ^ 1) * 8, ((j - 1) >> 1) & 1, 0x509)) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 16) {
              uint32_t o[16];
              tmem_ld16p(o_tm + lanes + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st16(o_tm + lanes + c0, o);
            }
            tmem_st_wait();
          }
        }
        sum = make_float2(0.f, 0.f);
        float over = -INFINITY;          // how far the tile passes the references
        const float2 neg = make_float2(-m, -m);
        const float to_v = m - M - kLift;
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          uint32_t s[32];
          load_s(s, c0);
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const float k = kk[c0 / 16 + g], f = weight_factor(vs[c0 / 16 + g], gain);
            float top = -INFINITY;
#pragma unroll
            for (int i = 8 * g; i < 8 * g + 8; i++) {
              float2 x = ffma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), make_float2(k, k), neg);
              top = fmaxf(top, fmaxf(x.x, x.y));
              x.x = ex2(x.x);
              x.y = ex2(x.y);
              sum = add2(sum, x);
              x = mul2(x, make_float2(f, f));
              w[c0 / 2 + i] = pack_half2(x.x, x.y);
            }
            over = fmaxf(over, fmaxf(top, top + (lv[c0 / 16 + g] + to_v)));
          }
        }
        if (move || !__any_sync(~0u, over > kSlack)) break;
        move = true;
      }
      if (!ok) break;
      l += sum.x + sum.y;
      tmem_st16(s_at, w);                // over columns that were read
      tmem_st16(s_at + 16, w + 16);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full + buf * 8);
    }
    if (ok && mbar_wait(o_done + ((tiles - 1) & 1) * 8, ((tiles - 1) >> 1) & 1, 0x505)) {
      tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : 0.f;
      // rows leave through shared memory (the key tiles, no longer in use) so that they are stored whole
      const uint32_t stage = k_sm + warp * (64 * D);
      // o is relative to M, l to m
      const float k = (m == kNone ? 0.f : ex2(M - m)) * inv;
      const int n_lo = nan_lo, n_hi = nan_hi;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t o[32];
        tmem_ld16p(o_tm + lanes + c0, o);
        tmem_ld16p(o_tm + lanes + c0 + 16, o + 16);
        tmem_ld_wait();
        if (n_hi >= 0) {
          // a NaN that was taken out of the edge tiles' values reaches the rows that see its token
          for (int key = max(first, n_lo * 64); key <= min(last, n_hi * 64 + 63); key++) {
            const int b = a.table[r * a.table_stride + key / T];
            if ((unsigned)b >= (unsigned)c.blocks) continue;
            const uint8_t* v = (const uint8_t*)c.v + b * c.block_stride + ((long long)kh * T + (key & (T - 1))) * D + c0;
#pragma unroll
            for (int i = 0; i < 32; i++)
              if ((v[i] & 0x7f) == 0x7f) o[i] = 0x7fffffffu;
          }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; e++)
            u[e] = float2_to_pair<BF16>(__uint_as_float(o[i + 2 * e]) * k, __uint_as_float(o[i + 2 * e + 1]) * k);
          const int ch = (c0 + i) / 8;
          sts128(stage + lane * (2 * D) + ((ch ^ (lane & 7)) << 4), u[0], u[1], u[2], u[3]);
        }
      }
      __syncwarp();
      constexpr int kChunks = D / 8, kRows = 32 / kChunks > 1 ? 32 / kChunks : 1;   // 16-byte chunks of a row; rows an instruction stores
      const long long mine = out_row * a.out_row + (long long)head * D;
#pragma unroll 4
      for (int i = 0; i < 32; i += kRows) {
        const int row = i + lane / kChunks % kRows, ch = lane % kChunks;
        const long long to = __shfl_sync(~0u, mine, row);
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(stage + row * (2 * D) + ((ch ^ (row & 7)) << 4)));
        if (warp * 32 + row < row_n) *(uint4*)((uint16_t*)a.out + to + ch * 8) = v;
      }
      if (a.lse && tid < row_n)
        a.lse[out_row * a.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
  } else if (warp < 8) {
    // ---------------- codes to fp16 tiles ----------------
    const int w = warp - 4;
    const int* table = a.table + r * a.table_stride;
    // table entry of 16-token group `lane` (< 4) of tile j, as it is; -1: none
    const auto entry = [&](int j) -> int {
      const int key = (j0 + j) * 64 + lane * 16;
      return lane < 4 && j < tiles && key < hi_key ? table[key / T] : -1;
    };
    const auto in_pool = [&](int b) { return (unsigned)b < (unsigned)c.blocks ? b : -1; };
    const int wrap = min(T, 64) - 1;      // tokens of a block that a tile's groups repeat after
    // warp w takes group w, 16 rows: lane row lane / 4 (and 8 more), 16 channels (lane % 4) of each slab
    const long long mine = ((long long)kh * T + ((w * 16 + lane / 4) & wrap)) * D + (lane & 3) * 16;
    uint4 kv[L::kK], vv[L::kK];
    const auto load = [&](uint4 (&x)[L::kK], const void* codes, int j, int ids) {
      const int id = __shfl_sync(~0u, ids, w), key0 = (j0 + j) * 64, left = id < 0 ? 0 : hi_key - key0 - w * 16;
      const uint8_t* at = (const uint8_t*)codes + mine + max(id, 0) * c.block_stride + (key0 & (T - 1)) * D;
#pragma unroll
      for (int i = 0; i < L::kK; i++) {
        const int slab = i % (D / 64), more = i / (D / 64) * 8;
        x[i] = make_uint4(0, 0, 0, 0);
        if (lane / 4 + more < left) x[i] = *(const uint4*)(at + more * D + slab * 64);
      }
    };
    // chunk pairs (lane % 4) * 2, + 1 of row lane / 4 of the group: the same place in the swizzle 8 rows on
    const uint32_t to0 = swz_at(w * 16 + lane / 4, (lane & 3) * 2), to1 = swz_at(w * 16 + lane / 4, (lane & 3) * 2 + 1);
    const auto store = [&](const uint4 (&x)[L::kK], uint32_t tile_at) {
#pragma unroll
      for (int i = 0; i < L::kK; i++) {
        const uint32_t at = tile_at + i % (D / 64) * 8192 + i / (D / 64) * 1024;
        uint32_t h[8];
        e4m3x4_to_half2x2(x[i].x, h[0], h[1]);
        e4m3x4_to_half2x2(x[i].y, h[2], h[3]);
        e4m3x4_to_half2x2(x[i].z, h[4], h[5]);
        e4m3x4_to_half2x2(x[i].w, h[6], h[7]);
        sts128(at + to0, h[0], h[1], h[2], h[3]);
        sts128(at + to1, h[4], h[5], h[6], h[7]);
      }
    };
    // 0 * NaN: a NaN value that some row does not see is taken out here, see the end
    const auto take_out = [&](int j) {
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < L::kK; i++) {
        uint32_t* v = (uint32_t*)&vv[i];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t nan = ((v[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          any |= nan;
          v[e] &= ~((nan >> 7) * 0xffu);
        }
      }
      if (any) {
        atomicMin(&nan_lo, j0 + j);
        atomicMax(&nan_hi, j0 + j);
      }
    };
    // kAhead tiles ahead the codes are called into L2, a line (128 bytes) a lane: half of the lanes
    // the keys, half the values of group w; its block id is read one tile before that
    constexpr int kAhead = 4, kLines = 16 * D / 128;
    const auto far_entry = [&](int j) -> int {
      const int key = (j0 + j) * 64 + w * 16;
      return j < tiles && key < hi_key ? table[key / T] : -1;
    };
    const auto call = [&](int j, int raw) {
      const int id = in_pool(raw), key0 = (j0 + j) * 64;
      const uint8_t* at = (const uint8_t*)(lane < 16 ? c.k : c.v) + id * c.block_stride +
                          ((long long)kh * T + ((key0 + w * 16) & (T - 1))) * D;
      if (id >= 0)
        for (int line = lane & 15; line < kLines; line += 16) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + line * 128));
    };
    int far = far_entry(1);
    for (int j = 1; j <= kAhead; j++) {
      call(j, far);
      far = far_entry(j + 1);
    }
    // one tile ahead: codes and scales; two tiles ahead: table entries
    int ids = in_pool(entry(0)), ahead = entry(1);
    const auto scale_of = [&](const float* scales, int id) { return scales[max(id, 0) * c.scale_stride + kh]; };
    load(kv, c.k, 0, ids);
    load(vv, c.v, 0, ids);
    float ks = scale_of(c.kscale, ids), vs = scale_of(c.vscale, ids);
    for (int j = 0; j < tiles; j++) {
      const int buf = j & 1, before = ((j >> 1) - 1) & 1;      // turn of tile j - 2 in the same buffers
      const int ids_next = in_pool(ahead);
      ahead = entry(j + 2);
      call(j + kAhead + 1, far);
      far = far_entry(j + kAhead + 2);
      if (j > 1 && !mbar_wait(s_full + buf * 8, before, 0x501)) break;   // QK j - 2 has read its keys
      store(kv, k_sm + buf * L::kTile);
      if (w == 0 && lane < 4) {
        ks_sm[j & 3][lane] = ids < 0 ? -1.f : ks;
        vs_sm[j & 3][lane] = ids < 0 ? 0.f : vs;
        lv_sm[j & 3][lane] = ids < 0 ? -INFINITY : __log2f(vs);
      }
      fence_proxy_async();
      mbar_arrive(k_full + buf * 8);
      load(kv, c.k, j + 1, ids_next);
      ks = scale_of(c.kscale, ids_next);
      vs = scale_of(c.vscale, ids_next);
      if (j > 1 && !mbar_wait(o_done + buf * 8, before, 0x502)) break;   // PV j - 2 its values
      const int key0 = (j0 + j) * 64;
      if (key0 < all_lo || key0 + 64 > all_hi) take_out(j);
      store(vv, v_sm + buf * L::kTile);
      fence_proxy_async();
      mbar_arrive(v_full + buf * 8);
      load(vv, c.v, j + 1, ids_next);
      ids = ids_next;
    }
  } else if (lane == 0) {
    // ---------------- MMA ----------------
    const uint64_t q_desc = sw128_desc(q_sm), k_desc = sw128_desc(k_sm), v_desc = sw128_mn_desc(v_sm, 8192);   // addresses count 16 bytes
    const auto qk = [&](int j) {
      const int buf = j & 1;
      if (!mbar_wait(k_full + buf * 8, (j >> 1) & 1, 0x504)) return false;
      tc_fence_after();
#pragma unroll
      for (int s = 0; s < D / 16; s++)
        tc_mma_f16(s_tm + buf * 64, q_desc + (s >> 2) * 1024 + (s & 3) * 2, k_desc + buf * (L::kTile / 16) + (s >> 2) * 512 + (s & 3) * 2,
                   idesc_f16_m128(64), s != 0);
      tc_commit(s_full + buf * 8);
      return true;
    };
    bool ok = qk(0) && (tiles < 2 || qk(1));
    for (int j = 0; j < tiles && ok; j++) {
      const int buf = j & 1, turn = (j >> 1) & 1;
      ok = mbar_wait(v_full + buf * 8, turn, 0x507) && mbar_wait(p_full + buf * 8, turn, 0x506);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int s = 0; s < 4; s++)
        tc_mma_f16_ts(o_tm, s_tm + buf * 64 + s * 8, v_desc + buf * (L::kTile / 16) + s * 128, idesc_f16_m128(D) | kBMnMajor, (j | s) != 0);
      tc_commit(o_done + buf * 8);
      // QK j + 2 takes the columns of P j: the order of MMAs with different accumulators is not promised
      if (j + 2 < tiles) ok = mbar_wait(o_done + buf * 8, turn, 0x508) && qk(j + 2);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }
}

template <bool BF16, int D>
static int launch_attn8_prompt(const Attn8Args& p, cudaStream_t st) {
  const auto kern = attn8_prompt_kernel<BF16, D>;
  if (smem_attr(kern, Pro<D>::kSmem) != cudaSuccess) return check_launch("attn_kv8 attr");
  const long long tiles = (long long)p.a.rows * (p.a.heads / p.c.heads) / 128 + p.a.requests;
  if (tiles * p.c.heads > 0x7fffffffll) return refuse(YK_EUNSUP, "attn_kv8: too many rows");
  launch_k(kern, (unsigned)(tiles * p.c.heads), kProThreads, Pro<D>::kSmem, st, p);
  note_launch();
  return check_launch("attn_kv8");
}
