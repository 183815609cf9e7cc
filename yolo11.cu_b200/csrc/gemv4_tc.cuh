// Products with a 4-bit weight matrix, many outputs or rows, on tcgen05 (included by gemv4.cu).
//
// The warp-MMA kernel spends most of its instructions around the products: x fragments, scales and zero
// points that every lane of a quad needs, sums of eight columns a lane.  Here a thread owns an output
// (a TMEM lane): it turns its row's codes into 16-bit integers in registers (about one instruction a
// code), stores them into TMEM as the A operand, and scales its own sums: one scale and zero point a
// group, no shuffles.  x is the B operand in shared memory, staged once for all 128 outputs.
//  * A chunk is 128 columns of 128 outputs; warps 0-3 take the first half of them, warps 4-7 the rest (a warp its
//    32 outputs' 64 bytes each, by cp.async), as two halves of 64 columns.
//    Half h goes to A buffer h % 2 and its sums (one accumulator for each group, or half a group) to D
//    buffer h % 2; a half's sums are read after the next half is stored, so the MMA runs behind.
//  * The next warps stage x: 8 columns in the order (0, 4, 1, 5, 2, 6, 3, 7) that the codes come out in.
//  * One thread of each of the last two warps issues one set's MMAs.
//  * Scales and zero points come 8 groups at a time where their rows allow it: a thread a row means a
//    line a lane, so each load costs the warp 32 lines.
// Measured: 16 e4m3 rows x 28672 outputs x 8192 columns, groups of 64 with zero points (129 MB) 81 us, 1.6 TB/s (warp
// MMAs: 102 us).  Two CTAs an SM take twice as long as one: an MMA of 16 columns of x ends only every 160
// cycles, whoever issues it; with the operand in shared memory instead the chain store -> MMA -> sums
// got longer (109 us).
template <int XT, int GB, int N>
struct GemvTc {
  static constexpr int kTeam = N / 16;                             // warps that stage a chunk of x together
  static constexpr int kTeams = N == 16 ? 4 : 2;                   // chunks in the making: a load's latency each
  static constexpr int kStageWarps = kTeam * kTeams;
  static constexpr int kThreads = (8 + kStageWarps + 2) * 32;
  static constexpr int kStages = 4, kXStages = 4;
  static constexpr int kUnits = GB == 1 ? 2 : 1;                   // accumulators of a half
  static constexpr int kD0 = 128;                                  // TMEM columns: A 2 x 2 x 32, then D 2 x 2 x kUnits x N
  static constexpr bool kOneD = 4 * kUnits * N > 384;              // (or 2 x kUnits x N: one D buffer each)
  static constexpr int kNeed = kD0 + (kOneD ? 2 : 4) * kUnits * N;
  static constexpr int kCols = kNeed <= 256 ? 256 : 512;
  static constexpr int kPlane = 128 * 16 + 32, kStage = 4 * kPlane;  // a 16-byte piece of 128 rows (banks apart), a chunk's four
  static constexpr int kRing = 2 * kStages * kStage;               // codes
  static constexpr int kX = N * 256;                               // x of a chunk
  static constexpr int kSmem = kRing + kXStages * kX + 1024;
  static constexpr int kPieces = 8;                                // 8-column pieces of x a staging thread and chunk
};

template <int XT, int GB, int N>
__global__ void __launch_bounds__(GemvTc<XT, GB, N>::kThreads, N == 16 ? 2 : 1) gemv4_tc_kernel(const __grid_constant__ Gemv4Args ga) {
  using S = GemvTc<XT, GB, N>;
  constexpr bool X8 = XT == YK_E4M3, F16 = XT != YK_BF16;
  extern __shared__ uint8_t gemv_tc_raw[];
  __shared__ __align__(8) uint64_t bars[4 + 4 + 2 * S::kXStages];
  __shared__ uint32_t tslot;
  __shared__ volatile int abort_flag;
  // scales of e4m3 x of a chunk at its number in turn % 8 (1 where there are none): x stages are free before the sums are read
  __shared__ __align__(16) float xs_sm[8][N];
  const YkGemv4& p = ga.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int K = p.k, chunks = (K + 127) / 128;
  const int n0 = blockIdx.x * 128;
  // set 0 has chunks 0 .. split - 1; split * 128 columns are a multiple of 8 groups
  const int split = min(chunks, ((chunks + 1) / 2 + 2 * GB - 1) / (2 * GB) * (2 * GB));
  const uint32_t base = (smem_u32(gemv_tc_raw) + 1023) & ~1023u;
  const uint32_t x_sm = base, ring = base + S::kXStages * S::kX;
  // A of (set of warps, buffer) is full; its MMA is done; x stage is full; is free
  const uint32_t a_full = smem_u32(&bars[0]), done = smem_u32(&bars[4]), x_full = smem_u32(&bars[8]),
                 x_free = smem_u32(&bars[8 + S::kXStages]);
  if (tid == 0) {
    for (int i = 0; i < 4; i++) {
      mbar_init(a_full + i * 8, 128);
      mbar_init(done + i * 8, 1);
    }
    for (int i = 0; i < S::kXStages; i++) {
      mbar_init(x_full + i * 8, S::kTeam * 32);
      mbar_init(x_free + i * 8, 1);
    }
    mbar_fence_init();
    abort_flag = 0;
  }
  pdl_wait();
  pdl_trigger();
  constexpr int kMmaWarp = 8 + S::kStageWarps;
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tslot), S::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  const auto a_at = [&](int set, int buf) { return tmem + (set * 2 + buf) * 32; };
  const auto d_at = [&](int set, int buf) {
    return tmem + S::kD0 + (S::kOneD ? set : set * 2 + buf) * (S::kUnits * N);
  };
  float2 tot[N / 2];
#pragma unroll
  for (int m = 0; m < N / 2; m++) tot[m] = make_float2(0.f, 0.f);

  if (warp < 8) {
    // ---------------- codes into TMEM, sums out of it ----------------
    const int set = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const long long n = min(n0 + row, p.n - 1);
    const uint16_t* scales = (const uint16_t*)p.wscale + n * p.group_row;
    const uint8_t* zeros = (const uint8_t*)p.wzero + n * p.group_row;
    const bool zero = ga.zero;
    const int c_first = set ? split : 0, mine = set ? chunks - split : split, groups = K / (32 * GB);
    const uint32_t slots = ring + set * (S::kStages * S::kStage), slot = slots + row * 16;
    // a warp copies its own 32 rows, four lanes a row's 64 bytes: 8 lines an instruction, not 32
    const int q_in = lane & 3, row_in = (warp & 3) * 32 + (lane >> 2);
    const uint8_t* w_in[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w_in[i] = (const uint8_t*)p.w + min((long long)n0 + row_in + 8 * i, p.n - 1ll) * p.w_row + q_in * 16;
    const auto issue = [&](int i) {
      if (i < mine) {
        const int k = (c_first + i) * 128;
        const uint32_t to = slots + (i % S::kStages) * S::kStage + q_in * S::kPlane + row_in * 16;
        const bool ok = k + q_in * 32 < K;
#pragma unroll
        for (int x = 0; x < 4; x++) cp_async_at<16>(to + x * 128, w_in[x] + (ok ? k / 2 : 0), ok);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; i++) issue(i);
    // scales and zero points of a half's units, as they are in memory, one half ahead; in eights
    // (s8, z8), the next eight on their way
    uint32_t s_next[S::kUnits], z_next[S::kUnits];
    uint4 s8, s8_next = make_uint4(0, 0, 0, 0);
    uint2 z8, z8_next = make_uint2(0x08080808u, 0x08080808u);
    const auto load8 = [&](int at) {
      if (at >= groups || !mine) return;
      s8_next = *(const uint4*)(scales + at);
      if (zero) z8_next = *(const uint2*)(zeros + at);
    };
    const auto load_scales = [&](int h) {
      const int k = (c_first + (h >> 1)) * 128 + (h & 1) * 64;
#pragma unroll
      for (int u = 0; u < S::kUnits; u++) {
        const int at = k / (32 * GB) + u;
        if (ga.s_vec) {
          if (at % 8 == 0 && (GB < 4 || (h & 1) == 0)) {
            s8 = s8_next;
            z8 = z8_next;
            load8(at + 8);
          }
          const uint32_t w = at & 4 ? (at & 2 ? s8.w : s8.z) : (at & 2 ? s8.y : s8.x);
          s_next[u] = at & 1 ? w >> 16 : w & 0xffffu;
          z_next[u] = (at & 4 ? z8.y : z8.x) >> (8 * (at & 3)) & 0xffu;
        } else {
          const bool ok = h < 2 * mine && at < groups;
          s_next[u] = ok ? scales[at] : 0;
          z_next[u] = zero && ok ? zeros[at] : 8;
        }
      }
    };
    if (ga.s_vec) load8(c_first * 4 / GB);
    load_scales(0);
    bool ok = true;
    float s_last[S::kUnits];
    // sums of half h (its scales in s_last), once its MMA is done
    const auto add_sums = [&](int h) {
      const int buf = h & 1, seq = (h & ~1) + set;           // of the chunk, among both sets' in turn
      if (!mbar_wait(done + (set * 2 + buf) * 8, (h >> 1) & 1, 0x601)) return false;
      tc_fence_after();
#pragma unroll
      for (int u = 0; u < S::kUnits; u++) {
#pragma unroll
        for (int m0 = 0; m0 < N; m0 += 16) {
          uint32_t d[16];
          tmem_ld16p(d_at(set, buf) + lanes + u * N + m0, d);
          tmem_ld_wait();
#pragma unroll
          for (int m = 0; m < 8; m++) {
            float2 f = make_float2(s_last[u], s_last[u]);
            if (X8) f = mul2(f, *(const float2*)&xs_sm[seq & 7][m0 + 2 * m]);
            float2& t = tot[m0 / 2 + m];
            t = ffma2(make_float2(__uint_as_float(d[2 * m]), __uint_as_float(d[2 * m + 1])), f, t);
          }
        }
      }
      tc_fence_before();       // before the next MMA into these columns
      return true;
    };
    for (int h = 0; h < 2 * mine && ok; h++) {
      const int i = h >> 1, buf = h & 1;
      if (buf == 0) {
        __syncwarp();                          // the stage that is filled next has been read
        issue(i + S::kStages - 1);
        cp_async_wait<S::kStages - 1>();
        __syncwarp();                          // every lane's pieces are there
      }
      if (S::kOneD && h > 0 && !add_sums(h - 1)) { ok = false; break; }
      float s_now[S::kUnits];
      Zero z[S::kUnits];
#pragma unroll
      for (int u = 0; u < S::kUnits; u++) {
        s_now[u] = XT == YK_BF16 || (X8 && ga.bf16) ? elem_to_float<true>(s_next[u]) : elem_to_float<false>(s_next[u]);
        z[u] = zero_of<F16>(z_next[u]);
      }
      load_scales(h + 1);
      const uint32_t from = slot + (i % S::kStages) * S::kStage + buf * 2 * S::kPlane;
#pragma unroll
      for (int q = 0; q < 2; q++) {            // 32 columns: 16 TMEM columns
        uint32_t v[4], a[16];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(from + q * S::kPlane));
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t o[4];
          codes8<F16>(v[e], z[S::kUnits == 2 ? q : 0], o);
#pragma unroll
          for (int x = 0; x < 4; x++) a[4 * e + x] = o[x];
        }
        tmem_st16(a_at(set, buf) + lanes + q * 16, a);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(a_full + (set * 2 + buf) * 8);
      if (!S::kOneD && h > 0 && !add_sums(h - 1)) { ok = false; break; }
#pragma unroll
      for (int u = 0; u < S::kUnits; u++) s_last[u] = s_now[u];
    }
    if (ok && mine && !add_sums(2 * mine - 1)) ok = false;
    if (!ok) abort_flag = 1;
    cp_async_wait<0>();
  } else if (warp < kMmaWarp) {
    // ---------------- x ----------------
    // chunks in turn, one of each set: team t takes numbers t, t + kTeams, ..; a lane 8 columns of every other row of its warp's 16
    const int team = (warp - 8) / S::kTeam, row0 = (warp - 8) % S::kTeam * 16 + (lane >> 4), ch = lane & 15;
    constexpr int kSize = X8 ? 1 : 2;
    const uint8_t* const x0 = (const uint8_t*)p.x + ((long long)row0 * p.x_row + ch * 8) * kSize;
    const long long step = 2 * p.x_row * kSize;
    const int m_xs = (warp - 8) % S::kTeam * 32 + lane;             // (lanes below N in all) reads a row's scale
    uint32_t raw[S::kPieces][2 * kSize];
    float xs = 1.f;
    const int turns = 2 * split;
    const auto chunk_at = [&](int seq) { return seq & 1 ? split + (seq >> 1) : seq >> 1; };   // (chunks on: none)
    const auto load = [&](int seq) {
      const int c = seq < turns ? chunk_at(seq) : chunks;
      const bool in_k = c * 128 + ch * 8 < K;
#pragma unroll
      for (int i = 0; i < S::kPieces; i++) {
        const uint8_t* x = x0 + i * step + c * 128 * kSize;
        const bool ok = in_k && row0 + 2 * i < p.rows;
        if (ga.x_vec) {
          if (X8) {
            const uint2 u = ok ? *(const uint2*)x : make_uint2(0, 0);
            raw[i][0] = u.x; raw[i][1] = u.y;
          } else {
            const uint4 u = ok ? *(const uint4*)x : make_uint4(0, 0, 0, 0);
            raw[i][0] = u.x; raw[i][1] = u.y; raw[i][2 * kSize - 2] = u.z; raw[i][2 * kSize - 1] = u.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2 * kSize; e++) {
            raw[i][e] = 0;
            if (ok)
              raw[i][e] = X8 ? x[4 * e] | x[4 * e + 1] << 8 | x[4 * e + 2] << 16 | (uint32_t)x[4 * e + 3] << 24
                             : ((const uint16_t*)x)[2 * e] | (uint32_t)((const uint16_t*)x)[2 * e + 1] << 16;
          }
        }
      }
      if (X8 && ga.xgroup && m_xs < N && c < chunks)
        xs = p.xscale[min(m_xs, p.rows - 1) * p.xscale_row + (ga.x_shift >= 0 ? c * 128 >> ga.x_shift : c * 128 / ga.xgroup)];
    };
    load(team);
    for (int seq = team; seq < turns; seq += S::kTeams) {
      if (chunk_at(seq) >= chunks) continue;
      const int stage = seq % S::kXStages;
      if (seq >= S::kXStages && !mbar_wait(x_free + stage * 8, (seq / S::kXStages - 1) & 1, 0x602)) { abort_flag = 1; break; }
#pragma unroll
      for (int i = 0; i < S::kPieces; i++) {
        const int m = row0 + 2 * i;
        uint32_t o[4];
        if (X8) {
          e4m3x4_to_half2x2(__byte_perm(raw[i][0], raw[i][1], 0x5140), o[0], o[1]);
          e4m3x4_to_half2x2(__byte_perm(raw[i][0], raw[i][1], 0x7362), o[2], o[3]);
        } else {
          o[0] = __byte_perm(raw[i][0], raw[i][2 * kSize - 2], 0x5410);
          o[1] = __byte_perm(raw[i][0], raw[i][2 * kSize - 2], 0x7632);
          o[2] = __byte_perm(raw[i][1], raw[i][2 * kSize - 1], 0x5410);
          o[3] = __byte_perm(raw[i][1], raw[i][2 * kSize - 1], 0x7632);
        }
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                         x_sm + stage * S::kX + (ch >> 3) * (N * 128) + m * 128 + (((ch & 7) ^ (m & 7)) << 4)),
                     "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
      }
      if (m_xs < N) xs_sm[seq & 7][m_xs] = xs;
      fence_proxy_async();
      mbar_arrive(x_full + stage * 8);
      load(seq + S::kTeams);
    }
  } else if (lane == 0) {
    // ---------------- MMA ----------------
    constexpr uint32_t idesc = idesc_f16_m128(N) | (F16 ? 0u : (1u << 7) | (1u << 10));     // bf16 A and B
    const uint64_t x_desc = sw128_desc(x_sm);
    const int set = warp - kMmaWarp;
    bool ok = true;
    const int mine = set ? chunks - split : split;
    for (int i = 0; i < mine && ok; i++) {
      const int stage = (2 * i + set) % S::kXStages;
      ok = mbar_wait(x_full + stage * 8, ((2 * i + set) / S::kXStages) & 1, 0x603);
#pragma unroll
      for (int half = 0; half < 2 && ok; half++) {
        ok = mbar_wait(a_full + (set * 2 + half) * 8, i & 1, 0x604);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < 4; s++)
          tc_mma_f16_ts(d_at(set, half) + (S::kUnits == 2 ? (s >> 1) * N : 0), a_at(set, half) + s * 8,
                        x_desc + (stage * S::kX + half * (N * 128)) / 16 + s * 2, idesc, S::kUnits == 2 ? s & 1 : s);
        tc_commit(done + (set * 2 + half) * 8);
        if (half == 1) tc_commit(x_free + stage * 8);
      }
    }
    if (!ok) abort_flag = 1;
  }
  // the two sets' sums meet: odd chunks' through shared memory (the ring, no longer in use)
  tc_fence_before();
  __syncthreads();
  float* meet = (float*)(gemv_tc_raw + (ring - smem_u32(gemv_tc_raw)));
  if (warp >= 4 && warp < 8) {
#pragma unroll
    for (int m = 0; m < N / 2; m++) {
      meet[(2 * m) * 128 + (tid & 127)] = tot[m].x;
      meet[(2 * m + 1) * 128 + (tid & 127)] = tot[m].y;
    }
  }
  __syncthreads();
  if (warp < 4 && n0 + tid < p.n && !abort_flag) {
    const float bias = p.bias ? p.bias[n0 + tid] : 0.f;
#pragma unroll
    for (int m = 0; m < N; m++) {
      if (m >= p.rows) break;
      float v = (m & 1 ? tot[m / 2].y : tot[m / 2].x) + meet[m * 128 + tid];
      if (X8 && !ga.xgroup) v *= p.xscale[m * p.xscale_row];
      v += bias;
      ((uint16_t*)p.y)[m * p.y_row + n0 + tid] = ga.bf16 ? float_to_elem<true>(v) : float_to_elem<false>(v);
    }
  }
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, S::kCols);
  }
}

template <int XT, int GB, int N>
static int launch_gemv4_tc(const Gemv4Args& a, cudaStream_t st) {
  using S = GemvTc<XT, GB, N>;
  const auto kern = gemv4_tc_kernel<XT, GB, N>;
  if (smem_attr(kern, S::kSmem) != cudaSuccess) return check_launch("gemv4 attr");
  launch_k(kern, (a.p.n + 127) / 128, S::kThreads, S::kSmem, st, a);
  note_launch();
  return check_launch("gemv4");
}
