// The next token from 16-bit scores (yk_sample).
#pragma once
#include "sample.cuh"

namespace yk {

// A 16-bit score has one of 65536 keys: each CTA of a row counts its scores by key, in 128 KB of shared memory as
// 16-bit counts by falling score ("place" = 65535 - key), two to a word.  With the counts every sum over a row is one
// over places, whose exact weights are evaluated once each, and both borders are found in the order itself:
//  * The warps of the row's cluster sum the places in reach of the largest score (2^-46 of its weight) in steps of 256,
//    over the counts of all CTAs, and tell all CTAs.
//  * Each CTA finds the step that holds a border, and goes through its places.
//  * Each CTA sums what stays of its own scores over the places that stay, which fills a table of their weights; the CTA
//    that holds the token then reads its scores once more, by warp.  Where more places stay than the table holds (scores
//    of both signs, for most magnitudes lie near 0), or without a limit, a CTA sums them score by score and by warp at once.
// An addition in shared memory takes a warp about 5 clocks, an exact weight about 50.  64 rows of 128000: 31 us (0.5 TB/s;
// by bins, with an exact weight for each score, 62), of which the counts take 5, the sums by step 6, a border 3, the pass
// through the token's CTA 7; the rest are some ten waits of the whole cluster or CTA for one another.  47 us if a row keeps
// scores of both signs; 35 without limits.
// Scores of a CTA at most: a count stays below 2^16, also where the start of the row moves a CTA's part by 256.  (64 rows of 128256 or
// 130048: 32 us by two CTAs each, which fill the SMs; 50 by four, two rounds, as from 130049 on.)
constexpr int kSamp16Slice = 65024;
constexpr int kSamp16Threads = 1024;
constexpr int kSamp16Table = 11264;            // places that stay, and one for all others
constexpr int kSamp16Smem = 65536 * 2 + kSamp16Table * 8;


// (out of line: where a kernel goes through its code once, fetching many copies of this took longer than the calls)
__device__ __noinline__ unsigned long long samp16_weight(float top, double c, double at_top, int mode, float l, const double* table) {
  SampWeights w;
  w.top = top;
  w.c = c;
  w.at_top = at_top;
  w.mode = mode;
  return w.of(l, table);
}

template <int DT>
__global__ void __launch_bounds__(kSamp16Threads, 1) sample16_kernel(const __grid_constant__ SampleArgs a) {
  using K = SampKey<DT>;
  using u64 = unsigned long long;
  constexpr int T = kSamp16Threads, kWarps = T / 32, kStep = 256;    // places of a warp's step
  extern __shared__ __align__(16) uint8_t samp_raw[];
  uint32_t* const counts = (uint32_t*)samp_raw;
  u64* const found_weight = (u64*)(samp_raw + 65536 * 2);            // of the places from the largest score's on
  __shared__ double table[512];
  __shared__ SampPart part[2][8];               // of the row's CTAs
  __shared__ u64 sum_mass[65536 / kStep];       // of the row's scores, by step of places
  __shared__ uint32_t sum_count[65536 / kStep];
  __shared__ u64 warp_mass[kWarps], warp_rest[kWarps];
  __shared__ uint32_t warp_a[kWarps], warp_b[kWarps];
  __shared__ u64 found_mass;
  __shared__ uint32_t found_place, found_take;
  const YkSample& p = a.p;
  if (a.split > 1) cluster_arrive();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, split = a.split;
  const int row = blockIdx.x / split, rank = split > 1 ? (int)cluster_rank() : 0;
  // the row begins `lead` scores behind a 16-byte boundary; a CTA's slices begin on one, so `first` may be negative
  const uint16_t* const scores = (const uint16_t*)p.logits + row * p.row;
  const int lead = (int)((uintptr_t)scores / 2 % 8);
  const int first = rank * a.slice - lead, size = max(0, min(a.slice, p.n - first)), begin = max(0, -first);
  const auto meet = [&] {
    __syncwarp();                               // (the cluster's barrier takes whole warps)
    if (split > 1) cluster_barrier(); else __syncthreads();
  };
  const auto tell = [&](int which, SampPart v) {
    if (tid < split) {
      const uint32_t to = smem_u32(&part[which][rank]), at = split > 1 ? cluster_map(to, tid) : to;
      st_cluster_u64(at, v.mass);
      st_cluster_u64(at + 8, v.rest);
      st_cluster_u32(at + 16, v.count);
      st_cluster_u32(at + 20, v.ties);
    }
    meet();
  };
  const auto count_at = [&](int place) { return counts[place >> 1] >> (place & 1) * 16 & 0xffffu; };
  for (int i = tid; i < 65536 / 8; i += T) ((uint4*)counts)[i] = make_uint4(0, 0, 0, 0);
  if (tid < 512) table[tid] = exp2((double)(tid / 16) / 32);
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  // eight scores from place i of the slice on, NaN for those beyond the row
  const auto load8 = [&](int i) {
    if (i >= begin && i + 8 <= size) return *(const uint4*)(scores + first + i);
    uint4 raw = make_uint4(~0u, ~0u, ~0u, ~0u);
    uint32_t* w = (uint32_t*)&raw;
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (i + e >= begin && i + e < size) w[e >> 1] ^= (scores[first + i + e] ^ 0xffffu) << (e & 1) * 16;
    return raw;
  };
  // places of two scores, but for -0 (one behind that of 0); a NaN's is before that of infinity or behind that of -infinity
  const auto places = [](uint32_t w) {
    uint32_t below;                             // of each half: its sign, 16 times
    asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(below) : "r"(w));
    return w ^ (0x7fff7fffu & ~below);
  };
  // the place of one of eight scores
  const auto place_of = [&](const uint4& raw, int e) {
    const uint32_t place = places(((const uint32_t*)&raw)[e >> 1]) >> (e & 1) * 16 & 0xffffu;
    return place - (place == 0x8000u);
  };
  // parameters, on their way meanwhile
  const float temperature = p.temperature ? p.temperature[row] : 1.f, u = p.u ? p.u[row] : 0.f;
  const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
  int top_k = p.top_k ? p.top_k[row] : 0;
  if (top_k <= 0 || top_k >= p.n) top_k = 0;
  const bool by_p = top_p < 1.f, limits = top_k || by_p;

  // ---- counts by place, the largest key
  uint32_t largest = DT == YK_BF16 ? 0xff80ff80u : 0xfc00fc00u;      // -infinity twice
  constexpr int kAhead = 4;                     // loads on their way
  for (int i0 = tid * 8; i0 < size; i0 += T * 8 * kAhead) {
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) raw[j] = load8(i0 + j * T * 8);
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (i0 + j * T * 8 >= size) break;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t w = ((const uint32_t*)&raw[j])[e], q = places(w);
        if (DT == YK_BF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(largest) : "r"(largest), "r"(w));
        else asm("max.f16x2 %0, %1, %2;" : "=r"(largest) : "r"(largest), "r"(w));
        if (!limits) continue;
        atomicAdd((uint32_t*)(samp_raw + (q & 0xfffeu) * 2), q & 1 ? 0x10000u : 1u);
        atomicAdd((uint32_t*)(samp_raw + (q >> 17) * 4), q & 0x10000u ? 0x10000u : 1u);
      }
    }
  }
  uint32_t top_key = max(K::of((uint16_t)largest), K::of((uint16_t)(largest >> 16)));
  const auto block_max = [&](uint32_t v) {
    v = __reduce_max_sync(~0u, v);
    __syncthreads();
    if (lane == 0) warp_a[warp] = v;
    __syncthreads();
    return __reduce_max_sync(~0u, warp_a[lane]);
  };
  top_key = block_max(top_key);
  if (tid == 0) {                               // both zeros at one place
    counts[0x3fff] += counts[0x4000] << 16;
    counts[0x4000] &= 0xffff0000u;
  }
  if (split > 1) {                              // every CTA of the row has started: its shared memory may be written
    __syncwarp();
    cluster_wait();
  }
  tell(0, {0, 0, top_key, 0});
  for (int i = 0; i < split; i++) top_key = max(top_key, part[0][i].count);
  const bool greedy = !(temperature > 0.f) || !p.u, any = top_key > K::kNone;
  if (!any || greedy) {
    // the lowest index of the largest score, in the first CTA that has one
    int who = 0;
    while (any && part[0][who].count != top_key) who++;
    if (rank != who) return;
    uint32_t at = 0xffffffffu;
    if (any)
      for (int i = tid * 8; i < size && at == 0xffffffffu; i += T * 8) {
        const uint4 raw = load8(i);
#pragma unroll
        for (int e = 7; e >= 0; e--)
          if (K::of((uint16_t)(((const uint32_t*)&raw)[e >> 1] >> (e & 1) * 16)) == top_key) at = (uint32_t)(first + i + e);
      }
    at = ~block_max(~at);
    if (tid == 0) {
      p.token[row] = any ? (int)at : -1;
      if (p.logprob) p.logprob[row] = any ? 0.f : -INFINITY;
      if (p.kept) p.kept[row] = any ? 1 : 0;
    }
    return;
  }
  const float top = K::value(top_key);
  SampWeights weights;
  weights.set(top, temperature);
  const auto weight = [&](int place) {
    return samp16_weight(weights.top, weights.c, weights.at_top, weights.mode, K::value(65535u - place), table);
  };
  const int top_place = 65535 - (int)top_key;
  const u64 least = min_p > 0.f ? min((u64)ceil(fmin((double)min_p, 1.0) * kSampOne), weight(top_place)) : 1ull;
  // places from `end` on have no weight: scores more than 46 ln 2 temperatures below the top
  int end = top_place + 1;
  if (top < INFINITY) {
    const float far = __double2float_rd((double)top - 46.0 / weights.c * 1.00001);
    const uint16_t b = DT == YK_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rd(far)) : __half_as_ushort(__float2half_rd(far));
    end = 65536 - (int)max(K::of(b), K::kNone + 1);
  }

  // Places before `cut` stay, and of the scores at it the first `take`.
  int cut = end;
  uint32_t take = 0;
  if (limits) {
    // sums by step of kStep places, from a multiple of 8 on, each by one warp of the row's
    const int start = top_place & ~7, steps = (end - start + kStep - 1) / kStep;
#pragma unroll 1
    for (int step = warp * split + rank; step < steps; step += kWarps * split) {
      const int place = start + step * kStep + lane * 8;
      uint32_t c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (place < end) {
        const uint32_t at = smem_u32(counts) + place * 2;
        for (int q0 = 0; q0 < split; q0 += 4) {   // (loads of four CTAs on their way together)
          uint32_t v[4][4];
#pragma unroll
          for (int q = 0; q < 4; q++) {
            if (q0 + q >= split) break;
            asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[q][0]), "=r"(v[q][1]), "=r"(v[q][2]), "=r"(v[q][3])
                         : "r"(split > 1 ? cluster_map(at, q0 + q) : at));
          }
#pragma unroll
          for (int q = 0; q < 4; q++) {
            if (q0 + q >= split) break;
#pragma unroll
            for (int e = 0; e < 8; e++) c[e] += v[q][e >> 1] >> (e & 1) * 16 & 0xffffu;
          }
        }
      }
      uint32_t count = 0, some = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (place + e < top_place || place + e >= end) c[e] = 0;   // (NaN are before infinity)
        count += c[e];
        some |= (c[e] != 0) << e;
      }
      u64 mass = 0;
      if (by_p)
        while (__any_sync(~0u, some != 0)) {      // places without a score take no evaluation
          const int at = some ? __ffs(some) - 1 : 8;
          uint32_t n = 0;
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (e == at) n = c[e];
          mass += n * weight(min(place + at, 65535));
          some &= some - 1;
        }
#pragma unroll
      for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
      count = __reduce_add_sync(~0u, count);
      if (lane < split) {
        const uint32_t m = smem_u32(&sum_mass[step]), n = smem_u32(&sum_count[step]);
        st_cluster_u64(split > 1 ? cluster_map(m, lane) : m, mass);
        st_cluster_u32(split > 1 ? cluster_map(n, lane) : n, count);
      }
    }
    meet();
    // lane i: the sums of steps 8 i .. 8 i + 7
    u64 mass = 0;
    uint32_t count = 0;
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (lane * 8 + i < steps) {
        mass += sum_mass[lane * 8 + i];
        count += sum_count[lane * 8 + i];
      }
    u64 mass_at = mass;
    uint32_t count_at = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u = __shfl_up_sync(~0u, mass_at, o);
      const uint32_t v = __shfl_up_sync(~0u, count_at, o);
      if (lane >= o) {
        mass_at += u;
        count_at += v;
      }
    }
    u64 upto = __shfl_sync(~0u, mass_at, 31);   // the weight of what stays so far
    mass_at -= mass;
    count_at -= count;
    // The place at which the sums of counts (turn 0) or weights reach `want`, and how many of its scores that takes:
    // first the step, then by a place a thread.
#pragma unroll 1
    for (int turn = top_k ? 0 : 1; turn < (by_p ? 2 : 1); turn++) {
      const u64 want = turn ? max(1ull, (u64)ceil(fmax((double)top_p, 0.0) * (double)upto)) : (u64)top_k;
      const u64 have = turn ? mass_at : count_at;
      const uint32_t hit = __ballot_sync(~0u, have < want && have + (turn ? mass : count) >= want);
      if (!hit) continue;                       // all of them stay
      const int who = __ffs(hit) - 1;
      u64 n_at = __shfl_sync(~0u, have, who), m_at = __shfl_sync(~0u, mass_at, who);
      int step = who * 8;
#pragma unroll 1
      for (;; step++) {
        const u64 m = sum_mass[step], n = turn ? m : sum_count[step];
        if (n_at + n >= want) break;
        n_at += n;
        m_at += m;
      }
      const int place = start + step * kStep + tid;
      u64 one = 0, n = 0, m = 0, n_to = 0, m_to = 0;   // of a score there, of all of them, with those before
      if (tid < kStep) {
        uint32_t c = 0;
        if (place >= top_place && place < end) {
          const uint32_t l = smem_u32(counts) + (place >> 1) * 4;
#pragma unroll 4
          for (int q = 0; q < split; q++) c += ld_cluster_u32(split > 1 ? cluster_map(l, q) : l) >> (place & 1) * 16 & 0xffffu;
        }
        if (by_p && __any_sync(~0u, c != 0)) one = weight(min(place, 65535));
        m_to = m = c * one;
        n_to = n = turn ? m : c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 u = __shfl_up_sync(~0u, n_to, o), v = __shfl_up_sync(~0u, m_to, o);
          if (lane >= o) {
            n_to += u;
            m_to += v;
          }
        }
        if (lane == 31) {
          warp_mass[warp] = n_to;
          warp_rest[warp] = m_to;
        }
      }
      __syncthreads();
      if (tid < kStep) {
        for (int i = 0; i < warp; i++) {
          n_to += warp_mass[i];
          m_to += warp_rest[i];
        }
        n_to += n_at - n;
        m_to += m_at - m;
        if (n_to < want && n_to + n >= want) {
          const uint32_t some = (uint32_t)(turn ? (want - n_to + one - 1) / one : want - n_to);
          found_place = (uint32_t)place;
          found_take = some;
          found_mass = m_to + some * one;
        }
      }
      __syncthreads();
      cut = (int)found_place;
      take = found_take;
      upto = found_mass;
    }
  }

  // ---- what stays of this CTA's scores, by place
  const u64 cut_w = take ? weight(cut) : 0;
  if (cut_w < least) take = 0;
  const uint32_t kept = cut - top_place, cut_place = take ? cut : ~0u;
  const int run = a.slice / kWarps, run_from = warp * run, run_to = min(size, run_from + run);   // of consecutive scores, a warp's
  const auto weight_at = [&](uint32_t place) {  // 0 at the cut
    const u64 w = place - (uint32_t)top_place < kept ? weight((int)place) : 0;
    return w < least ? 0 : w;
  };
  const bool listed = limits && kept < kSamp16Table;
  u64 mass = 0;
  uint32_t count = 0, ties = 0;
  if (listed) {
    for (int i0 = top_place; i0 <= cut; i0 += T) {
      const int i = i0 + tid;
      const uint32_t c = i < cut ? count_at(i) : 0;
      u64 w = 0;
      if (__any_sync(~0u, c != 0)) w = weight(min(i, 65535));
      if (w < least) w = 0;
      if (i <= cut) found_weight[i - top_place] = i < cut ? w : 0;   // (the last one: all others)
      mass += c * w;
      count += w ? c : 0;
    }
  } else {
    // without a limit, or where too many places stay for the table: each score by itself
#pragma unroll 1
    for (int i = run_from + lane * 8; i < run_to; i += 256) {
      const uint4 raw = load8(i);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t place = place_of(raw, e);
        u64 w = weights.of(K::value(65535u - place), table);
        if (place - (uint32_t)top_place >= kept || w < least) w = 0;
        mass += w;
        count += w != 0;
        ties += place == cut_place;
      }
    }
    ties = __reduce_add_sync(~0u, ties);
    if (lane == 0) warp_a[warp] = ties;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
  count = __reduce_add_sync(~0u, count);
  if (lane == 0) {
    warp_mass[warp] = mass;
    warp_b[warp] = count;
  }
  __syncthreads();
  mass = warp_mass[lane];
#pragma unroll
  for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
  tell(1, {mass, 0, __reduce_add_sync(~0u, warp_b[lane]), take ? count_at(cut) : 0});
  u64 total = 0, at = 0;                        // of the row; before this CTA
  uint32_t all = 0, ties_at = 0, tie_start = 0;
  u64 mine = 0;
  for (int q = 0; q < split; q++) {
    const uint32_t stay = min(part[1][q].ties, take - min(take, ties_at));
    const u64 v = part[1][q].mass + stay * cut_w;
    if (q == rank) {
      at = total;
      tie_start = ties_at;
      mine = v;
    }
    total += v;
    all += part[1][q].count + stay;
    ties_at += part[1][q].ties;
  }
  u64 target = u > 0.f ? (u64)fmin((double)u * (double)total, 9e18) : 0;
  target = min(target, total - 1);
  if (target < at || target - at >= mine) return;   // another CTA's
  // ---- by warp
  if (listed) {
    mass = 0;
#pragma unroll 1
    for (int i0 = run_from + lane * 8; i0 < run_to; i0 += 512) {
      uint4 raw[2];
#pragma unroll
      for (int j = 0; j < 2; j++) raw[j] = i0 + j * 256 < run_to ? load8(i0 + j * 256) : make_uint4(~0u, ~0u, ~0u, ~0u);
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const uint32_t place = place_of(raw[e >> 3], e & 7);
        mass += found_weight[min(place - top_place, kept)];
        ties += place == cut_place;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
    ties = __reduce_add_sync(~0u, ties);
    __syncthreads();
    if (lane == 0) {
      warp_mass[warp] = mass;
      warp_a[warp] = ties;
    }
    __syncthreads();
  }
  // lane i: warp i's
  ties = warp_a[lane];
  uint32_t tie_before = ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t b = __shfl_up_sync(~0u, tie_before, o);
    if (lane >= o) tie_before += b;
  }
  tie_before += tie_start - ties;
  mass = warp_mass[lane] + min(ties, take - min(take, tie_before)) * cut_w;
  u64 to = mass;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 b = __shfl_up_sync(~0u, to, o);
    if (lane >= o) to += b;
  }
  to += at;
  const uint32_t has = __ballot_sync(~0u, target < to && target >= to - mass);
  const int who = __ffs(has) - 1;
  at = __shfl_sync(~0u, to - mass, who);
  uint32_t tie = __shfl_sync(~0u, tie_before, who);
  // ---- that warp's run, a score a thread and turn: the first at which the sum passes the target
  const int run_end = min(size, (who + 1) * run);
  for (int i0 = who * run; i0 < run_end; i0 += T) {
    const int i = i0 + tid;
    const uint32_t k = i >= begin && i < run_end ? K::of(scores[first + i]) : K::kNone, place = 65535u - k;
    const bool same = place == cut_place;
    const uint32_t sames = __ballot_sync(~0u, same);
    u64 w = weight_at(place);
    __syncthreads();                            // the last turn's sums have been read
    if (lane == 0) warp_b[warp] = __popc(sames);
    __syncthreads();
    if (same) {
      const uint32_t ahead = tie + __popc(sames & ((1u << lane) - 1));
      uint32_t more = 0;
      for (int q = 0; q < warp; q++) more += warp_b[q];
      w = ahead + more < take ? cut_w : 0;
    }
    u64 s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 b = __shfl_up_sync(~0u, s, o);
      if (lane >= o) s += b;
    }
    if (lane == 31) warp_mass[warp] = s;
    __syncthreads();
    u64 sums = warp_mass[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 b = __shfl_up_sync(~0u, sums, o);
      if (lane >= o) sums += b;
    }
    const u64 ahead = __shfl_sync(~0u, sums, max(warp - 1, 0)), turn = __shfl_sync(~0u, sums, 31);
    s += at + (warp ? ahead : 0);
    if (s > target && s - w <= target) {        // one score of the row
      const float l = K::value(k);
      p.token[row] = first + i;
      if (p.logprob) p.logprob[row] = (float)((l == top ? 0.0 : ((double)l - (double)top) / (double)temperature) - log((double)total / kSampOne));
      if (p.kept) p.kept[row] = (int)all;
    }
    at += turn;
    if (at > target) return;
    tie += __reduce_add_sync(~0u, warp_b[lane]);
  }
}

}  // namespace yk
