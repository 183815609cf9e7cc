// The next token of each row of scores: temperature, top-k, top-p, min-p, from given random numbers (yk_sample).
#include "sample16.cuh"

namespace yk {

// A row's scores are read once, into the shared memory of a cluster, as keys.
// The borders of what stays:
//  * Scores are counted by bins of 1/64 octave of weight, together with the sum of where in its bin each lies: two 32-bit
//    additions in shared memory a score (64-bit ones take 6 to 150 times as long, and the counts need no weight).  A cluster's
//    CTAs sum a share of the bins each.  That gives the bin of the k-th score, and the weight up to each bin
//    within 10^-4: the bins in which the sum may reach top_p.
//  * One pass adds up the exact weights of all others, and lists the scores of those bins (some hundreds).
//  * Every CTA sorts the list and finds both borders in it.
//  * Where the list would be too long (thousands of equal scores), or a temperature so high that the ends of the floats weigh
//    alike (infinity), the borders are found digit by digit of the key instead: sums by digit of the keys that share the
//    digits so far, two or three turns a border.
// A chain of some twelve stages of 1 to 4 us, each the wait of a cluster for its slowest CTA: 1 x 32000 15 us; 200 x 151000
// of fp32 185 us, 5.4 rounds of two CTAs an SM (12 % of the copy rate; issue slots 55 % busy).
constexpr int kSampSlice = 32768;          // scores of a CTA at most
constexpr int kSampBins = 46 * 64;         // weights below 2^-46 count nothing
constexpr int kSampDigits = 2048;
constexpr int kSampThreads = 512;

template <int DT>
__global__ void __launch_bounds__(kSampThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  using K = SampKey<DT>;
  using key_t = typename K::type;
  using u64 = unsigned long long;
  constexpr int T = kSampThreads, kVec = 16 / sizeof(key_t), kWarps = T / 32;
  constexpr int kList = 2 * T;                       // of listed scores
  constexpr int kPer = (kSampBins + T - 1) / T;      // bins of a thread
  extern __shared__ __align__(16) uint8_t samp_raw[];
  key_t* const keys = (key_t*)samp_raw;
  __shared__ uint32_t hist[2 * kSampBins];           // counts, places; then the row's list; or two sums by digit
  __shared__ uint32_t own[kList];
  __shared__ uint8_t own_warp[kList];                // whose they are
  __shared__ double table[512];
  __shared__ SampPart part[3][8];                    // of the row's CTAs
  __shared__ u64 warp_mass[kWarps], warp_rest[kWarps];
  __shared__ uint32_t warp_a[kWarps], warp_b[kWarps];
  __shared__ float warp_lo[kWarps], warp_hi[kWarps];
  __shared__ u64 found_mass;
  __shared__ uint32_t border_key[5];
  __shared__ uint32_t found_bin, found_above, found_first, found_last, own_n;
  const YkSample& p = a.p;
  if (a.split > 1) cluster_arrive();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, split = a.split;
  const int row = blockIdx.x / split, rank = split > 1 ? (int)cluster_rank() : 0;
  // the row begins `lead` scores behind a 16-byte boundary; a CTA's slices begin on one, so `first` may be negative
  const int lead = (int)((uintptr_t)((const key_t*)p.logits + row * p.row) / sizeof(key_t) % kVec);
  const int first = rank * a.slice - lead, size = max(0, min(a.slice, p.n - first)), begin = max(0, -first);
  const auto meet = [&] {
    __syncwarp();                                    // (the cluster's barrier takes whole warps)
    if (split > 1) cluster_barrier(); else __syncthreads();
  };
  // this CTA's part to all of the row's, in turn `which`
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
  for (int i = tid; i < 512; i += T) table[i] = exp2((double)(i / 16) / 32);
  if (tid == 0) own_n = 0;
  for (int i = tid; i < 2 * kSampBins; i += T) hist[i] = 0;
  pdl_wait();
  pdl_trigger();

  // parameters, on their way meanwhile
  const float temperature = p.temperature ? p.temperature[row] : 1.f, u = p.u ? p.u[row] : 0.f;
  const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
  int top_k = p.top_k ? p.top_k[row] : 0;
  if (top_k <= 0 || top_k >= p.n) top_k = 0;

  // ---- scores into shared memory, the largest
  uint32_t top_key = K::kNone;
  {
    // 16 bytes a load, from the boundary before the row on: what comes before it there counts as NaN
    const key_t* from = (const key_t*)p.logits + row * p.row + first;
    constexpr int kAhead = 4;                        // loads on their way
    for (int i0 = tid * kVec; i0 < a.slice; i0 += T * kVec * kAhead) {
      uint4 raw[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const int i = i0 + j * T * kVec;
        if (i >= begin && i + kVec <= size) raw[j] = __ldcs((const uint4*)(from + i));
      }
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const int i = i0 + j * T * kVec;
        if (i >= a.slice) break;
        key_t* k = (key_t*)&raw[j];
        if (i < begin || i + kVec > size)
          for (int e = 0; e < kVec; e++) k[e] = i + e >= begin && i + e < size ? from[i + e] : (key_t)~0u;
#pragma unroll
        for (int e = 0; e < kVec; e++) {
          k[e] = (key_t)K::of(k[e]);
          top_key = max(top_key, (uint32_t)k[e]);
        }
        *(uint4*)(keys + i) = raw[j];
      }
    }
  }
  const auto block_max = [&](uint32_t v) {
    v = __reduce_max_sync(~0u, v);
    __syncthreads();
    if (lane == 0) warp_a[warp] = v;
    __syncthreads();
    return __reduce_max_sync(~0u, lane < kWarps ? warp_a[lane] : 0);
  };
  top_key = block_max(top_key);
  if (split > 1) {                                   // every CTA of the row has started: its shared memory may be written
    __syncwarp();
    cluster_wait();
  }
  tell(0, {0, 0, top_key, 0});
  for (int i = 0; i < split; i++) top_key = max(top_key, part[0][i].count);
  const bool greedy = !(temperature > 0.f) || !p.u;
  const bool any = top_key > K::kNone;
  if (!any || greedy) {
    // the lowest index of the largest score
    uint32_t at = 0xffffffffu;
    if (any)
      for (int i = tid; i < size; i += T)
        if (keys[i] == top_key) at = min(at, (uint32_t)(first + i));
    at = ~block_max(~at);
    tell(1, {0, 0, at, 0});
    for (int i = 0; i < split; i++) at = min(at, part[1][i].count);
    if (rank == 0 && tid == 0) {
      p.token[row] = any ? (int)at : -1;
      if (p.logprob) p.logprob[row] = any ? 0.f : -INFINITY;
      if (p.kept) p.kept[row] = any ? 1 : 0;
    }
    return;
  }
  const float top = K::value(top_key);
  SampWeights weights;
  weights.set(top, temperature);
  const auto weight = [&](uint32_t k) { return weights.of(K::value(k), table); };
  const u64 least = min_p > 0.f ? min((u64)ceil(fmin((double)min_p, 1.0) * kSampOne), weight(top_key)) : 1ull;
  const bool by_p = top_p < 1.f;

  // Keys above `cut` stay, and of those that equal it the first `take`.
  uint32_t cut = K::kNone, take = 0;
  bool limited = false;                              // by the cut
  bool by_list = false;                              // `mass` and `count` hold what of this warp's run stays, but for the list
  u64 mass = 0;
  uint32_t count = 0;
  const int run = a.slice / kWarps, from = warp * run, to = min(size, from + run);

  // 1/256 bins below the top, rounded (by the sum with 2^23); rises with falling scores
  const float c256 = (float)fmin(16384.0 * weights.c, 1e38);   // (times 0 is 0)
  const auto place = [&](uint32_t k) {
    return __float_as_uint(fminf(fmaf(top - K::value(k), c256, 8388608.f), 8388608.f + 256.f * kSampBins)) - 0x4b000000u;
  };
  const auto bin_of = [&](uint32_t k) { return (int)(place(k) >> 8); };
  bool open = top_k || by_p;                         // borders to find
  // (bins take differences of floats and count -infinity, the padding's too, as a score far below: not at flat temperatures)
  if (open && top < INFINITY && weights.steep()) {
    // ---- counts by bin
    for (int i = tid * kVec; i < a.slice; i += T * kVec) {     // (keys behind the last score are kNone: beyond the bins)
      const uint4 raw = *(const uint4*)(keys + i);
      const key_t* k = (const key_t*)&raw;
      uint32_t q[kVec];
#pragma unroll
      for (int e = 0; e < kVec; e++) q[e] = place(k[e]);
#pragma unroll
      for (int e = 0; e < kVec; e++) {
        if (q[e] >= kSampBins * 256) continue;
        atomicAdd(&hist[q[e] >> 8], 1u);
        if (by_p) atomicAdd(&hist[kSampBins + (q[e] >> 8)], q[e] & 255u);
      }
    }
    meet();
    if (split > 1) {
      // this CTA's share of the bins: the row's sums to all
      const int share = kSampBins / split;           // (46 * 64 is a multiple of 8)
      for (int i = tid; i < (by_p ? 2 : 1) * share; i += T) {
        const int b = i < share ? rank * share + i : kSampBins + rank * share + i - share;
        const uint32_t at = smem_u32(&hist[b]);
        uint32_t v = 0, part_of[8];
#pragma unroll
        for (int q = 0; q < 8; q++) part_of[q] = q < split ? ld_cluster_u32(cluster_map(at, q)) : 0;   // (on their way together)
#pragma unroll
        for (int q = 0; q < 8; q++) v += part_of[q];
        for (int q = 0; q < split; q++) st_cluster_u32(cluster_map(at, q), v);
      }
      meet();
    }
    // ---- thread t: kPer bins behind one another
    uint32_t n[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
      const int b = tid * kPer + e;
      n[e] = b < kSampBins ? hist[b] : 0;
      sum += n[e];
    }
    uint32_t above = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(~0u, above, o);
      if (lane >= o) above += v;
    }
    if (lane == 31) warp_a[warp] = above;
    if (tid == 0) {
      found_bin = found_first = kSampBins;
      found_last = kSampBins - 1;
      found_above = 0;
    }
    __syncthreads();
    above += __reduce_add_sync(~0u, lane < warp ? warp_a[lane] : 0) - sum;
    if (top_k) {
      uint32_t at = above;
#pragma unroll
      for (int e = 0; e < kPer; e++) {
        if (at < (uint32_t)top_k && at + n[e] >= (uint32_t)top_k) {
          found_bin = tid * kPer + e;
          found_above = at;
        }
        at += n[e];
      }
      __syncthreads();
    }
    const int bin_k = (int)found_bin;                // kSampBins: no score of a weight is left out by top-k
    const uint32_t above_k = found_above;
    int bin1 = bin_k, bin2 = bin_k;                  // bins below bin1 stay whole, those up to bin2 (and bin_k) are listed
    if (by_p) {
      // weights up to each bin, from below and from above: a bin's n scores at places f (in units of 1 / 256, half
      // a unit off at most and a tenth by the product's rounding) weigh 2^(-b / 64) (n - s sum f / 256 + at most n s^2 / 2),
      // s = ln 2 / 64
      constexpr float kS = 0.010830424696249145f, kOff = 2e-5f;
      float lo[kPer], hi[kPer], lo_sum = 0, hi_sum = 0;
#pragma unroll
      for (int e = 0; e < kPer; e++) {
        const int b = tid * kPer + e;
        lo[e] = hi[e] = 0;
        if (b <= bin_k && n[e]) {
          const float w = exp2f((float)b * -0.015625f), m = (float)n[e], f = (float)hist[kSampBins + b];
          lo[e] = w * (m - (kS / 256) * (f + 0.6f * m)) * (1 - kOff);
          hi[e] = w * (m - (kS / 256) * (f - 0.6f * m) + m * (kS * kS / 2)) * (1 + kOff);
          if (b == bin_k) {
            hi[e] = w * (float)(top_k - above_k) * (1 + kS / 256 + kOff);
            lo[e] = w * (float)(top_k - above_k) * (1 - kS * 1.01f - kOff);
          }
        }
        lo_sum += lo[e];
        hi_sum += hi[e];
      }
      float lo_at = lo_sum, hi_at = hi_sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float u = __shfl_up_sync(~0u, lo_at, o), v = __shfl_up_sync(~0u, hi_at, o);
        if (lane >= o) {
          lo_at += u;
          hi_at += v;
        }
      }
      if (lane == 31) {
        warp_lo[warp] = lo_at;
        warp_hi[warp] = hi_at;
      }
      __syncthreads();
      float lo_all = lane < kWarps ? warp_lo[lane] : 0, hi_all = lane < kWarps ? warp_hi[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float u = __shfl_up_sync(~0u, lo_all, o), v = __shfl_up_sync(~0u, hi_all, o);
        if (lane >= o) {
          lo_all += u;
          hi_all += v;
        }
      }
      const float lo_before = __shfl_sync(~0u, lo_all, max(warp - 1, 0)), hi_before = __shfl_sync(~0u, hi_all, max(warp - 1, 0));
      lo_at += (warp ? lo_before : 0) - lo_sum;
      hi_at += (warp ? hi_before : 0) - hi_sum;
      lo_all = __shfl_sync(~0u, lo_all, 31);
      hi_all = __shfl_sync(~0u, hi_all, 31);
      const float want_lo = fmaxf(top_p * lo_all * (1 - kOff), 1e-30f), want_hi = top_p * hi_all * (1 + kOff);
      // (bounds that miss a bin by these sums' own rounding are found out below)
      uint32_t at_hi = kSampBins, at_lo = kSampBins - 1;
#pragma unroll
      for (int e = kPer - 1; e >= 0; e--) {          // from the last bin down, so that the first one stays
        if (hi[e] > 0 && hi_at + hi_sum >= want_lo) at_hi = tid * kPer + e;
        if (lo[e] > 0 && lo_at + lo_sum >= want_hi) at_lo = tid * kPer + e;
        hi_sum -= hi[e];
        lo_sum -= lo[e];
      }
      at_hi = __reduce_min_sync(~0u, at_hi);
      at_lo = __reduce_min_sync(~0u, at_lo);
      if (lane == 0) {
        atomicMin(&found_first, at_hi);
        atomicMin(&found_last, at_lo);
      }
      __syncthreads();
      bin1 = (int)found_first;
      bin2 = max(bin1, min((int)found_last, bin_k));
    }
    // ---- exact weights of the bins that stay whole and (for top-p) of those that do not, and the list of the others
    u64 all = 0, rest = 0;
    // the smallest keys of bins below these five, a warp each, 33 parts a turn: bins fall as keys rise
    if (warp < 5) {
      const int b = warp == 0 ? bin1 : warp == 1 ? bin2 + 1 : warp == 2 ? bin_k : warp == 3 ? bin_k + 1 : kSampBins;
      uint32_t lo = 0, hi = top_key + 1u;            // (bins of lo and below are not, those of hi and above are)
      while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 32) / 33, m = lo + step * (lane + 1);
        const uint32_t yes = __ballot_sync(~0u, m >= hi || m < lo || bin_of(m) < b);
        const int i = yes ? __ffs(yes) - 1 : 32;     // the first that is
        const uint32_t next = lo + step * (i + 1);
        if (i < 32 && next < hi && next > lo) hi = next;
        lo += step * i;
      }
      if (lane == 0) border_key[warp] = hi;
    }
    __syncthreads();
    // keys from `whole` on stay, from `low` on are listed; so are those from k_low below k_high (bin_k may be bin2)
    const bool by_k = bin_k < kSampBins;
    const uint32_t whole = border_key[0], low = bin1 < kSampBins ? border_key[1] : whole;
    const uint32_t k_high = by_k ? border_key[2] : 0, k_low = by_k ? border_key[3] : 0;
    const uint32_t least_key = by_k ? min(k_low, low) : by_p ? border_key[4] : low;
    const auto note = [&](key_t k) {
      const uint32_t at = atomicAdd(&own_n, 1u);
      if (at < kList) {
        own[at] = k;
        own_warp[at] = (uint8_t)warp;
      }
    };
    for (int i = from + lane * kVec; i < from + run; i += 32 * kVec) {
      const uint4 raw = *(const uint4*)(keys + i);
      const key_t* k = (const key_t*)&raw;
      if (by_p && !by_k && least == 1 && weights.mode == 0) {
        // all weights count: no branch, but for the few that are listed
        u64 w[kVec];
        bool some = false;
#pragma unroll
        for (int e = 0; e < kVec; e++) w[e] = weights.of_near(K::value(k[e]), table);
#pragma unroll
        for (int e = 0; e < kVec; e++) {
          rest += w[e];
          if (k[e] >= whole) {
            all += w[e];
            count++;
          }
          some |= k[e] >= low && k[e] < whole;
        }
        if (some) {
#pragma unroll
          for (int e = 0; e < kVec; e++)
            if (k[e] >= low && k[e] < whole) {
              note(k[e]);
              rest -= w[e];
            }
        }
      } else {                                       // few do
#pragma unroll
        for (int e = 0; e < kVec; e++) {
          if (k[e] < least_key) continue;
          if ((k[e] < whole && k[e] >= low) || (k[e] < k_high && k[e] >= k_low)) {
            note(k[e]);
            continue;
          }
          const u64 w = weight(k[e]);
          rest += w;
          if (k[e] < whole) continue;
          all += w;
          if (w < least) continue;
          mass += w;
          count++;
        }
      }
    }
    rest -= all;
    if (by_p && !by_k && least == 1 && weights.mode == 0) mass = all;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      mass += __shfl_xor_sync(~0u, mass, o);
      all += __shfl_xor_sync(~0u, all, o);
      rest += __shfl_xor_sync(~0u, rest, o);
    }
    count = __reduce_add_sync(~0u, count);
    if (lane == 0) {
      warp_mass[warp] = all;
      warp_rest[warp] = rest;
    }
    __syncthreads();
    all = lane < kWarps ? warp_mass[lane] : 0;
    rest = lane < kWarps ? warp_rest[lane] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      all += __shfl_xor_sync(~0u, all, o);
      rest += __shfl_xor_sync(~0u, rest, o);
    }
    tell(2, {all, rest, own_n, 0});
    u64 before = 0, total = 0;                       // weight of the bins below bin1; of all but the list
    uint32_t m = 0;
    for (int q = 0; q < split; q++) {
      before += part[2][q].mass;
      total += part[2][q].mass + part[2][q].rest;
      m += min(part[2][q].count, kList + 1u);
    }
    by_list = true;
    if (m == 0 && !by_p) {
      open = false;                                  // top-k alone, and it leaves all that count
    } else if (m && m <= 32) {
      // ---- the row's list, sorted, by each warp for itself: lane i has place i
      uint32_t v = 0;
      if (lane < m) {
        uint32_t i = lane;
        int q = 0;
        while (i >= part[2][q].count) i -= part[2][q++].count;
        v = split > 1 ? ld_cluster_u32(cluster_map(smem_u32(own + i), q)) : own[i];
      }
#pragma unroll
      for (int k = 2; k <= 32; k *= 2) {
#pragma unroll
        for (int j = k / 2; j; j /= 2) {
          const uint32_t o = __shfl_xor_sync(~0u, v, j);
          v = ((lane & j) == 0) == ((lane & k) == 0) ? max(v, o) : min(v, o);
        }
      }
      open = false;
      uint32_t stay = m;                             // of the list, by top-k
      if (by_k) {
        stay = __popc(__ballot_sync(~0u, lane < m && bin_of(v) < bin_k)) + top_k - above_k;
        cut = __shfl_sync(~0u, v, stay - 1);
        take = stay - __popc(__ballot_sync(~0u, v > cut));
        limited = true;
      }
      if (by_p) {
        const u64 w = lane < stay ? weight(v) : 0;
        u64 in = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 u = __shfl_up_sync(~0u, in, o);
          if (lane >= o) in += u;
        }
        total += __shfl_sync(~0u, in, 31);
        const u64 want = max(1ull, (u64)ceil(fmax((double)top_p, 0.0) * (double)total));
        in += before;
        const uint32_t hit = __ballot_sync(~0u, in >= want && in - w < want && bin_of(v) <= bin2);
        if (hit == 0) {
          open = true;                               // (as below)
        } else {
          const int i = __ffs(hit) - 1;
          cut = __shfl_sync(~0u, v, i);
          take = i + 1 - __popc(__ballot_sync(~0u, v > cut));
          limited = true;
        }
      }
    } else if (m && m <= kList) {
      // ---- the row's list, sorted: thread t has places t and t + T
      uint32_t* const list = hist;
      for (uint32_t i = tid; i < m; i += T) {
        uint32_t at = i;
        int q = 0;
        while (at >= part[2][q].count) at -= part[2][q++].count;
        const uint32_t l = smem_u32(own + at);
        list[i] = split > 1 ? ld_cluster_u32(cluster_map(l, q)) : own[at];
      }
      uint32_t len = 32;
      while (len < m) len *= 2;
      for (uint32_t i = m + tid; i < len; i += T) list[i] = 0;
      __syncthreads();
      if (tid < len) {                               // whole warps
        uint32_t v[2];
        const uint32_t i1 = tid + T;
        const bool two = len > T;
        v[0] = list[tid];
        v[1] = two ? list[i1] : 0;
        const auto sync = [&] { asm volatile("bar.sync 1, %0;" ::"r"(min(len, (uint32_t)T)) : "memory"); };
        for (uint32_t k = 2; k <= len; k *= 2) {
          for (uint32_t j = k / 2; j; j /= 2) {
            if (j == T) {                            // both are this thread's
              const uint32_t x = max(v[0], v[1]), y = min(v[0], v[1]);
              v[0] = x;
              v[1] = y;
              continue;
            }
            uint32_t o[2] = {0, 0};
            if (j >= 32) {
              sync();
              list[tid] = v[0];
              if (two) list[i1] = v[1];
              sync();
              o[0] = list[tid ^ j];
              if (two) o[1] = list[i1 ^ j];
            } else {
              o[0] = __shfl_xor_sync(~0u, v[0], j);
              if (two) o[1] = __shfl_xor_sync(~0u, v[1], j);
            }
            // falling: of a pair the lower place has the larger one where bit k of the place is 0
            v[0] = ((tid & j) == 0) == ((tid & k) == 0) ? max(v[0], o[0]) : min(v[0], o[0]);
            if (two) v[1] = ((i1 & j) == 0) == ((i1 & k) == 0) ? max(v[1], o[1]) : min(v[1], o[1]);
          }
        }
        sync();
        list[tid] = v[0];
        if (two) list[i1] = v[1];
      }
      __syncthreads();
      // the first place of the list with a key of at most v
      const auto first_of = [&](uint32_t v) {
        uint32_t lo = 0, hi = m;
        while (lo < hi) {
          const uint32_t i = (lo + hi) / 2;
          if (list[i] > v) lo = i + 1; else hi = i;
        }
        return lo;
      };
      uint32_t stay = m;                             // of the list, by top-k
      if (by_k) {
        uint32_t lo = 0, hi = m;
        while (lo < hi) {
          const uint32_t i = (lo + hi) / 2;
          if (bin_of(list[i]) < bin_k) lo = i + 1; else hi = i;
        }
        stay = lo + (top_k - above_k);
        cut = list[stay - 1];
        take = stay - first_of(cut);
        limited = true;
      }
      open = false;
      if (by_p) {
        u64 w[2], sum = 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
          w[e] = 2 * tid + e < (int)stay ? weight(list[2 * tid + e]) : 0;
          sum += w[e];
        }
        u64 in = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 v = __shfl_up_sync(~0u, in, o);
          if (lane >= o) in += v;
        }
        if (lane == 31) warp_mass[warp] = in;
        if (tid == 0) found_bin = 0xffffffffu;
        __syncthreads();
        u64 sums = lane < kWarps ? warp_mass[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 v = __shfl_up_sync(~0u, sums, o);
          if (lane >= o) sums += v;
        }
        total += __shfl_sync(~0u, sums, 31);
        const u64 ahead = __shfl_sync(~0u, sums, max(warp - 1, 0));
        const u64 want = max(1ull, (u64)ceil(fmax((double)top_p, 0.0) * (double)total));
        u64 at = before + (warp ? ahead : 0) + in - sum;
#pragma unroll
        for (int e = 0; e < 2; e++) {
          if (at < want && at + w[e] >= want && bin_of(list[2 * tid + e]) <= bin2) found_bin = 2 * tid + e;
          at += w[e];
        }
        __syncthreads();
        if (found_bin == 0xffffffffu) {
          open = true;                               // (the bounds above leave this out; all CTAs agree on it)
        } else {
          cut = list[found_bin];
          take = found_bin + 1 - first_of(cut);
          limited = true;
        }
      }
    }
  }
  if (open) {
    // ---- digit by digit
    cut = K::kNone;
    take = count = 0;
    limited = by_list = false;
    mass = 0;
    meet();                                          // the list has been read
    uint32_t* const lo = hist;
    uint32_t* const hi = hist + kSampDigits;
    // One digit of a border.  The keys that stay so far and agree with `prefix` above this digit are summed by
    // digit over the row (their number, or their weights); from the largest digit down, the sums reach `want` (top_p of
    // the first level's total) in the digit that is returned.  `before` is what lies above it; returns -1 if the total stays below.
    const auto digit_of = [&](int level, uint32_t prefix, bool by_mass, u64& want, u64& before) {
      const int shift = K::shift(level), bits = K::bits(level), bins = 1 << bits;
      constexpr int kEach = kSampDigits / T;         // digits of a thread, from the top
      const auto agrees = [&](uint32_t k) { return level == 0 || k >> (shift + bits) == prefix; };
      for (int i = tid; i < bins; i += T) lo[i] = hi[i] = 0;
      if (tid == 0) found_bin = 0xffffffffu;
      __syncthreads();
      const auto add = [&](uint32_t k, u64 w) {
        const uint32_t bin = (k >> shift) & (bins - 1), l = (uint32_t)w, old = atomicAdd(&lo[bin], l);
        atomicAdd(&hi[bin], (uint32_t)(w >> 32) + (old + l < old));
      };
      for (int i = tid; i < size; i += T) {
        const uint32_t k = keys[i];
        if (k <= cut || !agrees(k)) continue;        // (those equal to the cut: below, as many as stay)
        if (by_mass) {
          const u64 w = weight(k);
          if (w) add(k, w);
        } else {
          atomicAdd(&lo[(k >> shift) & (bins - 1)], 1u);
        }
      }
      if (limited && by_mass && rank == 0 && tid == 0 && agrees(cut)) add(cut, weight(cut) * take);
      meet();
      u64 v[kEach], in = 0;
#pragma unroll
      for (int e = 0; e < kEach; e++) {
        const int bin = bins - 1 - kEach * tid - e;
        v[e] = 0;
        if (bin < 0) continue;
        const uint32_t l = smem_u32(&lo[bin]), h = smem_u32(&hi[bin]);
        if (split == 1) {
          v[e] = lo[bin] + ((u64)hi[bin] << 32);
        } else {
          for (int q = 0; q < split; q++)
            v[e] += ld_cluster_u32(cluster_map(l, q)) + (by_mass ? (u64)ld_cluster_u32(cluster_map(h, q)) << 32 : 0ull);
        }
        in += v[e];
      }
      u64 sum = in;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 b = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += b;
      }
      if (lane == 31) warp_mass[warp] = sum;
      __syncthreads();
      u64 warps = lane < kWarps ? warp_mass[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 b = __shfl_up_sync(~0u, warps, o);
        if (lane >= o) warps += b;
      }
      const u64 total = __shfl_sync(~0u, warps, 31), ahead = __shfl_sync(~0u, warps, max(warp - 1, 0));
      if (level == 0 && by_mass) want = max(1ull, (u64)ceil(fmax((double)top_p, 0.0) * (double)total));
      u64 at = (warp ? ahead : 0) + sum - in;
#pragma unroll
      for (int e = 0; e < kEach; e++) {
        if (at < want && at + v[e] >= want) {
          found_bin = bins - 1 - kEach * tid - e;
          found_mass = at;
        }
        at += v[e];
      }
      meet();                                        // found, and every CTA has read the sums
      before = found_mass;
      const int bin = (int)found_bin;
      __syncthreads();
      return bin;
    };
    const auto border = [&](bool by_mass, u64 want) {
      uint32_t prefix = 0;
      for (int level = 0; level < K::kLevels; level++) {
        u64 before;
        const int bin = digit_of(level, prefix, by_mass, want, before);
        if (bin < 0) return;                         // all of them stay
        want -= before;
        prefix = prefix << K::bits(level) | bin;
      }
      cut = prefix;
      const u64 w = by_mass ? weight(cut) : 1;
      take = (uint32_t)((want + w - 1) / w);
      limited = true;
    };
    if (top_k) border(false, top_k);
    if (by_p) border(true, 0);
  }

  // ---- what stays, by warp: a warp has a run of consecutive scores
  const u64 cut_w = limited ? weight(cut) : 0;
  if (cut_w < least) take = 0;
  uint32_t ties = 0;
  if (!by_list) {
    for (int i = from + lane; i < to; i += 32) {
      const uint32_t k = keys[i];
      ties += limited && k == cut;
      if (k <= cut) continue;
      const u64 w = weight(k);
      if (w < least) continue;
      mass += w;
      count++;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
    count = __reduce_add_sync(~0u, count);
    ties = __reduce_add_sync(~0u, ties);
  }
  __syncthreads();
  if (lane == 0) {
    warp_mass[warp] = mass;
    warp_a[warp] = count;
    warp_b[warp] = ties;
  }
  __syncthreads();
  if (by_list) {
    // of the bins that did not stay whole: the listed ones
    for (uint32_t i = tid; i < own_n; i += T) {
      const uint32_t k = own[i], of = own_warp[i];
      if (k < cut) continue;
      if (k == cut && limited) {
        atomicAdd(&warp_b[of], 1u);
        continue;
      }
      const u64 w = weight(k);
      if (w < least) continue;
      atomicAdd(&warp_mass[of], w);
      atomicAdd(&warp_a[of], 1u);
    }
    __syncthreads();
  }
  // lane i: warp i's
  mass = lane < kWarps ? warp_mass[lane] : 0;
  ties = lane < kWarps ? warp_b[lane] : 0;
  u64 cta_mass = mass;
#pragma unroll
  for (int o = 16; o; o >>= 1) cta_mass += __shfl_xor_sync(~0u, cta_mass, o);
  tell(1, {cta_mass, 0, __reduce_add_sync(~0u, lane < kWarps ? warp_a[lane] : 0), __reduce_add_sync(~0u, ties)});
  unsigned long long total = 0, start = 0;           // of the row; before this CTA
  uint32_t all = 0, ties_at = 0, tie_start = 0;
  for (int q = 0; q < split; q++) {
    if (q == rank) {
      start = total;
      tie_start = ties_at;
    }
    const uint32_t stay = min(part[1][q].ties, take - min(take, ties_at));
    total += part[1][q].mass + stay * cut_w;
    all += part[1][q].count + stay;
    ties_at += part[1][q].ties;
  }
  unsigned long long target = u > 0.f ? (unsigned long long)fmin((double)u * (double)total, 9e18) : 0;
  target = min(target, total - 1);
  // the first score at which the sum passes the target: its warp, then itself
  uint32_t tie_before = ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t b = __shfl_up_sync(~0u, tie_before, o);
    if (lane >= o) tie_before += b;
  }
  tie_before += tie_start - ties;
  mass += min(ties, take - min(take, tie_before)) * cut_w;
  unsigned long long end = mass;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long b = __shfl_up_sync(~0u, end, o);
    if (lane >= o) end += b;
  }
  end += start;
  const uint32_t has = __ballot_sync(~0u, lane < kWarps && target < end && target >= end - mass);
  if (!has) return;                                  // another CTA's (all of this one's warps see the same)
  const int who = __ffs(has) - 1;
  u64 at = __shfl_sync(~0u, end - mass, who);
  uint32_t tie = __shfl_sync(~0u, tie_before, who);
  // that warp's run, a score a thread and turn
  const int run_at = who * run, run_end = min(size, run_at + run);
  for (int i0 = run_at; i0 < run_end; i0 += T) {
    const uint32_t k = i0 + tid < run_end ? keys[i0 + tid] : 0;
    const bool same = limited && k == cut;
    const uint32_t sames = __ballot_sync(~0u, same);
    u64 w = k > cut ? weight(k) : 0;
    if (w < least) w = 0;
    __syncthreads();                                 // the last turn's sums have been read
    if (lane == 0) warp_b[warp] = __popc(sames);
    __syncthreads();
    if (same) {
      const uint32_t ahead = tie + __popc(sames & ((1u << lane) - 1));
      uint32_t more = 0;
      for (int i = 0; i < warp; i++) more += warp_b[i];
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
    u64 sums = lane < kWarps ? warp_mass[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 b = __shfl_up_sync(~0u, sums, o);
      if (lane >= o) sums += b;
    }
    const u64 ahead = __shfl_sync(~0u, sums, max(warp - 1, 0)), turn = __shfl_sync(~0u, sums, 31);
    s += at + (warp ? ahead : 0);
    if (s > target && s - w <= target) {             // one score of the row
      const float l = K::value(k);
      p.token[row] = first + i0 + tid;
      if (p.logprob) p.logprob[row] = (float)((l == top ? 0.0 : ((double)l - (double)top) / (double)temperature) - log((double)total / kSampOne));
      if (p.kept) p.kept[row] = (int)all;
    }
    at += turn;
    if (at > target) return;
    tie += __reduce_add_sync(~0u, lane < kWarps ? warp_b[lane] : 0);
  }
}

static int g_samp_split = 0, g_samp_kernel = 0;

template <int DT>
static int launch_sample(SampleArgs& a, cudaStream_t st) {
  const YkSample& p = a.p;
  constexpr int kVec = 16 / (DT == YK_F32 ? 4 : 2);
  const int sms = sm_count();
  // CTAs of a row: as many as the SMs have room for, each with scores for two a thread or more; and what one can hold.
  const auto split_for = [&](int most, bool whole) {
    int split = 1;
    while (split < 8 && (p.n > most * split || ((long long)p.rows * split * 2 <= (whole && split > 1 ? sms * 3 / 4 : sms) && p.n >= 4096 * split))) split *= 2;
    return split;
  };
  a.split = split_for(kSampSlice, false);
  bool by_place = false;
  if constexpr (DT != YK_F32) {
    // CTAs that count by place have an SM each (and clusters of 4 and 8 leave some without one).  From 16000 scores a CTA
    // on they take less time (64 x 128000: 31 us, by bins 62; 1 x 128000: 22 and 30; 64 x 32000: 22 and 29), below it
    // going through the places takes longer (1 x 32000: 20 and 19; 24 x 50000: 24 and 20; 1 x 4000: 20 and 11).
    const int split = split_for(kSamp16Slice, true);
    by_place = g_samp_kernel ? g_samp_kernel == 2 : p.n >= 16000 * split;
    if (by_place) a.split = split;
  }
  if (g_samp_split && p.n <= (by_place ? kSamp16Slice : kSampSlice) * g_samp_split) a.split = g_samp_split;
  const int width = p.n + (aligned16(p.logits) && p.row % kVec == 0 ? 0 : kVec - 1);   // with what may come before the row
  a.slice = ((width + a.split - 1) / a.split + 255) / 256 * 256;
  auto kern = sample_kernel<DT>;
  if constexpr (DT != YK_F32)
    if (by_place) kern = sample16_kernel<DT>;
  const int smem = by_place ? kSamp16Smem : a.slice * (DT == YK_F32 ? 4 : 2);
  if (smem_attr(kern, smem) != cudaSuccess) return check_launch("sample attr");
  launch_kc(kern, dim3((unsigned)((long long)p.rows * a.split)), by_place ? kSamp16Threads : kSampThreads, smem, a.split, st, a);
  note_launch();
  return check_launch("sample");
}

}  // namespace yk

using namespace yk;

extern "C" int yk_sample(const YkSample* p, yk_stream_t st) {
  if (!p || !p->logits || !p->token) return refuse(YK_EINVAL, "sample: null logits or token");
  if (p->dtype != YK_F16 && p->dtype != YK_BF16 && p->dtype != YK_F32) return refuse(YK_EUNSUP, "sample: dtype must be fp16, bf16 or fp32");
  if (p->rows < 0 || p->n < 1 || p->row < p->n) return refuse(YK_EINVAL, "sample: bad rows, n or row stride");
  if (p->n > 8 * kSampSlice || p->rows > 1 << 24) return refuse(YK_EUNSUP, "sample: at most 262144 scores a row and 2^24 rows");
  if ((uintptr_t)p->logits & (p->dtype == YK_F32 ? 3 : 1)) return refuse(YK_EINVAL, "sample: logits need the alignment of their type");
  if (((uintptr_t)p->temperature | (uintptr_t)p->top_k | (uintptr_t)p->top_p | (uintptr_t)p->min_p | (uintptr_t)p->u | (uintptr_t)p->token |
       (uintptr_t)p->logprob | (uintptr_t)p->kept) & 3)
    return refuse(YK_EINVAL, "sample: parameters and outputs need 4-byte alignment");
  if (p->rows == 0) return YK_OK;
  SampleArgs a{*p};
  cudaStream_t s = (cudaStream_t)st;
  return p->dtype == YK_F32 ? launch_sample<YK_F32>(a, s) : p->dtype == YK_BF16 ? launch_sample<YK_BF16>(a, s) : launch_sample<YK_F16>(a, s);
}

extern "C" int yk_test_sample(int split) {
  if (split < 0 || split > 8 || (split & (split - 1))) return YK_EINVAL;
  g_samp_split = split;
  return YK_OK;
}

extern "C" int yk_test_sample_kernel(int kernel) {
  if (kernel < 0 || kernel > 2) return YK_EINVAL;
  g_samp_kernel = kernel;
  return YK_OK;
}
