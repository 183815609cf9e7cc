// The next token of each row of scores: temperature, top-k, top-p, min-p, from given random numbers (yk_sample).
#include "text.cuh"

namespace yk {

struct SampleArgs {
  YkSample p;
  int split;         // CTAs of a row: a cluster
  int slice;         // scores of a CTA, a multiple of 8
  int vec;           // rows allow 16-byte loads
};

// A row's scores are read once, into the shared memory of a cluster, as keys whose order is that of the
// scores.  What stays (top-k, top-p, min-p) is always a beginning of one order, falling scores and equal ones by index, so
// it is described by a key and how many of the scores with that key stay.  Both borders are found
// digit by digit: counts (for top-p: weights) of the keys that share the digits so far, by digit, summed over the cluster.
// Weights are whole numbers, 2^44 for the largest, so that their sums do not depend on any order: the
// result is the same for every split.  They come from 64-bit exponentials: with 32 bits a sum over 10^5
// scores is off by about 10^-7 of the total, which would decide the token of one row in 10^2 to 10^4.
constexpr int kSampThreads = 1024, kSampWarps = kSampThreads / 32;
constexpr int kSampSlice = 32768;          // scores of a CTA at most
constexpr int kSampBins = 2048;
constexpr double kSampOne = 17592186044416.0;   // 2^44

struct SampPart {                          // what the CTAs of a row tell each other
  unsigned long long mass;
  unsigned int count, ties;
};

__device__ __forceinline__ void st_cluster_u64(uint32_t a, unsigned long long v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

// Keys: 0 for NaN and -infinity, else rising with the score; both zeros are equal.
template <int DT>
struct SampKey {
  using type = uint16_t;
  static constexpr int kBits = 16, kLevels = 2;
  __device__ static uint32_t of(uint16_t b) {
    const uint32_t inf = DT == YK_F16 ? 0x7c00u : 0x7f80u, m = b & 0x7fffu;
    if (m > inf || b == (0x8000u | inf)) return 0;
    if (m == 0) return 0x8000u;
    return b & 0x8000u ? (uint16_t)~b : b | 0x8000u;
  }
  __device__ static float value(uint32_t k) {
    const uint16_t b = k & 0x8000u ? (uint16_t)(k & 0x7fffu) : (uint16_t)~k;
    return elem_to_float<DT == YK_BF16>(b);
  }
  __device__ static constexpr int shift(int level) { return level == 0 ? 5 : 0; }
  __device__ static constexpr int bits(int level) { return level == 0 ? 11 : 5; }
};
template <>
struct SampKey<YK_F32> {
  using type = uint32_t;
  static constexpr int kBits = 32, kLevels = 3;
  __device__ static uint32_t of(uint32_t b) {
    const uint32_t m = b & 0x7fffffffu;
    if (m > 0x7f800000u || b == 0xff800000u) return 0;
    if (m == 0) return 0x80000000u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  __device__ static float value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
  __device__ static constexpr int shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
  __device__ static constexpr int bits(int level) { return level == 2 ? 10 : 11; }
};

// 2^44 exp((l - top) / temperature), rounded; c = log2(e) / temperature.
__device__ __forceinline__ unsigned long long samp_weight(float l, float top, double c) {
  if (l == top) return 1ull << 44;
  const double z = ((double)l - (double)top) * c;
  return z > -46.0 ? (unsigned long long)__double2ll_rn(exp2(z) * kSampOne) : 0ull;
}

template <int DT>
__global__ void __launch_bounds__(kSampThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  using K = SampKey<DT>;
  using key_t = typename K::type;
  constexpr int kVec = 16 / sizeof(key_t);
  extern __shared__ __align__(16) uint8_t samp_raw[];
  key_t* const keys = (key_t*)samp_raw;
  __shared__ uint32_t lo[kSampBins], hi[kSampBins];
  __shared__ SampPart part[2][8];                    // of the row's CTAs
  __shared__ unsigned long long warp_mass[kSampWarps];
  __shared__ uint32_t warp_a[kSampWarps], warp_b[kSampWarps];
  __shared__ unsigned long long found_mass;
  __shared__ uint32_t found_bin;
  const YkSample& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, split = a.split;
  const int row = blockIdx.x / split, rank = split > 1 ? (int)cluster_rank() : 0;
  const int first = rank * a.slice, size = max(0, min(a.slice, p.n - first));
  const auto meet = [&] { if (split > 1) cluster_barrier(); else __syncthreads(); };
  // this CTA's part to all of the row's, in turn `which`
  const auto tell = [&](int which, SampPart v) {
    if (tid < split) {
      const uint32_t to = smem_u32(&part[which][rank]), at = split > 1 ? cluster_map(to, tid) : to;
      st_cluster_u64(at, v.mass);
      st_cluster_u32(at + 8, v.count);
      st_cluster_u32(at + 12, v.ties);
    }
    meet();
  };
  pdl_wait();
  pdl_trigger();

  // ---- scores into shared memory, the largest
  uint32_t top_key = 0;
  {
    const key_t* from = (const key_t*)p.logits + row * p.row + first;
    if (a.vec) {
      for (int i = tid * kVec; i < size; i += kSampThreads * kVec) {
        key_t k[kVec];
        if (i + kVec <= size) {
          *(uint4*)k = *(const uint4*)(from + i);
        } else {
          for (int e = 0; e < kVec; e++) k[e] = i + e < size ? from[i + e] : 0;
        }
#pragma unroll
        for (int e = 0; e < kVec; e++) {
          k[e] = (key_t)(i + e < size ? K::of(k[e]) : 0);
          top_key = max(top_key, (uint32_t)k[e]);
        }
        *(uint4*)(keys + i) = *(const uint4*)k;
      }
    } else {
      for (int i = tid; i < (size + kVec - 1) / kVec * kVec; i += kSampThreads) {
        const key_t k = (key_t)(i < size ? K::of(from[i]) : 0);
        top_key = max(top_key, (uint32_t)k);
        keys[i] = k;
      }
    }
  }
  const auto block_max = [&](uint32_t v) {
    v = __reduce_max_sync(~0u, v);
    __syncthreads();
    if (lane == 0) warp_a[warp] = v;
    __syncthreads();
    return __reduce_max_sync(~0u, warp_a[lane]);
  };
  tell(0, {0, block_max(top_key), 0});
  for (int i = 0; i < split; i++) top_key = max(top_key, part[0][i].count);
  const float temperature = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !(temperature > 0.f) || !p.u;
  if (top_key == 0 || greedy) {
    // the lowest index of the largest score
    uint32_t at = 0xffffffffu;
    if (top_key)
      for (int i = tid; i < size; i += kSampThreads)
        if (keys[i] == top_key) at = min(at, (uint32_t)(first + i));
    at = ~block_max(~at);
    tell(1, {0, at, 0});
    for (int i = 0; i < split; i++) at = min(at, part[1][i].count);
    if (rank == 0 && tid == 0) {
      p.token[row] = top_key ? (int)at : -1;
      if (p.logprob) p.logprob[row] = top_key ? 0.f : -INFINITY;
      if (p.kept) p.kept[row] = top_key ? 1 : 0;
    }
    return;
  }
  const float top = K::value(top_key);
  const double c = 1.4426950408889634074 / (double)temperature;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const int top_k = p.top_k ? p.top_k[row] : 0;

  // Keys above `cut` stay, and of those that equal it the first `take`.
  uint32_t cut = 0, take = 0;
  bool limited = false;                              // by the cut
  // One digit of a border.  The keys that stay so far and agree with `prefix` above this digit are summed by
  // digit over the row (their number, or their weights); from the largest digit down, the sums reach `want` (top_p of
  // the first level's total) in the digit that is returned.  `before` is what lies above it; returns -1 if the total stays below.
  const auto digit_of = [&](int level, uint32_t prefix, bool by_mass, unsigned long long& want, unsigned long long& before) {
    const int shift = K::shift(level), bits = K::bits(level), bins = 1 << bits;
    const auto agrees = [&](uint32_t k) { return level == 0 || k >> (shift + bits) == prefix; };
    for (int i = tid; i < bins; i += kSampThreads) lo[i] = hi[i] = 0;
    if (tid == 0) found_bin = 0xffffffffu;
    __syncthreads();
    const auto add = [&](uint32_t k, unsigned long long w) {
      const uint32_t bin = (k >> shift) & (bins - 1), l = (uint32_t)w, old = atomicAdd(&lo[bin], l);
      atomicAdd(&hi[bin], (uint32_t)(w >> 32) + (old + l < old));
    };
    for (int i = tid; i < size; i += kSampThreads) {
      const uint32_t k = keys[i];
      if (k <= cut || !agrees(k)) continue;          // (those equal to the cut: below, as many as stay)
      if (by_mass) {
        const unsigned long long w = samp_weight(K::value(k), top, c);
        if (w) add(k, w);
      } else {
        atomicAdd(&lo[(k >> shift) & (bins - 1)], 1u);
      }
    }
    if (limited && by_mass && rank == 0 && tid == 0 && agrees(cut)) add(cut, samp_weight(K::value(cut), top, c) * take);
    meet();
    // thread t: the t-th two digits from the top
    unsigned long long v[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int bin = bins - 1 - 2 * tid - e;
      if (bin < 0) continue;
      const uint32_t l = smem_u32(&lo[bin]), h = smem_u32(&hi[bin]);
      if (split == 1) {
        v[e] = lo[bin] + ((unsigned long long)hi[bin] << 32);
      } else {
        for (int q = 0; q < split; q++)
          v[e] += ld_cluster_u32(cluster_map(l, q)) + (by_mass ? (unsigned long long)ld_cluster_u32(cluster_map(h, q)) << 32 : 0ull);
      }
    }
    unsigned long long sum = v[0] + v[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long b = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += b;
    }
    if (lane == 31) warp_mass[warp] = sum;
    __syncthreads();
    unsigned long long warps = warp_mass[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long b = __shfl_up_sync(~0u, warps, o);
      if (lane >= o) warps += b;
    }
    const unsigned long long total = __shfl_sync(~0u, warps, 31), above = __shfl_sync(~0u, warps, max(warp - 1, 0));
    if (level == 0 && by_mass) want = max(1ull, (unsigned long long)ceil((double)top_p * (double)total));
    unsigned long long at = (warp ? above : 0) + sum - v[0] - v[1];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (at < want && at + v[e] >= want) {
        found_bin = bins - 1 - 2 * tid - e;
        found_mass = at;
      }
      at += v[e];
    }
    meet();                                          // found, and every CTA has read the sums
    before = found_mass;
    const int bin = (int)found_bin;
    __syncthreads();
    return bin;
  };
  const auto border = [&](bool by_mass, unsigned long long want) {
    uint32_t prefix = 0;
    for (int level = 0; level < K::kLevels; level++) {
      unsigned long long before;
      const int bin = digit_of(level, prefix, by_mass, want, before);
      if (bin < 0) return;                           // all of them stay
      want -= before;
      prefix = prefix << K::bits(level) | bin;
    }
    cut = prefix;
    const unsigned long long w = by_mass ? samp_weight(K::value(cut), top, c) : 1;
    take = (uint32_t)((want + w - 1) / w);
    limited = true;
  };
  if (top_k > 0 && top_k < p.n) border(false, top_k);
  if (top_p < 1.f) border(true, 0);

  // ---- what stays, by warp: a warp has a run of consecutive scores
  const unsigned long long least = p.min_p && p.min_p[row] > 0.f ? (unsigned long long)ceil(fmin((double)p.min_p[row], 1.0) * kSampOne) : 1ull;
  const unsigned long long cut_w = limited ? samp_weight(K::value(cut), top, c) : 0;
  if (cut_w < least) take = 0;
  const int run = a.slice / kSampWarps, from = warp * run, to = min(size, from + run);
  unsigned long long mass = 0;
  uint32_t count = 0, ties = 0;
  for (int i = from + lane; i < to; i += 32) {
    const uint32_t k = keys[i];
    ties += limited && k == cut;
    if (k <= cut) continue;
    const unsigned long long w = samp_weight(K::value(k), top, c);
    if (w < least) continue;
    mass += w;
    count++;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
  count = __reduce_add_sync(~0u, count);
  ties = __reduce_add_sync(~0u, ties);
  __syncthreads();
  if (lane == 0) {
    warp_mass[warp] = mass;
    warp_a[warp] = count;
    warp_b[warp] = ties;
  }
  __syncthreads();
  // lane i: warp i's
  mass = warp_mass[lane];
  ties = warp_b[lane];
  unsigned long long cta_mass = mass;
#pragma unroll
  for (int o = 16; o; o >>= 1) cta_mass += __shfl_xor_sync(~0u, cta_mass, o);
  tell(1, {cta_mass, __reduce_add_sync(~0u, warp_a[lane]), __reduce_add_sync(~0u, ties)});
  unsigned long long total = 0, start = 0;           // of the row; before this CTA
  uint32_t all = 0, tie_at = 0, tie_start = 0;
  for (int q = 0; q < split; q++) {
    if (q == rank) {
      start = total;
      tie_start = tie_at;
    }
    const uint32_t stay = min(part[1][q].ties, take - min(take, tie_at));
    total += part[1][q].mass + stay * cut_w;
    all += part[1][q].count + stay;
    tie_at += part[1][q].ties;
  }
  const float u = p.u[row];
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
  const bool mine = target < end && target >= end - mass;
  if (!(__ballot_sync(~0u, mine) >> warp & 1)) return;
  unsigned long long at = __shfl_sync(~0u, end - mass, warp);
  uint32_t tie = __shfl_sync(~0u, tie_before, warp);
  for (int i0 = from; i0 < to; i0 += 32) {
    const uint32_t k = i0 + lane < to ? keys[i0 + lane] : 0;
    const bool same = limited && k == cut;
    const uint32_t sames = __ballot_sync(~0u, same);
    unsigned long long w = 0;
    if (k > cut) w = samp_weight(K::value(k), top, c);
    if (w < least) w = 0;
    if (same && tie + __popc(sames & ((1u << lane) - 1)) < take) w = cut_w;
    unsigned long long s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long b = __shfl_up_sync(~0u, s, o);
      if (lane >= o) s += b;
    }
    const uint32_t past = __ballot_sync(~0u, at + s > target);
    if (past) {
      if (lane == __ffs(past) - 1) {
        const float l = K::value(k);
        p.token[row] = first + i0 + lane;
        if (p.logprob) p.logprob[row] = (float)((l == top ? 0.0 : ((double)l - (double)top) / (double)temperature) - log((double)total / kSampOne));
        if (p.kept) p.kept[row] = (int)all;
      }
      return;
    }
    at += __shfl_sync(~0u, s, 31);
    tie += __popc(sames);
  }
}

static int g_samp_split = 0;

template <int DT>
static int launch_sample(SampleArgs& a, cudaStream_t st) {
  const YkSample& p = a.p;
  // CTAs of a row: as many as the SMs have room for, each with scores for two a thread; and what shared memory asks for
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  a.split = 1;
  while (a.split < 8 && (p.n > kSampSlice * a.split || ((long long)p.rows * a.split * 2 <= sms && p.n >= 4096 * a.split))) a.split *= 2;
  if (g_samp_split && p.n <= kSampSlice * g_samp_split) a.split = g_samp_split;
  a.slice = ((p.n + a.split - 1) / a.split + 255) / 256 * 256;
  a.vec = aligned16(p.logits) && p.row % (16 / (DT == YK_F32 ? 4 : 2)) == 0;
  const int smem = a.slice * (DT == YK_F32 ? 4 : 2);
  const auto kern = sample_kernel<DT>;
  if (smem_attr(kern, smem) != cudaSuccess) return check_launch("sample attr");
  launch_kc(kern, dim3((unsigned)((long long)p.rows * a.split)), kSampThreads, smem, a.split, st, a);
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
