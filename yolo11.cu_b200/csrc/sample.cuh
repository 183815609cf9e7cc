// Shared by the kernels of yk_sample: its arguments, keys whose order is that of the scores, exact weights.
#pragma once
#include "text.cuh"

namespace yk {

struct SampleArgs {
  YkSample p;
  int split;         // CTAs of a row: a cluster
  int slice;         // scores of a CTA, a multiple of 256
};

// What stays (top-k, top-p, min-p) is always a beginning of one order, falling scores and equal ones by index, so it
// is described by a key and how many of the scores with that key stay.
// Weights are whole numbers, 2^44 for the largest, so that their sums do not depend on any order: the
// result is the same for every split.  They come from 64-bit exponentials: with 32 bits a sum over 10^5
// scores is off by about 10^-7 of the total, which would decide the token of one row in 10^2 to 10^4.
constexpr double kSampOne = 17592186044416.0;   // 2^44

struct SampPart {                          // what the CTAs of a row tell each other
  unsigned long long mass, rest;
  unsigned int count, ties;
};

__device__ __forceinline__ void st_cluster_u64(uint32_t a, unsigned long long v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

// Keys rise with the score; NaN has the least one, that of -infinity (kNone), and both zeros are equal.
template <int DT>
struct SampKey {
  using type = uint16_t;
  static constexpr int kLevels = 2;
  static constexpr uint32_t kInf = DT == YK_F16 ? 0x7c00u : 0x7f80u, kNone = 0x7fffu - kInf;
  __device__ static uint32_t of(uint16_t b) {
    const uint32_t m = b & 0x7fffu;
    if (m > kInf) return kNone;
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
  static constexpr int kLevels = 3;
  static constexpr uint32_t kNone = 0x007fffffu;
  __device__ static uint32_t of(uint32_t b) {
    const uint32_t m = b & 0x7fffffffu;
    if (m > 0x7f800000u) return kNone;
    if (m == 0) return 0x80000000u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  __device__ static float value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
  __device__ static constexpr int shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
  __device__ static constexpr int bits(int level) { return level == 2 ? 10 : 11; }
};

// Weights 2^44 exp((l - top) / temperature), rounded.  A power of two by a table and a short series (Tang, 1989):
// z = (l - top) log2(e) / temperature = n / 32 + r, 2^z = 2^(n / 32) (1 + r ln 2 + ..), within 2^-47.  A sum with a large constant
// rounds to a whole number, and a float becomes a double by its bits, for conversions are slow.  No branch parts a warp, so
// that several are in work at once.  The table is there 16 times, side by side: a lane reads its own banks.
struct SampWeights {
  float top;
  double c, at_top;                        // log2(e) / temperature, -top c
  int mode;                                // 0 as above; 1: l - top first, for a far top or a tiny temperature; 2: top is infinite
  __device__ void set(float top_, float temperature) {
    top = top_;
    c = 1.4426950408889634074 / (double)temperature;
    at_top = -(double)top * c;
    mode = top == INFINITY ? 2 : fabs(at_top) < 512. && c < 1e20 ? 0 : 1;
  }
  __device__ __forceinline__ static unsigned long long power(double z, const double* table) {
    const double t = z + 211106232532992.0;          // 1.5 * 2^52 / 32
    const int n = __double2loint(t);
    const double r = z - (t - 211106232532992.0);
    const double p = r * fma(r, fma(r, fma(r, fma(r, 0.0013333558146428443423, 0.0096181291076284771619), 0.055504108664821579953),
                                    0.24022650695910071233), 0.69314718055994530942);
    const double w = table[(n & 31) * 16 + (threadIdx.x & 15)];
    const double s = __hiloint2double(__double2hiint(w) + ((n >> 5) + 44) * 0x100000, __double2loint(w));
    const unsigned long long v = (unsigned long long)__double_as_longlong(fma(s, p, s) + 4503599627370496.0) & 0xfffffffffffffull;
    return (uint32_t)__double2hiint(z) < 0xc0470000u ? v : 0ull;     // z > -46
  }
  // Neither -2^128, which of_near takes for -infinity, nor 2^128 below the top, where the difference of two floats ends, weighs
  // anything (2^-64 of the top at most).  Not so at flat temperatures (above 7.6 10^36; a top near -2^128: above 4 10^29).
  __device__ bool steep() const { return (340282366920938463463374607431768211456.0 + fmin((double)top, 0.0)) * c >= 64.; }
  // mode 0 (of 0 and subnormal numbers 10^-38 off; a NaN gives anything)
  __device__ __forceinline__ unsigned long long of_near(float l, const double* table) const {
    const uint32_t b = __float_as_uint(l);
    const double d = __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
    return power(fma(d, c, at_top), table);
  }
  __device__ __forceinline__ unsigned long long of(float l, const double* table) const {
    if (mode == 0) return of_near(l, table);
    if (mode == 2) return l == top ? 1ull << 44 : 0ull;
    return power(((double)l - (double)top) * c, table);
  }
};

}  // namespace yk
