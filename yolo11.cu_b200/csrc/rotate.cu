// Norm and rotary position of query and key heads (yk_qk_rotate).
#include "text.cuh"

namespace yk {

struct RotateArgs {
  YkQkRotate p;
  int items;         // 32-byte pieces of a row: (heads + kv_heads) * dim / 16
  uint32_t magic;    // ceil(2^32 / items): i / items = umulhi(i, magic) below 2^17
  int rows;          // of a CTA
  int after[4];      // pairs up to the end of each axis
};

// HBM bound: each row is read and written once.  A thread takes 16 channels of a head as two 16-byte chunks,
// such that the pairs that turn together are its own: chunks l and l + rot / 16 of the ones that
// turn, two neighbouring ones of the rest.  A head is dim / 16 neighbouring lanes: its sum of squares takes
// shuffles only.  The CTA's rows share one table of cosines and sines, made while the first rows are on their way:
// angle / 2 pi in 64 bits, less its whole turns, then 32 bits.
constexpr int kRotThreads = 256, kRotRows = 8;

template <bool BF16, int L, bool INTER, int V>
__global__ void __launch_bounds__(kRotThreads) rotate_kernel(const __grid_constant__ RotateArgs a) {
  __shared__ float2 turn[kRotRows * 128];            // [row][pair]
  __shared__ int there[kRotRows];
  const YkQkRotate& p = a.p;
  const int tid = threadIdx.x, l = tid % L, half = p.rot / 2, turning = p.rot / 16;
  const long long row0 = (long long)blockIdx.x * a.rows;
  const int rows = (int)min((long long)a.rows, p.rows - row0), all = rows * a.items;
  const bool turns = l < turning;
  const int c0 = turns ? l : turning + l, c1 = turns ? l + turning : turning + l + 1;   // chunks (the rest in twos)
  const int d0 = (turns ? c0 : 2 * turning + 2 * (l - turning)) * 8, d1 = turns ? c1 * 8 : d0 + 8;
  pdl_wait();
  pdl_trigger();
  uint4 w[2][2];                                     // weights of queries and of keys
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint16_t* weight = (const uint16_t*)(i ? p.k_weight : p.q_weight);
    w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
    if (weight) {
      w[i][0] = *(const uint4*)(weight + d0);
      w[i][1] = *(const uint4*)(weight + d1);
    }
  }
  for (int i0 = 0; i0 < all; i0 += kRotThreads * V) {
    uint4 x[V][2];
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int i = i0 + v * kRotThreads + tid, r = (int)__umulhi((uint32_t)i, a.magic), h = (i - r * a.items) / L;
      x[v][0] = x[v][1] = make_uint4(0, 0, 0, 0);
      if (i >= all) continue;
      const uint16_t* from = h < p.heads ? (const uint16_t*)p.q + (row0 + r) * p.q_row + h * (L * 16)
                                         : (const uint16_t*)p.k + (row0 + r) * p.k_row + (h - p.heads) * (L * 16);
      x[v][0] = __ldcs((const uint4*)(from + d0));
      x[v][1] = __ldcs((const uint4*)(from + d1));
    }
    if (i0 == 0) {
      for (int i = tid; i < rows * half; i += kRotThreads) {
        const int r = i / half, pair = i - r * half;
        const int axis = (pair >= a.after[0]) + (pair >= a.after[1]) + (pair >= a.after[2]);
        double t = (double)p.pos[axis * p.pos_axis + row0 + r] * (double)p.freqs[pair] * 0.15915494309189533577;   // 1 / 2 pi
        t -= rint(t);
        float s, c;
        sincospif(2.f * (float)t, &s, &c);
        turn[i] = make_float2(c, s);
      }
      if (tid < rows) there[tid] = p.pos[row0 + tid] >= 0;
      __syncthreads();
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int i = i0 + v * kRotThreads + tid, r = (int)__umulhi((uint32_t)i, a.magic), h = (i - r * a.items) / L;
      const bool key = h >= p.heads;
      float2 y[2][4];
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          y[c][e] = pair_to_float2<BF16>(((const uint32_t*)&x[v][c])[e]);
          ss = ffma2(y[c][e], mul2(y[c][e], make_float2(1.f / (L * 16), 1.f / (L * 16))), ss);
        }
      float m = ss.x + ss.y;
#pragma unroll
      for (int o = 1; o < L; o <<= 1) m += __shfl_xor_sync(~0u, m, o);
      if (key ? p.k_weight != nullptr : p.q_weight != nullptr) {
        const float inv = rsqrtf(m + p.eps);
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const uint4 wc = key ? w[1][c] : w[0][c];
#pragma unroll
          for (int e = 0; e < 4; e++) y[c][e] = mul2(y[c][e], mul2(make_float2(inv, inv), pair_to_float2<BF16>(((const uint32_t*)&wc)[e])));
        }
      }
      if (i >= all || !there[r]) continue;
      if (turns) {
        const float4* t0 = (const float4*)(turn + r * half + (INTER ? c0 * 4 : l * 8));
        const float4* t1 = INTER ? (const float4*)(turn + r * half + c1 * 4) : t0 + 2;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (INTER) {
            // chunk c holds pairs 4 c .. 4 c + 3, each in one register pair
            const float4 u = t0[e >> 1], s = t1[e >> 1];
            const float2 ta = e & 1 ? make_float2(u.z, u.w) : make_float2(u.x, u.y), tb = e & 1 ? make_float2(s.z, s.w) : make_float2(s.x, s.y);
            y[0][e] = make_float2(y[0][e].x * ta.x - y[0][e].y * ta.y, y[0][e].y * ta.x + y[0][e].x * ta.y);
            y[1][e] = make_float2(y[1][e].x * tb.x - y[1][e].y * tb.y, y[1][e].y * tb.x + y[1][e].x * tb.y);
          } else {
            // pairs 8 l + 2 e and 8 l + 2 e + 1: (c, s, c', s')
            const float4 u = e < 2 ? t0[e] : t1[e - 2];
            const float2 c = make_float2(u.x, u.z), s = make_float2(u.y, u.w), n = make_float2(-u.y, -u.w), b = y[0][e];
            y[0][e] = ffma2(y[0][e], c, mul2(y[1][e], n));
            y[1][e] = ffma2(y[1][e], c, mul2(b, s));
          }
        }
      }
      uint16_t* to = key ? (uint16_t*)p.k_out + (row0 + r) * p.k_out_row + (h - p.heads) * (L * 16)
                         : (uint16_t*)p.q_out + (row0 + r) * p.q_out_row + h * (L * 16);
#pragma unroll
      for (int c = 0; c < 2; c++) {
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = float2_to_pair<BF16>(y[c][e].x, y[c][e].y);
        *(uint4*)(to + (c ? d1 : d0)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
}

template <bool BF16, int L>
static void launch_rotate(const RotateArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.p.rows + a.rows - 1ll) / a.rows);
  if (a.p.interleaved) launch_k(rotate_kernel<BF16, L, true, 4>, grid, kRotThreads, 0, st, a);
  else launch_k(rotate_kernel<BF16, L, false, 4>, grid, kRotThreads, 0, st, a);
}
template <bool BF16>
static void launch_rotate(const RotateArgs& a, cudaStream_t st) {
  switch (a.p.dim) {
    case 32: return launch_rotate<BF16, 2>(a, st);
    case 64: return launch_rotate<BF16, 4>(a, st);
    case 128: return launch_rotate<BF16, 8>(a, st);
    default: return launch_rotate<BF16, 16>(a, st);
  }
}

}  // namespace yk

using namespace yk;

extern "C" int yk_qk_rotate(const YkQkRotate* p, yk_stream_t st) {
  if (!p || !p->q || !p->q_out || !p->pos || !p->freqs || (p->kv_heads && (!p->k || !p->k_out)))
    return refuse(YK_EINVAL, "qk_rotate: null pointer");
  if (p->dtype != YK_F16 && p->dtype != YK_BF16) return refuse(YK_EUNSUP, "qk_rotate: dtype must be fp16 or bf16");
  if (p->dim != 32 && p->dim != 64 && p->dim != 128 && p->dim != 256) return refuse(YK_EUNSUP, "qk_rotate: dim must be 32, 64, 128 or 256");
  if (p->rows < 0 || p->heads < 1 || p->kv_heads < 0) return refuse(YK_EINVAL, "qk_rotate: bad rows or heads");
  if (p->heads > 1024 || p->kv_heads > 1024 || p->heads + p->kv_heads > 1024) return refuse(YK_EUNSUP, "qk_rotate: at most 1024 heads");
  if (p->rot < 16 || p->rot > p->dim || p->rot % 16) return refuse(YK_EINVAL, "qk_rotate: rot must be a multiple of 16, at most dim");
  if (p->axes < 1 || p->axes > 4) return refuse(YK_EINVAL, "qk_rotate: axes must be 1 to 4");
  RotateArgs a{*p};
  int pairs = 0;
  for (int i = 0; i < 4; i++) {
    const int n = p->sections[i];
    if (n < 0 || n > p->rot / 2 || (i >= p->axes && n)) return refuse(YK_EINVAL, "qk_rotate: bad sections");
    a.after[i] = pairs += n;
  }
  if (p->axes == 1 && pairs == 0)
    for (int i = 0; i < 4; i++) a.after[i] = p->rot / 2;
  else if (pairs != p->rot / 2)
    return refuse(YK_EINVAL, "qk_rotate: sections must hold rot / 2 pairs in all");
  const long long qw = (long long)p->heads * p->dim, kw = (long long)p->kv_heads * p->dim;
  if ((p->q_row | p->q_out_row) % 8 || p->q_row < qw || p->q_out_row < qw || (p->axes > 1 && p->pos_axis < p->rows) ||
      (kw && ((p->k_row | p->k_out_row) % 8 || p->k_row < kw || p->k_out_row < kw)))
    return refuse(YK_EINVAL, "qk_rotate: row strides are multiples of 8 that hold a row, pos_axis at least rows");
  if (!aligned16(p->q) || !aligned16(p->q_out) || !aligned16(p->q_weight) || !aligned16(p->k_weight) ||
      (kw && (!aligned16(p->k) || !aligned16(p->k_out))))
    return refuse(YK_EINVAL, "qk_rotate: q, k, outputs and weights need 16-byte alignment");
  if (((uintptr_t)p->pos | (uintptr_t)p->freqs) & 3) return refuse(YK_EINVAL, "qk_rotate: pos and freqs need 4-byte alignment");
  if (!(p->eps >= 0.f)) return refuse(YK_EINVAL, "qk_rotate: bad eps");
  if (p->rows == 0) return YK_OK;
  a.items = (p->heads + p->kv_heads) * (p->dim / 16);
  a.magic = (uint32_t)((0x100000000ull + a.items - 1) / a.items);
  // a CTA's rows fill its four pieces a thread, while there are rows for two CTAs an SM
  a.rows = 1;
  while (a.rows < kRotRows && (a.rows + 1) * a.items <= 4 * kRotThreads && p->rows / (a.rows + 1) >= 296) a.rows++;
  if (p->dtype == YK_BF16) launch_rotate<true>(a, (cudaStream_t)st);
  else launch_rotate<false>(a, (cudaStream_t)st);
  note_launch();
  return check_launch("qk_rotate");
}
