// Norm and rotary position of query and key heads (yk_qk_rotate).
#include "text.cuh"

namespace yk {

struct RotateArgs {
  YkQkRotate p;
  int slots;                     // heads side by side in a warp; its other lanes take further rows
  int q_steps, steps;            // steps of a warp's rows: those of queries, and with those of keys
  long long each;                // steps of a warp
  int more;                      // warps with one more
  int warp_bytes;                // shared memory of a warp
  int after[4];                  // pairs up to the end of each axis
};

// HBM bound: each row is read and written once.  A lane takes 16 channels of a head as two 16-byte chunks, such that the
// pairs that turn together are its own: chunks l and l + rot / 16 of the ones that turn, two neighbouring ones of the
// rest.  A head is dim / 16 neighbouring lanes: its sum of squares takes shuffles only.  A lane stays at its channels for
// all heads of a row, so weight times cosine and weight times sine are made once a row and kept in registers:
// y = inv (w c) x + inv (+-w' s) x'.  Loading them for each head made the kernel wait for its instructions
// (12000 rows of 32 + 8 heads of 128: 57.8 us; 44.9 us now, 5.5 TB/s; a copy in this shape 41 us).
// The work is cut into steps of kRotV heads a lane.  Warps stay and take equal runs of steps, from any head of
// any row on, as a grid of whole rows leaves its last wave half empty (54 us); the next steps are loaded into shared
// memory meanwhile, kRotStages - 1 ahead.  A call of few steps has a warp for each (64 rows of the same: 3.7 us).
// Angles: the turns of a position are held modulo one in units of 2^-64, good to the last of them for frequencies up to 2^40 (1 / 2 pi
// comes in two doubles), so an angle is within 2^-31 of a turn at any position of 31 bits and needs no 64-bit floats for each
// row.  A cosine is rounded to 32 bits, and w c again.
constexpr int kRotWarps = 4, kRotBlocks = 5;    // of a CTA; CTAs an SM
constexpr int kRotV = 2, kRotStages = 3;
constexpr int kRotStage = kRotV * 1024 + 256;   // a step's data, and the positions of a warp's rows: [4][16]

template <bool BF16, int L, bool INTER>
__global__ void __launch_bounds__(kRotWarps * 32, kRotBlocks) rotate_kernel(const __grid_constant__ RotateArgs a) {
  extern __shared__ __align__(16) uint8_t rot_smem[];
  __shared__ unsigned long long freq[128];           // of each pair: turns a position, in units of 2^-64, less whole turns
  __shared__ __align__(16) float weights[2][L * 16];
  const YkQkRotate& p = a.p;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int l = lane % L, slot = lane / L % a.slots, r = lane / L / a.slots, rows = 32 / L / a.slots;
  const int half = p.rot / 2, turning = p.rot / 16;
  const bool turns = l < turning;
  const int d0 = (turns ? l : 2 * turning + 2 * (l - turning)) * 8, d1 = turns ? (l + turning) * 8 : d0 + 8;
  uint8_t* mine = rot_smem + warp * a.warp_bytes;
  const uint32_t stage0 = smem_u32(mine);
  float2* turn = (float2*)(mine + kRotStages * kRotStage);   // (cos, sin): [row of the warp][pair]
  const long long w = (long long)blockIdx.x * kRotWarps + warp;
  const long long begin = w * a.each + min(w, (long long)a.more);
  const int todo = (int)(a.each + (w < a.more ? 1 : 0));
  long long group = begin / a.steps, igroup = group; // of the step at work, of the step being loaded
  int at = (int)(begin - group * a.steps), iat = at;
  pdl_wait();
  pdl_trigger();
  int issued = 0;
  const auto issue = [&]() {
    if (issued < todo) {
      const long long row = igroup * rows + r;
      const uint32_t dst = stage0 + issued % kRotStages * kRotStage;
      const bool key = iat >= a.q_steps;
      const int heads = row < p.rows ? key ? p.kv_heads : p.heads : 0, h0 = (key ? iat - a.q_steps : iat) * kRotV * a.slots + slot;
      const uint16_t* from = (key ? (const uint16_t*)p.k + row * p.k_row : (const uint16_t*)p.q + row * p.q_row) + h0 * (L * 16);
#pragma unroll
      for (int v = 0; v < kRotV; v++) {
        const bool ok = h0 + v * a.slots < heads;
        cp_async_at<16>(dst + v * 1024 + lane * 16, from + v * a.slots * (L * 16) + d0, ok);
        cp_async_at<16>(dst + v * 1024 + 512 + lane * 16, from + v * a.slots * (L * 16) + d1, ok);
      }
      if (iat == 0 || issued == 0) {
        for (int i = lane; i < p.axes * 16; i += 32) {
          const long long pr = igroup * rows + i % 16;
          const bool ok = i % 16 < rows && pr < p.rows;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + kRotV * 1024 + i * 4),
              "l"(ok ? p.pos + i / 16 * p.pos_axis + pr : p.pos), "r"(ok ? 4 : 0) : "memory");
        }
      }
      issued++;
      if (++iat == a.steps) {
        iat = 0;
        igroup++;
      }
    }
    cp_async_commit();
  };
#pragma unroll 1
  for (int i = 0; i < kRotStages - 1; i++) issue();
  for (int i = threadIdx.x; i < half; i += kRotWarps * 32) {
    // 1 / 2 pi in two doubles: the product's rounding error and the second one's share are a part of their own, far below a turn
    const double f = p.freqs[i], h = f * 0.15915494309189533577, e = fma(f, 0.15915494309189533577, -h) + f * -9.839338337591243e-18;
    freq[i] = (unsigned long long)__double2ll_rn((h - rint(h)) * 18446744073709551616.) +
              (unsigned long long)__double2ll_rn(e * 18446744073709551616.);
  }
  for (int i = threadIdx.x; i < 2 * L * 16; i += kRotWarps * 32) {
    const uint16_t* weight = (const uint16_t*)(i < L * 16 ? p.q_weight : p.k_weight);
    weights[i / (L * 16)][i % (L * 16)] = weight ? elem_to_float<BF16>(weight[i % (L * 16)]) : 1.f;
  }
  __syncthreads();
  float2 A[2][4], B[2][4];                           // y = A x + B x', x' the other of a pair
  bool there = false;
#pragma unroll 1
  for (int step = 0; step < todo; step++) {
    cp_async_wait<kRotStages - 2>();
    __syncwarp();
    const uint8_t* stage = mine + step % kRotStages * kRotStage;
    issue();
    const long long row = group * rows + r;
    const bool key = at >= a.q_steps;
    if (step == 0 || at == 0) {
      const int* pos = (const int*)(stage + kRotV * 1024);
      there = row < p.rows && pos[r] >= 0;
      for (int i = lane; i < rows * half; i += 32) {
        const int tr = i / half, pair = i - tr * half;
        const int axis = (pair >= a.after[0]) + (pair >= a.after[1]) + (pair >= a.after[2]);
        const int t = (int)((freq[pair] * (unsigned long long)pos[axis * 16 + tr]) >> 32);
        float s, c;
        sincospif((float)t * 4.656612873e-10f, &s, &c);   // 2^-31
        turn[i] = make_float2(c, s);
      }
      __syncwarp();
    }
    if (step == 0 || at == 0 || at == a.q_steps) {
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float4 u = *(const float4*)(weights[key] + (c ? d1 : d0) + 2 * e);
          A[c][e] = make_float2(u.x, u.y);
          A[c][e + 1] = make_float2(u.z, u.w);
        }
      if (turns) {
        const float2* t = turn + r * half;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (INTER) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const float2 u = t[(c ? l + turning : l) * 4 + e], v = A[c][e];
              A[c][e] = make_float2(v.x * u.x, v.y * u.x);
              B[c][e] = make_float2(-v.y * u.y, v.x * u.y);
            }
          } else {
            const float4 u = *(const float4*)(t + l * 8 + 2 * e);
            const float2 c = make_float2(u.x, u.z), s = make_float2(u.y, u.w), w0 = A[0][e], w1 = A[1][e];
            A[0][e] = fmul2(w0, c);
            A[1][e] = fmul2(w1, c);
            B[0][e] = fmul2(w1, make_float2(-s.x, -s.y));
            B[1][e] = fmul2(w0, s);
          }
        }
      }
    }
    const bool normed = (key ? p.k_weight : p.q_weight) != nullptr;
    const int heads = there ? key ? p.kv_heads : p.heads : 0, h0 = (key ? at - a.q_steps : at) * kRotV * a.slots + slot;
    uint16_t* to = (key ? (uint16_t*)p.k_out + row * p.k_out_row : (uint16_t*)p.q_out + row * p.q_out_row) + h0 * (L * 16);
#pragma unroll
    for (int v = 0; v < kRotV; v++) {
      float2 y[2][4], z[2][4];
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const uint4 x = *(const uint4*)(stage + v * 1024 + c * 512 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; e++) y[c][e] = pair_to_float2<BF16>(((const uint32_t*)&x)[e]);
      }
      if (normed) {
        float2 ss = make_float2(0.f, 0.f), st = ss;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          ss = ffma2(y[0][e], y[0][e], ss);
          st = ffma2(y[1][e], y[1][e], st);
        }
        float m = (ss.x + st.x) + (ss.y + st.y);
#pragma unroll
        for (int o = 1; o < L; o <<= 1) m += __shfl_xor_sync(~0u, m, o);
        const float inv = rsqrtf(fmaf(m, 1.f / (L * 16), p.eps));
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int e = 0; e < 4; e++) y[c][e] = fmul2(y[c][e], make_float2(inv, inv));
      }
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) z[c][e] = fmul2(y[c][e], A[c][e]);
      if (turns) {
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int e = 0; e < 4; e++) z[c][e] = ffma2(INTER ? make_float2(y[c][e].y, y[c][e].x) : y[c ^ 1][e], B[c][e], z[c][e]);
      }
      if (h0 + v * a.slots < heads) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] = float2_to_pair<BF16>(z[c][e].x, z[c][e].y);
          *(uint4*)(to + v * a.slots * (L * 16) + (c ? d1 : d0)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
    if (++at == a.steps) {
      at = 0;
      group++;
    }
  }
}

template <bool BF16, int L, bool INTER>
static int launch_rotate(const RotateArgs& in, cudaStream_t st) {
  RotateArgs a = in;
  const YkQkRotate& p = a.p;
  const auto steps = [](int heads, int s) { return (heads + s * kRotV - 1) / (s * kRotV); };
  const auto lanes = [&](int s) { return (steps(p.heads, s) + steps(p.kv_heads, s)) * s; };
  // as many heads side by side as leave the fewest lanes without one
  a.slots = 32 / L;
  for (int s = 16 / L; s; s /= 2)
    if (lanes(s) < lanes(a.slots)) a.slots = s;
  const int rows = 32 / L / a.slots;
  a.q_steps = steps(p.heads, a.slots);
  a.steps = a.q_steps + steps(p.kv_heads, a.slots);
  const long long all = (p.rows + (long long)rows - 1) / rows * a.steps;
  a.warp_bytes = kRotStages * kRotStage + (rows * p.rot * 4 + 15) / 16 * 16;
  const int bytes = kRotWarps * a.warp_bytes;
  const int fit = (227 << 10) / (bytes + 2048 + L * 128), blocks = fit < kRotBlocks ? fit : kRotBlocks;
  const long long want = (all + kRotWarps - 1) / kRotWarps, most = (long long)blocks * sm_count();
  const unsigned grid = (unsigned)(want < most ? want : most);
  a.each = all / (grid * kRotWarps);
  a.more = (int)(all % (grid * kRotWarps));
  if (ensure_smem_attr((const void*)rotate_kernel<BF16, L, INTER>, bytes) != cudaSuccess) return check_launch("qk_rotate");
  launch_k(rotate_kernel<BF16, L, INTER>, grid, kRotWarps * 32, bytes, st, a);
  note_launch();
  return check_launch("qk_rotate");
}
template <bool BF16, int L>
static int launch_rotate(const RotateArgs& a, cudaStream_t st) {
  return a.p.interleaved ? launch_rotate<BF16, L, true>(a, st) : launch_rotate<BF16, L, false>(a, st);
}
template <bool BF16>
static int launch_rotate(const RotateArgs& a, cudaStream_t st) {
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
  if (p->rows > 1 && ((p->q_out == p->q && p->q_out_row != p->q_row) || (kw && p->k_out == p->k && p->k_out_row != p->k_row)))
    return refuse(YK_EINVAL, "qk_rotate: rows in place have one stride");
  if (!aligned16(p->q) || !aligned16(p->q_out) || !aligned16(p->q_weight) || !aligned16(p->k_weight) ||
      (kw && (!aligned16(p->k) || !aligned16(p->k_out))))
    return refuse(YK_EINVAL, "qk_rotate: q, k, outputs and weights need 16-byte alignment");
  if (((uintptr_t)p->pos | (uintptr_t)p->freqs) & 3) return refuse(YK_EINVAL, "qk_rotate: pos and freqs need 4-byte alignment");
  if (!(p->eps >= 0.f)) return refuse(YK_EINVAL, "qk_rotate: bad eps");
  if (p->rows == 0) return YK_OK;
  return p->dtype == YK_BF16 ? launch_rotate<true>(a, (cudaStream_t)st) : launch_rotate<false>(a, (cudaStream_t)st);
}
