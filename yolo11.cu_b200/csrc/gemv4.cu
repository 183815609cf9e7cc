// Products of a few rows with a 4-bit weight matrix (yk_gemv4).
#include "text.cuh"

namespace yk {

// One warp an output: its lanes walk the weight row in chunks of 32 weights (16 bytes), and
// each chunk meets up to 8 rows of x.
template <bool BF16, bool X8>
__global__ void __launch_bounds__(256) gemv4_kernel(const __grid_constant__ YkGemv4 p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long j = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (j >= p.n) return;
  const uint8_t* w = (const uint8_t*)p.w + j * p.w_row;
  for (int m0 = 0; m0 < p.rows; m0 += 8) {
    float acc[8] = {};
    for (int c = lane; c < p.k / 32; c += 32) {
      const uint4 v = *(const uint4*)(w + c * 16);
      const uint32_t* u = (const uint32_t*)&v;
      const int g = c * 32 / p.group;
      const float s = elem_to_float<BF16>(((const uint16_t*)p.wscale)[j * p.group_row + g]);
      const float z = p.wzero ? (float)((const uint8_t*)p.wzero)[j * p.group_row + g] : 8.f;
#pragma unroll
      for (int m = 0; m < 8; m++) {
        if (m0 + m >= p.rows) break;
        float d = 0.f;
        const long long xo = (m0 + m) * p.x_row + c * 32;
#pragma unroll
        for (int i = 0; i < 32; i++) {
          const float q = (float)((u[i >> 3] >> (4 * (i & 7))) & 15) - z;
          const float xv = X8 ? e4m3x2_to_float2(((const uint8_t*)p.x)[xo + i]).x
                              : elem_to_float<BF16>(((const uint16_t*)p.x)[xo + i]);
          d = fmaf(q, xv, d);
        }
        if (X8) d *= p.xscale[(m0 + m) * p.xscale_row + (p.xgroup ? c * 32 / p.xgroup : 0)];
        acc[m] = fmaf(d, s, acc[m]);
      }
    }
#pragma unroll
    for (int m = 0; m < 8; m++) {
      const float t = warp_sum(acc[m]);
      if (lane == 0 && m0 + m < p.rows)
        ((uint16_t*)p.y)[(m0 + m) * p.y_row + j] = float_to_elem<BF16>(t + (p.bias ? p.bias[j] : 0.f));
    }
  }
}

}  // namespace yk

using namespace yk;

extern "C" int yk_gemv4(const YkGemv4* p, yk_stream_t st) {
  if (!p || !p->x || !p->w || !p->wscale || !p->y) return refuse(YK_EINVAL, "gemv4: null pointer");
  if (p->dtype != YK_F16 && p->dtype != YK_BF16) return refuse(YK_EUNSUP, "gemv4: dtype must be fp16 or bf16");
  if (p->xtype != p->dtype && p->xtype != YK_E4M3)
    return refuse(YK_EUNSUP, "gemv4: xtype must be dtype or e4m3");
  if (p->rows < 1 || p->n < 1 || p->k < 1) return refuse(YK_EINVAL, "gemv4: rows, n and k must be positive");
  if (p->rows > 64) return refuse(YK_EUNSUP, "gemv4: at most 64 rows");
  if (p->group != 32 && p->group != 64 && p->group != 128)
    return refuse(YK_EUNSUP, "gemv4: group must be 32, 64 or 128");
  if (p->k % p->group) return refuse(YK_EINVAL, "gemv4: k must be a multiple of group");
  const bool x8 = p->xtype == YK_E4M3;
  if (x8 && (!p->xscale || p->xgroup < 0 || p->xgroup % p->group))
    return refuse(YK_EINVAL, "gemv4: e4m3 rows need scales, and an xgroup that is a multiple of group");
  if (!aligned16(p->w) || p->w_row % 16 || p->w_row < p->k / 2 || p->group_row < p->k / p->group ||
      p->x_row < 0 || p->y_row < p->n)
    return refuse(YK_EINVAL, "gemv4: weights need 16-byte alignment, strides at least a row");
  if (x8 && p->xscale_row < (p->xgroup ? (p->k + p->xgroup - 1) / p->xgroup : 1))
    return refuse(YK_EINVAL, "gemv4: xscale stride below its row");
  const auto kern = p->dtype == YK_BF16 ? (x8 ? gemv4_kernel<true, true> : gemv4_kernel<true, false>)
                                        : (x8 ? gemv4_kernel<false, true> : gemv4_kernel<false, false>);
  launch_k(kern, (p->n + 7) / 8, 256, 0, (cudaStream_t)st, *p);
  note_launch();
  return check_launch("gemv4");
}
