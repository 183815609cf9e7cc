// Residual addition, RMS norm and 8-bit output with scales (yk_rmsnorm8).
#include "text.cuh"

namespace yk {

// One CTA a row, the row in shared memory as fp32 between the three passes over it (sum of
// squares, group maxima, rounding): each element is read from and written to HBM once.
template <bool BF16>
__global__ void rmsnorm8_kernel(const __grid_constant__ YkRmsNorm8 p, int group, int groups) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ float row_sm[];      // [cols] then [groups]
  __shared__ float part[32];
  const int C = p.cols, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long r = blockIdx.x;
  float* scale_sm = row_sm + C;
  const uint16_t* x = (const uint16_t*)p.x + r * p.x_row;
  const uint16_t* add = p.add ? (const uint16_t*)p.add + r * p.add_row : nullptr;
  uint16_t* sum = p.sum ? (uint16_t*)p.sum + r * p.sum_row : nullptr;
  const float over_c = 1.f / (float)C;
  float ss = 0.f;
  for (int c = threadIdx.x; c < C; c += blockDim.x) {
    float h = elem_to_float<BF16>(x[c]);
    if (add) h += elem_to_float<BF16>(add[c]);
    if (sum) sum[c] = float_to_elem<BF16>(h);
    row_sm[c] = h;
    ss = fmaf(h, h * over_c, ss);   // the mean itself: the sum would overflow sooner
  }
  ss = warp_sum(ss);
  if (lane == 0) part[warp] = ss;
  __syncthreads();
  ss = warp_sum(lane < warps ? part[lane] : 0.f);
  const float inv = rsqrtf(ss + p.eps);
  const uint16_t* w = (const uint16_t*)p.weight;
  uint16_t* out = p.out ? (uint16_t*)p.out + r * p.out_row : nullptr;
  for (int c = threadIdx.x; c < C; c += blockDim.x) {
    const float y = row_sm[c] * inv * elem_to_float<BF16>(w[c]);
    row_sm[c] = y;
    if (out) out[c] = float_to_elem<BF16>(y);
  }
  if (!p.codes) return;
  __syncthreads();
  for (int g = warp; g < groups; g += warps) {
    float m = 0.f;
    for (int c = g * group + lane; c < min(C, (g + 1) * group); c += 32) m = fmaxf(m, finite_abs(row_sm[c]));
    m = warp_max(m);
    const float s = fmaxf(m / kE4m3Max, kMinScale);
    if (lane == 0) {
      p.scales[r * p.scales_row + g] = s;
      scale_sm[g] = 1.f / s;
    }
  }
  __syncthreads();
  uint8_t* codes = (uint8_t*)p.codes + r * p.codes_row;
  for (int c = threadIdx.x; c < C; c += blockDim.x)
    codes[c] = (uint8_t)float2_to_e4m3x2(row_sm[c] * scale_sm[c / group], 0.f);
}

}  // namespace yk

using namespace yk;

extern "C" int yk_rmsnorm8(const YkRmsNorm8* p, yk_stream_t st) {
  if (!p || !p->x || !p->weight) return refuse(YK_EINVAL, "rmsnorm8: null x or weight");
  if (!p->sum && !p->out && !p->codes) return refuse(YK_EINVAL, "rmsnorm8: no output");
  if (p->codes && !p->scales) return refuse(YK_EINVAL, "rmsnorm8: codes without scales");
  if (p->dtype != YK_F16 && p->dtype != YK_BF16) return refuse(YK_EUNSUP, "rmsnorm8: dtype must be fp16 or bf16");
  if (p->rows < 0 || p->cols < 1 || p->group < 0 || !(p->eps >= 0.f))
    return refuse(YK_EINVAL, "rmsnorm8: bad rows, cols, group or eps");
  if (p->cols > 32768 || (p->group && p->group < 16))
    return refuse(YK_EUNSUP, "rmsnorm8: at most 32768 columns, groups of at least 16");
  const int group = p->group && p->group < p->cols ? p->group : p->cols;
  const int groups = (p->cols + group - 1) / group;
  if (p->x_row < 0 || (p->add && p->add_row < 0) || (p->sum && p->sum_row < p->cols) ||
      (p->out && p->out_row < p->cols) || (p->codes && (p->codes_row < p->cols || p->scales_row < groups)))
    return refuse(YK_EINVAL, "rmsnorm8: an output's row stride is below its row, or an input's is negative");
  if (p->rows == 0) return YK_OK;
  const size_t smem = ((size_t)p->cols + groups) * sizeof(float);
  const int threads = p->cols <= 1024 ? 128 : p->cols <= 4096 ? 256 : 512;
  const auto kern = p->dtype == YK_BF16 ? rmsnorm8_kernel<true> : rmsnorm8_kernel<false>;
  if (smem_attr(kern, (int)smem) != cudaSuccess) return check_launch("rmsnorm8 attr");
  launch_k(kern, p->rows, threads, smem, (cudaStream_t)st, *p, group, groups);
  note_launch();
  return check_launch("rmsnorm8");
}
