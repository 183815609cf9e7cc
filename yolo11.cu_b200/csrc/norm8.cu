// Residual addition, RMS norm and 8-bit output with scales (yk_rmsnorm8).
#include "text.cuh"

namespace yk {

// HBM bound: x and add are read once and every output written once; the row stays in registers
// between the three passes over it (mean square, group maxima, rounding).
//
// rmsnorm8_vec_kernel: rows that allow 16-byte accesses.  A thread holds V chunks of 8 columns, chunk
// tid + i * threads, so that a group of 8 * 2^i columns (16 .. 256) lies in neighbouring lanes and its
// maximum takes shuffles only; one scale a row takes one block reduction.  Four rows share a block
// (a warp each) when a row is short.  Measured: 12,000 x 5120 bf16 with addition and a scale for each 128
// columns 71 us, 6.1 TB/s (the copy rate is 6.5); 8 x 2048 2.8 us, a launch.  Packed arithmetic and one filter
// for infinities a chunk instead of one an element took it from 98 us.  1 / scale is the hardware's approximation (one
// unit in the last place) and 1 / 448 a product: exact divisions cost up to 10 % (12,000 x 5120 without addition 46 -> 51 us)
// and move the error against 64 bits in its eleventh digit only; a code on a rounding boundary may differ from the
// other kernel's, as it may by the order of the squares' sum.
template <bool BF16, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512) rmsnorm8_vec_kernel(const __grid_constant__ YkRmsNorm8 p, int lanes, int shift) {
  __shared__ float part[2][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = WARP ? 1 : blockDim.x >> 5;
  const int id = WARP ? lane : threadIdx.x, size = WARP ? 32 : blockDim.x;
  const int chunks = p.cols / 8;
  const long long r = WARP ? (long long)blockIdx.x * 4 + warp : blockIdx.x;
  pdl_wait();
  pdl_trigger();
  if (WARP && r >= p.rows) return;
  const uint4* x = (const uint4*)((const uint16_t*)p.x + r * p.x_row);
  const uint4* add = p.add ? (const uint4*)((const uint16_t*)p.add + r * p.add_row) : nullptr;
  uint4 xv[V], av[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = id + i * size;
    xv[i] = c < chunks ? __ldcs(x + c) : make_uint4(0, 0, 0, 0);
    if (add) av[i] = c < chunks ? __ldcs(add + c) : make_uint4(0, 0, 0, 0);
  }
  uint4 wv[V];
#pragma unroll
  for (int i = 0; i < V; i++) wv[i] = id + i * size < chunks ? ((const uint4*)p.weight)[id + i * size] : make_uint4(0, 0, 0, 0);
  float2 h[V][4];
  const float over_c = 1.f / (float)p.cols;
  float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const uint32_t *xu = (const uint32_t*)&xv[i], *au = (const uint32_t*)&av[i];
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      h[i][e] = pair_to_float2<BF16>(xu[e]);
      if (add) h[i][e] = add2(h[i][e], pair_to_float2<BF16>(au[e]));
      o[e] = float2_to_pair<BF16>(h[i][e].x, h[i][e].y);
      ss2 = ffma2(h[i][e], mul2(h[i][e], make_float2(over_c, over_c)), ss2);   // the mean itself: the sum would overflow sooner
    }
    if (p.sum && id + i * size < chunks)
      ((uint4*)((uint16_t*)p.sum + r * p.sum_row))[id + i * size] = make_uint4(o[0], o[1], o[2], o[3]);
  }
  float ss = warp_sum(ss2.x + ss2.y);
  if (!WARP) {
    if (lane == 0) part[0][warp] = ss;
    __syncthreads();
    ss = part[0][0];
    for (int i = 1; i < warps; i++) ss += part[0][i];
  }
  const float inv = rsqrtf(ss + p.eps);
  float amax[V], row_max = 0.f;
  const auto amax8 = [&](int i, auto abs_of) {      // of chunk i; fmaxf leaves NaN out
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) m = fmaxf(m, fmaxf(abs_of(h[i][e].x), abs_of(h[i][e].y)));
    return id + i * size < chunks ? m : 0.f;
  };
#pragma unroll
  for (int i = 0; i < V; i++) {
    const uint32_t* wu = (const uint32_t*)&wv[i];
#pragma unroll
    for (int e = 0; e < 4; e++) h[i][e] = mul2(h[i][e], mul2(make_float2(inv, inv), pair_to_float2<BF16>(wu[e])));
    if (p.out && id + i * size < chunks)
      ((uint4*)((uint16_t*)p.out + r * p.out_row))[id + i * size] =
          make_uint4(float2_to_pair<BF16>(h[i][0].x, h[i][0].y), float2_to_pair<BF16>(h[i][1].x, h[i][1].y),
                     float2_to_pair<BF16>(h[i][2].x, h[i][2].y), float2_to_pair<BF16>(h[i][3].x, h[i][3].y));
    amax[i] = amax8(i, [](float v) { return fabsf(v); });
    if (amax[i] == INFINITY) amax[i] = amax8(i, finite_abs);
    row_max = fmaxf(row_max, amax[i]);
  }
  if (!p.codes) return;
  if (lanes == 0) {                       // one scale a row
    row_max = warp_max(row_max);
    if (!WARP) {
      if (lane == 0) part[1][warp] = row_max;
      __syncthreads();
      row_max = part[1][0];
      for (int i = 1; i < warps; i++) row_max = fmaxf(row_max, part[1][i]);
    }
  }
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = id + i * size;
    float m = lanes ? amax[i] : row_max;
#pragma unroll
    for (int o = 16; o; o >>= 1)
      if (lanes > o) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float s = fmaxf(m * (1.f / kE4m3Max), kMinScale), up = rcp_fast(s);
    if (c >= chunks) continue;
    if (lanes ? (c & (lanes - 1)) == 0 : c == 0) p.scales[r * p.scales_row + (c >> shift)] = s;
    float2 q[4];
#pragma unroll
    for (int e = 0; e < 4; e++) q[e] = mul2(h[i][e], make_float2(up, up));
    ((uint2*)((uint8_t*)p.codes + r * p.codes_row))[c] =
        make_uint2(float4_to_e4m3x4(q[0].x, q[0].y, q[1].x, q[1].y), float4_to_e4m3x4(q[2].x, q[2].y, q[3].x, q[3].y));
  }
}

// Any other columns, strides, alignment and groups: one CTA a row, the row in shared memory, a 2-byte
// access and (for the codes) a division an element.  Measured: 12,000 x 5119, else as above, 273 us; 64 x 5119 12.5 us.
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
  const bool bf = p->dtype == YK_BF16;
  cudaStream_t s = (cudaStream_t)st;
  const auto vec = [](const void* q, long long row) { return !q || (aligned16(q) && row % 8 == 0); };
  int lanes = 0;                            // lanes of a group, 0: one scale a row
  bool fits = p->cols % 8 == 0 && vec(p->x, p->x_row) && vec(p->add, p->add_row) && vec(p->sum, p->sum_row) &&
              vec(p->out, p->out_row) && vec(p->weight, 0) && ((uintptr_t)p->codes | (uintptr_t)p->codes_row) % 8 == 0;
  if (p->codes && groups > 1) {
    lanes = group / 8;
    fits = fits && group % 8 == 0 && lanes <= 32 && !(lanes & (lanes - 1));
  }
  if (fits) {
    const int shift = lanes ? __builtin_ctz(lanes) : 0;
    // a warp a row while its chunks are at most two a lane; else four chunks a thread (eight from
    // 16384 columns on): fewer threads leave more rows in flight on an SM
    const int chunks = p->cols / 8;
    if (chunks <= 64)
      launch_k(bf ? rmsnorm8_vec_kernel<true, 2, true> : rmsnorm8_vec_kernel<false, 2, true>, (unsigned)((p->rows + 3ll) / 4), 128, 0, s, *p, lanes, shift);
    else if (chunks <= 2048)
      launch_k(bf ? rmsnorm8_vec_kernel<true, 4, false> : rmsnorm8_vec_kernel<false, 4, false>, p->rows, (chunks + 127) / 128 * 32, 0, s, *p, lanes, shift);
    else
      launch_k(bf ? rmsnorm8_vec_kernel<true, 8, false> : rmsnorm8_vec_kernel<false, 8, false>, p->rows, 512, 0, s, *p, lanes, shift);
    note_launch();
    return check_launch("rmsnorm8");
  }
  const size_t smem = ((size_t)p->cols + groups) * sizeof(float);
  const int threads = p->cols <= 1024 ? 128 : p->cols <= 4096 ? 256 : 512;
  const auto kern = bf ? rmsnorm8_kernel<true> : rmsnorm8_kernel<false>;
  if (smem_attr(kern, (int)smem) != cudaSuccess) return check_launch("rmsnorm8 attr");
  launch_k(kern, p->rows, threads, smem, s, *p, group, groups);
  note_launch();
  return check_launch("rmsnorm8");
}
