// Attention over the paged 8-bit key/value cache (yk_attn_kv8).
#include "text.cuh"

namespace yk {

struct Attn8Args {
  YkKvCache c;
  YkAttnKv8 a;
};

// One warp a (row, query head): lanes own the channels, one key at a time.
template <bool BF16, int D>
__global__ void __launch_bounds__(256) attn8_kernel(const __grid_constant__ Attn8Args p) {
  pdl_wait();
  pdl_trigger();
  constexpr int V = D / 32;
  const YkAttnKv8& a = p.a;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int n = (int)(item / a.heads), h = (int)(item % a.heads);
  if (n >= a.rows) return;
  int lo = 0, hi = a.requests;    // the last request that starts at or before row n
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (a.cu[m] <= n) lo = m; else hi = m;
  }
  if (a.cu[lo] > n || a.cu[lo + 1] <= n) return;   // a row of no request
  const int r = lo, T = p.c.tokens, kh = h / (a.heads / p.c.heads);
  const long long cap = (long long)a.max_blocks * T;
  const int kv = (int)min((long long)max(0, a.kv_lens[r]), cap);
  int first = 0, last = kv - 1;
  if (a.causal) {
    const int pos = kv - a.cu[r + 1] + n;
    last = min(last, pos);
    if (a.window) first = max(0, pos - a.window + 1);
  }
  const uint16_t* qp = (const uint16_t*)a.q + n * a.q_row + h * D + lane * V;
  float q[V], o[V] = {};
#pragma unroll
  for (int i = 0; i < V; i++) q[i] = elem_to_float<BF16>(qp[i]) * a.scale;
  float m = -INFINITY, l = 0.f;
  for (int j = first; j <= last; j++) {
    const int b = a.table[r * a.table_stride + j / T];
    if ((unsigned)b >= (unsigned)p.c.blocks) continue;
    const long long at = b * p.c.block_stride + ((long long)kh * T + j % T) * D + lane * V;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) s = fmaf(q[i], e4m3x2_to_float2(((const uint8_t*)p.c.k)[at + i]).x, s);
    s = warp_sum(s) * p.c.kscale[b * p.c.scale_stride + kh];
    const float mn = fmaxf(m, s), corr = __expf(m - mn), w = __expf(s - mn);
    const float wv = w * p.c.vscale[b * p.c.scale_stride + kh];
    l = l * corr + w;
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = fmaf(wv, e4m3x2_to_float2(((const uint8_t*)p.c.v)[at + i]).x, o[i] * corr);
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t* op = (uint16_t*)a.out + n * a.out_row + h * D + lane * V;
#pragma unroll
  for (int i = 0; i < V; i++) op[i] = float_to_elem<BF16>(l > 0.f ? o[i] * inv : 0.f);
  if (a.lse && lane == 0) a.lse[(long long)n * a.heads + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace yk

using namespace yk;

extern "C" size_t yk_attn_kv8_workspace_bytes(int requests, int rows, int heads, int kv_heads, int dim) {
  return 16;
}

extern "C" int yk_attn_kv8(const YkKvCache* c, const YkAttnKv8* a, yk_stream_t st) {
  const int bad = check_cache(c);
  if (bad) return bad;
  if (!a || !a->cu || !a->kv_lens || !a->table || !a->ws) return refuse(YK_EINVAL, "attn_kv8: null pointer");
  if (a->dtype != YK_F16 && a->dtype != YK_BF16) return refuse(YK_EUNSUP, "attn_kv8: dtype must be fp16 or bf16");
  if (a->requests < 1 || a->rows < 0 || a->heads < 1 || a->heads % c->heads || a->max_blocks < 1 ||
      a->table_stride < a->max_blocks || a->window < 0 || !(a->scale >= 0.f))
    return refuse(YK_EINVAL, "attn_kv8: bad requests, rows, heads, table, window or scale");
  if (a->requests > 16384) return refuse(YK_EUNSUP, "attn_kv8: at most 16384 requests");
  if (a->window && !a->causal) return refuse(YK_EINVAL, "attn_kv8: a window needs causal");
  if (a->rows == 0) return YK_OK;
  if (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out) || a->q_row % 8 || a->out_row % 8 ||
      a->out_row < (long long)a->heads * c->dim || a->q_row < 0)
    return refuse(YK_EINVAL, "attn_kv8: q and out need 16-byte alignment and row strides that are multiples of 8");
  if (!aligned16(a->ws) || a->ws_bytes < yk_attn_kv8_workspace_bytes(a->requests, a->rows, a->heads, c->heads, c->dim))
    return refuse(YK_EINVAL, "attn_kv8: workspace too small or not 16-byte aligned");
  Attn8Args p{*c, *a};
  if (p.a.scale == 0.f) p.a.scale = 1.f / sqrtf((float)c->dim);
  const bool bf = a->dtype == YK_BF16;
  const auto kern = c->dim == 64 ? (bf ? attn8_kernel<true, 64> : attn8_kernel<false, 64>)
                    : c->dim == 128 ? (bf ? attn8_kernel<true, 128> : attn8_kernel<false, 128>)
                                    : (bf ? attn8_kernel<true, 256> : attn8_kernel<false, 256>);
  launch_k(kern, (unsigned)(((long long)a->rows * a->heads + 7) / 8), 256, 0, (cudaStream_t)st, p);
  note_launch();
  return check_launch("attn_kv8");
}
