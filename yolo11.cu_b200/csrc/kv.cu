// Paged 8-bit key/value cache: block tables and slots of a step (yk_kv_plan), and the write of
// new keys and values (yk_kv_append).
#include "text.cuh"

namespace yk {

// ---------------- plan ----------------
// Two exclusive prefix sums over the requests (rows, then blocks, as a request past the row
// limit takes none) and a scatter of 8 bytes a row.  Every CTA does both sums over all requests
// itself, in shared memory (8 bytes a request, read from L2): that costs less than a launch of
// its own, and the rows and table entries then spread over the grid without any exchange.
struct PlanArgs {
  YkKvPlan p;
  int finish;   // write cu, kv_lens, counts and the free head (block 0)
  int rows_too; // write slots, pos and table
};

__device__ __forceinline__ int plan_last_le(const int* a, int n, int v) {   // last i < n with a[i] <= v
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (a[m] <= v) lo = m; else hi = m;
  }
  return lo;
}

// Exclusive sum of one value a thread over the block; *total: the whole sum.
__device__ __forceinline__ long long block_exclusive(long long v, long long* part, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) part[warp] = s;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < warps ? part[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(~0u, w, o);
      if (lane >= o) w += u;
    }
    part[lane] = w;
  }
  __syncthreads();
  const long long before = (warp ? part[warp - 1] : 0) + s - v;
  *total = part[warps - 1];
  __syncthreads();   // part is used again
  return before;
}

__global__ void __launch_bounds__(1024) kv_plan_kernel(const __grid_constant__ PlanArgs a) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int plan_sm[];
  __shared__ long long part[32];
  __shared__ int stat[3];
  const YkKvPlan& p = a.p;
  const int R = p.requests, T = p.tokens;
  int* cu = plan_sm;            // [R + 1] rows before each request, at most p.rows
  int* boff = plan_sm + R + 1;  // [R + 1] blocks taken before each request
  const int per = (R + blockDim.x - 1) / blockDim.x;
  const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
  const int head = p.free_head ? max(0, min(*p.free_head, p.free_count)) : 0;
  const int avail = p.free_count - head;
  if (threadIdx.x < 3) stat[threadIdx.x] = 0;

  long long sum = 0, total;
  for (int r = r0; r < r1; r++) sum += max(0, p.fresh[r]);
  long long at = block_exclusive(sum, part, &total);
  // blocks needed by request r, whose rows start at `from`; -1: refused whatever is free
  const auto need_of = [&](int past, int fresh, long long from) -> int {
    if (past < 0 || fresh < 0 || (fresh && from + fresh > p.rows)) return -1;
    const long long end = (long long)past + fresh;
    if (end > (long long)p.max_blocks * T || end > 0x7fffffffll) return -1;
    return (int)((end + T - 1) / T - ((long long)past + T - 1) / T);
  };
  long long blocks = 0;
  for (int r = r0; r < r1; r++) {
    const int f = p.fresh[r];
    cu[r] = (int)min(at, (long long)p.rows);
    blocks += max(0, need_of(p.past[r], f, at));
    at += max(0, f);
  }
  if (threadIdx.x == 0) cu[R] = (int)min(total, (long long)p.rows);
  const long long all_rows = total;
  long long boffs = block_exclusive(blocks, part, &total);
  long long from = at;
  for (int r = r1 - 1; r >= r0; r--) from -= max(0, p.fresh[r]);
  int taken = 0, placed = 0, refused = 0;
  for (int r = r0; r < r1; r++) {
    const int f = p.fresh[r], need = need_of(p.past[r], f, from);
    boff[r] = (int)min(boffs, 0x7fffffffll);
    const bool ok = need == 0 || (need > 0 && boffs + need <= avail);
    if (ok && need > 0) taken = (int)(boffs + need);
    if (ok) placed += f; else refused++;
    boffs += max(0, need);
    from += max(0, f);
  }
  if (taken) atomicMax(&stat[0], taken);      // whole numbers: any order gives the same
  if (placed) atomicAdd(&stat[1], placed);
  if (refused) atomicAdd(&stat[2], refused);
  __syncthreads();
  const int n_taken = stat[0], n_rows = cu[R];

  if (a.rows_too) {
    const int warps = gridDim.x * (blockDim.x >> 5);
    const int gw = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    // a warp takes 128 consecutive rows; a lane's request only moves forward
    for (long long w0 = (long long)gw * 128; w0 < p.rows; w0 += (long long)warps * 128) {
      int r = -1, held = 0, past = 0, start = 0, base = 0;
      bool ok = false;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int n = (int)min(w0 + i * 32 + lane, (long long)p.rows);
        if (n >= p.rows) break;
        int slot = -1, pos = -1;
        if (n < n_rows) {
          int q = r < 0 ? plan_last_le(cu, R, n) : r;
          while (cu[q + 1] <= n) q++;
          if (q != r) {
            r = q;
            past = p.past[r];
            start = cu[r];
            const int need = need_of(past, p.fresh[r], start);
            base = boff[r];
            ok = need == 0 || (need > 0 && (long long)base + need <= avail);
            held = (int)(((long long)past + T - 1) / T);
          }
          if (past >= 0) pos = (int)min((long long)past + (n - start), 0x7fffffffll);
          if (ok) {
            const int b = pos / T;
            const int id = b < held ? p.table[(long long)r * p.table_stride + b]
                                    : p.free_blocks[head + base + (b - held)];
            if ((unsigned)id < (unsigned)p.blocks) slot = id * T + (pos & (T - 1));
          }
        }
        p.slots[n] = slot;
        if (p.pos) p.pos[n] = pos;
      }
    }
    const int threads = gridDim.x * blockDim.x;
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n_taken; e += threads) {
      const int r = plan_last_le(boff, R, (int)e);
      const int held = (int)(((long long)p.past[r] + T - 1) / T);
      p.table[(long long)r * p.table_stride + held + (e - boff[r])] = p.free_blocks[head + e];
    }
  }
  if (!a.finish || blockIdx.x) return;
  __syncthreads();   // kv_lens may be past: every read above comes first
  for (int r = threadIdx.x; r < R; r += blockDim.x) {
    const int past = p.past[r], f = p.fresh[r];
    const int need = need_of(past, f, cu[r]);
    const bool ok = need == 0 || (need > 0 && (long long)boff[r] + need <= avail);
    p.kv_lens[r] = ok ? past + f : past;
    p.cu[r] = cu[r];
  }
  if (threadIdx.x == 0) {
    p.cu[R] = n_rows;
    if (p.free_head) *p.free_head = head + n_taken;
    if (p.counts) {
      p.counts[0] = n_taken;
      p.counts[1] = stat[1];
      p.counts[2] = stat[2];
      p.counts[3] = (int)min(all_rows, 0x7fffffffll);
    }
  }
}

// ---------------- append ----------------
// A unit is the part of a block that the call fills: a run of rows with consecutive slots in one
// block.  Its items are (key or value, head).  The rows of a run share its items out among
// them, row j of n taking items j, j + n, ..., so one rule covers a decode step (runs of one row:
// each row's block of threads does all heads, a warp an item) and a prompt (runs of a whole
// block: one item a row, all threads together).
constexpr int kAppendThreads = 256;

struct AppendArgs {
  YkKvCache c;
  YkKvRows x;
  int window;   // rows of a CTA
};

// The smallest power of two s >= 2^-126 with 448 * s >= amax (448 = 1.75 * 2^8).
__device__ __forceinline__ float pow2_scale(float amax) {
  if (!(amax > 0.f)) return kMinScale;
  int e;
  const float f = frexpf(amax, &e);   // amax = f * 2^e, f in [0.5, 1)
  const int k = max(e - 9 + (f > 0.875f), -126);
  return __int_as_float((k + 127) << 23);
}

// Item (head, key or value) of the run of n rows from row `first` on, whose tokens start at
// `off` in their block, done by `size` threads of which this is number `id` (a warp, or the
// whole CTA: then `red` is the shared reduction buffer).  The x chunks that fit stay in
// registers between the maximum and the rounding; the rest is read again (from L2).
template <bool BF16, bool WHOLE>
__device__ __forceinline__ void append_item(const AppendArgs& a, int item, int first, int n, int slot,
                                            int id, float* red) {
  constexpr int kKeep = 8;
  const int size = WHOLE ? kAppendThreads : 32;
  const int T = a.c.tokens, D = a.c.dim, parts = D / 8;
  const int h = item >> 1, second = item & 1;
  const int block = slot / T, off = slot & (T - 1);
  const uint16_t* x = (const uint16_t*)(second ? a.x.v : a.x.k) +
                      (long long)h * (second ? a.x.v_head : a.x.k_head);
  const long long row = second ? a.x.v_row : a.x.k_row;
  uint8_t* codes = (uint8_t*)(second ? a.c.v : a.c.k) + block * a.c.block_stride + (long long)h * T * D;
  float* scale = (second ? a.c.vscale : a.c.kscale) + block * a.c.scale_stride + h;
  const int chunks = n * parts;
  const float before = off ? *scale : 0.f;
  const auto load = [&](int c) -> uint4 {
    const int j = c / parts;
    return *(const uint4*)(x + (first + j) * row + (c - j * parts) * 8);
  };
  uint4 keep[kKeep];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kKeep; i++) {
    const int c = i * size + id;
    keep[i] = c < chunks ? load(c) : make_uint4(0, 0, 0, 0);
  }
  const auto amax8 = [&](const uint4& v) {
    const uint32_t* u = (const uint32_t*)&v;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float2 f = pair_to_float2<BF16>(u[e]);
      m = fmaxf(m, fmaxf(finite_abs(f.x), finite_abs(f.y)));
    }
  };
#pragma unroll
  for (int i = 0; i < kKeep; i++) amax8(keep[i]);
  for (int c = kKeep * size + id; c < chunks; c += size) amax8(load(c));
  m = warp_max(m);
  if (WHOLE) {
    if ((id & 31) == 0) red[id >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < kAppendThreads / 32; i++) m = fmaxf(m, red[i]);
    __syncthreads();   // every thread has read red and `before`
  } else {
    __syncwarp();
  }
  const float s = fmaxf(pow2_scale(m), before), inv = 1.f / s;
  const auto store = [&](int c, const uint4& v) {
    const uint32_t* u = (const uint32_t*)&v;
    float2 f[4];
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = pair_to_float2<BF16>(u[e]);
    uint2 q;
    q.x = float4_to_e4m3x4(f[0].x * inv, f[0].y * inv, f[1].x * inv, f[1].y * inv);
    q.y = float4_to_e4m3x4(f[2].x * inv, f[2].y * inv, f[3].x * inv, f[3].y * inv);
    *(uint2*)(codes + (long long)off * D + c * 8) = q;
  };
#pragma unroll
  for (int i = 0; i < kKeep; i++) {
    const int c = i * size + id;
    if (c < chunks) store(c, keep[i]);
  }
  for (int c = kKeep * size + id; c < chunks; c += size) store(c, load(c));
  if (off && s > before) {   // the scale grew: the earlier tokens take the new one
    const float ratio = before / s;
    for (int c = id; c < off * D / 16; c += size) {
      uint4 v = *(const uint4*)(codes + c * 16);
      uint32_t* u = (uint32_t*)&v;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float2 lo = e4m3x2_to_float2(u[e]), hi = e4m3x2_to_float2(u[e] >> 16);
        u[e] = float4_to_e4m3x4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
      }
      *(uint4*)(codes + c * 16) = v;
    }
  }
  if (id == 0) *scale = s;
}

template <bool BF16>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[kAppendThreads / 32];
  __shared__ int sl[3 * 128];        // slots of the window and one block's tokens to either side
  __shared__ uint32_t follows[12];   // bit i: row lo + i is the next token of row lo + i - 1's run
  const int T = a.c.tokens, items = 2 * a.c.heads;
  const int w0 = blockIdx.x * a.window, w1 = min(a.x.rows, w0 + a.window);
  const int lo = max(0, w0 - T), hi = min(a.x.rows, w1 + T);
  for (int i = threadIdx.x; i < 3 * 128; i += blockDim.x) {
    const int s = lo + i < hi ? a.x.slots[lo + i] : -1;
    sl[i] = (unsigned)s < (unsigned)(a.c.blocks * T) ? s : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 3 * 128; i += blockDim.x) {
    const bool f = i > 0 && sl[i] > 0 && sl[i] == sl[i - 1] + 1 && (sl[i] & (T - 1));
    const uint32_t bits = __ballot_sync(~0u, f);
    if ((i & 31) == 0) follows[i >> 5] = bits;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  for (int i = w0 - lo; i < w1 - lo; i++) {
    const int s = sl[i];
    if (s < 0) continue;
    // rows of the run before and after row i (the same for every thread)
    int back = 0, ahead = 0;
    for (int j = i; j >= 0;) {         // consecutive set bits from i down
      const int ones = __clz(~(follows[j >> 5] << (31 - (j & 31))));
      const int got = min(ones, (j & 31) + 1);
      back += got;
      if (got <= (j & 31)) break;
      j -= got;
    }
    if (back >= items) continue;       // enough rows before this one share the items
    for (int j = i + 1; j < 3 * 128;) {   // and from i + 1 up
      const uint32_t w = ~(follows[j >> 5] >> (j & 31));
      const int got = min(w ? __ffs(w) - 1 : 32, 32 - (j & 31));
      ahead += got;
      if (got < 32 - (j & 31)) break;
      j += got;
    }
    const int n = back + ahead + 1, first = lo + i - back;
    if (n * (a.c.dim / 8) <= 64) {
      for (int it = back + warp * n; it < items; it += n * (kAppendThreads / 32))
        append_item<BF16, false>(a, it, first, n, s - back, threadIdx.x & 31, red);
    } else {
      for (int it = back; it < items; it += n)
        append_item<BF16, true>(a, it, first, n, s - back, threadIdx.x, red);
    }
  }
}

}  // namespace yk

using namespace yk;

extern "C" int yk_kv_plan(const YkKvPlan* p, yk_stream_t st) {
  if (!p || !p->past || !p->fresh || !p->table || !p->kv_lens || !p->cu)
    return refuse(YK_EINVAL, "kv_plan: null pointer");
  if (p->requests < 1 || p->rows < 0 || p->free_count < 0 || p->blocks < 1 || p->max_blocks < 1 ||
      p->table_stride < p->max_blocks || (p->rows && !p->slots) || (p->free_count && !p->free_blocks))
    return refuse(YK_EINVAL, "kv_plan: bad size, stride or null slots / free_blocks");
  if (p->tokens != 16 && p->tokens != 32 && p->tokens != 64 && p->tokens != 128)
    return refuse(YK_EUNSUP, "kv_plan: tokens of a block must be 16, 32, 64 or 128");
  if ((long long)p->blocks * p->tokens > 0x7fffffffll)
    return refuse(YK_EINVAL, "kv_plan: blocks * tokens must be below 2^31");
  if (p->requests > 16384) return refuse(YK_EUNSUP, "kv_plan: at most 16384 requests");
  const size_t smem = (2 * (size_t)p->requests + 2) * sizeof(int);
  if (smem_attr(kv_plan_kernel, (int)smem) != cudaSuccess) return check_launch("kv_plan attr");
  const int threads = std::min(1024, std::max(128, (std::max(p->requests, p->rows) + 31) / 32 * 32));
  const int grid = (int)std::max(1ll, std::min(148ll, ((long long)p->rows + 4095) / 4096));
  // With several CTAs, outputs that are inputs too (the free head, kv_lens over past) wait for a
  // launch of their own, so that no CTA reads them after they moved.
  const bool inplace = p->free_head || (p->kv_lens < p->past + p->requests && p->past < p->kv_lens + p->requests);
  const bool two = grid > 1 && inplace;
  PlanArgs a{*p, two ? 0 : 1, 1};
  launch_k(kv_plan_kernel, grid, threads, smem, (cudaStream_t)st, a);
  note_launch();
  if (two) {
    PlanArgs b{*p, 1, 0};
    launch_k(kv_plan_kernel, 1, threads, smem, (cudaStream_t)st, b);
    note_launch();
  }
  return check_launch("kv_plan");
}

extern "C" int yk_kv_append(const YkKvCache* c, const YkKvRows* x, yk_stream_t st) {
  const int bad = check_cache(c);
  if (bad) return bad;
  if (!x || x->rows < 0 || (x->rows && (!x->k || !x->v || !x->slots)))
    return refuse(YK_EINVAL, "kv_append: null pointer or negative rows");
  if (x->dtype != YK_F16 && x->dtype != YK_BF16) return refuse(YK_EUNSUP, "kv_append: dtype must be fp16 or bf16");
  if (!aligned16(x->k) || !aligned16(x->v) || x->k_row % 8 || x->v_row % 8 || x->k_head % 8 || x->v_head % 8)
    return refuse(YK_EINVAL, "kv_append: rows need 16-byte alignment and strides that are multiples of 8");
  if (x->rows == 0) return YK_OK;
  // about eight CTAs an SM, each of at most one block's rows
  int window = 1;
  while (window < c->tokens && x->rows / (2 * window) >= 148 * 8) window *= 2;
  AppendArgs a{*c, *x, window};
  const int grid = (x->rows + window - 1) / window;
  if (x->dtype == YK_BF16) launch_k(kv_append_kernel<true>, grid, kAppendThreads, 0, (cudaStream_t)st, a);
  else launch_k(kv_append_kernel<false>, grid, kAppendThreads, 0, (cudaStream_t)st, a);
  note_launch();
  return check_launch("kv_append");
}
