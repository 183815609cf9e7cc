// Paged 8-bit key/value cache: block tables and slots of a step (yk_kv_plan), and the write of
// new keys and values (yk_kv_append).
#include "text.cuh"

namespace yk {

// ---------------- plan ----------------
// Two exclusive prefix sums over the requests (rows, then blocks, as a request past the row
// limit takes none) and a scatter of 8 bytes a row.  Every CTA does both sums over all requests
// itself, in shared memory (8 bytes a request, read from L2): that costs less than a launch of
// its own, and the rows and table entries then spread over the grid without any exchange.
// Measured: 64 requests with one row each 4.5 us, 2048 requests with 736,000 rows 11.8 us (6.3 MB): latency
// bound (lengths, sums, then table or free list, one after the other).
struct PlanArgs {
  YkKvPlan p;
  int finish;   // write cu, kv_lens, counts and the free head (block 0)
  int rows_too; // write slots, pos and table
  int vec;      // slots and pos allow 16-byte stores
};

// The last i < n with a[i] <= v; a negative entry stands for its complement.
__device__ __forceinline__ int plan_last_le(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1, x = a[m];
    if ((x < 0 ? ~x : x) <= v) lo = m; else hi = m;
  }
  return lo;
}

// Exclusive sums of two values a thread over the block, in one go; totals: the whole sums.
struct Sums {
  long long a, b;
};
__device__ __forceinline__ Sums block_exclusive2(Sums v, Sums* part, Sums* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  Sums s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(~0u, s.a, o), b = __shfl_up_sync(~0u, s.b, o);
    if (lane >= o) { s.a += a; s.b += b; }
  }
  if (lane == 31) part[warp] = s;
  __syncthreads();
  if (warp == 0) {
    Sums w = lane < warps ? part[lane] : Sums{0, 0};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(~0u, w.a, o), b = __shfl_up_sync(~0u, w.b, o);
      if (lane >= o) { w.a += a; w.b += b; }
    }
    part[lane] = w;
  }
  __syncthreads();
  const Sums before = warp ? part[warp - 1] : Sums{0, 0};
  *total = part[warps - 1];
  return {before.a + s.a - v.a, before.b + s.b - v.b};
}

__global__ void __launch_bounds__(1024) kv_plan_kernel(const __grid_constant__ PlanArgs a) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int plan_sm[];
  __shared__ Sums part[32];
  __shared__ int stat[3];
  const YkKvPlan& p = a.p;
  const int R = p.requests, T = p.tokens, shift = 31 - __clz(T);
  int* cu = plan_sm;              // [R + 1] rows before each request, at most p.rows
  int* boff = cu + R + 1;         // [R] blocks needed before each request, ~ of that where it is refused
  int* past_sm = boff + R;        // [R]
  const int per = (R + blockDim.x - 1) / blockDim.x;
  const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
  const int head = p.free_head ? max(0, min(*p.free_head, p.free_count)) : 0;
  const int avail = p.free_count - head;
  if (threadIdx.x < 3) stat[threadIdx.x] = 0;

  // Both sums at once.  A refused request's need stays in the sum, so that none is overtaken.  A request
  // past the row limit counts too, but every later one that needs a block is past that limit itself.
  Sums sum = {0, 0}, total;
  for (int r = r0; r < r1; r++) {
    const int f = p.fresh[r], past = p.past[r];
    const long long end = (long long)past + f;
    const bool fits = past >= 0 && f >= 0 && end <= (long long)p.max_blocks * T && end <= 0x7fffffffll;
    const int need = fits ? (int)(((end + T - 1) >> shift) - (((long long)past + T - 1) >> shift)) : -1;
    cu[r] = max(0, f);
    boff[r] = need;
    past_sm[r] = past;
    sum.a += max(0, f);
    sum.b += max(0, need);
  }
  Sums at = block_exclusive2(sum, part, &total);
  if (threadIdx.x == 0) cu[R] = (int)min(total.a, (long long)p.rows);
  const long long all_rows = total.a;
  int taken = 0, placed = 0, refused = 0;
  for (int r = r0; r < r1; r++) {
    const int f = cu[r], need = boff[r];
    const bool ok = need >= 0 && !(f && at.a + f > p.rows) && (need == 0 || at.b + need <= avail);
    const int before = (int)min(at.b, 0x7fffffffll);
    cu[r] = (int)min(at.a, (long long)p.rows);
    boff[r] = ok ? before : ~before;
    if (ok && need > 0) taken = (int)(at.b + need);
    if (ok) placed += f; else refused++;
    at.a += f;
    at.b += max(0, need);
  }
  if (taken) atomicMax(&stat[0], taken);      // whole numbers: any order gives the same
  if (placed) atomicAdd(&stat[1], placed);
  if (refused) atomicAdd(&stat[2], refused);
  __syncthreads();
  const int n_taken = stat[0], n_rows = cu[R];

  if (a.rows_too) {
    const int threads = gridDim.x * blockDim.x, me = blockIdx.x * blockDim.x + threadIdx.x;
    // four consecutive rows a thread: mostly of one request and block, found once
    for (long long w0 = (long long)me * 4; w0 < p.rows; w0 += (long long)threads * 4) {
      int slot[4], pos[4];
      int r = -1, end = 0, past = 0, start = 0, b_off = -1, held = 0, b_have = -1, id = -1;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int n = (int)w0 + i;
        slot[i] = pos[i] = -1;
        if (w0 + i >= n_rows) continue;
        if (n >= end) {
          if (r < 0) r = plan_last_le(cu, R, n);
          while (cu[r + 1] <= n) r++;
          past = past_sm[r];
          start = cu[r];
          end = cu[r + 1];
          b_off = boff[r];
          held = (int)(((long long)past + T - 1) >> shift);
          b_have = -1;
        }
        if (past >= 0) pos[i] = (int)min((long long)past + (n - start), 0x7fffffffll);
        if (b_off < 0) continue;
        const int b = pos[i] >> shift;
        if (b != b_have) {
          id = b < held ? p.table[(long long)r * p.table_stride + b] : p.free_blocks[head + b_off + (b - held)];
          b_have = b;
        }
        if ((unsigned)id < (unsigned)p.blocks) slot[i] = id * T + (pos[i] & (T - 1));
      }
      if (a.vec && w0 + 4 <= p.rows) {
        *(int4*)(p.slots + w0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        if (p.pos) *(int4*)(p.pos + w0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (w0 + i < p.rows) {
            p.slots[w0 + i] = slot[i];
            if (p.pos) p.pos[w0 + i] = pos[i];
          }
      }
    }
    for (long long e = me; e < n_taken; e += threads) {
      const int r = plan_last_le(boff, R, (int)e);      // the last that starts there: not refused
      const int held = (int)(((long long)past_sm[r] + T - 1) >> shift);
      p.table[(long long)r * p.table_stride + held + (e - boff[r])] = p.free_blocks[head + e];
    }
  }
  if (!a.finish || blockIdx.x) return;
  // kv_lens may be past: each request's length is read before, by this thread
  for (int r = r0; r < r1; r++) {
    p.kv_lens[r] = boff[r] >= 0 ? past_sm[r] + cu[r + 1] - cu[r] : past_sm[r];
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
// HBM bound.  A unit is the part of a block that the call fills: a run of rows with consecutive
// slots in one block.  The rows of a run share its heads out among them, row j of n taking heads
// j * heads / n .. (j + 1) * heads / n - 1, so one rule covers a decode step (runs of one row: the
// row's CTA does all heads, a warp each) and a prompt (runs of a whole block: at most one head a row,
// the CTA's threads together).  Keys and values of a head go together: twice the bytes under way for
// the same two waits (maximum, scale).  Measured: 29,468 rows of 8 heads of 128 channels in bf16 54 us, 3.4 TB/s
// (four CTAs an SM; two: 66 us); 64 rows 3.6 us.
constexpr int kAppendThreads = 256;

struct AppendArgs {
  YkKvCache c;
  YkKvRows x;
  int window;   // rows of a CTA
};

// The smallest power of two s >= 2^-126 with 448 * s >= amax (448 = 1.75 * 2^8).
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);          // 1.f * 2^e: 2^(e - 8), twice that where 1.f > 1.75
  const int k = (int)(u >> 23) - 8 + ((u & 0x7fffff) > 0x600000);
  return __uint_as_float((uint32_t)max(k, 1) << 23);
}

// Head h of the run of n rows from row `first` on, whose tokens start at slot `slot`, done by a warp
// or the whole CTA (WHOLE; `red` is its reduction buffer); `id` is the thread's number among them.
// The first KEEP chunks a thread stay in registers between the maximum and the rounding; the rest
// is read again (from L2).
template <bool BF16, bool WHOLE, int KEEP>
__device__ __forceinline__ void append_head(const AppendArgs& a, int h, int first, int n, int slot, int id,
                                            float (*red)[kAppendThreads / 32]) {
  constexpr int size = WHOLE ? kAppendThreads : 32;
  const int T = a.c.tokens, D = a.c.dim, shift = 31 - __clz(D / 8);    // D / 8 chunks a row: a power of two
  const int block = slot >> (31 - __clz(T)), off = slot & (T - 1);
  const int chunks = n << shift;
  const uint16_t* x[2] = {(const uint16_t*)a.x.k + h * a.x.k_head, (const uint16_t*)a.x.v + h * a.x.v_head};
  const long long row[2] = {a.x.k_row, a.x.v_row};
  uint8_t* codes[2] = {(uint8_t*)a.c.k + block * a.c.block_stride + (long long)h * T * D,
                       (uint8_t*)a.c.v + block * a.c.block_stride + (long long)h * T * D};
  float* scale[2] = {a.c.kscale + block * a.c.scale_stride + h, a.c.vscale + block * a.c.scale_stride + h};
  const auto load = [&](int kv, int c) -> uint4 {
    return *(const uint4*)(x[kv] + (first + (c >> shift)) * row[kv] + (c & ((1 << shift) - 1)) * 8);
  };
  uint4 keep[2][KEEP];
  float before[2], m[2];
#pragma unroll
  for (int kv = 0; kv < 2; kv++) {
#pragma unroll
    for (int i = 0; i < KEEP; i++) {
      const int c = i * size + id;
      keep[kv][i] = c < chunks ? load(kv, c) : make_uint4(0, 0, 0, 0);
    }
    before[kv] = off ? *scale[kv] : 0.f;
  }
#pragma unroll
  for (int kv = 0; kv < 2; kv++) {
    uint32_t m2 = 0;
    const auto amax8 = [&](const uint4& v) {
      m2 = amax_pair<BF16>(amax_pair<BF16>(m2, v.x), v.y);
      m2 = amax_pair<BF16>(amax_pair<BF16>(m2, v.z), v.w);
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++) amax8(keep[kv][i]);
    for (int c = KEEP * size + id; c < chunks; c += size) amax8(load(kv, c));
    const float2 f = pair_to_float2<BF16>(m2);
    m[kv] = warp_max(fmaxf(f.x, f.y));
  }
  const auto meet = [&] {              // the warps' maxima
    if (WHOLE) {
      if ((id & 31) == 0) {
        red[0][id >> 5] = m[0];
        red[1][id >> 5] = m[1];
      }
      __syncthreads();
#pragma unroll
      for (int kv = 0; kv < 2; kv++)
#pragma unroll
        for (int i = 0; i < kAppendThreads / 32; i++) m[kv] = fmaxf(m[kv], red[kv][i]);
      __syncthreads();   // every thread has read red and `before`
    } else {
      __syncwarp();
    }
  };
  meet();
  if (m[0] == INFINITY || m[1] == INFINITY) {       // again, without the infinities
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
      float top = 0.f;
      for (int c = id; c < chunks; c += size) {
        const uint4 v = load(kv, c);
        const uint32_t* u = (const uint32_t*)&v;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 f = pair_to_float2<BF16>(u[e]);
          top = fmaxf(top, fmaxf(finite_abs(f.x), finite_abs(f.y)));
        }
      }
      m[kv] = warp_max(top);
    }
    meet();
  }
#pragma unroll
  for (int kv = 0; kv < 2; kv++) {
    const float s = fmaxf(pow2_scale(m[kv]), before[kv]);
    const uint32_t bits = __float_as_uint(s);       // a power of two, unless `before` was not
    const float inv = bits & 0x7fffff ? 1.f / s : __uint_as_float(0x7f000000u - bits);
    const auto store = [&](int c, const uint4& v) {
      const uint32_t* u = (const uint32_t*)&v;
      float2 f[4];
#pragma unroll
      for (int e = 0; e < 4; e++) f[e] = mul2(pair_to_float2<BF16>(u[e]), make_float2(inv, inv));
      *(uint2*)(codes[kv] + off * D + c * 8) = make_uint2(float4_to_e4m3x4(f[0].x, f[0].y, f[1].x, f[1].y),
                                                          float4_to_e4m3x4(f[2].x, f[2].y, f[3].x, f[3].y));
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++) {
      const int c = i * size + id;
      if (c < chunks) store(c, keep[kv][i]);
    }
    for (int c = KEEP * size + id; c < chunks; c += size) store(c, load(kv, c));
    if (off && s > before[kv]) {   // the scale grew: the earlier tokens take the new one
      const float ratio = before[kv] / s;
      for (int c = id; c < off * D / 16; c += size) {
        uint4 v = *(const uint4*)(codes[kv] + c * 16);
        uint32_t* u = (uint32_t*)&v;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 lo = e4m3x2_to_float2(u[e]), hi = e4m3x2_to_float2(u[e] >> 16);
          u[e] = float4_to_e4m3x4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
        }
        *(uint4*)(codes[kv] + c * 16) = v;
      }
    }
    if (id == 0) *scale[kv] = s;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[2][kAppendThreads / 32];
  __shared__ int sl[3 * 128];        // slots of the window and one block's tokens to either side
  __shared__ int4 job[128];
  __shared__ uint32_t follows[12];   // bit i: row lo + i is the next token of row lo + i - 1's run
  const int T = a.c.tokens, heads = a.c.heads;
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
  // each row of the window by a thread: rows of its run before it, rows of the run, its heads
  const int rows = w1 - w0;
  for (int j0 = threadIdx.x; j0 < rows; j0 += blockDim.x) {
    const int i = w0 - lo + j0;
    int back = 0, ahead = 0;
    for (int j = i; j >= 0;) {         // consecutive set bits from i down
      const int ones = __clz(~(follows[j >> 5] << (31 - (j & 31))));
      const int got = min(ones, (j & 31) + 1);
      back += got;
      if (got <= (j & 31)) break;
      j -= got;
    }
    for (int j = i + 1; j < 3 * 128;) {   // and from i + 1 up
      const uint32_t w = ~(follows[j >> 5] >> (j & 31));
      const int got = min(w ? __ffs(w) - 1 : 32, 32 - (j & 31));
      ahead += got;
      if (got < 32 - (j & 31)) break;
      j += got;
    }
    const int n = back + ahead + 1;
    const bool there = sl[i] >= 0;
    job[j0] = make_int4(back, n, there ? back * heads / n : 0, there ? (back + 1) * heads / n : 0);
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  for (int j = 0; j < rows; j++) {
    const int4 w = job[j];             // the same for every thread
    if (w.z >= w.w) continue;
    const int first = w0 + j - w.x, slot = sl[w0 - lo + j] - w.x;
    if (w.y * (a.c.dim / 8) <= 64) {
      for (int h = w.z + warp; h < w.w; h += kAppendThreads / 32)
        append_head<BF16, false, 2>(a, h, first, w.y, slot, threadIdx.x & 31, red);
    } else {
      for (int h = w.z; h < w.w; h++) append_head<BF16, true, 4>(a, h, first, w.y, slot, threadIdx.x, red);
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
  const size_t smem = (3 * (size_t)p->requests + 1) * sizeof(int);
  if (smem_attr(kv_plan_kernel, (int)smem) != cudaSuccess) return check_launch("kv_plan attr");
  const int threads = std::min(1024, std::max(64, (int)((std::max<long long>(p->requests, (p->rows + 3ll) / 4) + 31) / 32 * 32)));
  const int grid = (int)std::max(1ll, std::min(2 * 148ll, ((long long)p->rows + 4095) / 4096));
  // With several CTAs, outputs that are inputs too (the free head, kv_lens over past) wait for a
  // launch of their own, so that no CTA reads them after they moved.
  const bool inplace = p->free_head || (p->kv_lens < p->past + p->requests && p->past < p->kv_lens + p->requests);
  const bool two = grid > 1 && inplace;
  const int vec = aligned16(p->slots) && aligned16(p->pos);
  PlanArgs a{*p, two ? 0 : 1, 1, vec};
  launch_k(kv_plan_kernel, grid, threads, smem, (cudaStream_t)st, a);
  note_launch();
  if (two) {
    PlanArgs b{*p, 1, 0, vec};
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
  // rows of a CTA: as many as share one head of a full block, while that leaves two CTAs an SM
  int window = 1;
  while (window * 2 * c->heads <= c->tokens && x->rows / (2 * window) >= 148 * 2) window *= 2;
  AppendArgs a{*c, *x, window};
  const int grid = (x->rows + window - 1) / window;
  if (x->dtype == YK_BF16) launch_k(kv_append_kernel<true>, grid, kAppendThreads, 0, (cudaStream_t)st, a);
  else launch_k(kv_append_kernel<false>, grid, kAppendThreads, 0, (cudaStream_t)st, a);
  note_launch();
  return check_launch("kv_append");
}
