// Kernel-level C ABI of the B200 engine (libyolob200.so).
//
// One launcher per hot-path kernel family.  Every launcher is asynchronous on the given
// stream, takes plain pointers and view descriptors (no C++ or torch types), validates its
// arguments on the host and returns 0 on success or a negative YK_E* code (nothing is
// launched on error).  The engine's executor calls these for every op of a model graph; the
// parity tests call them one op at a time through ctypes.
//
// Tensors are NHWC fp16 "views" over a buffer of shape [batch][H][W][stride]:
// element (n, y, x, c) lives at ptr[((n*H + y)*W + x)*stride + coff + c].  This is the
// reference's (buffer, channel offset, C) view (engine/engine.cu:1254-1259) with the batch
// made explicit.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* yk_stream_t;   // == cudaStream_t

#define YK_OK 0
#define YK_EINVAL (-1)      // bad shape / alignment / argument
#define YK_ECUDA (-2)       // CUDA launch error (see yk_last_cuda_error)
#define YK_ETIMEOUT (-3)    // a kernel's bounded wait gave up (device error word set)
#define YK_EUNSUP (-4)      // shape outside what the kernels implement

typedef struct {
  void* ptr;          // fp16 buffer base (NOT offset by coff)
  int batch, H, W;    // logical shape of the view
  int stride;         // channels per pixel of the underlying buffer
  int coff;           // first channel of the view
  int C;              // channels in the view
} YkView;

typedef struct {
  const void* weight;   // fp16 OHWI [Cout][k][k][Cin/groups]
  const float* bias;    // fp32 [Cout]
  int k, s, p;          // square kernel, stride, padding
  int groups;           // 1 (dense) or == Cin == Cout (depthwise)
  int act;              // 0 identity, 1 SiLU
  int Cin, Cout;
  int tile;             // tensor-core N tile (0 = heuristic, else 32/64/128/256)
  int msub;             // stacked 128-row sub-tiles per CTA tile (0 = heuristic, 1/2/4)
  int algo;             // 0 heuristic, 1 implicit GEMM (TMA im2col / gather), 2 halo patches
                        // (3x3 stride 1 pad 1, Cin % 64 == 0; tile 64/128/256, msub 1/2),
                        // 3 implicit GEMM with transposed tiles (128 output channels x
                        // 128*msub pixels per MMA; Cin >= 64; msub 1/2; tile 256: two
                        // 128-channel MMAs share the pixel operand, msub 2 only; msub 4:
                        // two 256-pixel MMAs share the weight operand),
                        // 4 halo patches with transposed tiles (as 2 but Cin % 32 == 0;
                        // tile = output channels per MMA, 64 or 128; msub 1/2),
                        // 5 halo patches with the 3 horizontal taps folded into the MMA's N
                        // (3x3 stride 1 pad 1, Cin % 32 == 0; tile 32/64 output channels,
                        // N = 3*tile; msub 1/2 for tile 32, 1 for 64),
                        // 6 CTA pairs: one M = 256 MMA over two SMs' shared memory, 256
                        // output channels x 256 pixels per pair (Cin >= 64; tile, msub
                        // ignored)
} YkConv;

// Convolution with bias, activation, optional residual (y = act(conv(x)+b) + res) written
// into y's channel slice.  Dense convs with Cin % 8 == 0 run on the tcgen05 implicit-GEMM
// kernel; Cin == 3 (first conv) and depthwise convs run on dedicated direct kernels.
// Replaces the CONV dispatch of runOp (engine/engine.cu:1263-1336).
int yk_conv(const YkView* x, const YkView* y, const YkView* res, const YkConv* p, yk_stream_t st);

// im2col of a thin input (x->C <= 8) for a k x k / stride s / pad p conv: row (n, oy, ox) of
// col gets the k*k*x->C taps in (ky, kx, c) order, zero past the image and past k*k*C
// (col->C >= k*k*x->C, a multiple of 8).  With it the first conv (Cin = 3, k*k*C = 27 -> 32)
// runs as a 1x1 tensor-core GEMM.  Replaces the reference's direct k_conv0 (engine/engine.cu:487-532).
int yk_im2col(const YkView* x, const YkView* col, int k, int s, int p, yk_stream_t st);

// 5x5 stride-1 pad-2 max pool (SPPF), engine/engine.cu:672-695.
int yk_maxpool5(const YkView* x, const YkView* y, yk_stream_t st);
// The SPPF chain y1 = pool5(x), y2 = pool5(y1), y3 = pool5(y2) in one pass over x.
int yk_maxpool5x3(const YkView* x, const YkView* y1, const YkView* y2, const YkView* y3, yk_stream_t st);
// Nearest 2x upsample, engine/engine.cu:697-708.
int yk_upsample2(const YkView* x, const YkView* y, yk_stream_t st);
// Pixel shuffle r=2 from quadrant channel blocks, engine/engine.cu:713-725.
int yk_ps2(const YkView* x, const YkView* y, yk_stream_t st);
// Channel-slice copy, engine/engine.cu:727-732.
int yk_copyc(const YkView* x, const YkView* y, yk_stream_t st);
// y = a + b, engine/engine.cu:663-670.
int yk_add(const YkView* a, const YkView* b, const YkView* y, yk_stream_t st);
// PSA attention: per image and head, out = softmax(q k^T / sqrt(kd)) v over the H*W tokens;
// qkv channel layout per head [q kd | k kd | v hd].  Replaces engine/engine.cu:1363-1404.
int yk_attn(const YkView* qkv, const YkView* y, int heads, int kd, int hd, yk_stream_t st);

// Letterbox one BGR u8 HWC frame (device memory, sh x sw) into batch slot `slot` of the
// S x S x 3 input view y (RGB, /255, pad 114, bilinear as cv2 INTER_LINEAR's formula).
// Geometry (scale, top, left) is computed on the host as in engine/engine.cu:1704-1713
// and returned through the optional out pointers.  Kernel: engine/engine.cu:968-998.
int yk_letterbox(const uint8_t* bgr, int sh, int sw, const YkView* y, int slot,
                 float* scale_out, int* top_out, int* left_out, yk_stream_t st);
// The same for n equal-size frames in one launch: frame i (BGR u8 HWC, sh x sw, device
// memory) starts at bgr + i * frame_stride bytes and fills slot slot0 + i.  All frames
// share one geometry, returned as by yk_letterbox.  Replaces one k_preprocess launch per
// frame (engine/engine.cu:1704-1713, serve.cpp's per-frame yolo_preprocess loop).
// Source rows up to about 34,000 pixels wide (YK_EUNSUP beyond).
int yk_letterbox_batch(const uint8_t* bgr, size_t frame_stride, int n, int sh, int sw,
                       const YkView* y, int slot0, float* scale_out, int* top_out,
                       int* left_out, yk_stream_t st);

// Classification head (task "classify").  Global average pool of x [B][H][W][C] into
// y [B][1][1][C], fp32 sums (engine/engine.cu:735-744, k_gap); C % 8 == 0, 16-byte views.
int yk_gap(const YkView* x, const YkView* y, yk_stream_t st);
// Channel softmax of x [B][1][1][C] into y (not in place), fp32 max / exp sum
// (engine/engine.cu:746-785, k_softmax_ch).
int yk_softmax(const YkView* x, const YkView* y, yk_stream_t st);
// Classify preprocessing of one BGR u8 HWC frame (device memory, sh x sw) into batch slot
// `slot` of the S x S x 3 input view y: shortest edge resized to S with the antialiased
// triangle filter, centre crop, RGB, /255 (torchvision Resize + CenterCrop + ToTensor;
// engine/engine.cu:1000-1046, k_preprocess_cls + clsGeom).  geom_out (optional, 4 ints)
// receives the resized height, width and the crop's top, left.
int yk_preprocess_cls(const uint8_t* bgr, int sh, int sw, const YkView* y, int slot,
                      int* geom_out, yk_stream_t st);

// Detection head levels for decode / NMS / masks.
typedef struct {
  YkView box;     // 64 channels: 4 sides x 16 DFL bins
  YkView cls;     // >= nc channels (multiple of 8; pad logits ignored)
  YkView coef;    // segment: nm mask coefficients; ptr == NULL for detect
  int stride;     // 8, 16, 32
} YkLevel;

// Oriented boxes (task "obb").  Workspace bytes for batch x anchors.
size_t yk_obb_workspace_bytes(int batch, int anchors);
// Decode of every anchor: levels[i].coef is the ANGLE view (channel 0 real); cls views hold
// nc logits zero-padded to a multiple of 8.  Records cx, cy, w, h (letterbox px), score,
// cls, theta (engine/engine.cu:908-960, k_decode_obb).
int yk_decode_obb(const YkLevel* levels, int nlevels, int batch, int nc, float conf, void* ws,
                  yk_stream_t st);
// Rotated NMS over ALL candidates (the reference keeps the first 2048): score order (ties by
// anchor), same-class probiou >= iou drops the later box, dropped boxes still suppress
// (ultralytics fast-NMS; engine/engine.cu:1160-1252).  outdets [batch][max_out][7] as the
// decode records, outcnt / rawcnt per image (survivors / candidates).
int yk_nms_obb(int batch, int anchors, float iou, int max_out, void* ws, float* outdets,
               int* outcnt, int* rawcnt, yk_stream_t st);

// Device workspace of the post-processing chain, sized by yk_post_workspace_bytes.
typedef struct {
  void* ws;          // device scratch
  size_t ws_bytes;
  float* outdets;    // device [batch][max_out][6]: x1 y1 x2 y2 score cls (letterbox px)
  int* outidx;       // device [batch][max_out]: anchor index of each survivor
  int* outcnt;       // device [batch]: survivors
  int* rawcnt;       // device [batch]: conf-passing candidates before NMS
} YkPost;

size_t yk_post_workspace_bytes(int batch, int anchors);
// Decode (engine/engine.cu:848-906): per anchor best class over nc, score = sigmoid,
// keep if score >= conf, DFL box.  Candidates keep anchor order (no atomics).
int yk_decode(const YkLevel* levels, int nlevels, int batch, int nc, float conf,
              const YkPost* post, yk_stream_t st);
// NMS (engine/engine.cu:1051-1123, made exact and deterministic): every candidate is
// considered (no 1024 cap); order = score desc, anchor index asc; same-class IoU > iou
// suppresses; at most max_out survivors per image.
int yk_nms(int batch, int anchors, float iou, int max_out, const YkPost* post, yk_stream_t st);
// Masks for NMS survivors (engine/engine.cu:1129-1158): logit = coef . proto, crop to the
// box scaled to proto resolution (half-open), mask = logit > 0.  masks: [batch][max_out][Ph][Pw].
int yk_masks(const YkLevel* levels, int nlevels, const YkView* proto, int in_h, int in_w,
             int max_out, const YkPost* post, uint8_t* masks, yk_stream_t st);

// Decode + NMS with no allocation at all (no counterpart in the reference).  For callers
// that cannot call cudaMalloc — code under a fixed device-memory budget, plugins whose host
// framework owns all allocations, loops that must never enter the allocator — the scratch
// lives in one static 8 MiB device array inside the library instead of a YkPost workspace.
// Same arguments and results as yk_decode + yk_nms; outputs as in YkPost ([batch][max_out][6],
// [batch][max_out], [batch], [batch]).  Limit: batch * per-image scratch <= 8 MiB (about
// 9 images of 8400 anchors at 640, 3 images at 1024); larger requests return YK_EINVAL with
// the reason in yk_last_cuda_error.  The first call on each device looks up the array's
// device address (cudaGetSymbolAddress), so make that first call before any stream capture.
// All calls on a device share the one array and it keeps the last call's contents: calls
// whose kernels overlap on the GPU (other streams, other threads) race and corrupt each other.
// The looked-up address is kept for the life of the process: resetting a device
// (cudaDeviceReset) while the library stays loaded is not supported by this entry point.
int yk_decode_nms_static(const YkLevel* levels, int nlevels, int batch, int nc, float conf,
                         float iou, int max_out, float* outdets, int* outidx, int* outcnt,
                         int* rawcnt, yk_stream_t st);

// ---------------------------------------------------------------------------------------
// Text decoder (no counterpart in the reference): the operators of one step of a decoder that
// answers about a frame or its detections, over ragged batches of requests.  Lengths, tables
// and slots are device arrays, nothing is read back and nothing is allocated, so a whole step
// is one CUDA graph.  8-bit values are e4m3 codes (1 sign, 4 exponent, 3 fraction bits, largest
// 448, no infinity); a value is code * scale.  A refused call (YK_EINVAL, YK_EUNSUP) launches
// nothing and says why in yk_last_cuda_error().
#define YK_F16 0
#define YK_BF16 1
#define YK_E4M3 2
#define YK_F32 3

// Key/value cache in 8 bits: a pool of blocks of `tokens` tokens, one scale for each (block,
// head).  Channel d of token t of head h in block b is code b*block_stride + (h*tokens + t)*dim
// + d of k and v, its scale entry b*scale_stride + h of kscale and vscale.  Slot s of the pool
// is token s % tokens of block s / tokens.
typedef struct {
  void* k;                 // e4m3 codes, 16-byte aligned
  void* v;
  float* kscale;           // positive
  float* vscale;
  long long block_stride;  // codes from block to block, >= heads*tokens*dim, multiple of 16
  long long scale_stride;  // scales from block to block, >= heads
  int blocks;              // blocks of the pool (blocks * tokens < 2^31)
  int heads;               // key/value heads
  int tokens;              // tokens of a block: 16, 32, 64 or 128
  int dim;                 // channels of a head: 64, 128 or 256
} YkKvCache;

// Block tables and slots of a step from the requests' lengths.  Request r holds past[r] tokens
// in the blocks table[r][0 .. ceil(past/tokens)) and adds fresh[r].  In request order, each
// takes the blocks it needs more from free_blocks (from entry *free_head on, when given) and
// appends them to its table row.  Row n of the step is token past + j of its request r, with
// n = cu[r] + j: pos[n] is that position and slots[n] its place in the pool.
// A request is refused, and takes no block, when its needs and those of all requests before it pass
// the free blocks (one that needs none still goes on): after the first that does not fit, each later
// one that needs a block is refused too, so that none is overtaken, even where enough are left for it.
// It is also refused when its tokens pass max_blocks blocks or a length is negative (a negative fresh
// counts as no rows), which does not hold up the ones after it, and when its rows pass `rows`.  Its
// kv_lens stays past and its rows' slots are -1; so are the slots of rows past the last
// request's (their pos too), and of tokens whose table entry lies outside the pool.
typedef struct {
  const int* past;         // [requests]
  const int* fresh;        // [requests]
  const int* free_blocks;  // [free_count] block ids
  int* free_head;          // NULL (0), or in/out: the first free entry; moved past those taken
  int* table;              // in/out [requests][table_stride]; only the new entries are written
  int* kv_lens;            // out [requests]: past + fresh, or past if refused; may be `past`
  int* cu;                 // out [requests + 1]: rows before each request (at most `rows`)
  int* slots;              // out [rows]
  int* pos;                // out [rows], or NULL
  int* counts;             // out [4]: blocks taken, rows placed, requests refused, rows; or NULL
  long long table_stride;  // >= max_blocks
  int requests;            // 1 .. 16384
  int rows;                // rows of slots and pos
  int free_count;
  int blocks;              // blocks of the pool
  int max_blocks;          // table entries of a request
  int tokens;              // tokens of a block: 16, 32, 64 or 128
} YkKvPlan;
int yk_kv_plan(const YkKvPlan* p, yk_stream_t st);

// New keys and values, one row a token: head h of row n at n*k_row + h*k_head.
typedef struct {
  const void* k;           // fp16 or bf16, 16-byte aligned
  const void* v;
  const int* slots;        // [rows]; a row whose slot lies outside the pool is left out
  long long k_row, v_row, k_head, v_head;   // elements, multiples of 8
  int rows;
  int dtype;               // YK_F16 or YK_BF16
} YkKvRows;
// Quantises rows into the cache.  The rows of one block are consecutive and ascend (as
// yk_kv_plan's slots do); tokens before them in the block are kept, tokens after them are not
// used.  Each (block, head) gets the smallest power-of-two scale that holds its finite new
// values (at least 2^-126), or keeps its scale where that is larger and the block has earlier
// tokens; those are rounded to the new scale where it grew.  Infinite values become +-448, NaN
// stays NaN.
int yk_kv_append(const YkKvCache* c, const YkKvRows* x, yk_stream_t st);

// Attention of a step's rows over the cache: rows cu[r] .. cu[r+1]-1 are request r's last
// tokens, query head h reads key/value head h / (heads / c->heads).  causal: row i of a request
// of q rows sees keys j <= kv_lens[r] - q + i, with a window w > 0 only j > kv_lens[r] - q + i
// - w; else every key.  A row that sees no key gives zeros (lse -inf); keys in blocks outside
// the pool are not seen.  What the cache holds past kv_lens is never used.  Scores, their maximum and
// the weights' sum are in 32 bits.  The weights meet the values as fp16, rounded once; for fp16 rows of a
// request with at most 8 rows a key head, in a call of few rows, as two parts of fp16 (22 bits).
typedef struct {
  const void* q;           // head h of row n at n*q_row + h*dim; fp16 or bf16, 16-byte aligned
  void* out;               // likewise, with out_row
  float* lse;              // [rows][heads]: log of the sum of the weights, or NULL
  const int* cu;           // [requests + 1]
  const int* kv_lens;      // [requests]
  const int* table;        // [requests][table_stride] block ids
  void* ws;                // yk_attn_kv8_workspace_bytes, 16-byte aligned, zeroed before its first
  size_t ws_bytes;         // use (each call leaves it so); calls that overlap need one each
  long long q_row, out_row;   // elements, multiples of 8
  long long table_stride;
  int max_blocks;          // table entries of a request
  int requests;            // 1 .. 16384
  int rows;                // rows * heads below 2^31
  int heads;               // query heads, a multiple of c->heads
  int dtype;               // YK_F16 or YK_BF16 (q and out)
  int causal;
  int window;              // 0: none
  float scale;             // of the products; 0: 1 / sqrt(dim)
} YkAttnKv8;
size_t yk_attn_kv8_workspace_bytes(int requests, int rows, int heads, int kv_heads, int dim);
int yk_attn_kv8(const YkKvCache* c, const YkAttnKv8* a, yk_stream_t st);

// h = x + add, y = h / sqrt(mean(h^2) + eps) * weight over each row, in 32 bits; sum = h and
// out = y rounded to dtype, codes = y / scale rounded to e4m3 with one scale for each `group`
// columns: the largest finite |y| / 448 (at least 2^-126).  sum may be x or add itself.
typedef struct {
  const void* x;
  const void* add;         // or NULL
  void* sum;               // or NULL
  const void* weight;      // [cols]
  void* out;               // or NULL
  void* codes;             // e4m3, or NULL
  float* scales;           // [rows][scales_row], with codes
  long long x_row, add_row, sum_row, out_row, codes_row, scales_row;   // elements
  int rows, cols;          // cols up to 32768
  int group;               // columns of a scale, at least 16 (the last group may be shorter); 0: the
                           // whole row
  int dtype;               // YK_F16 or YK_BF16: x, add, sum, weight, out
  float eps;
} YkRmsNorm8;
int yk_rmsnorm8(const YkRmsNorm8* p, yk_stream_t st);

// y[m][j] = sum_k x[m][k] * (q[j][k] - zero) * scale + bias[j] for up to 64 rows: 4-bit weights
// q (0..15), byte i of a row holds column 2i in its low and 2i+1 in its high half; scale and zero
// for each `group` columns.  x is fp16 / bf16, or e4m3 codes with a scale for each xgroup columns
// (yk_rmsnorm8's output).  32-bit sums, one rounding to dtype.
typedef struct {
  const void* x;
  const float* xscale;     // e4m3: [rows][xscale_row]
  const void* w;           // [n][w_row bytes], 16-byte aligned
  const void* wscale;      // [n][group_row] of dtype
  const void* wzero;       // [n][group_row] bytes 0..15, or NULL (8)
  const float* bias;       // [n] or NULL
  void* y;                 // [rows][y_row]
  long long x_row, xscale_row, w_row, group_row, y_row;   // elements; w_row: bytes, multiple of 16
  int rows;                // 1 .. 64
  int n;                   // outputs
  int k;                   // columns, a multiple of group
  int group;               // 32, 64 or 128
  int xgroup;              // e4m3: a multiple of group, or 0: one scale a row
  int xtype;               // dtype, or YK_E4M3
  int dtype;               // YK_F16 or YK_BF16: wscale, y (and x)
} YkGemv4;
int yk_gemv4(const YkGemv4* p, yk_stream_t st);

// Norm of each query and key head, and its rotary position, in one pass: h = a head's row (dim channels),
// y = h / sqrt(mean(h^2) + eps) * weight in 32 bits (without a weight: y = h), then pair i < rot/2 turns by
// the angle pos[axis of i][n] * freqs[i]: (a, b) -> (a cos - b sin, b cos + a sin), rounded once to dtype.
// The pair is channels (i, i + rot/2), or (2i, 2i + 1) if interleaved; channels from rot on do not turn.
// The first sections[0] pairs follow axis 0, the next sections[1] axis 1, and so on (time, row, column of
// an image's tokens).  Whole turns are taken off in whole numbers: an angle is within 2^-31 of a turn at any position, with
// frequencies up to 2^40.  Rows whose pos on axis 0 is negative are left as they are.  Outputs may be the inputs themselves.
typedef struct {
  const void* q;           // head h of row n at n*q_row + h*dim; fp16 or bf16, 16-byte aligned
  const void* k;           // likewise with k_row; NULL with kv_heads 0
  void* q_out;             // likewise with q_out_row; q itself with its stride, or apart from it
  void* k_out;
  const void* q_weight;    // [dim] of dtype, or NULL: no norm
  const void* k_weight;
  const int* pos;          // axis a of row n at a*pos_axis + n
  const float* freqs;      // [rot / 2] radians a position, finite
  long long q_row, k_row, q_out_row, k_out_row;   // elements, multiples of 8
  long long pos_axis;
  int rows;
  int heads;               // query heads
  int kv_heads;            // key heads (0: queries only); heads + kv_heads at most 1024
  int dim;                 // 32, 64, 128 or 256
  int rot;                 // channels that turn: a multiple of 16, at most dim
  int axes;                // 1 .. 4
  int sections[4];         // pairs of each axis, rot / 2 in all; with one axis all zeros serve too
  int interleaved;
  int dtype;               // YK_F16 or YK_BF16
  float eps;
} YkQkRotate;
int yk_qk_rotate(const YkQkRotate* p, yk_stream_t st);

// Matrices of 4-bit floats (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with a scale for each group
// of columns of a row: YK_NVFP4 has groups of 16 with e4m3 scales, YK_MXFP4 groups of 32 with powers of two
// (one byte e: 2^(e - 127), 255: NaN).  A value is code * scale of its group * scale of the whole matrix.
// Byte i of a row holds column 2i in its low and 2i + 1 in its high half.  Scales lie in blocks of 128
// rows x 4 groups, 512 bytes each, along the groups first: with B = ceil(groups / 4), the scale of row r
// and group g is byte ((r / 128) * B + g / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + g % 4.
#define YK_NVFP4 0
#define YK_MXFP4 1
// Bytes of the scales of rows x cols: whole blocks.  0 if an argument is out of range.
size_t yk_fp4_scale_bytes(int rows, int cols, int format);
// Rounds rows to 4 bits.  t = largest finite |x| of the group / (6 scale); the group's scale is t rounded to
// e4m3, between 2^-9 and 448 (YK_NVFP4), or the smallest power of two >= t between 2^-96 and 2^96 (YK_MXFP4);
// codes are x / (group's scale * scale) rounded to nearest, ties to even, at most 6 (infinities too).  A group
// with a NaN has a NaN scale and codes 0.  Codes of columns past the last up to a multiple of 8, scales of groups past
// the last up to a multiple of 4 and of rows past the last up to a multiple of 128 are 0.
typedef struct {
  const void* x;           // [rows][x_row] of dtype
  void* codes;             // [rows][codes_row bytes], 16-byte aligned
  void* scales;            // yk_fp4_scale_bytes, 16-byte aligned
  void* values;            // [rows][values_row]: what the codes stand for, rounded to dtype; or NULL
  long long x_row, values_row;   // elements
  long long codes_row;     // bytes, a multiple of 16
  int rows, cols;
  int format;              // YK_NVFP4 or YK_MXFP4
  int dtype;               // YK_F16 or YK_BF16
  float scale;             // of the whole matrix, 2^-30 .. 2^30; 0: 1
} YkQuantFp4;
int yk_quant_fp4(const YkQuantFp4* p, yk_stream_t st);

// y[m][j] = alpha * sum_k x[m][k] w[j][k] + bias[j] of two such matrices of one format, or, with w2, a gated
// pair: g = alpha * x w^T, y = g / (1 + exp(-g)) * (alpha2 * x w2^T).  alpha takes the scales of the whole
// matrices.  Sums in 32 bits, one rounding to dtype.  Any rows, n and k; with an odd k the last byte's high half
// has to be 0 in x or w, and scales of groups past the last up to a multiple of 4 no NaN (yk_quant_fp4 writes both so).
typedef struct {
  const void* x;           // [rows][x_row bytes], 16-byte aligned
  const void* xscale;      // yk_fp4_scale_bytes(rows, k, format), 16-byte aligned
  const void* w;           // [n][w_row bytes]
  const void* wscale;      // yk_fp4_scale_bytes(n, k, format)
  const void* w2;          // as w, or NULL: not gated
  const void* w2scale;
  const float* bias;       // [n] or NULL; not with w2
  void* y;                 // [rows][y_row]
  long long x_row, w_row;  // bytes, multiples of 16 (of 128: up to a fifth faster)
  long long y_row;         // elements
  int rows, n, k;
  int format;              // YK_NVFP4 or YK_MXFP4
  int dtype;               // YK_F16 or YK_BF16: y
  float alpha, alpha2;     // 0: 1
} YkGemmFp4;
int yk_gemm_fp4(const YkGemmFp4* p, yk_stream_t st);

// The next token of each row of scores.  weight_i = exp((l_i - max) / temperature) (a score of NaN or -infinity has
// none; if the largest is +infinity, those that are have weight 1 and the others none).  In the order of falling scores,
// equal ones by index, stay the first top_k; of these the shortest beginning whose weight reaches top_p
// of theirs; and of these the ones of at least min_p times the largest weight.  The token is the first, by index, at which
// the sum of the weights that stay passes u times their total.  Weights and sums are exact to 2^-44 of the
// largest weight, whatever the launch.  A temperature that is not positive takes the largest score, the
// lowest index among equal ones.  A row without any weight gives token -1, log probability -infinity, 0 kept.
typedef struct {
  const void* logits;      // [rows][row]: fp16, bf16 or fp32
  const float* temperature;// [rows], or NULL: 1
  const int* top_k;        // [rows]: 0 or less: all; or NULL
  const float* top_p;      // [rows]: 1 or more, or NaN: all; 0 or less: one; or NULL
  const float* min_p;      // [rows]: 0 or less, or NaN: all; or NULL
  const float* u;          // [rows] in [0, 1) (a smaller one or NaN counts as 0, a larger as the last token); NULL: largest score
  int* token;              // out [rows]
  float* logprob;          // out [rows]: log of the token's weight over the total of those that stay; or NULL
  int* kept;               // out [rows]: how many stay (of a weight that is not 0); or NULL
  long long row;           // elements, >= n
  int rows;
  int n;                   // scores of a row, 1 .. 262144
  int dtype;               // YK_F16, YK_BF16 or YK_F32
} YkSample;
int yk_sample(const YkSample* p, yk_stream_t st);

// Device error word (bounded-wait timeouts) of the current device; cleared by the call.
int yk_fetch_device_error(void);
// Test hook for the bounded-wait failure path (no counterpart in the reference, which has no
// bounded waits): wait_ns sets the wait budget of every kernel on the current device (0 =
// the default 2 s); withhold = 1 makes block 0 of the next tensor-core conv launches on the
// TMA path skip its first stage load, so that block's MMA wait runs out, the device error
// word is set and the kernel unwinds (no trap, no hang: the wait is bounded).  Synchronous;
// call yk_test_inject(0, 0) to restore normal operation.
int yk_test_inject(int withhold, unsigned long long wait_ns);
// Test hook: CTAs per image of the NMS launch (thread-block cluster size 1, 2, 4 or 8; 0
// restores the default, the largest power of two up to 8 with batch x size <= the SM count).
// Results do not depend on it; tests compare every size bit for bit.
int yk_test_nms_cluster(int size);
// Test hook: the kernel behind yk_attn_kv8 (1: keys split over all CTAs, 2: 128-row tiles, 0: the
// library's rule); tests compare both with the definition.
int yk_test_attn_kv8(int kernel);
// Test hook: the kernel behind yk_gemm_fp4 (1: whole tiles, 2: columns split over `split` = 1, 2, 4 or 8
// CTAs; 0: the library's rules, each for itself); tests compare all with the definition.
int yk_test_gemm_fp4(int kernel, int split);
// Test hook: CTAs of a row in yk_sample (1, 2, 4 or 8; 0: the library's rule, as where a row needs more).
// Results do not depend on it; tests compare all bit for bit.
int yk_test_sample(int split);
// Test hook: 16-bit scores in yk_sample counted by bins of weight (1) or by place (2); 0: the library's rule.
int yk_test_sample_kernel(int kernel);
const char* yk_last_cuda_error(void);
// Number of kernels this library launched since load (all devices) — a host-side counter.
long long yk_launch_count(void);

#ifdef __cplusplus
}
#endif
