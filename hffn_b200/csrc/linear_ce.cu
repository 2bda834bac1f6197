// Linear softmax cross entropy over a large vocabulary: the loss of hidden states h [n, d] under the head w [vocab, d]
//   z_tv = h_t . w_v,   lse_t = log sum_v exp z_tv,   loss_t = lse_t - z_{t, target_t}
// and its gradients
//   g_tv = c_t (exp(z_tv - lse_t) - [v = target_t]),   dh_t = sum_v g_tv w_v,   dw_v = sum_t g_tv h_t
// without the [n, vocab] logits: the forward reduces each tile of logits to a maximum and a sum of exponentials per
// row, and the backward recomputes the logits of one piece of the vocabulary at a time into g.
//
// The sums leave the target's own logit out, so that with the odds o = sum_{v != target} exp(z_v - z_target)
//   loss = log(1 + o),   g_target = -c o / (1 + o),
// both without a difference of nearly equal numbers where the target is well predicted (o small): lse - z and p - 1 would
// leave of a loss of 1e-5 two digits, and p - 1 of logits summed once more in another order fewer. g_target is the
// forward's; the other entries of g are as close, relative to themselves, as their logits are absolutely.
//
// Only kept rows exist for the products: rows whose target is ignored (or out of range) are left out when the hidden
// states are gathered, so they cost nothing and whatever they hold (infinities, NaN) reaches no sum. How many are
// kept is known on the device alone; every kernel reads it there, so a call can be captured and replayed.
//
// The products (2 n vocab d operations each: the logits twice, dh, dw) bound everything from a few hundred tokens on;
// below that the head's bytes do. All run in one persistent tcgen05 kernel shape on pairs of SMs (cta_group::2): a
// tile of 256 x 256 accumulators, 128 rows in each SM's TMEM, each SM loading its own 128 rows of A and half of B, so
// that an SM takes 32 KB from L2 per 64 values of K for 256 x 256 x 64 products of the pair. Two accumulator buffers let
// the epilogue of one tile run under the products of the next.
//
// Types. bfloat16: products of the inputs as they are; g is held in bfloat16, off by at most 2^-8 of an entry, as the
// gradients' own storage. It holds p - [v = target] where all tokens have one c, which is applied to dh and dw in float32
// (the target's entry of a token that is not well predicted, the largest, is then close to -1, which is exact), and c
// with it where they differ (a c h in bfloat16 beside it would round twice). float32: three fp16 products per product, of
// operands held as two fp16 parts (hi = rn(x 2^e), lo = rn(x 2^e - hi); hi hi + hi lo + lo hi, the rest is below 2^-22),
// 2^e a power of two that brings the largest finite entry to [2^14, 2^15): entries down to 2^-17 of the largest keep 22
// bits, smaller ones are held to 2^-39 of it. For the logits every row of h and of w has a scale of its own, which is a
// factor of its logits, so that no token or id takes bits from another, however large. dh sums over the rows of w, and dw
// over those of h: there one scale has to serve the operand, whose parts the backward makes once more (rows_kernel: 59 us
// of 2048 x 1024 x 50304). g holds 2^14 (p - [v = target]); c_t is applied in float32 afterwards (dh: per row; dw: one
// factor, or rows of h scaled by their c_t beforehand where they differ). Sums: the tensor core's float32 accumulation
// truncates at every step, so what ends in float32 (float32 gradients, losses) is summed in registers from accumulators of
// few steps each (chunk_of).
//
// Measured (ncu, products alone): bfloat16 8192 x 2048 x 12800 logits 261 us, g 266 us, dh and dw 546 us (1.57 to 1.65
// PFLOP/s, 96 to 97 % of the tensor pipe's cycles); float32 2048 x 1024 x 25344 218, 245 and 449 us (86, 74 and 93 %).
// The kernels that sum in registers (all float32 ones, bfloat16 logits) use all 168 registers that 320 threads leave, and
// spill 72 to 200 bytes a thread.
// Back to back for a second or more the card's power limit sets the rate: 1.42 PFLOP/s for 8192 x 2048 x 50304 logits,
// what the library's plain product sustains.
#include <cuda_fp16.h>

#include <algorithm>

#include "tc_ptx.cuh"

namespace hffn {
namespace ce {

using namespace tc;

constexpr int kTile = 256;                           // rows and columns of a pair's tile
constexpr int kBlockK = 64;                          // values of K in a stage: 128 bytes, the swizzle's row
constexpr int kThreads = 320;                        // warp 0: loads, warp 1: products, warps 2 to 9: epilogue
constexpr int kEpilogueWarps = 8;
constexpr int kGroupRows = 32;                       // row tiles of logits that share their pass over the vocabulary
constexpr int kOperandBytes = 128 * kBlockK * 2;     // one SM's share of one operand part in a stage
constexpr int kStageBytes = 6 * 2 * kOperandBytes;   // all stages of one SM
constexpr int kOutBytes = 4096;                      // an epilogue warp's 32 rows x 32 columns on their way out
constexpr int kSmem = 1024 + kStageBytes + kEpilogueWarps * kOutBytes + 256;
constexpr int64_t kPieceBytes = int64_t(256) << 20;  // of g: the piece of the vocabulary the backward holds at a time
constexpr int kPieceMin = 4096;
constexpr int kMaxDevices = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kErrLoad = 401, kErrProduct = 402, kErrEpilogue = 403;

__device__ int g_error;   // first error code of a wait that ran out (0: none)

__host__ __device__ inline int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// What the forward leaves for the backward, in one buffer.
struct State {
  int32_t* kept;       // [1] rows kept
  uint32_t* arrived;   // [1] blocks of the losses that are done
  uint32_t* largest;   // [2] float32, backward: bits of the largest finite |entry| of the kept rows and of the head
  int32_t* failed;     // [1] not 0: a wait of the call ran out, tiles are missing from its results, which become NaN
  int32_t* row_of;     // [n] the input row of each kept row
  int32_t* place_of;   // [n] the kept row of each input row; -1: left out
  int32_t* target;     // [n]
  float2* sums;        // [n] of each kept row the largest logit and the sum of exponentials relative to it
  float* own;          // [n] p - 1 of its target
  void* hidden[2];     // [n_pad, d] the kept rows (float32: their fp16 parts, each row at a scale of its own)
  float* hidden_inverse;   // [n_pad] float32: the inverse scales of those rows
  void* head[2];       // [vocab, d] float32: the head's fp16 parts, each row at a scale of its own
  float* inverse;      // [vocab] float32: the inverse scales of those rows
  float* raw;          // [n, d] float32, few rows: the kept rows as they are. Their parts and the head's, for which the
                       // backward has room, are made there
  int64_t bytes;
};

struct Carve {
  uint8_t* base;
  int64_t at = 0;
  template <typename T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + at);
    at += round_up(count * (int64_t)sizeof(T), 256);
    return p;
  }
};

// Few rows: their logits are computed on the CUDA cores, straight from the head (few_kernel), where that is faster than
// the tensor cores' tiles. float32: up to 16 rows, in passes of 8, since it spares making the head's fp16 parts (a pass
// of reads and one of writes before the products): vocabulary 50304, whole calls, 4, 8 and 16 rows here against 17 in
// tiles: d 512 31, 50 and 74 us against 79, d 1024 50, 80 and 122 against 131, d 2048 91, 140 and 219 against 245; 32 rows
// of 1024 would take 228. bfloat16: one row against two in tiles: 23 us against 24, 32 against 37 and 51 against 58 (two
// rows of 1024 here: 42). The rows have to fit the kernel's shared memory.
constexpr int kFewRows = 8, kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int64_t kFewBytes = 96 << 10;

// Rows of one pass.
static int few_rows(int dtype, int64_t n) {
  return dtype == HFFN_BF16 ? 1 : n <= kFewRows / 2 ? kFewRows / 2 : kFewRows;
}

static bool is_few(int dtype, int64_t n, int d) {
  return n <= (dtype == HFFN_F32 ? 2 * kFewRows : 1) && (int64_t)few_rows(dtype, n) * d * 4 <= kFewBytes;
}

static void take_head(Carve& c, void* (&head)[2], float*& inverse, int d, int vocab) {
  for (int part = 0; part < 2; ++part) head[part] = c.take<uint16_t>((int64_t)vocab * d);
  inverse = c.take<float>(vocab);
}

static State state_at(void* base, int dtype, int64_t n, int d, int vocab) {
  Carve c{static_cast<uint8_t*>(base)};
  const int64_t n_pad = round_up(n, kTile);
  State s = {};
  s.kept = c.take<int32_t>(5);
  s.arrived = reinterpret_cast<uint32_t*>(s.kept + 1);
  s.largest = reinterpret_cast<uint32_t*>(s.kept + 2);
  s.failed = s.kept + 4;
  s.row_of = c.take<int32_t>(n_pad);
  s.place_of = c.take<int32_t>(n_pad);
  s.target = c.take<int32_t>(n_pad);
  s.sums = c.take<float2>(n_pad);
  s.own = c.take<float>(n_pad);
  for (int part = 0; part < (dtype == HFFN_F32 ? 2 : 1); ++part) s.hidden[part] = c.take<uint16_t>(n_pad * d);
  if (dtype == HFFN_F32) {
    s.hidden_inverse = c.take<float>(n_pad);
    if (is_few(dtype, n, d)) s.raw = c.take<float>(n * d);
    else take_head(c, s.head, s.inverse, d, vocab);
  }
  s.bytes = c.at;
  return s;
}

// The gradient of the losses as the caller gave it: c_t of a kept row.
struct Upstream {
  const float* grad_loss;
  int reduction;
  __device__ __forceinline__ float of(const State& s, int row, int kept) const {
    if (reduction == HFFN_REDUCE_NONE) return grad_loss[s.row_of[row]];
    return reduction == HFFN_REDUCE_MEAN ? grad_loss[0] / (float)kept : grad_loss[0];
  }
};

// Programmatic dependent launch: a kernel of a call is started while its predecessor still runs (its prologue and its
// launch then overlap the predecessor's end) and touches global memory only after this, when the predecessor has
// completed. In a plain launch both are no-ops.
__device__ __forceinline__ void depend() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- scales of the fp16 parts -------------------------------------------------------------------------------------
// The exponent e of an operand's scale 2^e from the bits of its largest finite magnitude.
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
  if (bits == 0) return 0;
  return min(14 - ((int)(bits >> 23) - 127), 110);
}

__device__ __forceinline__ float power_of_two(int e) { return ldexpf(1.f, e); }

__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
  return bits < 0x7f800000u ? bits : 0u;
}

// Eight values as fp16 parts, 16 bytes each; two at a time, since the single conversions run at a quarter of the rate.
__device__ __forceinline__ void split8(const float* x, uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2 high = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
    const float2 back = __half22float2(high);
    const __half2 low = __floats2half2_rn(x[2 * j] - back.x, x[2 * j + 1] - back.y);
    h[j] = *reinterpret_cast<const uint32_t*>(&high);
    l[j] = *reinterpret_cast<const uint32_t*>(&low);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

__device__ __forceinline__ void store_parts(const float (&x)[8], __half* hi, __half* lo) {
  uint4 h, l;
  split8(x, h, l);
  *reinterpret_cast<uint4*>(hi) = h;
  *reinterpret_cast<uint4*>(lo) = l;
}

// ---- which rows are kept ------------------------------------------------------------------------------------------
constexpr int kGatherThreads = 256;
constexpr int kGatherWarps = kGatherThreads / 32;

__device__ __forceinline__ bool is_kept(int64_t target, int64_t ignore, int vocab) {
  return target != ignore && target >= 0 && target < vocab;
}

__device__ __forceinline__ int block_count(int mine, int* shared) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = mine;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kGatherWarps; ++w) total += shared[w];
  return total;
}

// Raises a largest magnitude by a whole warp's; most find it raised already, and spare the atomic.
__device__ __forceinline__ void raise_largest(uint32_t* largest, uint32_t bits) {
  bits = __reduce_max_sync(0xffffffffu, bits);
  if ((threadIdx.x & 31) == 0 && bits > *const_cast<volatile uint32_t*>(largest)) atomicMax(largest, bits);
}

// A block owns `span` consecutive input rows. It counts the kept rows before them (from the targets alone, so that no block
// waits for another), places its own, and copies them (bfloat16; float32: a second kernel stores their parts).
template <typename T>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const T* hidden, int64_t stride,
                                                                const int64_t* targets, int64_t ignore, int n, int d,
                                                                int vocab, int span, bool aligned, float* losses,
                                                                State s) {
  __shared__ int shared[kGatherWarps];
  depend();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * span, last = min(n, first + span);
  int mine = 0;
  for (int t = threadIdx.x; t < first; t += kGatherThreads) mine += is_kept(targets[t], ignore, vocab);
  int place = block_count(mine, shared);
  T* out = static_cast<T*>(s.hidden[0]);
  for (int base = first; base < last; base += 32) {      // every warp walks all rows and takes every eighth kept one
    const int t = base + lane;
    const int64_t target = t < last ? targets[t] : ignore;
    const bool keep = t < last && is_kept(target, ignore, vocab);
    const unsigned mask = __ballot_sync(0xffffffffu, keep);
    if (warp == 0 && t < last) {
      const int at = place + __popc(mask & ((1u << lane) - 1u));
      s.place_of[t] = keep ? at : -1;
      if (keep) {
        s.row_of[at] = t;
        s.target[at] = (int)target;
      } else {
        losses[t] = target == ignore ? 0.f : NAN;
      }
    }
    int at = place;
    if (sizeof(T) == 2)
      for (unsigned left = mask; left; left &= left - 1, ++at) {
        if ((at & (kGatherWarps - 1)) != warp) continue;
        const T* from = hidden + (int64_t)(base + __ffs(left) - 1) * stride;
        T* to = out + (int64_t)at * d;
        if (aligned)
          for (int i = lane; i < d / 8; i += 32)
            reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(from)[i];
        else
          for (int i = lane; i < d; i += 32) to[i] = from[i];
      }
    place += __popc(mask);
  }
  if (last == n && threadIdx.x == 0) {
    *s.kept = place;
    *s.arrived = 0;
    *s.failed = 0;
  }
}

__device__ __forceinline__ void load8(const float* from, bool aligned, float (&x)[8]) {
  if (aligned) {
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(from);
    *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(from + 4);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = from[j];
  }
}

// One warp: the fp16 parts of a row times `scale`, from value `first` on.
__device__ __forceinline__ void split_row(const float* from, bool aligned, int first, int d, float scale, __half* hi,
                                          __half* lo) {
  for (int i = first + 8 * (threadIdx.x & 31); i < d; i += 256) {
    float x[8];
    load8(from + i, aligned, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= scale;
    store_parts(x, hi + i, lo + i);
  }
}

// float32: the fp16 parts of the head and of the kept rows (from `hidden`, or from the state where `hidden` is NULL) for
// the logits, one warp a row, each row at a scale of its own. for_backward: also the largest magnitudes of both.
__global__ void __launch_bounds__(256) split_kernel(const float* hidden, int64_t stride, bool aligned, const float* head,
                                                    int d, int vocab, bool for_backward, State s) {
  depend();
  int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  const bool of_head = row < vocab;
  if (!of_head) row -= vocab;
  if (!of_head && row >= *s.kept) return;
  const float* from = of_head          ? head + (int64_t)row * d
                      : hidden != NULL ? hidden + (int64_t)s.row_of[row] * stride
                                       : s.raw + (int64_t)row * d;
  aligned = aligned || of_head;
  // the first kHeld values of a row stay in registers between the two passes over it (50304 rows of 1024: 61 us, 79 with
  // a second read)
  constexpr int kHeld = 4 * 256;
  const int lane = threadIdx.x & 31;
  float x[kHeld / 256][8];
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < kHeld / 256; ++k) {
    const int i = 256 * k + 8 * lane;
    if (i < d) load8(from + i, aligned, x[k]);
  }
#pragma unroll
  for (int k = 0; k < kHeld / 256; ++k)
    if (256 * k + 8 * lane < d)
#pragma unroll
      for (int j = 0; j < 8; ++j) bits = max(bits, finite_bits(x[k][j]));
  for (int i = kHeld + lane; i < d; i += 32) bits = max(bits, finite_bits(from[i]));
  bits = __reduce_max_sync(0xffffffffu, bits);
  const int e = scale_exponent(bits);
  const float scale = power_of_two(e);
  if (lane == 0) (of_head ? s.inverse : s.hidden_inverse)[row] = power_of_two(-e);
  if (for_backward) raise_largest(s.largest + of_head, bits);
  const int64_t at = (int64_t)row * d;
  __half* hi = static_cast<__half*>(of_head ? s.head[0] : s.hidden[0]) + at;
  __half* lo = static_cast<__half*>(of_head ? s.head[1] : s.hidden[1]) + at;
#pragma unroll
  for (int k = 0; k < kHeld / 256; ++k) {
    const int i = 256 * k + 8 * lane;
    if (i >= d) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[k][j] *= scale;
    store_parts(x[k], hi + i, lo + i);
  }
  split_row(from, aligned, kHeld, d, scale, hi, lo);
}

// float32: eight values of a kept row times c, from its parts.
__device__ __forceinline__ void kept_values(const State& s, int row, int i, int d, float c, float (&x)[8]) {
  const uint4 hi = *reinterpret_cast<const uint4*>(static_cast<const __half*>(s.hidden[0]) + (int64_t)row * d + i);
  const uint4 lo = *reinterpret_cast<const uint4*>(static_cast<const __half*>(s.hidden[1]) + (int64_t)row * d + i);
  const float inverse = s.hidden_inverse[row];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    x[j] = c * ((__half2float(reinterpret_cast<const __half*>(&hi)[j]) +
                 __half2float(reinterpret_cast<const __half*>(&lo)[j])) * inverse);
}

// float32, a gradient of its own for each token: the largest magnitude of the rows c_t h_t.
__global__ void __launch_bounds__(256) scaled_largest_kernel(State s, Upstream upstream, uint32_t* largest, int d) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), kept = *s.kept;
  if (row >= kept) return;
  uint32_t bits = 0;
  for (int i = 8 * (threadIdx.x & 31); i < d; i += 256) {
    float x[8];
    kept_values(s, row, i, d, upstream.of(s, row, kept), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) bits = max(bits, finite_bits(x[j]));
  }
  raise_largest(largest, bits);
}

// float32: the operands that dh and dw sum over, as fp16 parts at one scale each: `width` rows of the head, then of the
// first `rows` kept rows h_t, or c_t h_t where each token has a gradient of its own (`each`), padded with zeros to a whole
// stage of K. One warp a row.
__global__ void __launch_bounds__(256) rows_kernel(const float* head, int width, __half* head_hi, __half* head_lo, State s,
                                                   Upstream upstream, bool each, int rows,
                                                   const uint32_t* rows_largest, __half* rows_hi, __half* rows_lo,
                                                   int d) {
  depend();
  int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row < width) {
    const int64_t at = (int64_t)row * d;
    split_row(head + at, true, 0, d, power_of_two(scale_exponent(s.largest[1])), head_hi + at, head_lo + at);
    return;
  }
  row -= width;
  const int kept = *s.kept;
  if (row >= min(rows, (int)round_up(kept, kBlockK))) return;
  const float scale = power_of_two(scale_exponent(*rows_largest));
  const float c = row < kept && each ? upstream.of(s, row, kept) : 1.f;
  for (int i = 8 * (threadIdx.x & 31); i < d; i += 256) {
    float x[8] = {};
    if (row < kept) kept_values(s, row, i, d, c, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= scale;
    store_parts(x, rows_hi + (int64_t)row * d + i, rows_lo + (int64_t)row * d + i);
  }
}

// ---- products -----------------------------------------------------------------------------------------------------
// kStats: logits reduced to statistics. kGrad: logits turned into g. kGradients: dh and dw of one piece from g.
enum Epilogue { kStats = 0, kGrad = 1, kGradients = 2 };

// One product C[m, n] = sum_k A[m, k] B[n, k]; kept: which of the three extents counts kept rows and is read on the
// device. An operand is K-major (its rows hold consecutive k) or MN-major (its rows hold consecutive m or n): the logits'
// are both K-major, dh (job 0 of kGradients) has B MN-major (the head as it is), dw (job 1) both (g and the hidden
// states as they are).
struct Job {
  int m, n, k;
  int kept;                // 0: m, 2: k
  int splits;              // parts of K, each a result of its own
  int b_row;               // first row of B's tensor map that belongs to the product
};

struct Maps {
  CUtensorMap a[2][2], b[2][2];   // [job][part]
  CUtensorMap out[2];             // kGrad: g's parts; kGradients: dh's slots, dw
};

struct Args {
  State s;
  Job job[2];
  int jobs;
  int d, vocab;
  int v0, width;           // the piece of the vocabulary
  int64_t n_pad;
  float2* stats;           // kStats: [2 per column tile][n_pad] maximum and sum of exponentials, the target's left out
  float* picked;           // kStats: [n_pad] the target's logit
  Upstream upstream;
  int add;                 // kGradients: dh adds to its slots (a later piece)
  const uint32_t* dw_rows_largest;   // float32: of the rows dw sums (h, or c h)
  int dw_upstream;                   // dw's rows lack their c, which is the same for all
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// The address of the first SM's copy of a shared-memory location, for accesses from either SM of the pair.
__device__ __forceinline__ uint32_t at_leader(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A tile load into this SM's shared memory, counted on the leader's barrier.
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(leader_bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// Tells the leader that an accumulator has been read. What it orders are tensor-memory loads, which have been waited
// for; no release at cluster scope, which waited for the thread's earlier stores too (2300 cycles per accumulator).
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// Matrix descriptors over TMA's 128-byte swizzle. K-major: rows of 64 k (128 bytes), groups of 8 rows 1024 bytes apart.
// MN-major: blocks of 64 m (128 bytes) x 64 k, 8192 bytes apart; within a block groups of 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn) {
  const uint64_t leading = mn ? (8192 >> 4) : 1;
  return (uint64_t)((addr >> 4) & 0x3FFF) | (leading << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}

__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(add));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The extents of a launch's products, with the number of kept rows filled in.
struct Extent {
  int m_tiles, n_tiles, blocks, tiles;   // blocks of K
};

__device__ __forceinline__ Extent extent_of(const Job& j, int kept) {
  Extent x;
  x.m_tiles = ((j.kept == 0 ? kept : j.m) + kTile - 1) / kTile;
  x.n_tiles = (j.n + kTile - 1) / kTile;
  x.blocks = ((j.kept == 2 ? kept : j.k) + kBlockK - 1) / kBlockK;
  x.tiles = x.m_tiles * x.n_tiles * j.splits;
  return x;
}

struct Tile {
  int job, m, n, split, first, last;     // blocks [first, last) of K
};

// Logits: all row tiles of a group before the next column tile, so that a tile of the head is read from HBM once per
// group while the group's hidden states stay in L2. Gradients: the column tiles of a row tile together (they share A,
// the long operand).
template <int EPI>
__device__ __forceinline__ Tile tile_of(int index, const Extent (&x)[2], const Args& e) {
  Tile t;
  t.job = EPI == kGradients && index >= x[0].tiles ? 1 : 0;
  if (t.job) index -= x[0].tiles;
  const Extent& q = t.job ? x[1] : x[0];
  if constexpr (EPI == kGradients) {
    t.n = index % q.n_tiles;
    index /= q.n_tiles;
    t.m = index % q.m_tiles;
    t.split = index / q.m_tiles;
    const int splits = e.job[t.job].splits;
    t.first = (int)((int64_t)q.blocks * t.split / splits);
    t.last = (int)((int64_t)q.blocks * (t.split + 1) / splits);
  } else {
    const int group = index / (kGroupRows * q.n_tiles), rest = index - group * kGroupRows * q.n_tiles;
    const int rows = min(kGroupRows, q.m_tiles - group * kGroupRows);
    t.n = rest / rows;
    t.m = group * kGroupRows + rest % rows;
    t.split = 0;
    t.first = 0;
    t.last = q.blocks;
  }
  return t;
}

// A warp's 32 x 32 block of a result on its way to global memory: rows of 64 or 128 bytes in the swizzle TMA reads, so
// that a row's 16-byte pieces fall in different banks across rows, then one tile store. Stored by each thread for its
// own row instead, every 16 bytes of a warp's store touch another line: 32 passes through the L1 per instruction, which
// bounded g (d 1024, bfloat16: 906 us against 647 for the same logits without a store).
struct BlockOut {
  uint8_t* base;
  int lane;
  int half;              // place of the last block
  bool whole;            // the last block was of 4 KB

  // Room for a block of 4 KB, or of 2 KB while another one of 2 KB before it is still read out; its place.
  template <int BYTES>
  __device__ __forceinline__ int begin() {
    if (BYTES == kOutBytes || whole) {
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    } else {
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    }
    __syncwarp();
    whole = BYTES == kOutBytes;
    return half = whole ? 0 : half ^ (kOutBytes / 2);
  }
  template <int ROW_BYTES>
  __device__ __forceinline__ void put(int offset, int piece, uint4 v) const {
    const int at = ROW_BYTES == 64 ? piece ^ ((lane >> 1) & 3) : piece ^ (lane & 7);
    *reinterpret_cast<uint4*>(base + offset + lane * ROW_BYTES + at * 16) = v;
  }
  __device__ __forceinline__ void written() const {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
  }
  __device__ __forceinline__ void store(const CUtensorMap* map, int offset, int x, int y) const {
    if (lane == 0)
      asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                   "r"(smem_u32(base + offset)), "r"(x), "r"(y)
                   : "memory");
  }
  __device__ __forceinline__ void add(const CUtensorMap* map, int offset, int x, int y) const {
    if (lane == 0)
      asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                   "r"(smem_u32(base + offset)), "r"(x), "r"(y)
                   : "memory");
  }
  __device__ __forceinline__ void end() const {
    if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void finish() const {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
};

__device__ __forceinline__ uint4 pack_bf16(const float* x) {
  uint4 v;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
    w[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return v;
}

// The rows of a tile, one thread each: 32 columns at a time.
template <int PARTS, int EPI>
struct RowEpilogue {
  const Maps& maps;
  const Args& e;
  BlockOut& out;
  const Tile& t;
  int row, first_row;       // of the product: this thread's, the warp's first
  bool live;                // the row exists
  int target;
  float factor;             // of the accumulators
  float below;              // logits of float32: the part of it at most 1, applied before the columns' scales, so that
                            // ordinary logits of a tiny and a huge row do not overflow on the way
  float top, sum;           // kStats
  float4 inverse;           // logits of float32: the inverse scales of this lane's 4 of the warp's 128 columns
  float2 sums;              // kGrad
  float lse2, c;

  __device__ __forceinline__ RowEpilogue(const Maps& maps_, const Args& args, BlockOut& out_, const Tile& tile,
                                         int warp_row, int first_col, int kept)
      : maps(maps_), e(args), out(out_), t(tile) {
    first_row = t.m * kTile + warp_row;
    row = first_row + out.lane;
    factor = 1.f;
    if constexpr (EPI == kGradients) {
      if (t.job == 1) {
        if (PARTS == 2) factor = power_of_two(-14 - scale_exponent(*e.dw_rows_largest));
        if (e.dw_upstream && kept > 0) factor *= e.upstream.of(e.s, 0, kept);
      }
    } else {
      live = row < kept;
      target = live ? e.s.target[row] : -1;
      if (PARTS == 2) {
        const float inverse_row = live ? e.s.hidden_inverse[row] : 1.f;
        below = fminf(inverse_row, 1.f);
        factor = fmaxf(inverse_row, 1.f);
      }
      top = -INFINITY;
      sum = 0.f;
      if (PARTS == 2) {
        const int v = e.v0 + first_col + 4 * out.lane;       // the array is padded to a multiple of 64
        inverse = v < e.vocab ? __ldg(reinterpret_cast<const float4*>(e.s.inverse + v)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (EPI == kGrad) {
        sums = live ? e.s.sums[row] : make_float2(0.f, 1.f);
        lse2 = (sums.x + logf(sums.y)) * kLog2e;
        c = PARTS == 2 ? 16384.f : live && e.upstream.reduction == HFFN_REDUCE_NONE ? e.upstream.of(e.s, row, kept) : 1.f;
        sums.y = c / sums.y;
      }
    }
  }

  // The sums are complete. Logits of float32: their columns' scales, by way of shared memory where every lane reads them
  // (once the stores of the last tile have been read out of it).
  __device__ __forceinline__ void begin(float (&total)[128]) {
    if constexpr (PARTS == 2 && EPI != kGradients) {
      if (EPI == kGrad) out.template begin<kOutBytes>();
      __syncwarp();
      reinterpret_cast<float4*>(out.base)[out.lane] = inverse;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 128; j += 4) {
        const float4 x = *reinterpret_cast<const float4*>(out.base + 4 * j);
        total[j] = total[j] * below * x.x;
        total[j + 1] = total[j + 1] * below * x.y;
        total[j + 2] = total[j + 2] * below * x.z;
        total[j + 3] = total[j + 3] * below * x.w;
      }
      __syncwarp();
    }
  }

  __device__ __forceinline__ void columns(float (&v)[32], int col) {
    if constexpr (EPI == kGradients) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= factor;
    }
    if constexpr (EPI == kStats) {
      if (col + 32 > e.vocab) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col + j >= e.vocab) v[j] = -INFINITY;
      }
      const int at = target - col;
      if (__any_sync(0xffffffffu, at >= 0 && at < 32)) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (at == j) {
            e.picked[row] = v[j] * factor;
            v[j] = -INFINITY;              // the sums are those of the others
          }
      }
      // `factor` is a power of two, so it goes into the exponents' and the maximum's multiplications unrounded
      float most = v[0];
#pragma unroll
      for (int j = 1; j < 32; ++j) most = fmaxf(most, v[j]);
      most = fmaxf(top, most * factor);
      const float factor2 = factor * kLog2e;
      // a row of -inf so far has nothing to rescale; NaN logits reach the sum through their exponentials. The rounding
      // of `base` (1e-6 of a logit of 16) is the same in all 32 exponents: it is taken out of their sum.
      const bool none = most == -INFINITY;
      const float base = none ? 0.f : most * kLog2e;
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 32; ++j) part[j & 3] += exp2_fast(fmaf(v[j], factor2, -base));
      const float more = (part[0] + part[1]) + (part[2] + part[3]);
      sum = none ? sum + more
                 : fmaf(sum, exp2_fast((top - most) * kLog2e), more * exp2_fast(-fmaf(most, kLog2e, -base)));
      top = most;
    } else if constexpr (EPI == kGrad) {
      const int at = target - e.v0 - col;
      // float32: relative to the largest logit, whose difference is exact where p is large (an argument rounded at
      // the size of the logit puts 1e-6 on p, and p - 1 may be small); `factor` and c are powers of two
#pragma unroll
      for (int j = 0; j < 32; ++j)
        v[j] = PARTS == 2 ? exp2_fast(fmaf(v[j], factor, -sums.x) * kLog2e) * sums.y
                          : c * exp2_fast(fmaf(v[j], kLog2e, -lse2));
      if (__any_sync(0xffffffffu, at >= 0 && at < 32)) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (at == j) v[j] = c * e.s.own[row];
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = live ? v[j] : 0.f;
      const int at_block = out.template begin<PARTS * kOutBytes / 2>();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (PARTS == 2) {
          uint4 hi, lo;
          split8(v + 8 * q, hi, lo);
          out.template put<64>(0, q, hi);
          out.template put<64>(kOutBytes / 2, q, lo);
        } else {
          out.template put<64>(at_block, q, pack_bf16(v + 8 * q));
        }
      }
      out.written();
      out.store(&maps.out[0], at_block, col, first_row);
      if (PARTS == 2) out.store(&maps.out[1], kOutBytes / 2, col, first_row);
      out.end();
    } else {
      if (col >= e.d || (t.job == 1 && first_row >= e.width)) return;
      int at_block = 0;
      if (PARTS == 2 || t.job == 0) {
        out.template begin<kOutBytes>();
#pragma unroll
        for (int q = 0; q < 8; ++q)
          out.template put<128>(0, q, *reinterpret_cast<const uint4*>(v + 4 * q));
      } else {
        at_block = out.template begin<kOutBytes / 2>();
#pragma unroll
        for (int q = 0; q < 4; ++q) out.template put<64>(at_block, q, pack_bf16(v + 8 * q));
      }
      out.written();
      if (t.job == 1) out.store(&maps.out[1], at_block, col, e.v0 + first_row);
      else if (e.add) out.add(&maps.out[0], 0, col, t.split * (int)e.n_pad + first_row);
      else out.store(&maps.out[0], 0, col, t.split * (int)e.n_pad + first_row);
      out.end();
    }
  }

  __device__ __forceinline__ void finish(int column_part) {
    if constexpr (EPI == kStats)
      if (live) e.stats[column_part * e.n_pad + row] = make_float2(top, sum);
  }
};

template <int PARTS>
struct Stages {
  static constexpr int kCount = 6 / PARTS;
  static constexpr int kBytes = PARTS * 2 * kOperandBytes;   // of one SM
};

// A position in a ring of `count` slots whose barriers' phases alternate.
struct Ring {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int count) {
    if (++at == count) {
      at = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
  return elected != 0;
}

// What the thread of a warp whose wait ran out leaves: the device's error code, the call's mark, the other warps' sign.
__device__ __forceinline__ void give_up(const State& s, volatile int* abort_flag, int code) {
  atomicCAS(&g_error, 0, code);
  *reinterpret_cast<volatile int32_t*>(s.failed) = 1;
  *abort_flag = 1;
}

// A bounded wait of a whole warp: every lane gets the same answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, kWaitNs));
}

template <int EPI, int JOB>
struct Major {
  static constexpr bool kA = EPI == kGradients && JOB == 1, kB = EPI == kGradients;   // MN-major
};

// The loads of one tile's K. The whole warp runs the loop and one lane issues, with the tensor maps at addresses known
// when compiled: from one lane alone, or with a map picked at run time, a stage's three or four loads took 550 cycles to
// issue, longer than its products (dh 8192 x 2048 x 12800: 801 cycles a stage, 586 for the logits).
template <int PARTS, int EPI, int JOB>
__device__ __forceinline__ bool load_stages(const Maps& maps, const Args& e, const Tile& t, uint32_t rank, uint8_t* smem,
                                            uint64_t* full, uint64_t* empty, Ring& ring, volatile int* abort_flag) {
  using M = Major<EPI, JOB>;
  const int m = t.m * kTile + (int)rank * 128, n = t.n * kTile + (int)rank * 128, b_row = e.job[JOB].b_row;
  for (int kb = t.first; kb < t.last; ++kb) {
    if (!warp_wait(&empty[ring.at], ring.phase ^ 1, abort_flag)) return false;
    if (elect_one()) {
      if (rank == 0) mbar_expect_tx(&full[ring.at], 2 * Stages<PARTS>::kBytes);
      const uint32_t bar = at_leader(&full[ring.at]);
      uint8_t* dst = smem + ring.at * Stages<PARTS>::kBytes;
      const int k = kb * kBlockK;
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        if constexpr (M::kA) {
          load_tile(dst, &maps.a[JOB][part], bar, m, k);
          load_tile(dst + 8192, &maps.a[JOB][part], bar, m + 64, k);
        } else {
          load_tile(dst, &maps.a[JOB][part], bar, k, m);
        }
        dst += kOperandBytes;
        if constexpr (M::kB) {
          load_tile(dst, &maps.b[JOB][part], bar, n, b_row + k);
          load_tile(dst + 8192, &maps.b[JOB][part], bar, n + 64, b_row + k);
        } else {
          load_tile(dst, &maps.b[JOB][part], bar, k, b_row + n);
        }
        dst += kOperandBytes;
      }
    }
    __syncwarp();
    ring.next(Stages<PARTS>::kCount);
  }
  return true;
}

// Stages of K per accumulator, 0: all. A step of 16 values truncates by half a unit of the sum so far on average.
// float32: 2 stages, 24 steps, of which each stage's 8 with the low parts come first, so that it is the 4 of hi hi per
// stage that cost (4 stages with the parts interleaved: dh of 46 tokens 1.2e-6 off, plain float32 sums 0.4e-6). Losses of
// bfloat16 logits: 8 stages, 32 steps (8 x 511 tokens of 1024: 2.5e-7 off, plain sums 2.3e-7; 16 stages 5.2e-7 and no
// faster; 4 stages 1.2e-7 but 8 to 15 % slower), and 4 where one row tile leaves the time to reading the head (few
// losses average less, and that of a well predicted token is a small difference of logits). bfloat16 gradients need none: an
// error of a recomputed logit is one of p relative to itself, where g is rounded to 2^-8 of itself (p - 1 of the target,
// where it would be more, is the forward's), and dh and dw are rounded to 2^-8 afterwards.
template <int PARTS, int EPI>
__device__ __forceinline__ int chunk_of(int kept) {
  return PARTS == 2 ? 2 : EPI == kStats ? (kept <= kTile ? 4 : 8) : 0;
}

// The products of one tile.
template <int PARTS, int EPI, int JOB>
__device__ __forceinline__ bool multiply_stages(const Tile& t, int kept, uint32_t tmem_base, uint8_t* smem,
                                                uint64_t* full, uint64_t* empty, uint64_t* tfull, uint64_t* tempty,
                                                Ring& ring, Ring& acc, volatile int* abort_flag) {
  using M = Major<EPI, JOB>;
  constexpr uint32_t format = PARTS == 2 ? 0 : 1;   // fp16, bfloat16
  constexpr uint32_t idesc = (1u << 4) | (format << 7) | (format << 10) | ((uint32_t)M::kA << 15) |
                             ((uint32_t)M::kB << 16) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
  constexpr uint32_t a_step = M::kA ? 2048 : 32, b_step = M::kB ? 2048 : 32;   // bytes of 16 k
  int chunk = chunk_of<PARTS, EPI>(kept);
  if (chunk == 0) chunk = t.last - t.first;
  for (int first = t.first; first < t.last; first += chunk) {
    if (!warp_wait(&tempty[acc.at], acc.phase ^ 1, abort_flag)) return false;
    fence_after();
    const uint32_t d_tmem = tmem_base + acc.at * kTile;
    const int last = min(first + chunk, t.last);
    for (int kb = first; kb < last; ++kb) {
      if (!warp_wait(&full[ring.at], ring.phase, abort_flag)) return false;
      fence_after();
      if (elect_one()) {
        const uint32_t base = smem_u32(smem + ring.at * Stages<PARTS>::kBytes);
        auto multiply = [&](uint32_t a, uint32_t b, bool fresh) {
#pragma unroll
          for (int k = 0; k < kBlockK / 16; ++k)
            mma_pair(d_tmem, operand_desc(base + a * kOperandBytes + a_step * k, M::kA),
                     operand_desc(base + b * kOperandBytes + b_step * k, M::kB), idesc, !fresh || kb != first || k != 0);
        };
        if constexpr (PARTS == 2) {
          multiply(0, 3, true);      // hi lo
          multiply(2, 1, false);     // lo hi
          multiply(0, 1, false);
        } else {
          multiply(0, 1, true);
        }
        commit_pair(&empty[ring.at]);
        if (kb == last - 1) commit_pair(&tfull[acc.at]);
      }
      __syncwarp();
      ring.next(Stages<PARTS>::kCount);
    }
    acc.next(2);
  }
  return true;
}

template <int PARTS, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args e) {
  constexpr int STAGES = Stages<PARTS>::kCount;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStageBytes + kEpilogueWarps * kOutBytes);   // used in the leader
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;                                                                    // used in the leader
  uint64_t* done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * kEpilogueWarps);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tmem_base = *tmem_slot;
  depend();

  const int kept = *e.s.kept;
  const Extent extent[2] = {extent_of(e.job[0], kept), extent_of(e.job[1], kept)};
  const int tiles = extent[0].tiles + (EPI == kGradients && e.jobs > 1 ? extent[1].tiles : 0);
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 0) {
    // ---------------- loads ----------------
    Ring ring;
    bool ok = true;
    for (int index = pair; index < tiles && ok; index += pairs) {
      const Tile t = tile_of<EPI>(index, extent, e);
      if (EPI == kGradients && t.job == 1)
        ok = load_stages<PARTS, EPI, 1>(maps, e, t, rank, smem, full, empty, ring, abort_flag);
      else
        ok = load_stages<PARTS, EPI, 0>(maps, e, t, rank, smem, full, empty, ring, abort_flag);
    }
    if (!ok && lane == 0) {
      give_up(e.s, abort_flag, kErrLoad);
      // the loads in flight land within microseconds; nothing waits on them any more, so this SM gives them time
      const uint64_t start = global_ns();
      while (global_ns() - start < 10000000ull) {
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------- products ----------------
      Ring ring, acc;
      bool ok = true;
      for (int index = pair; index < tiles && ok; index += pairs) {
        const Tile t = tile_of<EPI>(index, extent, e);
        if (EPI == kGradients && t.job == 1)
          ok = multiply_stages<PARTS, EPI, 1>(t, kept, tmem_base, smem, full, empty, tfull, tempty, ring, acc,
                                              abort_flag);
        else
          ok = multiply_stages<PARTS, EPI, 0>(t, kept, tmem_base, smem, full, empty, tfull, tempty, ring, acc,
                                              abort_flag);
      }
      if (lane == 0) {
        if (!ok) {
          give_up(e.s, abort_flag, kErrProduct);
        }
      }
      __syncwarp();
      // every product has been computed before the TMEM is freed (tcgen05.commit tracks the elected lane's products)
      if (elect_one()) {
        commit_pair(done);
        const uint64_t start = global_ns();
        while (!mbar_try_wait(done, 0) && global_ns() - start < kWaitNs) {
        }
      }
    }
  } else {
    // ---------------- epilogue: a TMEM lane (row) per thread, two warps per lane quarter sharing the columns ----------
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * 128;
    const int warp_row = (int)rank * 128 + quarter * 32;
    BlockOut block{smem + kStageBytes + (warp - 2) * kOutBytes, lane, 0, false};
    const uint32_t release[2] = {at_leader(&tempty[0]), at_leader(&tempty[1])};
    constexpr bool kChunks = PARTS == 2 || EPI == kStats;
    const int chunk = chunk_of<PARTS, EPI>(kept);
    Ring acc;
    bool ok = true;
    for (int index = pair; index < tiles && ok; index += pairs) {
      const Tile t = tile_of<EPI>(index, extent, e);
      const int col = t.n * kTile + half * 128;
      RowEpilogue<PARTS, EPI> out(maps, e, block, t, warp_row, col, kept);
      auto release_buffer = [&] {
        fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(release[acc.at]);
        acc.next(2);
      };
      if constexpr (kChunks) {
        float total[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) total[j] = 0.f;
        for (int first = t.first; first < t.last; first += chunk) {
          if (!(ok = warp_wait(&tfull[acc.at], acc.phase, abort_flag))) break;
          fence_after();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v[32];
            tmem_ld32(lane_base + acc.at * kTile + 32 * c, v);
#pragma unroll
            for (int j = 0; j < 32; ++j) total[32 * c + j] += v[j];
          }
          release_buffer();
        }
        if (!ok) break;
        out.begin(total);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = total[32 * c + j];
          out.columns(v, col + 32 * c);
        }
      } else {
        const bool any = t.first < t.last;
        if (any && !(ok = warp_wait(&tfull[acc.at], acc.phase, abort_flag))) break;
        fence_after();
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float v[32];
          if (any) {
            tmem_ld32(lane_base + acc.at * kTile + 32 * c, v);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
          out.columns(v, col + 32 * c);
        }
        if (any) release_buffer();
      }
      out.finish(2 * t.n + half);
    }
    block.finish();
    if (!ok && lane == 0) {
      give_up(e.s, abort_flag, kErrEpilogue);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  cluster_sync();      // neither SM leaves while the other may still reach its memory or its barriers
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base));
  }
}

// ---- per-row kernels ----------------------------------------------------------------------------------------------
__device__ __forceinline__ void merge(float& top, float& sum, float top2, float sum2) {
  const float most = fmaxf(top, top2);
  if (most > -INFINITY) sum = sum * exp2f((top - most) * kLog2e) + sum2 * exp2f((top2 - most) * kLog2e);
  else sum += sum2;
  top = most;
}

// ---- few rows -----------------------------------------------------------------------------------------------------
// The logits of up to ROWS kept rows (the groups of blockIdx.y) reduced to statistics: bound by reading the head once. A
// warp takes BATCH rows of the head at a time, 16 bytes a lane and row, against the hidden rows in shared memory
// (float32, in planes of 16-byte pieces, so that neighbouring lanes read neighbouring pieces), then adds its BATCH x ROWS
// sums across its lanes by halving: lane l ends with the sum of index l / (32 / (BATCH x ROWS)).
template <typename T>
__device__ __forceinline__ void widen(uint4 bits, float (&x)[16 / sizeof(T)]) {
  const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      x[j] = __uint_as_float(w[j]);
    } else {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
}

template <typename T, int ROWS, int BATCH>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const T* hidden, int64_t stride, const T* head,
                                                          const int64_t* targets, int64_t ignore, int n, int d, int vocab,
                                                          float2* stats, int64_t n_pad, float* picked, float* losses,
                                                          State s) {
  constexpr int kVector = 16 / sizeof(T), kPlanes = kVector / 4, kSums = ROWS * BATCH;
  static_assert(kSums <= 32 && (kSums & (kSums - 1)) == 0, "one sum a lane at most");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  float* rows = reinterpret_cast<float*>(smem_raw);                       // [ROWS][kPlanes][d / kPlanes]
  __shared__ int row_of[32], target_of[32], kept_rows;
  __shared__ float2 shared[kFewWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = blockIdx.y * ROWS;
  depend();
  if (warp == 0) {
    const int64_t target = lane < n ? targets[lane] : ignore;
    const bool keep = lane < n && is_kept(target, ignore, vocab);
    const unsigned mask = __ballot_sync(0xffffffffu, keep);
    const int at = __popc(mask & ((1u << lane) - 1u));
    const bool writes = blockIdx.x == 0 && blockIdx.y == 0;
    if (keep) {
      row_of[at] = lane;
      target_of[at] = (int)target;
      if (writes) {
        s.row_of[at] = lane;
        s.target[at] = (int)target;
      }
    }
    if (writes && lane < n) {
      s.place_of[lane] = keep ? at : -1;
      if (!keep) losses[lane] = target == ignore ? 0.f : NAN;
    }
    if (lane == 0) {
      kept_rows = __popc(mask);
      if (writes) {
        *s.kept = kept_rows;
        *s.arrived = 0;
        *s.failed = 0;
      }
    }
  }
  __syncthreads();
  const int kept = kept_rows;
  if (first >= kept) return;
  for (int i = threadIdx.x; i < ROWS * d; i += kFewThreads) {
    const int r = i / d, c = i % d;
    const T v = first + r < kept ? hidden[row_of[first + r] * stride + c] : from_f<T>(0.f);
    rows[(r * kPlanes + c / 4 % kPlanes) * (d / kPlanes) + c / kVector * 4 + c % 4] = to_f<T>(v);
    if (blockIdx.x == 0 && first + r < kept) {
      if constexpr (sizeof(T) == 4) s.raw[(int64_t)first * d + i] = v;
      else static_cast<T*>(s.hidden[0])[(int64_t)first * d + i] = v;
    }
  }
  __syncthreads();

  constexpr int kCopies = 32 / kSums;                    // lanes that end with the same sum
  const int index = lane / kCopies, row = index % ROWS, batch_row = index / ROWS;
  const int target = first + row < kept ? target_of[first + row] : -1;
  float top = -INFINITY, sum = 0.f;
  const int step = gridDim.x * kFewWarps * BATCH;
  for (int v0 = (blockIdx.x * kFewWarps + warp) * BATCH; v0 < vocab; v0 += step) {
    float acc[kSums] = {};
#pragma unroll 2
    for (int c = lane * kVector; c < d; c += 32 * kVector) {
      uint4 bits[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b)
        bits[b] = __ldcs(reinterpret_cast<const uint4*>(head + (int64_t)min(v0 + b, vocab - 1) * d + c));
      float w[BATCH][kVector];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) widen<T>(bits[b], w[b]);
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int p = 0; p < kPlanes; ++p) {
          const float4 h = *reinterpret_cast<const float4*>(rows + (r * kPlanes + p) * (d / kPlanes) + c / kPlanes);
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            float& a = acc[b * ROWS + r];
            a = fmaf(h.x, w[b][4 * p], a);
            a = fmaf(h.y, w[b][4 * p + 1], a);
            a = fmaf(h.z, w[b][4 * p + 2], a);
            a = fmaf(h.w, w[b][4 * p + 3], a);
          }
        }
    }
#pragma unroll
    for (int o = 16, count = kSums; o > 0; o >>= 1) {
      if (count > 1) {
        count /= 2;
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < kSums / 2; ++i)
          if (i < count) {
            const float own = upper ? acc[i + count] : acc[i], sent = upper ? acc[i] : acc[i + count];
            acc[i] = own + __shfl_xor_sync(0xffffffffu, sent, o);
          }
      } else {
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
      }
    }
    const int v = v0 + batch_row;
    if (v < vocab) {
      const float z = acc[0];
      if (v == target) picked[first + row] = z;
      else merge(top, sum, z, z == z ? 1.f : z);      // no maximum keeps a NaN: it stays in the sum
    }
  }
  shared[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x < ROWS && first + threadIdx.x < kept) {
    top = -INFINITY;
    sum = 0.f;
    for (int w = 0; w < kFewWarps; ++w)
      for (int b = 0; b < BATCH; ++b) {
        const float2 part = shared[w][(b * ROWS + threadIdx.x) * kCopies];
        merge(top, sum, part.x, part.y);
      }
    stats[blockIdx.x * n_pad + first + threadIdx.x] = make_float2(top, sum);
  }
}

// ---- losses -------------------------------------------------------------------------------------------------------
// lse, loss and the target's p - 1 of the kept rows from their targets' logits and the parts' maxima and sums of the other
// logits: 32 rows a block, its 32 warps sharing the parts.
// The block that finishes last also adds up the losses where their sum or mean is asked for (float64, the same order
// whichever block that is). The blocks after the `row_blocks` (bfloat16) zero the kept rows up to a whole stage of K of
// the dw product.
__global__ void __launch_bounds__(1024) losses_kernel(State s, const float2* stats, int64_t n_pad, int parts,
                                                      const float* picked, float* losses, int n, int reduction,
                                                      float* loss, int row_blocks, int row_bytes) {
  __shared__ float2 shared[32][33];
  depend();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * 32 + lane, kept = *s.kept;
  if (blockIdx.x >= row_blocks) {
    const int64_t step = (int64_t)(gridDim.x - row_blocks) * 1024, end = round_up(kept, kBlockK) * row_bytes / 16;
    for (int64_t i = (int64_t)kept * row_bytes / 16 + (blockIdx.x - row_blocks) * 1024 + threadIdx.x; i < end; i += step)
      static_cast<uint4*>(s.hidden[0])[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  if (blockIdx.x * 32 < kept) {
    float top = -INFINITY, sum = 0.f;
    if (row < kept) {
      for (int i = warp; i < parts; i += 256) {
        float2 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = i + 32 * j < parts ? stats[(i + 32 * j) * n_pad + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) merge(top, sum, v[j].x, v[j].y);
      }
    }
    shared[warp][lane] = make_float2(top, sum);
    __syncthreads();
    float2 v = shared[lane][warp];           // row `warp` of the block, one part a lane
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float top2 = __shfl_xor_sync(0xffffffffu, v.x, o), sum2 = __shfl_xor_sync(0xffffffffu, v.y, o);
      merge(v.x, v.y, top2, sum2);
    }
    const int mine = blockIdx.x * 32 + warp;
    if (lane == 0 && mine < kept) {
      const float z = picked[mine];
      float of_row;
      if (z >= v.x) {
        const float odds = v.y * expf(v.x - z);
        of_row = log1pf(odds) + (z - z);              // an infinite logit of the target: NaN
        s.sums[mine] = make_float2(z, 1.f + odds);
        s.own[mine] = -odds / (1.f + odds);
      } else {
        const float total = v.y + expf(z - v.x);
        of_row = (v.x - z) + logf(total);
        s.sums[mine] = make_float2(v.x, total);
        s.own[mine] = -v.y / total;
      }
      if (*s.failed) {
        of_row = s.own[mine] = NAN;
        s.sums[mine] = make_float2(0.f, NAN);
      }
      losses[s.row_of[mine]] = of_row;
    }
  }
  if (reduction == HFFN_REDUCE_NONE) return;
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(s.arrived, 1u) == (unsigned)row_blocks - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double* sums = reinterpret_cast<double*>(shared);
  double sum = 0;
  for (int t = threadIdx.x; t < n; t += 1024) sum += (double)__ldcg(losses + t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < 32; ++w) sum += sums[w];
    *loss = (float)(reduction == HFFN_REDUCE_MEAN ? sum / max(1, kept) : sum);
  }
}

// dh of each input row: the sum of its kept row's slots (in order), or zeros. One warp a row. After a wait that ran out:
// NaN for the kept rows, and for all of dw (`weight_count` entries, none where it is not wanted).
template <typename T>
__global__ void __launch_bounds__(256) scatter_kernel(State s, const float* slots, int splits, int64_t n_pad,
                                                      Upstream upstream, T* grad_hidden, T* grad_weight,
                                                      int64_t weight_count, int n, int d) {
  depend();
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const bool failed = *s.failed != 0;
  if (failed)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < weight_count; i += (int64_t)gridDim.x * 256)
      grad_weight[i] = from_f<T>(NAN);
  if (t >= n || grad_hidden == nullptr) return;
  const int at = s.place_of[t];
  float factor = 1.f;      // what g lacks
  if (at >= 0 && (sizeof(T) == 4 || upstream.reduction != HFFN_REDUCE_NONE)) factor = upstream.of(s, at, *s.kept);
  if (sizeof(T) == 4) factor *= power_of_two(-14 - scale_exponent(s.largest[1]));
  if (failed && at >= 0) factor = NAN;
  for (int i = 4 * lane; i < d; i += 128) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at >= 0)
      for (int k = 0; k < splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(slots + (k * n_pad + at) * d + i);
        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
      }
    __align__(16) T out[4] = {from_f<T>(sum.x * factor), from_f<T>(sum.y * factor), from_f<T>(sum.z * factor),
                              from_f<T>(sum.w * factor)};
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(grad_hidden + (int64_t)t * d + i) = *reinterpret_cast<const float4*>(out);
    else
      *reinterpret_cast<uint2*>(grad_hidden + (int64_t)t * d + i) = *reinterpret_cast<const uint2*>(out);
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
static int parts_of(int dtype) { return dtype == HFFN_F32 ? 2 : 1; }

// Columns of g held at a time: the vocabulary in equal pieces of whole tiles, each at most kPieceBytes but at least
// kPieceMin columns (a shorter K would spend dh's time on adding its results to the last piece's).
static int piece_width(int dtype, int64_t n, int vocab) {
  const int64_t row = 2 * parts_of(dtype) * round_up(n, kTile);
  const int64_t width = std::max<int64_t>(kPieceMin, kPieceBytes / row);
  const int64_t pieces = ceil_div(vocab, width);
  return (int)round_up(ceil_div(vocab, pieces), kTile);
}

static int sm_pairs() {
  static int pairs[kMaxDevices] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) return 74;
  if (pairs[device] == 0) {
    int sms = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    pairs[device] = std::max(1, sms / 2);
  }
  return pairs[device];
}

// Parts of K of the dh product: as many as it takes to give every pair of SMs a tile, each part 1024 values at least.
// From n alone, so that the result does not depend on the device.
static int hidden_splits(int dtype, int64_t n, int d, int vocab) {
  const int64_t tiles = ceil_div(n, kTile) * ceil_div(d, kTile);
  const int64_t most = std::max<int64_t>(1, piece_width(dtype, n, vocab) / 1024);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, 74 / tiles));
}

// A row-major matrix in boxes of box_columns x box_rows; the swizzle is that of a box row's bytes (64 or 128).
static int make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t rows, int64_t columns,
                    int64_t ld, int box_columns, int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) {
    set_error("cuTensorMapEncodeTiled unavailable");
    return HFFN_ERR_CUDA;
  }
  const int element = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * element)};
  const cuuint32_t box[2] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows};
  const cuuint32_t step[2] = {1, 1};
  const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box_columns * element == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for a [%lld, %lld] operand", (int)r, (long long)rows,
              (long long)columns);
    return HFFN_ERR_CUDA;
  }
  return HFFN_OK;
}

static CUtensorMapDataType part_type(int dtype) {
  return dtype == HFFN_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// An operand part (fp16 or bfloat16) in boxes of 64 columns (K-major: k, 128 rows; MN-major: m or n, 64 rows of k).
static int operand_map(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t columns, int64_t ld,
                       int box_rows) {
  return make_map(map, part_type(dtype), base, rows, columns, ld, kBlockK, box_rows);
}

// Raises a kernel's limit of dynamic shared memory, once per device.
template <auto kernel>
static int allow_shared_memory(int bytes) {
  static bool done[kMaxDevices] = {};
  int device = -1;
  cudaGetDevice(&device);
  const bool known = device >= 0 && device < kMaxDevices;
  if (known && done[device]) return HFFN_OK;
  const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (r != cudaSuccess) {
    set_error("linear_ce: %s", cudaGetErrorString(r));
    return HFFN_ERR_CUDA;
  }
  if (known) done[device] = true;
  return HFFN_OK;
}

// Launches a kernel that may start while the kernel before it in the stream, one of the same call, still runs.
template <auto kernel, typename... A>
static void launch_next(unsigned grid, unsigned threads, size_t shared, cudaStream_t st, A... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = st;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, kernel, args...);     // its error is the next launch_status'
}

// next: the kernel before it in the stream is one of the same call.
template <int PARTS, int EPI>
static int launch_products(const Maps& maps, const Args& e, int64_t most_tiles, bool next, cudaStream_t st) {
  HFFN_TRY((allow_shared_memory<product_kernel<PARTS, EPI>>(kSmem)));
  const int pairs = (int)std::min<int64_t>(sm_pairs(), most_tiles);
  if (next) launch_next<product_kernel<PARTS, EPI>>(2 * pairs, kThreads, kSmem, st, maps, e);
  else product_kernel<PARTS, EPI><<<2 * pairs, kThreads, kSmem, st>>>(maps, e);
  return launch_status("linear_ce product");
}

// The logits' operands: rows of the kept hidden states and of the head, both K-major.
static int logits_job(Maps& maps, Args& e, int dtype, const void* weight, int64_t n, int d, int vocab) {
  const void* head[2] = {dtype == HFFN_F32 ? e.s.head[0] : weight, e.s.head[1]};
  for (int part = 0; part < parts_of(dtype); ++part) {
    HFFN_TRY(operand_map(&maps.a[0][part], dtype, e.s.hidden[part], e.n_pad, d, d, 128));
    HFFN_TRY(operand_map(&maps.b[0][part], dtype, head[part], vocab, d, d, 128));
  }
  e.job[0] = {(int)n, e.width, d, 0, 1, e.v0};
  e.job[1] = {};
  e.jobs = 1;
  return HFFN_OK;
}

constexpr int kFewBlocks = 148 * 3;    // of the few-row kernel: 24 warps an SM (8 float32 rows: 16, its registers allow two)

template <typename T, int ROWS, int BATCH>
static int launch_few(const T* hidden, int64_t stride, const T* head, const int64_t* targets, int64_t ignore, int n,
                      int d, int vocab, float2* stats, int64_t n_pad, float* picked, float* losses, const State& s,
                      int blocks, cudaStream_t st) {
  HFFN_TRY((allow_shared_memory<few_kernel<T, ROWS, BATCH>>((int)kFewBytes)));
  few_kernel<T, ROWS, BATCH><<<dim3(blocks, (unsigned)ceil_div(n, ROWS)), kFewThreads, ROWS * d * 4, st>>>(
      hidden, stride, head, targets, ignore, n, d, vocab, stats, n_pad, picked, losses, s);
  return launch_status("linear_ce few rows");
}

struct ForwardWork {
  float2* stats;
  float *picked, *losses;
  int64_t bytes;
};

static ForwardWork forward_work(void* base, int dtype, int64_t n, int d, int vocab) {
  Carve c{static_cast<uint8_t*>(base)};
  const int64_t n_pad = round_up(n, kTile);
  ForwardWork w;
  w.stats = c.take<float2>((is_few(dtype, n, d) ? kFewBlocks : 2 * ceil_div(vocab, kTile)) * n_pad);
  w.picked = c.take<float>(n_pad);
  w.losses = c.take<float>(n_pad);
  w.bytes = c.at;
  return w;
}

struct BackwardWork {
  void* g[2];
  float* slots;
  uint32_t* largest;      // float32, a gradient for each token: of c h
  void* rows[2];          // float32, [n_pad, d]: the fp16 parts of the rows dw sums
  void* head[2];          // float32, [piece_width, d]: those of the rows dh sums
  void* logits_head[2];   // float32, few rows: the state's `head` and `inverse`
  float* logits_inverse;
  int64_t bytes;
};

static BackwardWork backward_work(void* base, int dtype, int64_t n, int d, int vocab) {
  Carve c{static_cast<uint8_t*>(base)};
  const int64_t n_pad = round_up(n, kTile);
  BackwardWork w = {};
  for (int part = 0; part < parts_of(dtype); ++part) w.g[part] = c.take<uint16_t>(n_pad * piece_width(dtype, n, vocab));
  w.slots = c.take<float>(hidden_splits(dtype, n, d, vocab) * n_pad * d);
  if (dtype == HFFN_F32) {
    w.largest = c.take<uint32_t>(1);
    for (int part = 0; part < 2; ++part) w.rows[part] = c.take<uint16_t>(n_pad * d);
    for (int part = 0; part < 2; ++part) w.head[part] = c.take<uint16_t>((int64_t)piece_width(dtype, n, vocab) * d);
    if (is_few(dtype, n, d)) take_head(c, w.logits_head, w.logits_inverse, d, vocab);
  }
  w.bytes = c.at;
  return w;
}

static int check(int dtype, int64_t n, int32_t d, int32_t vocab) {
  HFFN_REQUIRE(dtype == HFFN_F32 || dtype == HFFN_BF16, "unknown dtype %d", dtype);
  HFFN_REQUIRE(n >= 1 && n <= (int64_t(1) << 24), "token count %lld out of range [1, 2^24]", (long long)n);
  HFFN_REQUIRE(d >= 8 && d % 8 == 0 && d <= 32768, "hidden size %d: a multiple of 8 up to 32768", d);
  HFFN_REQUIRE(vocab >= 1 && vocab <= (1 << 24), "vocabulary %d out of range [1, 2^24]", vocab);
  HFFN_REQUIRE(ceil_div(n, kTile) * ceil_div(vocab, kTile) < (int64_t(1) << 30), "too many tokens times rows");
  return HFFN_OK;
}

template <typename T>
static int forward(const void* hidden, int64_t stride, const void* weight, const int64_t* targets, int64_t ignore,
                   int reduction, bool for_backward, float* loss, void* state, void* work, int n, int d, int vocab,
                   cudaStream_t st) {
  constexpr int PARTS = sizeof(T) / 2;
  constexpr int dtype = PARTS == 2 ? HFFN_F32 : HFFN_BF16;
  const ForwardWork w = forward_work(work, dtype, n, d, vocab);
  Args e = {};
  e.s = state_at(state, dtype, n, d, vocab);
  e.d = d;
  e.vocab = e.width = vocab;
  e.n_pad = round_up(n, kTile);
  e.stats = w.stats;
  e.picked = w.picked;
  float* losses = reduction == HFFN_REDUCE_NONE ? loss : w.losses;
  const T *rows = static_cast<const T*>(hidden), *head = static_cast<const T*>(weight);
  int parts = 0;
  if (is_few(dtype, n, d)) {
    parts = (int)std::min<int64_t>(kFewBlocks, ceil_div(vocab, kFewWarps * 4));
    auto few = launch_few<T, PARTS == 1 ? 1 : kFewRows, PARTS == 1 ? 8 : 4>;
    if constexpr (PARTS == 2)
      if (few_rows(dtype, n) < kFewRows) few = launch_few<T, kFewRows / 2, 4>;
    HFFN_TRY(few(rows, stride, head, targets, ignore, n, d, vocab, w.stats, e.n_pad, w.picked, losses, e.s, parts, st));
  } else {
    const int span = (int)std::max<int64_t>(16, ceil_div(n, 512)), gather = (int)ceil_div(n, span);
    const bool aligned = (reinterpret_cast<uintptr_t>(hidden) & 15) == 0 && stride * (int64_t)sizeof(T) % 16 == 0;
    if (PARTS == 2 && cudaMemsetAsync(e.s.largest, 0, 8, st) != cudaSuccess) return launch_status("linear_ce");
    gather_kernel<T><<<gather, kGatherThreads, 0, st>>>(rows, stride, targets, ignore, n, d, vocab, span, aligned, losses,
                                                        e.s);
    if constexpr (PARTS == 2)
      launch_next<split_kernel>((unsigned)ceil_div((int64_t)vocab + n, 8), 256, 0, st, rows, stride, aligned, head, d,
                                vocab, for_backward, e.s);
    Maps maps;
    HFFN_TRY(logits_job(maps, e, dtype, weight, n, d, vocab));
    HFFN_TRY((launch_products<PARTS, kStats>(maps, e, ceil_div(n, kTile) * ceil_div(vocab, kTile), true, st)));
    parts = 2 * (int)ceil_div(vocab, kTile);
  }
  const int row_blocks = (int)ceil_div(n, 32);
  launch_next<losses_kernel>(row_blocks + (PARTS == 1 ? 4 : 0), 1024, 0, st, e.s, w.stats, e.n_pad, parts, w.picked,
                             losses, n, reduction, loss, row_blocks, 2 * d);
  return launch_status("linear_ce_forward");
}

template <typename T>
static int backward(const void* weight, int reduction, const float* grad_loss, void* grad_hidden, void* grad_weight,
                    void* state, void* work, int n, int d, int vocab, cudaStream_t st) {
  constexpr int PARTS = sizeof(T) / 2;
  constexpr int dtype = PARTS == 2 ? HFFN_F32 : HFFN_BF16;
  if (grad_hidden == nullptr && grad_weight == nullptr) return HFFN_OK;
  const BackwardWork w = backward_work(work, dtype, n, d, vocab);
  const int width = piece_width(dtype, n, vocab), splits = hidden_splits(dtype, n, d, vocab);
  Args e = {};
  e.s = state_at(state, dtype, n, d, vocab);
  e.d = d;
  e.vocab = vocab;
  e.n_pad = round_up(n, kTile);
  e.upstream = {grad_loss, reduction};
  bool prepared = false;             // a kernel of this call precedes the products
  if constexpr (PARTS == 2) {
    if (is_few(dtype, n, d)) {       // the forward has made no parts
      e.s.head[0] = w.logits_head[0];
      e.s.head[1] = w.logits_head[1];
      e.s.inverse = w.logits_inverse;
      if (cudaMemsetAsync(e.s.largest, 0, 8, st) != cudaSuccess) return launch_status("linear_ce");
      split_kernel<<<(unsigned)ceil_div((int64_t)vocab + n, 8), 256, 0, st>>>(
          nullptr, 0, true, static_cast<const float*>(weight), d, vocab, true, e.s);
      prepared = true;
    }
  }
  const void* rows[2] = {e.s.hidden[0], e.s.hidden[1]};    // what dw sums
  e.dw_upstream = reduction != HFFN_REDUCE_NONE;
  const bool each = reduction == HFFN_REDUCE_NONE;
  if (PARTS == 2 && grad_weight != nullptr) {
    rows[0] = w.rows[0];
    rows[1] = w.rows[1];
    e.dw_rows_largest = each ? w.largest : e.s.largest;
    if (each) {
      if (cudaMemsetAsync(w.largest, 0, 4, st) != cudaSuccess) return launch_status("linear_ce");
      scaled_largest_kernel<<<(unsigned)ceil_div(n, 8), 256, 0, st>>>(e.s, e.upstream, w.largest, d);
      prepared = true;
    }
  }
  const void* head[2] = {PARTS == 2 ? w.head[0] : weight, w.head[1]};     // what dh sums
  const int64_t row_tiles = ceil_div(n, kTile), wide = ceil_div(d, kTile);
  for (int v0 = 0; v0 < vocab; v0 += width) {
    e.v0 = v0;
    e.width = std::min(width, vocab - v0);
    e.add = v0 > 0;
    const int64_t columns = ceil_div(e.width, kTile);
    if constexpr (PARTS == 2) {
      const float* from = static_cast<const float*>(weight) + (int64_t)v0 * d;
      const int wide_rows = grad_hidden != nullptr ? e.width : 0;
      const int kept_rows = grad_weight != nullptr && v0 == 0 ? (int)e.n_pad : 0;
      const int64_t all = (int64_t)wide_rows + kept_rows;
      __half *head_hi = static_cast<__half*>(w.head[0]), *head_lo = static_cast<__half*>(w.head[1]);
      __half *rows_hi = static_cast<__half*>(w.rows[0]), *rows_lo = static_cast<__half*>(w.rows[1]);
      const unsigned blocks = (unsigned)ceil_div(all, 8);
      if (all > 0 && prepared)
        launch_next<rows_kernel>(blocks, 256, 0, st, from, wide_rows, head_hi, head_lo, e.s, e.upstream, each,
                                 kept_rows, e.dw_rows_largest, rows_hi, rows_lo, d);
      else if (all > 0)
        rows_kernel<<<blocks, 256, 0, st>>>(from, wide_rows, head_hi, head_lo, e.s, e.upstream, each, kept_rows,
                                            e.dw_rows_largest, rows_hi, rows_lo, d);
      prepared = prepared || all > 0;
    }
    Maps maps;
    HFFN_TRY(logits_job(maps, e, dtype, weight, n, d, vocab));
    for (int part = 0; part < PARTS; ++part)
      HFFN_TRY(make_map(&maps.out[part], part_type(dtype), w.g[part], e.n_pad, width, width, 32, 32));
    HFFN_TRY((launch_products<PARTS, kGrad>(maps, e, row_tiles * columns, prepared, st)));
    e.jobs = 0;
    int64_t tiles = 0;
    if (grad_hidden != nullptr) {
      const int j = e.jobs++;
      for (int part = 0; part < PARTS; ++part) {
        HFFN_TRY(operand_map(&maps.a[j][part], dtype, w.g[part], e.n_pad, e.width, width, 128));
        HFFN_TRY(operand_map(&maps.b[j][part], dtype, head[part], PARTS == 2 ? e.width : vocab, d, d, kBlockK));
      }
      HFFN_TRY(make_map(&maps.out[0], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, w.slots, splits * e.n_pad, d, d, 32, 32));
      e.job[j] = {n, d, e.width, 0, splits, PARTS == 2 ? 0 : v0};
      tiles += row_tiles * wide * splits;
    }
    if (grad_weight != nullptr) {
      // job 1 is dw: without dh, job 0 is empty
      if (e.jobs == 0) e.job[e.jobs++] = {};
      for (int part = 0; part < PARTS; ++part) {
        HFFN_TRY(operand_map(&maps.a[1][part], dtype, w.g[part], e.n_pad, e.width, width, kBlockK));
        HFFN_TRY(operand_map(&maps.b[1][part], dtype, rows[part], e.n_pad, d, d, kBlockK));
      }
      HFFN_TRY(make_map(&maps.out[1], PARTS == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                        grad_weight, vocab, d, d, 32, 32));
      e.job[1] = {e.width, d, n, 2, 1, 0};
      e.jobs = 2;
      tiles += columns * wide;
    }
    if (tiles > 0) HFFN_TRY((launch_products<PARTS, kGradients>(maps, e, tiles, true, st)));
    prepared = true;
  }
  launch_next<scatter_kernel<T>>(grad_hidden != nullptr ? (unsigned)ceil_div(n, 8) : 1u, 256, 0, st, e.s,
                                 (const float*)w.slots, splits, e.n_pad, e.upstream, static_cast<T*>(grad_hidden),
                                 static_cast<T*>(grad_weight), grad_weight != nullptr ? (int64_t)vocab * d : (int64_t)0, n,
                                 d);
  return launch_status("linear_ce_backward");
}

// Makes the current device's context current for the calling thread too, where that has made no CUDA call yet (a
// framework's backward thread): the tensor maps are encoded by the driver, which asks for one.
static int bind_context() {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  if (e != cudaSuccess) {
    set_error("linear_ce: %s", cudaGetErrorString(e));
    return HFFN_ERR_CUDA;
  }
  return HFFN_OK;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace ce
}  // namespace hffn

using namespace hffn;

extern "C" {

int64_t hffn_linear_ce_state_bytes(int dtype, int64_t n, int32_t d, int32_t vocab) {
  if (ce::check(dtype, n, d, vocab) != HFFN_OK) return -1;
  return ce::state_at(nullptr, dtype, n, d, vocab).bytes;
}

int64_t hffn_linear_ce_forward_workspace(int dtype, int64_t n, int32_t d, int32_t vocab) {
  if (ce::check(dtype, n, d, vocab) != HFFN_OK) return -1;
  return ce::forward_work(nullptr, dtype, n, d, vocab).bytes;
}

int64_t hffn_linear_ce_backward_workspace(int dtype, int64_t n, int32_t d, int32_t vocab) {
  if (ce::check(dtype, n, d, vocab) != HFFN_OK) return -1;
  return ce::backward_work(nullptr, dtype, n, d, vocab).bytes;
}

int hffn_linear_ce_forward(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                           const int64_t* targets, int64_t ignore_index, int reduction, int for_backward, float* loss,
                           void* state, void* work, int64_t n, int32_t d, int32_t vocab, void* stream) {
  HFFN_TRY(ce::check(dtype, n, d, vocab));
  HFFN_REQUIRE(reduction == HFFN_REDUCE_NONE || reduction == HFFN_REDUCE_MEAN || reduction == HFFN_REDUCE_SUM,
               "unknown reduction %d", reduction);
  HFFN_REQUIRE(hidden && weight && targets && loss && state && work, "null pointer argument");
  HFFN_REQUIRE(hidden_stride >= d || n == 1, "hidden rows overlap");
  HFFN_REQUIRE(ce::aligned16(weight) && ce::aligned16(state) && ce::aligned16(work),
               "weight, state and work must be 16-byte aligned");
  HFFN_TRY(bind_stream_device(stream));
  HFFN_TRY(ce::bind_context());
  auto run = dtype == HFFN_F32 ? ce::forward<float> : ce::forward<__nv_bfloat16>;
  return run(hidden, hidden_stride, weight, targets, ignore_index, reduction, for_backward != 0, loss, state, work,
             (int)n, d, vocab, static_cast<cudaStream_t>(stream));
}

int hffn_linear_ce_backward(int dtype, const void* weight, int reduction, const float* grad_loss, void* grad_hidden,
                            void* grad_weight, void* state, void* work, int64_t n, int32_t d, int32_t vocab,
                            void* stream) {
  HFFN_TRY(ce::check(dtype, n, d, vocab));
  HFFN_REQUIRE(reduction == HFFN_REDUCE_NONE || reduction == HFFN_REDUCE_MEAN || reduction == HFFN_REDUCE_SUM,
               "unknown reduction %d", reduction);
  HFFN_REQUIRE(weight && grad_loss && state && work, "null pointer argument");
  HFFN_REQUIRE(ce::aligned16(weight) && ce::aligned16(state) && ce::aligned16(work) && ce::aligned16(grad_hidden) &&
                   ce::aligned16(grad_weight),
               "weight, gradients, state and work must be 16-byte aligned");
  HFFN_TRY(bind_stream_device(stream));
  HFFN_TRY(ce::bind_context());
  auto run = dtype == HFFN_F32 ? ce::backward<float> : ce::backward<__nv_bfloat16>;
  return run(weight, reduction, grad_loss, grad_hidden, grad_weight, state, work, (int)n, d, vocab,
             static_cast<cudaStream_t>(stream));
}

int hffn_linear_ce_error(int32_t* value, int clear) {
  HFFN_REQUIRE(value != nullptr, "null pointer argument");
  cudaError_t e = cudaMemcpyFromSymbol(value, ce::g_error, sizeof(int32_t));
  if (e == cudaSuccess && clear) {
    const int32_t zero = 0;
    e = cudaMemcpyToSymbol(ce::g_error, &zero, sizeof(int32_t));
  }
  if (e != cudaSuccess) {
    set_error("hffn_linear_ce_error: %s", cudaGetErrorString(e));
    return HFFN_ERR_CUDA;
  }
  return HFFN_OK;
}

}  // extern "C"
