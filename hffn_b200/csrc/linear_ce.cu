// Linear softmax cross entropy over a large vocabulary: the loss of hidden states h [n, d] under the head w [vocab, d]
//   z_tv = h_t . w_v,   lse_t = log sum_v exp z_tv,   loss_t = lse_t - z_{t, target_t}
// and its gradients
//   g_tv = c_t (exp(z_tv - lse_t) - [v = target_t]),   dh_t = sum_v g_tv w_v,   dw_v = sum_t g_tv h_t
// without the [n, vocab] logits: the forward reduces each tile of logits to a maximum and a sum of exponentials per
// row, and the backward recomputes the logits of one piece of the vocabulary at a time into g.
//
// Only kept rows exist for the products: rows whose target is ignored (or out of range) are left out when the hidden
// states are gathered, so they cost nothing and whatever they hold (infinities, NaN) reaches no sum. How many are
// kept is known on the device alone; every kernel reads it there, so a call can be captured and replayed.
#include <algorithm>

#include "common.cuh"

namespace hffn {
namespace ce {

constexpr int kRowTile = 256;                        // kept rows are padded to whole tiles (of zeros)
constexpr int64_t kPieceBytes = int64_t(256) << 20;  // of g: the piece of the vocabulary the backward holds at a time
constexpr int kPieceMin = 4096;

__host__ __device__ inline int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// What the forward leaves for the backward, in one buffer.
struct State {
  int32_t* kept;       // [1] rows kept
  int32_t* row_of;     // [n] the input row of each kept row
  int32_t* place_of;   // [n] the kept row of each input row; -1: ignored, -2: target out of range
  int32_t* target;     // [n]
  float* lse;          // [n]
  void* hidden;        // [n_pad, d] the kept rows
  int64_t bytes;
};

static State state_at(void* base, int dtype, int64_t n, int d) {
  uint8_t* p = static_cast<uint8_t*>(base);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    uint8_t* q = p + at;
    at += round_up(bytes, 256);
    return q;
  };
  State s;
  const int64_t n_pad = round_up(n, kRowTile);
  s.kept = reinterpret_cast<int32_t*>(take(4));
  s.row_of = reinterpret_cast<int32_t*>(take(4 * n_pad));
  s.place_of = reinterpret_cast<int32_t*>(take(4 * n_pad));
  s.target = reinterpret_cast<int32_t*>(take(4 * n_pad));
  s.lse = reinterpret_cast<float*>(take(4 * n_pad));
  s.hidden = take(n_pad * d * (dtype == HFFN_F32 ? 4 : 2));
  s.bytes = at;
  return s;
}

// ---- which rows are kept ------------------------------------------------------------------------------------------
constexpr int kGatherThreads = 256;

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
  for (int w = 0; w < kGatherThreads / 32; ++w) total += shared[w];
  return total;
}

// A block owns `span` consecutive input rows: it counts the kept rows before them (from the targets alone, so that no
// block waits for another), places its own and copies them. The last block pads the kept rows to a whole tile of zeros.
template <typename T>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const T* hidden, int64_t stride, const int64_t* targets,
                                                                int64_t ignore, int n, int d, int vocab, int span,
                                                                State s) {
  __shared__ int shared[kGatherThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * span, last = min(n, first + span);
  int mine = 0;
  for (int t = threadIdx.x; t < first; t += kGatherThreads) mine += is_kept(targets[t], ignore, vocab);
  int place = block_count(mine, shared);
  T* out = static_cast<T*>(s.hidden);
  for (int base = first; base < last; base += 32) {      // every warp walks all rows and copies every eighth
    const int t = base + lane;
    const int64_t target = t < last ? targets[t] : ignore;
    const bool keep = t < last && is_kept(target, ignore, vocab);
    const unsigned mask = __ballot_sync(0xffffffffu, keep);
    const int at = place + __popc(mask & ((1u << lane) - 1u));
    if (warp == 0 && t < last) {
      s.place_of[t] = keep ? at : (target == ignore ? -1 : -2);
      if (keep) {
        s.row_of[at] = t;
        s.target[at] = (int)target;
      }
    }
    int k = 0;
    for (unsigned left = mask; left; left &= left - 1, ++k) {
      if (((place + k) & (kGatherThreads / 32 - 1)) != warp) continue;
      const T* from = hidden + (int64_t)(base + __ffs(left) - 1) * stride;
      T* to = out + (int64_t)(place + k) * d;
      for (int i = lane; i < d; i += 32) to[i] = from[i];
    }
    place += __popc(mask);
  }
  if (last == n) {
    if (threadIdx.x == 0) *s.kept = place;
    const int64_t end = round_up(place, kRowTile) * d;
    for (int64_t i = (int64_t)place * d + threadIdx.x; i < end; i += kGatherThreads) out[i] = from_f<T>(0.f);
  }
}

// ---- products -----------------------------------------------------------------------------------------------------
// C[m, n] = sum_k A[m, k] B[n, k], either operand with any strides, 64 x 64 tiles, 4 x 4 values a thread.
enum { kStats = 0, kGrad = 1, kGradHidden = 2, kGradWeight = 3 };

struct Args {
  State s;
  int v0;                  // first vocabulary row of the piece
  int width;               // rows of the piece
  float2* stats;           // [row tiles of the vocabulary][n_pad] maximum and sum of exponentials
  float* picked;           // [n] the target's logit
  const float* upstream;   // [n] c_t by kept row
  float* g;                // [n_pad, width]
  float* dh;               // [n_pad, d]
  void* dw;                // [vocab, d]
  int add;
};

constexpr int kTile = 64, kStep = 16;

template <typename A, typename B, typename T, int EPI>
__global__ void __launch_bounds__(256) product_kernel(const A* a, int64_t am, int64_t ak, const B* b, int64_t bn,
                                                      int64_t bk, int M, int N, int K, int kept_dim, Args e, int d) {
  const int kept = *e.s.kept;
  if (kept_dim == 0) M = kept;       // the dimension that counts tokens
  else K = kept;
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  if (m0 >= M) return;
  __shared__ float as[kStep][kTile + 1], bs[kStep][kTile + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      const int r = i / kStep, k = i % kStep;
      as[k][r] = m0 + r < M && k0 + k < K ? to_f<A>(a[(m0 + r) * am + (k0 + k) * ak]) : 0.f;
      bs[k][r] = n0 + r < N && k0 + k < K ? to_f<B>(b[(n0 + r) * bn + (k0 + k) * bk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += as[k][ty * 4 + i] * bs[k][tx * 4 + j];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty * 4 + i;
    if constexpr (EPI == kStats) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + tx * 4 + j < N) top = fmaxf(top, acc[i][j]);
#pragma unroll
      for (int s = 8; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int v = n0 + tx * 4 + j;
        if (v < N) sum += expf(acc[i][j] - top);
        if (m < M && v < N && v == e.s.target[m]) e.picked[m] = acc[i][j];
      }
#pragma unroll
      for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      if (m < M && tx == 0) e.stats[(int64_t)blockIdx.x * gridDim.y * kTile + m] = make_float2(top, sum);
    } else {
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = n0 + tx * 4 + j;
        if (c >= N) continue;
        if constexpr (EPI == kGrad) {
          const float p = expf(acc[i][j] - e.s.lse[m]);
          e.g[(int64_t)m * e.width + c] = e.upstream[m] * (p - (e.v0 + c == e.s.target[m] ? 1.f : 0.f));
        } else if constexpr (EPI == kGradHidden) {
          float* at = e.dh + (int64_t)m * d + c;
          *at = acc[i][j] + (e.add ? *at : 0.f);
        } else {
          static_cast<T*>(e.dw)[(int64_t)(e.v0 + m) * d + c] = from_f<T>(acc[i][j]);
        }
      }
    }
  }
}

// ---- per-row kernels ----------------------------------------------------------------------------------------------
// lse and loss of each input row from the tiles' maxima and sums, one warp a row.
__global__ void __launch_bounds__(256) losses_kernel(State s, const float2* stats, int64_t ld, int tiles,
                                                     const float* picked, float* losses, int n) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= n) return;
  const int at = s.place_of[t];
  if (at < 0) {
    if (lane == 0) losses[t] = at == -1 ? 0.f : NAN;
    return;
  }
  float top = -INFINITY, sum = 0.f;
  for (int i = lane; i < tiles; i += 32) {
    const float2 v = stats[i * ld + at];
    const float m = fmaxf(top, v.x);
    if (m > -INFINITY) sum = sum * expf(top - m) + v.y * expf(v.x - m);
    else sum += v.y;
    top = m;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float top2 = __shfl_xor_sync(0xffffffffu, top, o), sum2 = __shfl_xor_sync(0xffffffffu, sum, o);
    const float m = fmaxf(top, top2);
    if (m > -INFINITY) sum = sum * expf(top - m) + sum2 * expf(top2 - m);
    else sum += sum2;
    top = m;
  }
  if (lane == 0) {
    const float lse = top + logf(sum);
    s.lse[at] = lse;
    losses[t] = lse - picked[at];
  }
}

// The sum or the mean of the rows' losses (float64, a fixed order): one block.
__global__ void __launch_bounds__(1024) reduce_kernel(State s, const float* losses, int n, int mean, float* loss) {
  __shared__ double shared[32];
  double sum = 0;
  for (int t = threadIdx.x; t < n; t += 1024) sum += (double)losses[t];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < 32; ++w) sum += shared[w];
    *loss = (float)(mean ? sum / max(1, *s.kept) : sum);
  }
}

// c_t of each kept row.
__global__ void __launch_bounds__(256) upstream_kernel(State s, const float* grad_loss, int reduction, float* upstream) {
  const int at = blockIdx.x * 256 + threadIdx.x, kept = *s.kept;
  if (at >= kept) return;
  upstream[at] = reduction == HFFN_REDUCE_NONE ? grad_loss[s.row_of[at]]
                 : reduction == HFFN_REDUCE_MEAN ? grad_loss[0] / (float)kept : grad_loss[0];
}

// dh of each input row: its kept row's, or zeros.
template <typename T>
__global__ void __launch_bounds__(256) scatter_kernel(State s, const float* dh, T* grad_hidden, int n, int d) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= n) return;
  const int at = s.place_of[t];
  for (int i = lane; i < d; i += 32) grad_hidden[(int64_t)t * d + i] = from_f<T>(at < 0 ? 0.f : dh[(int64_t)at * d + i]);
}

// ---- host side ----------------------------------------------------------------------------------------------------
static int piece_width(int64_t n, int vocab) {
  const int64_t width = std::max<int64_t>(kPieceMin, kPieceBytes / 4 / round_up(n, kRowTile) / 256 * 256);
  const int64_t pieces = ceil_div(vocab, width);
  return (int)std::min<int64_t>(vocab, round_up(ceil_div(vocab, pieces), 256));
}

static int64_t forward_bytes(int64_t n, int vocab) {
  const int64_t n_pad = round_up(n, kRowTile);
  return round_up(8 * n_pad * ceil_div(vocab, kTile), 256) + 2 * round_up(4 * n_pad, 256);
}

static int64_t backward_bytes(int64_t n, int d, int vocab) {
  const int64_t n_pad = round_up(n, kRowTile);
  return round_up(4 * n_pad, 256) + round_up(4 * n_pad * piece_width(n, vocab), 256) + round_up(4 * n_pad * d, 256);
}

static int check(int dtype, int64_t n, int32_t d, int32_t vocab) {
  HFFN_REQUIRE(dtype == HFFN_F32 || dtype == HFFN_BF16, "unknown dtype %d", dtype);
  HFFN_REQUIRE(n >= 1 && n <= (int64_t(1) << 24), "token count %lld out of range [1, 2^24]", (long long)n);
  HFFN_REQUIRE(d >= 8 && d % 8 == 0 && d <= 32768, "hidden size %d: a multiple of 8 up to 32768", d);
  HFFN_REQUIRE(vocab >= 1 && vocab <= (1 << 24), "vocabulary %d out of range [1, 2^24]", vocab);
  return HFFN_OK;
}

template <typename T>
static int forward(const void* hidden, int64_t stride, const void* weight, const int64_t* targets, int64_t ignore,
                   int reduction, float* loss, const State& s, uint8_t* work, int n, int d, int vocab, cudaStream_t st) {
  const int64_t n_pad = round_up(n, kRowTile);
  const int tiles = (int)ceil_div(vocab, kTile);
  Args e = {};
  e.s = s;
  e.width = vocab;
  e.stats = reinterpret_cast<float2*>(work);
  e.picked = reinterpret_cast<float*>(work + round_up(8 * n_pad * tiles, 256));
  float* losses = reduction == HFFN_REDUCE_NONE ? loss : e.picked + round_up(4 * n_pad, 256) / 4;
  const int span = (int)std::max<int64_t>(16, ceil_div(n, 512));
  gather_kernel<T><<<(unsigned)ceil_div(n, span), kGatherThreads, 0, st>>>(static_cast<const T*>(hidden), stride, targets,
                                                                          ignore, n, d, vocab, span, s);
  product_kernel<T, T, T, kStats><<<dim3(tiles, (unsigned)(n_pad / kTile)), 256, 0, st>>>(
      static_cast<const T*>(s.hidden), d, 1, static_cast<const T*>(weight), d, 1, n, vocab, d, 0, e, d);
  losses_kernel<<<(unsigned)ceil_div(n, 8), 256, 0, st>>>(s, e.stats, n_pad, tiles, e.picked, losses, n);
  if (reduction != HFFN_REDUCE_NONE)
    reduce_kernel<<<1, 1024, 0, st>>>(s, losses, n, reduction == HFFN_REDUCE_MEAN, loss);
  return launch_status("linear_ce_forward");
}

template <typename T>
static int backward(const void* weight, int reduction, const float* grad_loss, void* grad_hidden, void* grad_weight,
                    const State& s, uint8_t* work, int n, int d, int vocab, cudaStream_t st) {
  const int64_t n_pad = round_up(n, kRowTile);
  const int width = piece_width(n, vocab);
  float* upstream = reinterpret_cast<float*>(work);
  Args e = {};
  e.s = s;
  e.upstream = upstream;
  e.g = reinterpret_cast<float*>(work + round_up(4 * n_pad, 256));
  e.dh = e.g + round_up(4 * n_pad * width, 256) / 4;
  e.dw = grad_weight;
  upstream_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, st>>>(s, grad_loss, reduction, upstream);
  const T *w = static_cast<const T*>(weight), *h = static_cast<const T*>(s.hidden);
  for (int v0 = 0; v0 < vocab; v0 += width) {
    e.v0 = v0;
    e.width = std::min(width, vocab - v0);
    e.add = v0 > 0;
    const T* piece = w + (int64_t)v0 * d;
    const unsigned rows = (unsigned)(n_pad / kTile), cols = (unsigned)ceil_div(e.width, kTile);
    const unsigned wide = (unsigned)ceil_div(d, kTile);
    product_kernel<T, T, T, kGrad><<<dim3(cols, rows), 256, 0, st>>>(h, d, 1, piece, d, 1, n, e.width, d, 0, e, d);
    if (grad_hidden != nullptr)
      product_kernel<float, T, T, kGradHidden><<<dim3(wide, rows), 256, 0, st>>>(e.g, e.width, 1, piece, 1, d, n, d,
                                                                                 e.width, 0, e, d);
    if (grad_weight != nullptr)
      product_kernel<float, T, T, kGradWeight><<<dim3(wide, cols), 256, 0, st>>>(e.g, 1, e.width, h, 1, d, e.width, d,
                                                                                 n, 1, e, d);
  }
  if (grad_hidden != nullptr)
    scatter_kernel<T><<<(unsigned)ceil_div(n, 8), 256, 0, st>>>(s, e.dh, static_cast<T*>(grad_hidden), n, d);
  return launch_status("linear_ce_backward");
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace ce
}  // namespace hffn

using namespace hffn;

extern "C" {

int64_t hffn_linear_ce_state_bytes(int dtype, int64_t n, int32_t d, int32_t vocab) {
  if (ce::check(dtype, n, d, vocab) != HFFN_OK) return -1;
  return ce::state_at(nullptr, dtype, n, d).bytes;
}

int64_t hffn_linear_ce_forward_workspace(int dtype, int64_t n, int32_t d, int32_t vocab) {
  if (ce::check(dtype, n, d, vocab) != HFFN_OK) return -1;
  return ce::forward_bytes(n, vocab);
}

int64_t hffn_linear_ce_backward_workspace(int dtype, int64_t n, int32_t d, int32_t vocab) {
  if (ce::check(dtype, n, d, vocab) != HFFN_OK) return -1;
  return ce::backward_bytes(n, d, vocab);
}

int hffn_linear_ce_forward(int dtype, const void* hidden, int64_t hidden_stride, const void* weight,
                           const int64_t* targets, int64_t ignore_index, int reduction, float* loss, void* state,
                           void* work, int64_t n, int32_t d, int32_t vocab, void* stream) {
  HFFN_TRY(ce::check(dtype, n, d, vocab));
  HFFN_REQUIRE(reduction == HFFN_REDUCE_NONE || reduction == HFFN_REDUCE_MEAN || reduction == HFFN_REDUCE_SUM,
               "unknown reduction %d", reduction);
  HFFN_REQUIRE(hidden && weight && targets && loss && state && work, "null pointer argument");
  HFFN_REQUIRE(hidden_stride >= d || n == 1, "hidden rows overlap");
  HFFN_REQUIRE(ce::aligned16(weight) && ce::aligned16(state) && ce::aligned16(work),
               "weight, state and work must be 16-byte aligned");
  HFFN_TRY(bind_stream_device(stream));
  const ce::State s = ce::state_at(state, dtype, n, d);
  auto run = dtype == HFFN_F32 ? ce::forward<float> : ce::forward<__nv_bfloat16>;
  return run(hidden, hidden_stride, weight, targets, ignore_index, reduction, loss, s, static_cast<uint8_t*>(work),
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
  const ce::State s = ce::state_at(state, dtype, n, d);
  auto run = dtype == HFFN_F32 ? ce::backward<float> : ce::backward<__nv_bfloat16>;
  return run(weight, reduction, grad_loss, grad_hidden, grad_weight, s, static_cast<uint8_t*>(work), (int)n, d, vocab,
             static_cast<cudaStream_t>(stream));
}

}  // extern "C"
