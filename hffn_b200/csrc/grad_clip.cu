// The global gradient norm over many tensors, and clipping by it:
//   norm = sqrt(sum over every entry x of every tensor of x^2),   out = x min(1, max_norm / (norm + 1e-6)).
// Memory bound: the norm reads every entry once, the scaling reads and writes every entry once more. 64 M float32
// entries into other buffers: norm 48 us (5.4 TB/s), scaling 75 us (6.9 TB/s, the end of the tensors still in L2); 582 M
// bfloat16 entries into float32: 213 us (5.5 TB/s) and 558 us (6.3 TB/s).
//
// The tensors' addresses travel as a kernel parameter (no copy to the device, nothing kept between calls, and a captured
// graph holds them by value): up to kTableMax tensors per launch. A tensor is cut into chunks of kChunk entries; the
// blocks walk the chunks of all tensors, so hundreds of small tensors cost one launch. Every block leaves one partial
// sum; the next kernel's blocks each add the partials in the same fixed order, so the factor is the same in every
// block and on every call, without atomics.
//
// Squares and sums are float64: a float32 square overflows from 1.8e19 and loses entries below 1e-19, which gradients
// under a loss scale reach.
#include <algorithm>
#include <exception>
#include <vector>

#include "common.cuh"

namespace hffn {
namespace clip {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;             // entries a block takes at a time
// Blocks of one launch, the fastest of 4 to 16 per SM (582 M bfloat16 entries): the norm 213 us with 4 (265 with 8), the
// scaling 558 us with 16 (597 with 8).
constexpr int kNormBlocks = 148 * 4, kScaleBlocks = 148 * 16;
constexpr int kTableMax = 1000;          // 32 bytes each: within the 32764 bytes of kernel parameters
constexpr int kMaxTensors = 64000;

struct Entry {
  const void* in;
  void* out;
  int64_t count;
  int32_t first_chunk;     // chunks of the tensors before this one
  int16_t in_type, out_type;
};

template <int N>
struct Table {
  int32_t tensors, chunks;
  Entry entry[N];
};

// The tensor that owns `chunk`: the last whose first chunk is at or before it.
template <int N>
__device__ __forceinline__ int owner(const Table<N>& table, int chunk) {
  int low = 0, high = table.tensors - 1;
  while (low < high) {
    const int mid = (low + high + 1) >> 1;
    if (table.entry[mid].first_chunk <= chunk) low = mid;
    else high = mid - 1;
  }
  return low;
}

// The sum of one double per thread, the same in every thread, in a fixed order.
__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) shared[warp] = v;
  __syncthreads();
  double total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += shared[w];
  return total;
}

// 16 bytes of a tensor as float32.
template <typename T>
struct Vector {
  static constexpr int kCount = 16 / sizeof(T);
  uint4 bits;
  __device__ __forceinline__ float operator[](int i) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&bits);
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A whole, aligned chunk is loaded before the first entry is used: 128 bytes (float32) in flight per thread.
template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int count) {
  constexpr int kVectors = kChunk / kThreads / Vector<T>::kCount;
  double sum[2] = {0, 0};
  if (count == kChunk && aligned16(p)) {
    Vector<T> x[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) x[i].bits = reinterpret_cast<const uint4*>(p)[i * kThreads + threadIdx.x];
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int j = 0; j < Vector<T>::kCount; ++j) {
        const double v = (double)x[i][j];
        sum[j & 1] += v * v;
      }
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += kThreads) {
      const double v = (double)to_f<T>(p[i]);
      sum[0] += v * v;
    }
  }
  return sum[0] + sum[1];
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4) squares_kernel(const __grid_constant__ Table<N> table, double* partial) {
  __shared__ double shared[kThreads / 32];
  double sum = 0;
  for (int chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
    const Entry& e = table.entry[owner(table, chunk)];
    const int64_t at = (int64_t)(chunk - e.first_chunk) * kChunk;
    const int count = (int)(e.count - at < kChunk ? e.count - at : kChunk);
    sum += e.in_type == HFFN_F32 ? chunk_squares((const float*)e.in + at, count)
                                 : chunk_squares((const __nv_bfloat16*)e.in + at, count);
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The norm of the partial sums, the same bits in every thread of every block.
__device__ __forceinline__ float norm_of(const double* partial, int partials, double* shared) {
  double sum = 0;
  for (int i = threadIdx.x; i < partials; i += kThreads) sum += partial[i];
  return (float)sqrt(block_sum(sum, shared));
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* partial, int partials, float* norm) {
  __shared__ double shared[kThreads / 32];
  const float v = norm_of(partial, partials, shared);
  if (threadIdx.x == 0) *norm = v;
}

__device__ __forceinline__ uint32_t bf16_pair(float low, float high) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(low, high);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four entries of a tensor as float32.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = v;
  else *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pair(v.x, v.y), bf16_pair(v.z, v.w));
}

// Four entries at a time whatever the types, so that a warp's loads and its stores are both without gaps.
template <typename I, typename O>
__device__ __forceinline__ void chunk_scale(const I* in, O* out, int count, float factor) {
  if (count == kChunk && aligned16(in) && aligned16(out)) {
    constexpr int kVectors = kChunk / kThreads / 4;
    float4 x[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) x[i] = load4(in + (i * kThreads + threadIdx.x) * 4);
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      store4(out + (i * kThreads + threadIdx.x) * 4,
             make_float4(x[i].x * factor, x[i].y * factor, x[i].z * factor, x[i].w * factor));
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += kThreads) out[i] = from_f<O>(to_f<I>(in[i]) * factor);
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ Table<N> table, const double* partial,
                                                         int partials, float max_norm, float* norm) {
  __shared__ double shared[kThreads / 32];
  const float total = norm_of(partial, partials, shared);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  const float ratio = max_norm / (total + 1e-6f);
  const float factor = ratio > 1.0f ? 1.0f : ratio;      // a NaN norm passes through
  // last chunks first: the norm's pass has left those in L2
  for (int chunk = table.chunks - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
    const Entry& e = table.entry[owner(table, chunk)];
    if (factor == 1.0f && e.in == e.out) continue;       // nothing changes
    const int64_t at = (int64_t)(chunk - e.first_chunk) * kChunk;
    const int count = (int)(e.count - at < kChunk ? e.count - at : kChunk);
    if (e.in_type == HFFN_F32) {
      const float* in = (const float*)e.in + at;
      if (e.out_type == HFFN_F32) chunk_scale(in, (float*)e.out + at, count, factor);
      else chunk_scale(in, (__nv_bfloat16*)e.out + at, count, factor);
    } else {
      const __nv_bfloat16* in = (const __nv_bfloat16*)e.in + at;
      if (e.out_type == HFFN_F32) chunk_scale(in, (float*)e.out + at, count, factor);
      else chunk_scale(in, (__nv_bfloat16*)e.out + at, count, factor);
    }
  }
}

static int64_t size_of(int type) { return type == HFFN_F32 ? 4 : 2; }

struct Tensors {
  int32_t count;
  const void* const* in;
  void* const* out;            // NULL: none
  const int64_t* numel;
  const int32_t* in_type;
  const int32_t* out_type;
};

static int check_tensors(const Tensors& t) {
  HFFN_REQUIRE(t.count >= 0, "negative tensor count");
  HFFN_REQUIRE(t.count == 0 || (t.in && t.numel && t.in_type), "null tensor list");
  HFFN_REQUIRE(t.count <= kMaxTensors, "%d tensors: at most %d", t.count, kMaxTensors);
  int64_t entries = 0;
  for (int i = 0; i < t.count; ++i) {
    HFFN_REQUIRE(t.numel[i] >= 0 && (entries += t.numel[i]) <= (int64_t(1) << 40), "tensor %d: bad entry count", i);
    HFFN_REQUIRE(t.in_type[i] == HFFN_F32 || t.in_type[i] == HFFN_BF16, "tensor %d: unknown dtype", i);
    HFFN_REQUIRE(t.numel[i] == 0 || t.in[i], "tensor %d: null pointer", i);
    HFFN_REQUIRE(((uintptr_t)t.in[i] & (size_of(t.in_type[i]) - 1)) == 0, "tensor %d: misaligned", i);
    if (t.out == nullptr) continue;
    HFFN_REQUIRE(t.out_type[i] == HFFN_F32 || t.out_type[i] == HFFN_BF16, "output %d: unknown dtype", i);
    HFFN_REQUIRE(t.numel[i] == 0 || t.out[i], "output %d: null pointer", i);
    HFFN_REQUIRE(((uintptr_t)t.out[i] & (size_of(t.out_type[i]) - 1)) == 0, "output %d: misaligned", i);
  }
  return HFFN_OK;
}

// What one block writes no other block may read or write: the outputs are disjoint, and an output overlaps no input but
// its own, which it then equals.
static int check_overlap(const Tensors& t) {
  struct Range {
    uintptr_t begin, end;
    int32_t tensor;
    bool written;
  };
  std::vector<Range> ranges;
  try {
    ranges.reserve(2 * (size_t)t.count);
  } catch (const std::exception& e) {
    set_error("clip_grad_norm: %s", e.what());
    return HFFN_ERR_CUDA;
  }
  for (int i = 0; i < t.count; ++i) {
    if (t.numel[i] == 0) continue;
    const uintptr_t in = (uintptr_t)t.in[i], out = (uintptr_t)t.out[i];
    ranges.push_back({out, out + (uintptr_t)(t.numel[i] * size_of(t.out_type[i])), i, true});
    if (in != out || t.in_type[i] != t.out_type[i])
      ranges.push_back({in, in + (uintptr_t)(t.numel[i] * size_of(t.in_type[i])), i, false});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t end = 0, written_end = 0;    // of the ranges so far: all of them, and those that are written
  for (const Range& r : ranges) {
    HFFN_REQUIRE(r.begin >= written_end && (!r.written || r.begin >= end),
                 "tensor %d shares memory with another of the call that is written", r.tensor);
    end = std::max(end, r.end);
    if (r.written) written_end = std::max(written_end, r.end);
  }
  return HFFN_OK;
}

// The launches of a call: tables of up to kTableMax non-empty tensors.
template <typename F>
static int for_each_table(const Tensors& t, F&& launch) {
  static thread_local Table<kTableMax> table;
  int at = 0;
  while (at < t.count) {
    table.tensors = 0;
    int64_t chunks = 0;
    for (; at < t.count && table.tensors < kTableMax; ++at) {
      if (t.numel[at] == 0) continue;
      table.entry[table.tensors++] = {t.in[at], t.out ? t.out[at] : nullptr, t.numel[at], (int32_t)chunks,
                                      (int16_t)t.in_type[at], (int16_t)(t.out ? t.out_type[at] : 0)};
      chunks += ceil_div(t.numel[at], kChunk);
    }
    table.chunks = (int32_t)chunks;
    if (table.tensors > 0) HFFN_TRY(launch(table));
  }
  return HFFN_OK;
}

// Calls `launch` with the smallest of the table sizes that holds the tensors: the parameters of a launch are copied with
// it, so a short list should not carry 32 KB.
template <int N>
static const Table<N>& cut(const Table<kTableMax>& table) {
  static thread_local Table<N> small;
  small.tensors = table.tensors;
  small.chunks = table.chunks;
  std::copy(table.entry, table.entry + table.tensors, small.entry);
  return small;
}

static int launch_squares(const Tensors& t, double* work, int* partials, cudaStream_t s) {
  *partials = 0;
  return for_each_table(t, [&](const Table<kTableMax>& table) {
    const int blocks = std::min(table.chunks, kNormBlocks);
    double* out = work + *partials;
    *partials += blocks;
    if (table.tensors <= 64) squares_kernel<64><<<blocks, kThreads, 0, s>>>(cut<64>(table), out);
    else squares_kernel<kTableMax><<<blocks, kThreads, 0, s>>>(table, out);
    return launch_status("grad_norm");
  });
}

}  // namespace clip
}  // namespace hffn

using namespace hffn;

extern "C" {

int64_t hffn_grad_norm_workspace(int32_t count) {
  if (count < 0) return -1;
  const int64_t launches = count > 0 ? ceil_div(count, clip::kTableMax) : 1;
  return launches * clip::kNormBlocks * (int64_t)sizeof(double);
}

int hffn_grad_norm(int32_t count, const void* const* tensors, const int64_t* numel, const int32_t* dtypes, float* norm,
                   void* work, void* stream) {
  const clip::Tensors t{count, tensors, nullptr, numel, dtypes, nullptr};
  HFFN_TRY(clip::check_tensors(t));
  HFFN_REQUIRE(norm && work, "null pointer argument");
  HFFN_REQUIRE(((uintptr_t)work & 7) == 0, "work must be 8-byte aligned");
  HFFN_TRY(bind_stream_device(stream));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int partials = 0;
  HFFN_TRY(clip::launch_squares(t, static_cast<double*>(work), &partials, s));
  clip::norm_kernel<<<1, clip::kThreads, 0, s>>>(static_cast<const double*>(work), partials, norm);
  return launch_status("grad_norm");
}

int hffn_clip_grad_norm(int32_t count, const void* const* tensors, void* const* outs, const int64_t* numel,
                        const int32_t* dtypes, const int32_t* out_dtypes, float max_norm, float* norm, void* work,
                        void* stream) {
  const clip::Tensors t{count, tensors, outs, numel, dtypes, out_dtypes};
  HFFN_REQUIRE(count <= 0 || (outs && out_dtypes), "null output list");
  HFFN_TRY(clip::check_tensors(t));
  HFFN_REQUIRE(max_norm >= 0, "max_norm must be at least 0");
  HFFN_REQUIRE(norm && work, "null pointer argument");
  HFFN_REQUIRE(((uintptr_t)work & 7) == 0, "work must be 8-byte aligned");
  HFFN_TRY(clip::check_overlap(t));
  HFFN_TRY(bind_stream_device(stream));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const double* partial = static_cast<const double*>(work);
  int partials = 0;
  HFFN_TRY(clip::launch_squares(t, static_cast<double*>(work), &partials, s));
  if (partials == 0) {
    clip::norm_kernel<<<1, clip::kThreads, 0, s>>>(partial, 0, norm);
    return launch_status("clip_grad_norm");
  }
  return clip::for_each_table(t, [&](const clip::Table<clip::kTableMax>& table) {
    const int blocks = std::min(table.chunks, clip::kScaleBlocks);
    if (table.tensors <= 64)
      clip::scale_kernel<64><<<blocks, clip::kThreads, 0, s>>>(clip::cut<64>(table), partial, partials, max_norm, norm);
    else
      clip::scale_kernel<clip::kTableMax><<<blocks, clip::kThreads, 0, s>>>(table, partial, partials, max_norm, norm);
    norm = nullptr;            // the first launch stores it
    return launch_status("clip_grad_norm");
  });
}

}  // extern "C"
