// The global norm of many gradients and their clipping, n = scale * sqrt(sum g^2), g <- g * scale * min(1, max_norm / (n + eps)).
// No counterpart in the reference, whose backward leaves the optimiser to its caller; the layer's backward writes dense
// gradients of both expert tables (flash_moe/ops/triton/flash_expert.py:653-745), so this pass over them is long.
//
// Memory-bound: every gradient is read once for the norm and, only where the factor is not 1, read and written once more.
// One launch covers up to kTensors tensors: their addresses travel as a kernel parameter, nothing is copied to the device.  The
// chunks of all tensors form one list of which each CTA has a contiguous piece, so the sums are formed in a fixed order.
#include <algorithm>
#include <cfloat>
#include <new>

#include "common.cuh"

namespace fmoe {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kTensors = 96;
constexpr int kThreads = 256;
// Eight 16-byte loads a thread, and a grid of two CTAs an SM, each with two chunks on the way.  The gradients of four blocks of width
// 1024 (371 MB, bfloat16): 71 us for the sums (5.2 TB/s; behind a pass that wrote, whose lines are still on their way to memory;
// 59 us and 6.3 TB/s by itself) and 111 to scale (6.7 TB/s).  Sums alone and the whole call, measured
// together: 32 KiB with 2 CTAs an SM 78 and 186, with 4 86 and 203; 16 KiB with 2 88 and 203, with 4 82 and 191; 8 KiB with 4 86 and 199.
constexpr int kChunkBytes = 32768;
constexpr int kLoads = kChunkBytes / 16 / kThreads;

struct TensorList {
  void* ptr[kTensors];
  int64_t numel[kTensors];
  int64_t first[kTensors + 1];  // chunks in front of the tensor
  uint8_t dtype[kTensors];
  int count;
};

// the tensor that chunk c belongs to
__device__ __forceinline__ int find_tensor(const TensorList& l, int64_t c) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A CTA's walk over its chunks, up or down, with the next chunk's pieces on the way while the present one is worked on.  Pieces are
// raw 16 bytes whatever the type; a tensor that does not start at one is read value by value.
struct Walk {
  const TensorList& l;
  int tensor;
  uint4 q[kLoads];
  char* at;   // the chunk
  int bytes;  // of it
  uint8_t dtype;
  bool pieces;

  __device__ __forceinline__ Walk(const TensorList& list, int64_t c) : l(list), tensor(find_tensor(list, c)) {}
  __device__ __forceinline__ void fetch(int64_t c) {
    while (c >= l.first[tensor + 1]) ++tensor;
    while (c < l.first[tensor]) --tensor;
    dtype = l.dtype[tensor];
    const int64_t offset = (c - l.first[tensor]) * kChunkBytes;
    const int64_t left = l.numel[tensor] * (dtype == FMOE_DTYPE_F32 ? 4 : 2) - offset;
    at = static_cast<char*>(l.ptr[tensor]) + offset;
    bytes = static_cast<int>(left < kChunkBytes ? left : kChunkBytes);
    pieces = (reinterpret_cast<uintptr_t>(at) & 15u) == 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int b = (i * kThreads + threadIdx.x) * 16;
      q[i] = make_uint4(0, 0, 0, 0);
      if (pieces && b + 16 <= bytes) q[i] = ld16(at + b);
    }
  }
  // values that are not in a whole piece: from(index), then every kThreads
  __device__ __forceinline__ int rest(int size) const { return (pieces ? bytes / 16 * 16 / size : 0) + threadIdx.x; }
};

template <typename T> __device__ __forceinline__ float chunk_squares(const Walk& w) {
  constexpr int VEC = Vec16<T>::N;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    float f[VEC];
    unpack16<T>(w.q[i], f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j & 3] = fmaf(f[j], f[j], acc[j & 3]);
  }
  const T* p = reinterpret_cast<const T*>(w.at);
  for (int e = w.rest(sizeof(T)); e < static_cast<int>(w.bytes / sizeof(T)); e += kThreads) {
    const float f = to_f32<T>(p[e]), oldest = acc[0];  // the four sums in turn: as short as those of whole pieces
    acc[0] = acc[1];
    acc[1] = acc[2];
    acc[2] = acc[3];
    acc[3] = fmaf(f, f, oldest);
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

__device__ __forceinline__ double cta_sum(double v) {
  __shared__ double sums[kThreads / 32];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) v += sums[i];
  return v;
}

__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ TensorList l, double* part) {
  const int64_t chunks = l.first[l.count];
  const int64_t c0 = chunks * blockIdx.x / gridDim.x, c1 = chunks * (blockIdx.x + 1) / gridDim.x;
  double sum = 0.0;  // float32 inside a chunk, 64 bits over the chunks
  if (c0 < c1) {
    Walk next(l, c0);
    next.fetch(c0);
    for (int64_t c = c0; c < c1; ++c) {
      const Walk now = next;
      if (c + 1 < c1) next.fetch(c + 1);
      float v;
      if (now.dtype == FMOE_DTYPE_F32) v = chunk_squares<float>(now);
      else if (now.dtype == FMOE_DTYPE_BF16) v = chunk_squares<__nv_bfloat16>(now);
      else v = chunk_squares<__half>(now);
      sum += v;
    }
  }
  sum = cta_sum(sum);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

struct NormArgs {
  const double* part;
  int parts;
  float scale;
  const float* device_scale;  // nullable: multiplies scale
  float* norm;
};

__device__ __forceinline__ float scale_of(const NormArgs& a) {
  return a.device_scale != nullptr ? a.scale * *a.device_scale : a.scale;
}
__device__ __forceinline__ float norm_of(const NormArgs& a, float scale) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < a.parts; i += kThreads) sum += a.part[i];
  return static_cast<float>(sqrt(cta_sum(sum)) * fabs(static_cast<double>(scale)));
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const NormArgs a) {
  const float n = norm_of(a, scale_of(a));
  if (threadIdx.x == 0) *a.norm = n;
}

template <typename T> __device__ __forceinline__ void chunk_scale(const Walk& w, float factor) {
  constexpr int VEC = Vec16<T>::N;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int b = (i * kThreads + threadIdx.x) * 16;
    float f[VEC];
    unpack16<T>(w.q[i], f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] *= factor;
    if (w.pieces && b + 16 <= w.bytes) *reinterpret_cast<uint4*>(w.at + b) = pack16<T>(f);
  }
  T* p = reinterpret_cast<T*>(w.at);
  for (int e = w.rest(sizeof(T)); e < static_cast<int>(w.bytes / sizeof(T)); e += kThreads) p[e] = from_f32<T>(to_f32<T>(p[e]) * factor);
}

// Chunks in the opposite order of the sums: what those read last is in the L2 cache still.
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ TensorList l, const NormArgs a, float max_norm,
                                                             float eps) {
  const float scale = scale_of(a);
  const float n = norm_of(a, scale);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = n;
  const float ratio = max_norm / (n + eps);
  const float factor = (ratio > 1.f ? 1.f : ratio) * scale;  // a NaN stays
  if (factor == 1.f) return;
  const int64_t chunks = l.first[l.count];
  const int64_t c0 = chunks * blockIdx.x / gridDim.x, c1 = chunks * (blockIdx.x + 1) / gridDim.x;
  if (c0 == c1) return;
  Walk next(l, c1 - 1);
  next.fetch(c1 - 1);
  for (int64_t c = c1 - 1; c >= c0; --c) {
    const Walk now = next;
    if (c > c0) next.fetch(c - 1);
    if (now.dtype == FMOE_DTYPE_F32) chunk_scale<float>(now, factor);
    else if (now.dtype == FMOE_DTYPE_BF16) chunk_scale<__nv_bfloat16>(now, factor);
    else chunk_scale<__half>(now, factor);
  }
}

constexpr int kGridCap = kB200Sms * 2;  // whatever the device: the workspace may have been sized while another was current
int launches(int count) { return (count + kTensors - 1) / kTensors; }

// apart: no two tensors may share memory, where they are written: one would be scaled twice
int check_tensors(void* const* grads, const int64_t* numels, const int32_t* dtypes, int count, bool apart) {
  struct Range {
    uintptr_t lo, hi;
  };
  Range* r = new (std::nothrow) Range[count];
  if (r == nullptr) return FMOE_ERR_BAD_ARG;
  int n = 0, rc = FMOE_OK;
  for (int i = 0; i < count && rc == FMOE_OK; ++i) {
    if (numels[i] < 0 || dtypes[i] < FMOE_DTYPE_F32 || dtypes[i] > FMOE_DTYPE_F16 || (numels[i] > 0 && grads[i] == nullptr)) rc = FMOE_ERR_BAD_ARG;
    else if (numels[i] > 0) {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(grads[i]);
      if (lo % dtype_size(dtypes[i]) != 0) rc = FMOE_ERR_ALIGNMENT;
      r[n++] = {lo, lo + static_cast<uintptr_t>(numels[i]) * dtype_size(dtypes[i])};
    }
  }
  if (rc == FMOE_OK && apart) {
    std::sort(r, r + n, [](const Range& a, const Range& b) { return a.lo < b.lo; });
    for (int i = 1; i < n; ++i)
      if (r[i].lo < r[i - 1].hi) rc = FMOE_ERR_BAD_ARG;
  }
  delete[] r;
  return rc;
}

void fill(TensorList* l, void* const* grads, const int64_t* numels, const int32_t* dtypes, int count) {
  l->count = count;
  l->first[0] = 0;
  for (int i = 0; i < count; ++i) {
    l->ptr[i] = grads[i];
    l->numel[i] = numels[i];
    l->dtype[i] = static_cast<uint8_t>(dtypes[i]);
    const int64_t elems = kChunkBytes / dtype_size(dtypes[i]);
    l->first[i + 1] = l->first[i] + (numels[i] + elems - 1) / elems;
  }
}

int grid_of(const TensorList& l) {
  const int64_t chunks = l.first[l.count];
  return static_cast<int>(chunks < 1 ? 1 : chunks < kGridCap ? chunks : kGridCap);
}

}  // namespace

size_t grad_norm_workspace_bytes(int count) {
  return count <= 0 ? 0 : static_cast<size_t>(launches(count)) * kGridCap * sizeof(double);
}

int launch_grad_norm(void* const* grads, const int64_t* numels, const int32_t* dtypes, int count, bool clip, float max_norm,
                     float eps, float scale, const float* device_scale, float* norm, void* ws, size_t ws_bytes,
                     cudaStream_t stream) {
  if (count < 0 || norm == nullptr || (count > 0 && (grads == nullptr || numels == nullptr || dtypes == nullptr))) return FMOE_ERR_BAD_ARG;
  if (!(scale >= 0.f && scale <= FLT_MAX) || (clip && (!(max_norm >= 0.f) || !(eps >= 0.f)))) return FMOE_ERR_BAD_ARG;
  if (count == 0) {
    FMOE_CUDA_TRY(cudaMemsetAsync(norm, 0, sizeof(float), stream));
    return FMOE_OK;
  }
  if (ws == nullptr || ws_bytes < grad_norm_workspace_bytes(count)) return FMOE_ERR_WORKSPACE;
  if (!aligned16(ws)) return FMOE_ERR_ALIGNMENT;
  const int rc = check_tensors(grads, numels, dtypes, count, clip);
  if (rc != FMOE_OK) return rc;
  double* part = static_cast<double*>(ws);
  int parts = 0;
  TensorList l;
  for (int i = 0; i < count; i += kTensors) {
    fill(&l, grads + i, numels + i, dtypes + i, std::min(kTensors, count - i));
    const int grid = grid_of(l);
    grad_squares_kernel<<<grid, kThreads, 0, stream>>>(l, part + parts);
    FMOE_LAUNCH_CHECK();
    parts += grid;
  }
  const NormArgs a = {part, parts, scale, device_scale, norm};
  if (!clip) {
    grad_norm_kernel<<<1, kThreads, 0, stream>>>(a);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
  }
  for (int i = 0; i < count; i += kTensors) {
    if (count > kTensors) fill(&l, grads + i, numels + i, dtypes + i, std::min(kTensors, count - i));
    grad_scale_kernel<<<grid_of(l), kThreads, 0, stream>>>(l, a, max_norm, eps);
    FMOE_LAUNCH_CHECK();
  }
  return FMOE_OK;
}

}  // namespace fmoe
