// How often each expert was selected, and the loss that evens it out.  No counterpart in the reference, which returns the router's
// logits for its caller to build one (flash_moe/modules/flash_moe.py:103-105).
//
// With p_h = softmax(logits[h]) the router's probability of expert e = (i, j) is p_0[i] p_1[j].  C[i, j] counts the selections, and
//   loss = nk^2 sum_e (C_e / sum C) mean_t p_0[t, i] p_1[t, j] = (nk^2 / (T sum C)) sum_t s_t,   s_t = p_0[t] C p_1[t]^T.
// The [T, nk^2] probabilities never exist.  With G_0 = p_1 C^T and G_1 = p_0 C the gradient is
//   dlogits[h, t] = upstream (nk^2 / (T sum C)) p_h[t] (G_h[t] - s_t).
// The rows of p sum to 1, so a constant taken off C shifts G_h and s_t alike: C is used without its (whole) mean, which keeps
// the bits of the differences where the counts are nearly even.
#include "common.cuh"

namespace fmoe {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;

__global__ void __launch_bounds__(256) expert_counts_kernel(const int64_t* indices, const uint8_t* mask, int64_t pairs, int k,
                                                            int64_t N, unsigned long long* counts, int32_t* status) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < pairs; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t e = indices[i];
    if (mask != nullptr && mask[i / k] == 0) continue;
    if (e >= 0 && e < N) atomicAdd(counts + e, 1ull);
    else if (e != -1 && status != nullptr) atomicOr(status, FMOE_STATUS_BAD_EXPERT_ID);
  }
}

// What the loss keeps of the counts: one block for both directions.
struct Prepared {
  double coef;    // nk^2 / (T sum C), 0 where there is no token or no selection
  double sum;     // sum C
  double tokens;  // unmasked
  float mean;     // what was taken off
  int pad;
};
constexpr int kParts = 64;
struct Part {
  double sum, tokens;
};

__global__ void __launch_bounds__(256) balance_sums_kernel(const int64_t* counts, int n, const uint8_t* mask, int64_t T, Part* part) {
  __shared__ double s[2][8];
  double c = 0.0, m = 0.0;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += kParts * 256) c += static_cast<double>(counts[i]);
  if (mask != nullptr)
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < T; i += kParts * 256) m += mask[i] != 0;
  for (int d = 16; d > 0; d >>= 1) {
    c += __shfl_xor_sync(kFull, c, d);
    m += __shfl_xor_sync(kFull, m, d);
  }
  if ((threadIdx.x & 31) == 0) {
    s[0][threadIdx.x >> 5] = c;
    s[1][threadIdx.x >> 5] = m;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) {
      c += s[0][i];
      m += s[1][i];
    }
    part[blockIdx.x] = {c, m};
  }
}

__global__ void __launch_bounds__(256) balance_prepare_kernel(const int64_t* counts, int nk, bool masked, int64_t T, const Part* part,
                                                              Prepared* head, float* c0, float* c1) {
  double sum = 0.0, tokens = 0.0;
  for (int i = 0; i < kParts; ++i) {
    sum += part[i].sum;
    tokens += part[i].tokens;
  }
  if (!masked) tokens = static_cast<double>(T);
  const int n = nk * nk;
  const double mean = rint(sum / n);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    head->coef = sum > 0.0 && tokens > 0.0 ? static_cast<double>(n) / (sum * tokens) : 0.0;
    head->sum = sum;
    head->tokens = tokens;
    head->mean = static_cast<float>(mean);
  }
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
    const float v = static_cast<float>(static_cast<double>(counts[i]) - mean);
    c1[i] = v;                          // [key of half 0][key of half 1]: G_1 reads it along the rows
    c0[(i % nk) * nk + i / nk] = v;     // transposed, for G_0
  }
}

constexpr int kTile = 8;  // tokens of a CTA, one warp each for the softmax

// p[h][t][i] of the CTA's tokens, zero for masked ones and behind the last
template <typename T>
__device__ void softmax_tile(const T* logits, int64_t ts, int64_t hs, const uint8_t* mask, int64_t t0, int64_t ntok, int nk, float* p) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t t = t0 + w;
  const bool live = t < ntok && (mask == nullptr || mask[t] != 0);
  for (int h = 0; h < 2; ++h) {
    float* row = p + (h * kTile + w) * nk;
    if (!live) {
      for (int i = lane; i < nk; i += 32) row[i] = 0.f;
      continue;
    }
    const T* src = logits + t * ts + h * hs;
    float top = -INFINITY, sum = 0.f;
    for (int i = lane; i < nk; i += 32) top = fmaxf(top, to_f32<T>(src[i]));
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
    for (int i = lane; i < nk; i += 32) sum += row[i] = expf(to_f32<T>(src[i]) - top);
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
    for (int i = lane; i < nk; i += 32) row[i] /= sum;
  }
  __syncthreads();
}

// g[t] += sum_j c[j][i] p[t][j] for column i of this thread
__device__ __forceinline__ void product(const float* c, const float* p, int nk, int i, float (&g)[kTile]) {
  for (int t = 0; t < kTile; ++t) g[t] = 0.f;
  for (int j = 0; j < nk; ++j) {
    const float v = c[static_cast<int64_t>(j) * nk + i];
    for (int t = 0; t < kTile; ++t) g[t] = fmaf(v, p[t * nk + j], g[t]);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) balance_forward_kernel(const T* logits, int64_t ts, int64_t hs, const uint8_t* mask, int64_t ntok,
                                                              int nk, const float* c0, float* token_s, double* part) {
  extern __shared__ float p[];
  __shared__ float sums[8][kTile];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTile;
  softmax_tile<T>(logits, ts, hs, mask, t0, ntok, nk, p);
  float s[kTile] = {};
  for (int i = threadIdx.x; i < nk; i += 256) {
    float g[kTile];
    product(c0, p + kTile * nk, nk, i, g);
    for (int t = 0; t < kTile; ++t) s[t] = fmaf(p[t * nk + i], g[t], s[t]);
  }
  for (int t = 0; t < kTile; ++t) {
    for (int d = 16; d > 0; d >>= 1) s[t] += __shfl_xor_sync(kFull, s[t], d);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5][t] = s[t];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int t = 0; t < kTile; ++t) {
      float v = 0.f;
      for (int w = 0; w < 8; ++w) v += sums[w][t];
      if (t0 + t < ntok) token_s[t0 + t] = v;
      all += v;
    }
    part[blockIdx.x] = all;
  }
}

__global__ void __launch_bounds__(256) balance_loss_kernel(const Prepared* head, const double* part, int64_t parts, float* loss) {
  __shared__ double sums[8];
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < parts; i += 256) v += part[i];
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) v += sums[i];
    *loss = static_cast<float>(head->coef * (v + static_cast<double>(head->mean) * head->tokens));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) balance_backward_kernel(const T* logits, int64_t ts, int64_t hs, const uint8_t* mask, int64_t ntok,
                                                               int nk, const Prepared* head, const float* c0, const float* c1,
                                                               const float* token_s, const float* upstream, T* dlogits) {
  extern __shared__ float p[];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTile;
  softmax_tile<T>(logits, ts, hs, mask, t0, ntok, nk, p);
  const float scale = static_cast<float>(head->coef * static_cast<double>(*upstream));
  for (int h = 0; h < 2; ++h)
    for (int i = threadIdx.x; i < nk; i += 256) {
      float g[kTile];
      product(h == 0 ? c0 : c1, p + (1 - h) * kTile * nk, nk, i, g);
      for (int t = 0; t < kTile; ++t) {
        if (t0 + t >= ntok) break;
        const bool live = mask == nullptr || mask[t0 + t] != 0;
        dlogits[((t0 + t) * 2 + h) * nk + i] =
            from_f32<T>(live ? p[(h * kTile + t) * nk + i] * (g[t] - token_s[t0 + t]) * scale : 0.f);
      }
    }
}

size_t matrix_bytes(int nk) { return align_up(static_cast<size_t>(nk) * nk * sizeof(float), 256); }
constexpr int kMaxKeys = 2048;

template <typename T>
int forward_typed(const void* logits, int64_t ts, int64_t hs, const uint8_t* mask, int64_t ntok, int nk, const float* c0,
                  const Prepared* head, float* token_s, double* part, float* loss, cudaStream_t stream) {
  const int64_t tiles = (ntok + kTile - 1) / kTile;
  const int smem = 2 * kTile * nk * 4;
  if (tiles > 0) {
    FMOE_CUDA_TRY(allow_smem(balance_forward_kernel<T>, smem));
    balance_forward_kernel<T><<<static_cast<unsigned>(tiles), 256, smem, stream>>>(static_cast<const T*>(logits), ts, hs, mask, ntok, nk, c0, token_s, part);
    FMOE_LAUNCH_CHECK();
  }
  balance_loss_kernel<<<1, 256, 0, stream>>>(head, part, tiles, loss);
  FMOE_LAUNCH_CHECK();
  return FMOE_OK;
}

template <typename T>
int backward_typed(const void* logits, int64_t ts, int64_t hs, const uint8_t* mask, int64_t ntok, int nk, const Prepared* head,
                   const float* c0, const float* c1, const float* token_s, const float* upstream, void* dlogits, cudaStream_t stream) {
  const int64_t tiles = (ntok + kTile - 1) / kTile;
  const int smem = 2 * kTile * nk * 4;
  FMOE_CUDA_TRY(allow_smem(balance_backward_kernel<T>, smem));
  balance_backward_kernel<T><<<static_cast<unsigned>(tiles), 256, smem, stream>>>(static_cast<const T*>(logits), ts, hs, mask, ntok, nk, head, c0, c1,
                                                                                 token_s, upstream, static_cast<T*>(dlogits));
  FMOE_LAUNCH_CHECK();
  return FMOE_OK;
}

}  // namespace

int launch_expert_counts(const int64_t* indices, const uint8_t* mask, int64_t T, int k, int64_t N, int64_t* counts, int32_t* status,
                         cudaStream_t stream) {
  if (T < 0 || k < 0 || N < 0) return FMOE_ERR_BAD_ARG;
  if (N > 0 && counts == nullptr) return FMOE_ERR_BAD_ARG;
  if (N > 0) FMOE_CUDA_TRY(cudaMemsetAsync(counts, 0, static_cast<size_t>(N) * 8, stream));
  if (T == 0 || k == 0) return FMOE_OK;
  if (indices == nullptr) return FMOE_ERR_BAD_ARG;
  const int64_t want = (T * k + 255) / 256, cap = static_cast<int64_t>(device_sm_count()) * 8;
  expert_counts_kernel<<<static_cast<unsigned>(want < cap ? want : cap), 256, 0, stream>>>(
      indices, mask, T * k, k, N, reinterpret_cast<unsigned long long*>(counts), status);
  FMOE_LAUNCH_CHECK();
  return FMOE_OK;
}

size_t balance_prepared_bytes(int nk) { return nk <= 0 || nk > kMaxKeys ? 0 : 256 + 2 * matrix_bytes(nk); }
size_t balance_workspace_bytes(int64_t T) {
  return T < 0 ? 0 : kParts * sizeof(Part) + static_cast<size_t>((T + kTile - 1) / kTile) * sizeof(double);
}

int launch_balance_forward(const void* logits, int64_t ts, int64_t hs, int dtype, const int64_t* counts, const uint8_t* mask, int64_t T,
                           int nk, float* loss, float* token_s, void* prepared, size_t prepared_bytes, void* ws, size_t ws_bytes,
                           cudaStream_t stream) {
  if (T < 0 || nk <= 0 || counts == nullptr || loss == nullptr) return FMOE_ERR_BAD_ARG;
  if (nk > kMaxKeys) return FMOE_ERR_UNSUPPORTED;
  if (T > 0 && (logits == nullptr || token_s == nullptr)) return FMOE_ERR_BAD_ARG;
  if (prepared == nullptr || prepared_bytes < balance_prepared_bytes(nk) || ws == nullptr || ws_bytes < balance_workspace_bytes(T)) return FMOE_ERR_WORKSPACE;
  Prepared* head = static_cast<Prepared*>(prepared);
  float* c0 = reinterpret_cast<float*>(static_cast<char*>(prepared) + 256);
  float* c1 = reinterpret_cast<float*>(static_cast<char*>(prepared) + 256 + matrix_bytes(nk));
  Part* sums = static_cast<Part*>(ws);
  double* part = reinterpret_cast<double*>(sums + kParts);
  balance_sums_kernel<<<kParts, 256, 0, stream>>>(counts, nk * nk, mask, T, sums);
  FMOE_LAUNCH_CHECK();
  balance_prepare_kernel<<<(nk * nk + 1023) / 1024, 256, 0, stream>>>(counts, nk, mask != nullptr, T, sums, head, c0, c1);
  FMOE_LAUNCH_CHECK();
  switch (dtype) {
    case FMOE_DTYPE_F32: return forward_typed<float>(logits, ts, hs, mask, T, nk, c0, head, token_s, part, loss, stream);
    case FMOE_DTYPE_BF16: return forward_typed<__nv_bfloat16>(logits, ts, hs, mask, T, nk, c0, head, token_s, part, loss, stream);
    case FMOE_DTYPE_F16: return forward_typed<__half>(logits, ts, hs, mask, T, nk, c0, head, token_s, part, loss, stream);
    default: return FMOE_ERR_BAD_ARG;
  }
}

int launch_balance_backward(const void* logits, int64_t ts, int64_t hs, int dtype, const uint8_t* mask, int64_t T, int nk,
                            const float* token_s, const void* prepared, size_t prepared_bytes, const float* upstream, void* dlogits,
                            cudaStream_t stream) {
  if (T < 0 || nk <= 0) return FMOE_ERR_BAD_ARG;
  if (nk > kMaxKeys) return FMOE_ERR_UNSUPPORTED;
  if (T == 0) return FMOE_OK;
  if (logits == nullptr || token_s == nullptr || upstream == nullptr || dlogits == nullptr) return FMOE_ERR_BAD_ARG;
  if (prepared == nullptr || prepared_bytes < balance_prepared_bytes(nk)) return FMOE_ERR_WORKSPACE;
  const Prepared* head = static_cast<const Prepared*>(prepared);
  const float* c0 = reinterpret_cast<const float*>(static_cast<const char*>(prepared) + 256);
  const float* c1 = reinterpret_cast<const float*>(static_cast<const char*>(prepared) + 256 + matrix_bytes(nk));
  switch (dtype) {
    case FMOE_DTYPE_F32: return backward_typed<float>(logits, ts, hs, mask, T, nk, head, c0, c1, token_s, upstream, dlogits, stream);
    case FMOE_DTYPE_BF16: return backward_typed<__nv_bfloat16>(logits, ts, hs, mask, T, nk, head, c0, c1, token_s, upstream, dlogits, stream);
    case FMOE_DTYPE_F16: return backward_typed<__half>(logits, ts, hs, mask, T, nk, head, c0, c1, token_s, upstream, dlogits, stream);
    default: return FMOE_ERR_BAD_ARG;
  }
}

}  // namespace fmoe
