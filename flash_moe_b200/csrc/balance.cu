// How often each expert was selected, and the loss that evens it out.  No counterpart in the reference, which returns the router's
// logits for its caller to build one (flash_moe/modules/flash_moe.py:103-105).
//
// With p_h = softmax(logits[h]) the router's probability of expert e = (i, j) is p_0[i] p_1[j].  C[i, j] counts the selections, and
//   loss = nk^2 sum_e (C_e / sum C) mean_t p_0[t, i] p_1[t, j] = (nk^2 / (T sum C)) sum_t s_t,   s_t = p_0[t] C p_1[t]^T.
// The [T, nk^2] probabilities never exist.  With G_0 = p_1 C^T and G_1 = p_0 C the gradient is
//   dlogits[h, t] = upstream (nk^2 / (T sum C)) p_h[t] (G_h[t] - s_t).
// The rows of p sum to 1, so a constant taken off C shifts G_h and s_t alike: C is used without its (whole) mean, which keeps
// the bits of the differences where the counts are nearly even.
//
// The two products run on the tensor cores (tcgen05) with float16 operands.  A float16 holds 11 bits, and none below 2^-24, so:
//   a probability p, times 2^15, is the sum of two of them to within 2^-23 of it, or 2^-40 in all where p < 2^-17; p < 2^-40 is 0;
//   a count, less the mean, is such a sum exactly up to 2^22 (up to 2048 the second is zero and its product is left out), above
//   to within 2^-23 of it, or 2^-39 of the largest.
// hi C_hi + lo C_hi + hi C_lo, without lo C_lo, less than 2^-22 p C, in one float32 accumulator is what a float32 product would give,
// but for the absolute 2^-40 C a key: where only experts that improbable were selected, of counts whose rounded mean is 0, the loss
// and what it would pull on are below 2^-40 nk^2 and are not told from 0.  Pieces of bfloat16 would keep them, five products instead of two.
//
// Launches: row statistics (maximum and 1 / sum of both halves) beside the sums of the counts; the centred counts as float16
// pieces in the order in which shared memory wants them; the product with s_t and the loss; for the gradient one more product
// kernel, which needs nothing from memory but the logits, five numbers a token and the pieces.

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace fmoe {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;

// ------------------------------------------------------------------------------------------------ counts
// Popular experts are selected again and again: at a Zipf exponent of 1.1 one id of a million takes an eighth of the selections,
// and additions to one address follow one another (56 us for 524288 selections, all by global atomics).  So each CTA adds in
// a small table in shared memory first, an id in one of two places of its own; an id that finds both taken by others goes to
// global memory, and at the end so does each place of the table.  Whole numbers: the order changes nothing.
constexpr int kCountThreads = 512;
constexpr int kCountPlaces = 4096;

__device__ __forceinline__ void count_one(int64_t e, int64_t N, int* ids, unsigned* seen, unsigned long long* counts, int32_t* status) {
  if (e < 0 || e >= N) {
    if (e != -1 && status != nullptr) atomicOr(status, FMOE_STATUS_BAD_EXPERT_ID);
    return;
  }
  if (e < 0x7FFFFFFF) {
    const int id = static_cast<int>(e);
    const unsigned place = (static_cast<unsigned>(id) * 2654435761u) >> 20;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned at = place ^ i;
      int owner = *static_cast<volatile int*>(ids + at);
      if (owner == -1) owner = atomicCAS(ids + at, -1, id);
      if (owner == -1 || owner == id) {
        atomicAdd(seen + at, 1u);
        return;
      }
    }
  }
  atomicAdd(counts + e, 1ull);
}

// Walks over selections i, i + step, ...: reads kAhead ids, and the mask of their tokens, before the first is used.  The token moves
// on by whole and left-over slots, without a division a selection.
template <int kAhead, typename Use>
__device__ __forceinline__ void each_selection(const int64_t* indices, const uint8_t* mask, int64_t i, int64_t end, int64_t step, int k,
                                               Use&& use) {
  int64_t token = 0, tokens = 0;
  int slot = 0, slots = 0;
  if (mask != nullptr) {
    token = i / k;
    slot = static_cast<int>(i % k);
    tokens = step / k;
    slots = static_cast<int>(step % k);
  }
  while (i < end) {
    int64_t e[kAhead];
    uint8_t keep[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool in = i + u * step < end;
      e[u] = in ? indices[i + u * step] : -1;
      keep[u] = 1;
      if (mask != nullptr) {
        if (in) keep[u] = mask[token];
        token += tokens;
        slot += slots;
        if (slot >= k) {
          slot -= k;
          ++token;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (keep[u] != 0) use(e[u]);
    i += kAhead * step;
  }
}

// One cluster of CTAs clears the counts itself where the call is small: a launch less.
template <bool CLEAR>
__global__ void __launch_bounds__(kCountThreads) expert_counts_kernel(const int64_t* indices, const uint8_t* mask, int64_t pairs, int k,
                                                                      int64_t N, unsigned long long* counts, int32_t* status) {
  __shared__ int ids[kCountPlaces];
  __shared__ unsigned seen[kCountPlaces];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kCountThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kCountThreads;
  for (int i = threadIdx.x; i < kCountPlaces; i += kCountThreads) {
    ids[i] = -1;
    seen[i] = 0;
  }
  if (CLEAR) {
    for (int64_t i = first; i < N; i += step) counts[i] = 0;
    ptx::cluster_sync();
  } else {
    __syncthreads();
  }
  each_selection<4>(indices, mask, first, pairs, step, k, [&](int64_t e) { count_one(e, N, ids, seen, counts, status); });
  __syncthreads();
  for (int i = threadIdx.x; i < kCountPlaces; i += kCountThreads)
    if (seen[i] != 0) atomicAdd(counts + ids[i], static_cast<unsigned long long>(seen[i]));
}

// Many selections of not too many experts: every CTA counts all its selections in shared memory, in 16 bits an expert, and the
// eight CTAs of a cluster add theirs up before they go to global memory, each a part of the experts and in ascending order.
// At 4.2 million selections of 65536 experts the tables above are mostly taken by others.  What is left of its 21 us there is
// 34 MB of ids (5 us), the atomics in shared memory and 120 CTAs' worth of counters on their way to global memory.
constexpr int kHistCtas = 8;
constexpr int kHistThreads = 1024;
constexpr int kHistExperts = 102400;      // 200 KB
constexpr int64_t kHistMost = 65535;      // selections of a CTA before a counter could overflow

__device__ __forceinline__ unsigned ld_cluster_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared::cluster.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}

__global__ void __launch_bounds__(kHistThreads, 1) expert_histogram_kernel(const int64_t* indices, const uint8_t* mask, int64_t pairs, int k,
                                                                           int N, unsigned long long* counts, int32_t* status) {
  extern __shared__ uint4 hist[];
  unsigned* words = reinterpret_cast<unsigned*>(hist);
  const int quads = (N + 7) / 8;  // 16 bytes, eight experts
  const uint32_t rank = ptx::cluster_ctarank();
  const int64_t p0 = pairs * blockIdx.x / gridDim.x, p1 = pairs * (blockIdx.x + 1) / gridDim.x;
  // all CTAs of a cluster go round equally often
  const int64_t most = pairs / gridDim.x + 1;
  for (int64_t done = 0; done < most; done += kHistMost) {
    for (int i = threadIdx.x; i < quads; i += kHistThreads) hist[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int64_t end = p0 + done + kHistMost < p1 ? p0 + done + kHistMost : p1;
    each_selection<8>(indices, mask, p0 + done + threadIdx.x, end, kHistThreads, k, [&](int64_t e) {
      if (e >= 0 && e < N) atomicAdd(words + (e >> 1), 1u << ((e & 1) * 16));
      else if (e != -1 && status != nullptr) atomicOr(status, FMOE_STATUS_BAD_EXPERT_ID);
    });
    ptx::cluster_sync();
    // a lane per expert: a warp adds to 256 consecutive bytes, a quarter of the sectors that a lane per 16 bytes would touch
    const int e0 = N * static_cast<int64_t>(rank) / kHistCtas, e1 = N * static_cast<int64_t>(rank + 1) / kHistCtas;
    const uint32_t base = ptx::smem_u32(hist);
    for (int e = e0 + threadIdx.x; e < e1; e += kHistThreads) {
      unsigned sum = 0;
#pragma unroll
      for (int r = 0; r < kHistCtas; ++r) sum += ld_cluster_u16(ptx::map_to_cta(base + e * 2, r));
      if (sum != 0) atomicAdd(counts + e, static_cast<unsigned long long>(sum));
    }
    ptx::cluster_sync();  // nobody clears, or leaves, while others read
  }
}

// ------------------------------------------------------------------------------------------------ statistics and counts
constexpr int kParts = 64;  // CTAs that sum the counts
constexpr int kMaxKeys = 2048;
constexpr int kTileTokens = 128;
constexpr int kChunk = 256;  // columns of a product that one CTA accumulates, at most

inline int padded_keys(int nk) { return (nk + 63) / 64 * 64; }

struct Part {
  double sum;
  long long top, tokens;
};

// What both directions keep of the counts, in front of their pieces.
struct Prepared {
  double coef;        // nk^2 / (T sum C), 0 where there is no token or no selection
  double tokens;      // unmasked
  float mean;         // what was taken off
  float unscale;      // accumulator -> G: 2^(shift - 15)
  int second;         // whether the second pieces of the counts are needed
  unsigned finished;  // CTAs of the forward product that have ended
};
constexpr size_t kHeadBytes = 256;

// exp(x - top) / 2^d, with one small d for all values of a row whose largest is top: by the exponential of base 2, at
// x log2 e - c, where c is top log2 e rounded and d what it was rounded by, which the row's sum has as well.  One multiply-add and
// one exponential; values below 2^-126 become 0.  From 2^30 on d would overflow: neighbours of type float are 64 or more apart
// there, so x = top is all that counts, and a power of two in the place of log2 e, for which c is exact, gives 1 for it and 0 for
// the others, 256 below it.
struct RowExp {
  float a, c;
  __device__ __forceinline__ explicit RowExp(float top) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23 & 255u) - 127;
    a = e < 30 ? 1.44269504f : __uint_as_float(static_cast<uint32_t>(32 - e + 127) << 23);
    c = __fmul_rn(a, top);
  }
  __device__ __forceinline__ RowExp() : a(0.f), c(0.f) {}
  __device__ __forceinline__ float operator()(float x) const {
    float v;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"(fmaf(x, a, -c)));
    return v;
  }
};

template <typename T> __device__ __forceinline__ uint32_t minus_infinity() { return 0xFF800000u; }
template <> __device__ __forceinline__ uint32_t minus_infinity<__nv_bfloat16>() { return 0xFF80FF80u; }
template <> __device__ __forceinline__ uint32_t minus_infinity<__half>() { return 0xFC00FC00u; }

// A piece of a row: 8 or 4 logits, 16 bytes, from a column on, by loads of W bytes: 16 where rows are made of aligned pieces, 8 or 4
// where they are made of such, and 2 for an odd number of 16-bit keys, where every other row starts in the middle of a word: there
// the words that hold the piece are read, five of them, and shifted.  What lies behind the row's end, or in a row that is not
// read, is minus infinity: its exponential is 0 and no use of the values has to ask.  Each load is one predicated instruction into
// the register that holds the fill: with a branch, the compiler may copy the value where the ways meet, and a copy waits for it.
template <typename T, int W> struct Piece {
  static constexpr int N = Vec16<T>::N;
  static constexpr int kRegs = W == 2 ? 6 : 4;
  uint32_t w[kRegs];  // W = 2: five words, and 2 * columns to the row's end + whether the piece starts in the middle of the first
  __device__ __forceinline__ void load(const T* at, int left, bool read) {  // `left` columns to the row's end
    const uint32_t none = minus_infinity<T>();
#pragma unroll
    for (int i = 0; i < kRegs; ++i) w[i] = none;
    if constexpr (W == 16) {
      asm volatile(
          "{\n\t"
          ".reg .pred p;\n\t"
          "setp.ne.s32 p, %5, 0;\n\t"
          "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t"
          "}\n"
          : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3])
          : "l"(__cvta_generic_to_global(at)), "r"(static_cast<int>(read && left > 0)));
    } else if constexpr (W == 8) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.s32 p, %3, 0;\n\t"
            "@p ld.global.v2.u32 {%0, %1}, [%2];\n\t"
            "}\n"
            : "+r"(w[2 * i]), "+r"(w[2 * i + 1])
            : "l"(__cvta_generic_to_global(at + i * (N / 2))), "r"(static_cast<int>(read && left > i * (N / 2))));
    } else {
      const char* from = reinterpret_cast<const char*>(at);
      int odd = 0;
      if (W == 2) {
        odd = static_cast<int>(reinterpret_cast<uintptr_t>(at) >> 1) & 1;
        from -= 2 * odd;  // an aligned word that holds a value of the row
        w[kRegs - 1] = static_cast<uint32_t>((left > 0 && read ? left : 0) * 2 + odd);
      }
#pragma unroll
      for (int i = 0; i < (W == 2 ? 5 : 4); ++i) {
        bool in = read && left > i * (N / 4) - odd;
        if (W == 2) in = in && left > 0 && i * 2 - odd < 8;
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.s32 p, %2, 0;\n\t"
            "@p ld.global.u32 %0, [%1];\n\t"
            "}\n"
            : "+r"(w[i])
            : "l"(__cvta_generic_to_global(from + 4 * i)), "r"(static_cast<int>(in)));
      }
    }
  }
  __device__ __forceinline__ void get(float* f) const {
    uint4 q = make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (W == 2) {
      if (w[5] & 1u)
        q = make_uint4(__funnelshift_r(w[0], w[1], 16), __funnelshift_r(w[1], w[2], 16), __funnelshift_r(w[2], w[3], 16),
                       __funnelshift_r(w[3], w[4], 16));
    }
    unpack16<T>(q, *reinterpret_cast<float (*)[N]>(f));
    if constexpr (W == 2) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i >= static_cast<int>(w[5] >> 1)) f[i] = -INFINITY;
    }
  }
  // the larger of each two values; the other one where one is a NaN
  __device__ __forceinline__ void join_max(const Piece& o) {
    static_assert(W != 2, "its words are not values yet");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(fmaxf(__uint_as_float(w[i]), __uint_as_float(o.w[i])));
      } else {
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        const T2 m = __hmax2(*reinterpret_cast<const T2*>(&w[i]), *reinterpret_cast<const T2*>(&o.w[i]));
        w[i] = *reinterpret_cast<const uint32_t*>(&m);
      }
    }
  }
};
template <typename T, int W> __device__ __forceinline__ void store_values(T* at, int left, const float* f) {
  constexpr int N = Vec16<T>::N;
  const uint4 q = pack16<T>(*reinterpret_cast<const float (*)[N]>(f));
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (W == 16) {
    if (left > 0) *reinterpret_cast<uint4*>(at) = q;
  } else if constexpr (W == 8) {
    if (left > 0) *reinterpret_cast<uint2*>(at) = make_uint2(q.x, q.y);
    if (left > N / 2) *reinterpret_cast<uint2*>(at + N / 2) = make_uint2(q.z, q.w);
  } else if constexpr (W == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (left > i * (N / 4)) *reinterpret_cast<uint32_t*>(at + i * (N / 4)) = w[i];
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(at);
    const bool odd = (reinterpret_cast<uintptr_t>(at) & 2u) != 0;
    if (left >= N && odd) {  // a value, three words, a value
      p[0] = static_cast<uint16_t>(w[0]);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint32_t*>(p + 2 * i + 1) = __funnelshift_r(w[i], w[i + 1], 16);
      p[7] = static_cast<uint16_t>(w[3] >> 16);
    } else if (left >= N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(p + 2 * i) = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (left > i) p[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
    }
  }
}

// such loads of one and two values: what is not read stays as it was
__device__ __forceinline__ void load_if(bool read, const float* at, float& x, float& y) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.s32 p, %3, 0;\n\t"
      "@p ld.global.v2.f32 {%0, %1}, [%2];\n\t"
      "}\n"
      : "+f"(x), "+f"(y)
      : "l"(__cvta_generic_to_global(at)), "r"(static_cast<int>(read)));
}
__device__ __forceinline__ void load_if(bool read, const float* at, float& x) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.s32 p, %2, 0;\n\t"
      "@p ld.global.f32 %0, [%1];\n\t"
      "}\n"
      : "+f"(x)
      : "l"(__cvta_generic_to_global(at)), "r"(static_cast<int>(read)));
}
// (maximum, 1 / sum of exp(x - maximum)) of each half; 0, 0 for masked tokens, which are not read: no sum has an inverse of 0
// Eight lanes share a row, so a warp has four tokens at a time and a lane enough values for its part of the reductions.  HELD: the
// 16-byte pieces that a lane holds of each half; what longer rows have beside them is read again for the sum.  Memory-bound: 131072
// tokens x 256 keys, bfloat16, 134 MB in 27 us (4.9 TB/s), with 65 % of the issue slots busy with maxima and exponentials.
template <typename T, int W, int HELD>
__global__ void __launch_bounds__(256, 4) balance_stats_kernel(const T* logits, int64_t ts, int64_t hs, const uint8_t* mask, int64_t ntok,
                                                            int nk, float4* stats, const int64_t* counts, Part* part) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x < kParts) {
    __shared__ double sums[8];
    __shared__ long long tops[8], tokens[8];
    const int n = nk * nk;
    double c = 0.0;
    long long top = 0, m = 0;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += kParts * 256) {
      const long long v = counts[i];
      c += static_cast<double>(v);
      top = v > top ? v : top;
    }
    if (mask != nullptr)
      for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < ntok; i += kParts * 256) m += mask[i] != 0;
    for (int d = 16; d > 0; d >>= 1) {
      c += __shfl_xor_sync(kFull, c, d);
      m += __shfl_xor_sync(kFull, m, d);
      const long long o = __shfl_xor_sync(kFull, top, d);
      top = o > top ? o : top;
    }
    if (lane == 0) {
      sums[warp] = c;
      tops[warp] = top;
      tokens[warp] = m;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 8; ++i) {
        c += sums[i];
        m += tokens[i];
        top = tops[i] > top ? tops[i] : top;
      }
      part[blockIdx.x] = {c, top, mask != nullptr ? m : blockIdx.x == 0 ? static_cast<long long>(ntok) : 0ll};
    }
  }
  constexpr int N = Vec16<T>::N;
  const int sub = lane & 7;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 32;
  auto reads = [&](int64_t t) { return t < ntok && (mask == nullptr || mask[t] != 0); };
  bool ahead = reads((static_cast<int64_t>(blockIdx.x) * 8 + warp) * 4 + (lane >> 3));
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * 8 + warp) * 4; t0 < ntok; t0 += step) {
    const int64_t t = t0 + (lane >> 3);
    const bool live = ahead;
    const T* row[2] = {logits + t * ts, logits + t * ts + hs};
    Piece<T, W> q[2][HELD];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int u = 0; u < HELD; ++u) q[h][u].load(row[h] + (u * 8 + sub) * N, nk - (u * 8 + sub) * N, live);
    ahead = reads(t + step);
    float top[2], sum[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[N];
      top[h] = -INFINITY;
      if constexpr (W == 2) {
        auto join = [&](const Piece<T, W>& v) {
          v.get(f);
#pragma unroll
          for (int i = 0; i < N; ++i) top[h] = fmaxf(top[h], f[i]);
        };
#pragma unroll
        for (int u = 0; u < HELD; ++u) join(q[h][u]);
        if (live)
          for (int c = (HELD * 8 + sub) * N; c < nk; c += 8 * N) {
            Piece<T, W> v;
            v.load(row[h] + c, nk - c, true);
            join(v);
          }
      } else {
        Piece<T, W> m = q[h][0];
#pragma unroll
        for (int u = 1; u < HELD; ++u) m.join_max(q[h][u]);
        if (live)
          for (int c = (HELD * 8 + sub) * N; c < nk; c += 8 * N) {
            Piece<T, W> v;
            v.load(row[h] + c, nk - c, true);
            m.join_max(v);
          }
        m.get(f);
#pragma unroll
        for (int i = 0; i < N; ++i) top[h] = fmaxf(top[h], f[i]);
      }
    }
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(kFull, top[0], d));
      top[1] = fmaxf(top[1], __shfl_xor_sync(kFull, top[1], d));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
      const RowExp exp_of(top[h]);
      auto join = [&](const Piece<T, W>& v) {
        float f[N];
        v.get(f);
#pragma unroll
        for (int i = 0; i < N; ++i) part[i & 3] += exp_of(f[i]);
      };
#pragma unroll
      for (int u = 0; u < HELD; ++u) join(q[h][u]);
      if (live)
        for (int c = (HELD * 8 + sub) * N; c < nk; c += 8 * N) {
          Piece<T, W> v;
          v.load(row[h] + c, nk - c, true);
          join(v);
        }
      sum[h] = (part[0] + part[1]) + (part[2] + part[3]);
    }
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) {
      sum[0] += __shfl_xor_sync(kFull, sum[0], d);
      sum[1] += __shfl_xor_sync(kFull, sum[1], d);
    }
    if (sub == 0 && t < ntok)
      stats[t] = live ? make_float4(top[0], 1.f / sum[0], top[1], 1.f / sum[1]) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// Matrix h [row n][column k]: what multiplies p_(1-h)[k] in G_h[n], so h = 0 is C and h = 1 its transpose.  Stored in blocks of 64
// columns, [k / 64][n][64], each row 128 bytes with its 16-byte pieces swizzled as the tensor core reads them: a block of rows is
// copied to shared memory as it is.  Each 32 rows, the columns of the product, are in the order in which four threads read eight
// neighbouring columns each out of tensor memory (ptx::tmem_ld_32x256): column 8 q + 2 j + b is at 8 j + 2 q + b.
__global__ void __launch_bounds__(256) balance_prepare_kernel(const int64_t* counts, int nk, int padded, const Part* part, Prepared* head,
                                                              uint4* pieces) {
  pdl_launch_dependents();
  pdl_wait();
  // every warp adds the parts itself, in the same order
  const int lane = threadIdx.x & 31;
  static_assert(kParts == 64, "two parts a lane");
  double sum = part[lane].sum + part[lane + 32].sum;
  long long tokens = part[lane].tokens + part[lane + 32].tokens;
  long long top = part[lane].top > part[lane + 32].top ? part[lane].top : part[lane + 32].top;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    sum += __shfl_xor_sync(kFull, sum, d);
    tokens += __shfl_xor_sync(kFull, tokens, d);
    const long long o = __shfl_xor_sync(kFull, top, d);
    top = o > top ? o : top;
  }
  const double n = static_cast<double>(nk) * nk;
  const double mean = rint(sum / n);
  const double most = fmax(static_cast<double>(top) - mean, mean);
  int shift = 0;  // the largest value becomes at most 2^15, a float16
  if (most > 32768.0) shift = ilogb(most) - 14;
  const bool second = most > 2048.0;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    head->coef = sum > 0.0 && tokens > 0 ? n / (sum * static_cast<double>(tokens)) : 0.0;
    head->tokens = static_cast<double>(tokens);
    head->mean = static_cast<float>(mean);
    head->unscale = static_cast<float>(ldexp(1.0, shift - 15));
    head->second = second;
    head->finished = 0;
  }
  const long long taken = static_cast<long long>(mean);
  const float scale = ldexpf(1.f, -shift);
  const int64_t per = static_cast<int64_t>(padded) * padded / 8;  // 16-byte pieces of one matrix
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= 2 * per) return;
  const int h = at >= per;
  const int64_t local = at - h * per;
  int row, col;  // of the matrix; neighbouring threads read neighbouring counts
  if (h == 0) {
    row = static_cast<int>(local / (padded / 8));
    col = static_cast<int>(local % (padded / 8)) * 8;
  } else {
    row = static_cast<int>(local % padded);
    col = static_cast<int>(local / padded) * 8;
  }
  float hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = col + i;
    float v = 0.f, rest = 0.f;
    if (row < nk && k < nk) {
      const long long c = h == 0 ? counts[static_cast<int64_t>(row) * nk + k] : counts[static_cast<int64_t>(k) * nk + row];
      const float d = static_cast<float>(c - taken) * scale;  // 24 bits, of which the two pieces keep 22
      v = round_to<__half>(d);
      rest = d - v;
    }
    hi[i] = v;
    lo[i] = rest;
  }
  const int at_row = (row & ~31) | (((row >> 1) & 3) << 3) | (((row >> 3) & 3) << 1) | (row & 1);
  const int64_t slot = (static_cast<int64_t>(col / 64) * padded + at_row) * 8 + (((col % 64) / 8) ^ (at_row & 7));
  pieces[(2 * h) * per + slot] = pack16<__half>(hi);
  if (second) pieces[(2 * h + 1) * per + slot] = pack16<__half>(lo);
}

// ------------------------------------------------------------------------------------------------ product
// One CTA per SM works through items of 128 tokens x up to 256 columns of G_h (forward: h = 0; backward: both, next to each other
// so that the second finds the logits in the L2 cache).  Warp roles, each a loop over the items of the CTA:
//   0      copies the blocks of the counts' pieces into the ring
//   1      issues the products of a stage: three of 128 x columns x 64, into one of two accumulators
//   2..5   epilogue, a warp for 32 tokens: probabilities p_h from the logits, with the accumulator
//   6..13  make the stage's two pieces of p_(1-h), 128 x 64 each, from the logits
// Both kinds of readers of the logits have the next ones on the way while they work on the present ones.
//
// At 131072 tokens x 256 keys, bfloat16, it takes 50 us forward (134 MB of logits, 17 GF three times) and 93 us backward (268 MB, 34 GF
// three times), the tensor pipe busy 55 % of the time in both.  In a program that measured parts of it the backward took 98 us, without
// its epilogue's stores 82, without its epilogue 72, with nothing but the copies and the products 61: the warps that make and read
// probabilities hide behind the products in part only.  Measured and not kept: pairs of CTAs that hold the counts' pieces in shared
// memory for all items (forward and backward 102 us on average, this form 83 at the time: fewer stages are left for the
// probabilities), a second team of readers for every other item (backward 102 and 106 us with one and two chunks of logits on the
// way), logits fetched two stages ahead, streaming stores.  Small calls are a chain of latencies: 4096 x 128, 8 + 8 us.
// Every wait is bounded; one that runs out raises FMOE_STATUS_WAIT_TIMEOUT and the CTA drains and leaves.
constexpr int kMakers = 8, kReaders = 4;  // warps
constexpr int kProductThreads = (2 + kReaders + kMakers) * 32;
constexpr int kPieceBytes = kTileTokens * 128;  // one piece of the probabilities
constexpr int kMaxStages = 4;

// a stage of the ring and the parity of its use
struct RingCursor {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
};

struct ProductArgs {
  const void* logits;
  int64_t ts, hs, ntok;
  const float4* stats;
  float* token_s;  // [partial sums][T]
  const Prepared* head;
  const uint4* pieces;
  double* part;           // forward: [items][kReaders]
  float* loss;            // forward
  unsigned* finished;     // forward
  const float* upstream;  // backward
  void* dlogits;          // backward: [T, 2, nk]
  int32_t* status;
  int nk, padded, stages, items;
  int width, chunks;  // columns of an item, items side by side
  int partials;       // sums that make up s_t
};

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
               : "memory");
}

template <typename T, int W, bool BACKWARD>
__global__ void __launch_bounds__(kProductThreads, 1) balance_product_kernel(const ProductArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[3 * kMaxStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ double sums[kProductThreads / 32];
  __shared__ int last;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - raw);
  volatile int* abort_flag = &abort_word;
  const uint32_t b_bytes = static_cast<uint32_t>(a.width) * 128u;
  const uint32_t stage_bytes = 2u * kPieceBytes + 2u * b_bytes;
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto ready_bar = [&](int s) { return bar0 + s * 8; };                   // the probabilities' pieces
  auto full_bar = [&](int s) { return bar0 + (kMaxStages + s) * 8; };     // the counts' pieces
  auto empty_bar = [&](int s) { return bar0 + (2 * kMaxStages + s) * 8; };
  auto tfull_bar = [&](int i) { return bar0 + (3 * kMaxStages + i) * 8; };
  auto tempty_bar = [&](int i) { return bar0 + (3 * kMaxStages + 2 + i) * 8; };
  const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int blocks = a.padded / 64;

  if (warp == 0 && ptx::elect_one()) {
    for (int s = 0; s < a.stages; ++s) {
      ptx::mbar_init(ready_bar(s), kMakers);
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(tfull_bar(i), 1);
      ptx::mbar_init(tempty_bar(i), kReaders);
    }
    abort_word = 0;
    ptx::mbar_fence_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  pdl_wait();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const bool second = a.head->second != 0;
  struct Item {
    int64_t t0;
    int h, chunk, n0, columns;
  };
  auto item_of = [&](int i) {
    Item it;
    it.h = BACKWARD ? i & 1 : 0;
    const int j = BACKWARD ? i >> 1 : i;
    it.chunk = j % a.chunks;
    it.t0 = static_cast<int64_t>(j / a.chunks) * kTileTokens;
    it.n0 = it.chunk * a.width;
    it.columns = a.padded - it.n0 < a.width ? a.padded - it.n0 : a.width;
    return it;
  };

  // whole warps wait, and give up together
  auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(kFull, ptx::mbar_wait_bounded(bar, parity, abort_flag)) != 0; };

  if (warp == 0) {
    bool ok = true;
    uint32_t use = 0;  // stages used so far
    RingCursor ring;
    for (int i = blockIdx.x; i < a.items && ok; i += gridDim.x) {
      const Item it = item_of(i);
      const int64_t per = static_cast<int64_t>(a.padded) * a.padded / 8;
      const uint32_t bytes = static_cast<uint32_t>(it.columns) * 128u;
      for (int kb = 0; kb < blocks; ++kb, ++use, ring.next(a.stages)) {
        const int s = ring.stage;
        ok = wait(empty_bar(s), ring.parity ^ 1u);
        if (!ok) break;
        if (ptx::elect_one()) {
          const uint4* src = a.pieces + 2 * it.h * per + (static_cast<int64_t>(kb) * a.padded + it.n0) * 8;
          const uint32_t dst = base + s * stage_bytes + 2 * kPieceBytes;
          ptx::mbar_arrive_expect_tx(full_bar(s), second ? 2 * bytes : bytes);
          bulk_copy(dst, src, bytes, full_bar(s));
          if (second) bulk_copy(dst + b_bytes, src + per, bytes, full_bar(s));
        }
        __syncwarp();
      }
    }
    if (!ok) {  // let the copies already requested land before the CTA goes away (bounded)
      const uint32_t first = use > static_cast<uint32_t>(a.stages) ? use - a.stages : 0;
      for (uint32_t u = first; u < use; ++u) ptx::mbar_wait_drain(full_bar(u % a.stages), (u / a.stages) & 1u);
    }
  } else if (warp == 1) {
    bool ok = true;
    uint32_t round = 0;
    RingCursor ring;
    for (int i = blockIdx.x; i < a.items && ok; i += gridDim.x, ++round) {
      const Item it = item_of(i);
      const uint32_t acc = round & 1u;
      ok = wait(tempty_bar(acc), ((round >> 1) & 1u) ^ 1u);
      // float16 operands, float32 accumulator, 128 rows
      const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(it.columns >> 3) << 17) | (8u << 24);
      for (int kb = 0; kb < blocks && ok; ++kb, ring.next(a.stages)) {
        const int s = ring.stage;
        ok = wait(full_bar(s), ring.parity) && wait(ready_bar(s), ring.parity);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t st = base + s * stage_bytes;
        const uint64_t hi = ptx::umma_desc_kmajor_sw128(st), lo = ptx::umma_desc_kmajor_sw128(st + kPieceBytes);
        const uint64_t c_hi = ptx::umma_desc_kmajor_sw128(st + 2 * kPieceBytes);
        const uint64_t c_lo = ptx::umma_desc_kmajor_sw128(st + 2 * kPieceBytes + b_bytes);
        if (ptx::elect_one()) {
          const uint32_t d = tmem + acc * kChunk;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            ptx::umma_bf16_ss(d, hi + 2 * kk, c_hi + 2 * kk, idesc, (kb | kk) != 0 ? 1u : 0u);
            ptx::umma_bf16_ss(d, lo + 2 * kk, c_hi + 2 * kk, idesc, 1u);
            if (second) ptx::umma_bf16_ss(d, hi + 2 * kk, c_lo + 2 * kk, idesc, 1u);
          }
          ptx::umma_commit(empty_bar(s));
          if (kb == blocks - 1) ptx::umma_commit(tfull_bar(acc));
        }
        __syncwarp();
      }
    }
  } else if (warp < 2 + kReaders) {
    bool ok = true;
    uint32_t round = 0;
    const int quarter = warp & 3;  // the lanes of tensor memory that this warp may read
    // 32 rows x 32 columns at a time.  A thread has eight neighbouring columns, 8 (lane % 4) on, of the rows lane / 4 + 8 r in
    // tensor memory as in global memory: nothing changes hands, and an instruction touches eight lines, where a thread per row would
    // touch 32.
    constexpr int N = Vec16<T>::N, kLoads = 8 / N, kRows = 4;
    const int64_t stride = 8 * a.ts, out_stride = 16 * static_cast<int64_t>(a.nk);
    const float unscale = a.head->unscale;
    const float scale = BACKWARD ? static_cast<float>(a.head->coef * static_cast<double>(*a.upstream)) : 0.f;
    // what an item's tokens are read with; two chunks of logits are on the way, the next item's behind this one's
    struct Source {
      const T* rows;
      int left;       // columns from the thread's first to the row's end
      unsigned live;  // a bit a row
    };
    struct Stats {
      float top[kRows], inv[kRows], s[kRows];
    };
    auto stats_of = [&](int i, Stats& w) {
      const Item it = item_of(i);
      const int64_t first = it.t0 + quarter * 32 + (lane >> 2);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const bool in = i < a.items && first + 8 * r < a.ntok;
        w.top[r] = w.inv[r] = w.s[r] = 0.f;
        load_if(in, reinterpret_cast<const float*>(a.stats + first + 8 * r) + 2 * it.h, w.top[r], w.inv[r]);
        if (BACKWARD) load_if(in, a.token_s + first + 8 * r, w.s[r]);
      }
      if (BACKWARD && a.partials > 1) {  // calls of few tokens alone: no hurry
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          if (i < a.items && first + 8 * r < a.ntok)
            for (int c = 1; c < a.partials; ++c) w.s[r] += a.token_s[static_cast<int64_t>(c) * a.ntok + first + 8 * r];
      }
    };
    auto source_of = [&](int i, const Stats& w) {
      const Item it = item_of(i);
      Source f;
      const int ahead = it.n0 + (lane & 3) * 8;
      f.rows = static_cast<const T*>(a.logits) + (it.t0 + quarter * 32 + (lane >> 2)) * a.ts + it.h * a.hs + ahead;
      f.left = a.nk - ahead;
      f.live = 0;
#pragma unroll
      for (int r = 0; r < kRows; ++r) f.live |= w.inv[r] != 0.f ? 1u << r : 0u;
      return f;
    };
    auto fetch = [&](const Source& f, int r, int c, Piece<T, W> (&to)[kLoads]) {
      const T* at = f.rows + r * stride + c;
#pragma unroll
      for (int k = 0; k < kLoads; ++k) to[k].load(at + k * N, f.left - c - k * N, (f.live >> r & 1u) != 0);
    };
    Piece<T, W> q[2][kRows][kLoads];
    Stats stats;
    stats_of(blockIdx.x, stats);
    Source now = source_of(blockIdx.x, stats);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      fetch(now, r, 0, q[0][r]);
      fetch(now, r, 32, q[1][r]);
    }
    for (int i = blockIdx.x; i < a.items && ok; i += gridDim.x, ++round) {
      const Item it = item_of(i);
      const uint32_t acc = round & 1u;
      const int64_t first = it.t0 + quarter * 32 + (lane >> 2);
      T* outs = BACKWARD ? static_cast<T*>(a.dlogits) + (first * 2 + it.h) * a.nk + it.n0 + (lane & 3) * 8 : nullptr;
      const int left = now.left;
      // p (G - s) scale = e (acc weight + sum)
      RowExp exp_of[kRows];
      float weight[kRows], sum[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float inv = stats.inv[r];
        exp_of[r] = RowExp(stats.top[r]);
        weight[r] = inv * unscale;
        sum[r] = 0.f;
        if (BACKWARD) {
          weight[r] = inv != 0.f ? inv * scale : 0.f;
          sum[r] = -stats.s[r] * weight[r];
          weight[r] *= unscale;
        }
      }
      stats_of(i + gridDim.x, stats);
      ok = wait(tfull_bar(acc), (round >> 1) & 1u);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t taddr = tmem + acc * kChunk + (static_cast<uint32_t>(quarter * 32) << 16);
      for (int c = 0; c < it.columns; c += 64) {
        int to = c + 64;
        if (to == it.columns) {  // the next item's first two chunks
          to = 0;
          now = source_of(i + gridDim.x, stats);
        }
#pragma unroll
        for (int chunk = 0; chunk < 2; ++chunk)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t g[16];
            ptx::tmem_ld_32x256(taddr + (static_cast<uint32_t>(16 * half) << 16) + c + 32 * chunk, g);
            float p[2][8];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int r = 2 * half + u;
#pragma unroll
              for (int k = 0; k < kLoads; ++k) q[chunk][r][k].get(&p[u][k * N]);
              fetch(now, r, to + 32 * chunk, q[chunk][r]);
#pragma unroll
              for (int k = 0; k < 8; ++k) p[u][k] = exp_of[r](p[u][k]);
            }
            ptx::tmem_ld_wait(g);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int r = 2 * half + u;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float v = __uint_as_float(g[4 * (k >> 1) + 2 * u + (k & 1)]);
                if (BACKWARD) p[u][k] *= fmaf(v, weight[r], sum[r]);
                else sum[r] = fmaf(p[u][k], v, sum[r]);
              }
              if (BACKWARD && first + 8 * r < a.ntok) {
#pragma unroll
                for (int k = 0; k < kLoads; ++k)
                  store_values<T, W>(outs + r * out_stride + c + 32 * chunk + k * N, left - c - 32 * chunk - k * N, &p[u][k * N]);
              }
            }
          }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(tempty_bar(acc));
      if (!BACKWARD) {
        double all = 0.0;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          sum[r] += __shfl_xor_sync(kFull, sum[r], 1);
          sum[r] += __shfl_xor_sync(kFull, sum[r], 2);
          sum[r] *= weight[r];
          if ((lane & 3) == 0 && first + 8 * r < a.ntok) a.token_s[static_cast<int64_t>(it.chunk) * a.ntok + first + 8 * r] = sum[r];
          all += sum[r];
        }
        for (int d = 16; d > 2; d >>= 1) all += __shfl_xor_sync(kFull, all, d);
        if (lane == 0) a.part[static_cast<int64_t>(i) * kReaders + warp - 2] = all;
      }
    }
  } else {
    bool ok = true;
    RingCursor ring;
    // thread -> rows r0, r0 + 32, ... and a fixed 16-byte place (8 columns) of each 64-column block
    const int id = threadIdx.x - (2 + kReaders) * 32, piece = id & 7, r0 = id >> 3;
    const int place = piece ^ (r0 & 7);
    constexpr int kStep = kMakers * 4, kRows = kTileTokens / kStep;
    constexpr int N = Vec16<T>::N, kLoads = 8 / N;
    struct Rows {
      const T* first;  // the thread's first row, at its place of the first block
      float top[kRows], inv[kRows];
    };
    Rows now, next;
    Piece<T, W> x[kRows][kLoads];
    auto tokens = [&](int i, Rows& w) {
      const Item it = item_of(i);
      const int64_t t0 = it.t0 + r0;
      w.first = static_cast<const T*>(a.logits) + t0 * a.ts + (1 - it.h) * a.hs + piece * 8;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        w.top[r] = w.inv[r] = 0.f;
        load_if(i < a.items && t0 + r * kStep < a.ntok, reinterpret_cast<const float*>(a.stats + t0 + r * kStep) + 2 * (1 - it.h),
                w.top[r], w.inv[r]);
      }
    };
    const int64_t stride = kStep * a.ts;
    auto fetch = [&](int kb, const Rows& w) {
      const T* at = w.first + kb * 64;
      const int left = a.nk - kb * 64 - piece * 8;  // columns from here to the row's end
#pragma unroll
      for (int r = 0; r < kRows; ++r, at += stride)
#pragma unroll
        for (int k = 0; k < kLoads; ++k) x[r][k].load(at + k * N, left - k * N, w.inv[r] != 0.f);
    };
    tokens(blockIdx.x, now);
    fetch(0, now);
    for (int i = blockIdx.x; i < a.items && ok; i += gridDim.x) {
      tokens(i + gridDim.x, next);
      RowExp exp_of[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) exp_of[r] = RowExp(now.top[r]);
      for (int kb = 0; kb < blocks; ++kb, ring.next(a.stages)) {
        float p[kRows][8];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float weight = now.inv[r] * 32768.f;
#pragma unroll
          for (int k = 0; k < kLoads; ++k) x[r][k].get(&p[r][k * N]);
#pragma unroll
          for (int k = 0; k < 8; ++k) p[r][k] = exp_of[r](p[r][k]) * weight;
        }
        if (kb + 1 < blocks) fetch(kb + 1, now);
        else fetch(0, next);
        ok = wait(empty_bar(ring.stage), ring.parity ^ 1u);
        if (!ok) break;
        uint4* dst = reinterpret_cast<uint4*>(gen + ring.stage * stage_bytes) + r0 * 8 + place;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const __half2 h = __floats2half2_rn(p[r][2 * k], p[r][2 * k + 1]);
            const float2 f = __half22float2(h);
            const __half2 l = __floats2half2_rn(p[r][2 * k] - f.x, p[r][2 * k + 1] - f.y);
            hi[k] = *reinterpret_cast<const uint32_t*>(&h);
            lo[k] = *reinterpret_cast<const uint32_t*>(&l);
          }
          dst[r * kStep * 8] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          dst[r * kStep * 8 + kPieceBytes / 16] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        ptx::fence_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ready_bar(ring.stage));
      }
      now = next;
    }
  }

  __syncwarp();
  ptx::tc_fence_before();
  __threadfence();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && abort_word != 0 && a.status != nullptr) atomicOr(a.status, FMOE_STATUS_WAIT_TIMEOUT);
  if (BACKWARD) return;
  // the CTA that ends last adds the items' sums, in their order
  if (threadIdx.x == 0) last = atomicAdd(a.finished, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (int i = threadIdx.x; i < kReaders * a.items; i += kProductThreads) v += static_cast<const volatile double*>(a.part)[i];
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  if (lane == 0) sums[warp] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kProductThreads / 32; ++i) v += sums[i];
    *a.loss = static_cast<float>(a.head->coef * (v + static_cast<double>(a.head->mean) * a.head->tokens));
  }
}

size_t matrix_bytes(int nk) { return static_cast<size_t>(padded_keys(nk)) * padded_keys(nk) * 2; }
int64_t token_tiles(int64_t T) { return (T + kTileTokens - 1) / kTileTokens; }

// bytes of the loads that rows of these sizes and addresses allow: 16, 8, 4 or, for 16-bit types, 2
template <typename T> int load_width(const ProductArgs& a, const void* out) {
  const uintptr_t bits = (static_cast<uintptr_t>(a.nk) | static_cast<uintptr_t>(a.ts) | static_cast<uintptr_t>(a.hs)) * sizeof(T) |
                         reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(out);
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

// Columns of an item: as few as 64 while the items still fit the SMs side by side, since an item's latency is what small calls
// cost; each item makes the probabilities of its tokens again.  Forward and backward, bfloat16, us, with this width and with 256
// columns: 128 tokens x 128 keys 7.5 + 6.7 and 8.6 + 7.5, 128 x 512 12.0 + 11.0 and 15.6 + 14.6, 2368 x 256 9.6 + 9.4 and 11.8 +
// 11.4, 512 x 1024 18.6 + 18.4 and 22.4 + 21.5; where only the forward's items fit, 4096 x 256, 10.4 + 10.2 and 11.9 + 11.6.
// The number of SMs is that of a B200 whatever the device has: what the forward leaves of s_t depends on the width.
constexpr int kSideBySide = 148;
int item_width(int64_t T, int nk, int halves) {
  const int padded = padded_keys(nk);
  int width = padded < kChunk ? padded : kChunk;
  for (int w = 64; w < width; w *= 2)
    if (token_tiles(T) * ((padded + w - 1) / w) * halves <= kSideBySide) return w;
  return width;
}
int chunks_of(int nk, int width) { return (padded_keys(nk) + width - 1) / width; }
// what the forward leaves of s_t: a sum for each item's columns
int partial_sums(int64_t T, int nk) { return chunks_of(nk, item_width(T, nk, 1)); }

template <typename T, bool BACKWARD> int launch_product(ProductArgs a, cudaStream_t stream) {
  const int bytes = load_width<T>(a, a.dlogits);
  a.width = item_width(a.ntok, a.nk, BACKWARD ? 2 : 1);
  a.chunks = chunks_of(a.nk, a.width);
  a.partials = partial_sums(a.ntok, a.nk);
  const int stage = 2 * kPieceBytes + 2 * a.width * 128;
  a.stages = 224 * 1024 / stage;
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  const int smem = a.stages * stage + 1024;
  const int64_t items = token_tiles(a.ntok) * a.chunks * (BACKWARD ? 2 : 1);
  if (items > 0x7FFFFFFF / kReaders - 65536) return FMOE_ERR_UNSUPPORTED;
  a.items = static_cast<int>(items);
  const int grid = a.items < device_sm_count() ? a.items : device_sm_count();
  auto run = [&](auto* kern) -> int {
    FMOE_CUDA_TRY(allow_smem(kern, smem));
    FMOE_CUDA_TRY(launch_pdl(BACKWARD ? 0 : 32, kern, dim3(grid), dim3(kProductThreads), smem, stream, 1, a));
    return FMOE_OK;
  };
  if (bytes == 16) return run(balance_product_kernel<T, 16, BACKWARD>);
  if (bytes == 8) return run(balance_product_kernel<T, 8, BACKWARD>);
  if constexpr (sizeof(T) == 2)
    if (bytes == 2) return run(balance_product_kernel<T, 2, BACKWARD>);
  return run(balance_product_kernel<T, 4, BACKWARD>);
}

template <typename T>
int forward_typed(ProductArgs a, const uint8_t* mask, const int64_t* counts, Prepared* head, float4* stats, Part* part, cudaStream_t stream) {
  const int64_t want = (a.ntok + 31) / 32, cap = static_cast<int64_t>(device_sm_count()) * 16;
  const int64_t grid = want > cap ? cap : want < kParts ? kParts : want;
  constexpr int kLine = 8 * Vec16<T>::N;  // columns of eight lanes' pieces
  const int bytes = load_width<T>(a, nullptr);
  auto* kern = a.nk <= kLine ? balance_stats_kernel<T, 16, 1> : a.nk <= 2 * kLine ? balance_stats_kernel<T, 16, 2> : balance_stats_kernel<T, 16, 4>;
  if (bytes == 8) kern = a.nk <= 2 * kLine ? balance_stats_kernel<T, 8, 2> : balance_stats_kernel<T, 8, 4>;
  if (bytes == 4) kern = a.nk <= 2 * kLine ? balance_stats_kernel<T, 4, 2> : balance_stats_kernel<T, 4, 4>;
  if constexpr (sizeof(T) == 2)
    if (bytes == 2) kern = a.nk <= 2 * kLine ? balance_stats_kernel<T, 2, 2> : balance_stats_kernel<T, 2, 4>;
  kern<<<static_cast<unsigned>(grid), 256, 0, stream>>>(static_cast<const T*>(a.logits), a.ts, a.hs, mask, a.ntok, a.nk, stats, counts, part);
  FMOE_LAUNCH_CHECK();
  const int64_t pieces = static_cast<int64_t>(a.padded) * a.padded / 4;
  FMOE_CUDA_TRY(launch_pdl(32, balance_prepare_kernel, dim3(static_cast<unsigned>((pieces + 255) / 256)), dim3(256), 0, stream, 1, counts,
                           a.nk, a.padded, part, head, const_cast<uint4*>(a.pieces)));
  return launch_product<T, false>(a, stream);
}

}  // namespace

namespace {
// Clusters of the histogram that the device runs at once (its GPCs have SMs left over: 15 of 18 on this one); cached per device.
int histogram_clusters() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (cache[dev] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(device_sm_count() / kHistCtas * kHistCtas);
    cfg.blockDim = dim3(kHistThreads);
    cfg.dynamicSmemBytes = kHistExperts * 2;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = kHistCtas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (allow_smem(expert_histogram_kernel, kHistExperts * 2) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, expert_histogram_kernel, &cfg) != cudaSuccess)
      return 0;
    cache[dev] = n;
  }
  return cache[dev];
}

template <typename... KArgs, typename... Args>
int launch_cluster(void (*kern)(KArgs...), int ctas, int threads, int width, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = width;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FMOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...));
  return FMOE_OK;
}
}  // namespace

int launch_expert_counts(const int64_t* indices, const uint8_t* mask, int64_t T, int k, int64_t N, int64_t* counts, int32_t* status,
                         cudaStream_t stream) {
  if (T < 0 || k < 0 || N < 0) return FMOE_ERR_BAD_ARG;
  if (N > 0 && counts == nullptr) return FMOE_ERR_BAD_ARG;
  if (T == 0 || k == 0) {
    if (N > 0) FMOE_CUDA_TRY(cudaMemsetAsync(counts, 0, static_cast<size_t>(N) * 8, stream));
    return FMOE_OK;
  }
  if (indices == nullptr) return FMOE_ERR_BAD_ARG;
  unsigned long long* out = reinterpret_cast<unsigned long long*>(counts);
  const int64_t pairs = T * k;
  if (pairs <= 32768 && N <= 131072) {
    // the widest cluster that every device takes; in a graph, us, with 2, 4 and 8 CTAs: 64 selections of 256 experts 2.8, 2.7, 2.7; 2048 of
    // 4096 4.1, 3.6, 3.6; 4096 of 16384 6.0, 4.6, 4.1; 2048 of 65536 8.3, 5.9, 4.9; 32768 of 131072 24, 14.5, 9.3
    constexpr int kCtas = 8;
    return launch_cluster(expert_counts_kernel<true>, kCtas, kCountThreads, kCtas, 0, stream, indices, mask, pairs, k, N, out, status);
  }
  FMOE_CUDA_TRY(cudaMemsetAsync(counts, 0, static_cast<size_t>(N) * 8, stream));
  // measured, whole call, Zipf exponent 0.7, tables and histogram: 16384 experts, 262144 selections 10.4 and 12.1 us, 1048576 17.8 and
  // 13.6; 65536 experts, 1048576 selections 17.7 and 17.7, 4194304 32.1 and 22.0; 256 experts, 524288 selections 13.8 and 9.9
  const int clusters = pairs >= (1 << 19) && N <= kHistExperts && pairs >= 32 * N ? histogram_clusters() : 0;
  if (clusters > 0) {
    const int smem = static_cast<int>((N + 7) / 8) * 16;
    return launch_cluster(expert_histogram_kernel, clusters * kHistCtas, kHistThreads, kHistCtas, smem, stream, indices, mask, pairs, k,
                          static_cast<int>(N), out, status);
  }
  const int64_t want = (pairs + 4 * kCountThreads - 1) / (4 * kCountThreads), cap = device_sm_count();
  expert_counts_kernel<false><<<static_cast<unsigned>(want < cap ? want : cap), kCountThreads, 0, stream>>>(indices, mask, pairs, k, N, out, status);
  FMOE_LAUNCH_CHECK();
  return FMOE_OK;
}

size_t balance_prepared_bytes(int nk) { return nk <= 0 || nk > kMaxKeys ? 0 : kHeadBytes + 4 * matrix_bytes(nk); }
size_t balance_stats_floats(int64_t T, int nk) { return T <= 0 || nk <= 0 || nk > kMaxKeys ? 0 : static_cast<size_t>(T) * (4 + partial_sums(T, nk)); }
size_t balance_workspace_bytes(int64_t T, int nk) {
  if (T < 0 || nk <= 0 || nk > kMaxKeys) return 0;
  return kParts * sizeof(Part) + static_cast<size_t>(token_tiles(T)) * partial_sums(T, nk) * kReaders * sizeof(double);
}

int launch_balance_forward(const void* logits, int64_t ts, int64_t hs, int dtype, const int64_t* counts, const uint8_t* mask, int64_t T,
                           int nk, float* loss, float* stats, void* prepared, size_t prepared_bytes, void* ws, size_t ws_bytes,
                           int32_t* status, cudaStream_t stream) {
  if (T < 0 || nk <= 0 || counts == nullptr || loss == nullptr) return FMOE_ERR_BAD_ARG;
  if (nk > kMaxKeys) return FMOE_ERR_UNSUPPORTED;
  if (T == 0) {
    FMOE_CUDA_TRY(cudaMemsetAsync(loss, 0, sizeof(float), stream));
    return FMOE_OK;
  }
  if (logits == nullptr || stats == nullptr) return FMOE_ERR_BAD_ARG;
  if (prepared == nullptr || prepared_bytes < balance_prepared_bytes(nk) || ws == nullptr || ws_bytes < balance_workspace_bytes(T, nk)) return FMOE_ERR_WORKSPACE;
  if (!aligned16(stats) || !aligned16(prepared) || !aligned16(ws)) return FMOE_ERR_ALIGNMENT;
  Prepared* head = static_cast<Prepared*>(prepared);
  Part* part = static_cast<Part*>(ws);
  ProductArgs a = {};
  a.logits = logits;
  a.ts = ts;
  a.hs = hs;
  a.ntok = T;
  a.stats = reinterpret_cast<const float4*>(stats);
  a.token_s = stats + 4 * T;
  a.head = head;
  a.pieces = reinterpret_cast<const uint4*>(static_cast<char*>(prepared) + kHeadBytes);
  a.part = reinterpret_cast<double*>(part + kParts);
  a.loss = loss;
  a.finished = &head->finished;
  a.status = status;
  a.nk = nk;
  a.padded = padded_keys(nk);
  float4* st = reinterpret_cast<float4*>(stats);
  switch (dtype) {
    case FMOE_DTYPE_F32: return forward_typed<float>(a, mask, counts, head, st, part, stream);
    case FMOE_DTYPE_BF16: return forward_typed<__nv_bfloat16>(a, mask, counts, head, st, part, stream);
    case FMOE_DTYPE_F16: return forward_typed<__half>(a, mask, counts, head, st, part, stream);
    default: return FMOE_ERR_BAD_ARG;
  }
}

int launch_balance_backward(const void* logits, int64_t ts, int64_t hs, int dtype, int64_t T, int nk, const float* stats,
                            const void* prepared, size_t prepared_bytes, const float* upstream, void* dlogits, int32_t* status,
                            cudaStream_t stream) {
  if (T < 0 || nk <= 0) return FMOE_ERR_BAD_ARG;
  if (nk > kMaxKeys) return FMOE_ERR_UNSUPPORTED;
  if (T == 0) return FMOE_OK;
  if (logits == nullptr || stats == nullptr || upstream == nullptr || dlogits == nullptr) return FMOE_ERR_BAD_ARG;
  if (prepared == nullptr || prepared_bytes < balance_prepared_bytes(nk)) return FMOE_ERR_WORKSPACE;
  if (!aligned16(stats) || !aligned16(prepared)) return FMOE_ERR_ALIGNMENT;
  ProductArgs a = {};
  a.logits = logits;
  a.ts = ts;
  a.hs = hs;
  a.ntok = T;
  a.stats = reinterpret_cast<const float4*>(stats);
  a.token_s = const_cast<float*>(stats) + 4 * T;
  a.head = static_cast<const Prepared*>(prepared);
  a.pieces = reinterpret_cast<const uint4*>(static_cast<const char*>(prepared) + kHeadBytes);
  a.upstream = upstream;
  a.dlogits = dlogits;
  a.status = status;
  a.nk = nk;
  a.padded = padded_keys(nk);
  switch (dtype) {
    case FMOE_DTYPE_F32: return launch_product<float, true>(a, stream);
    case FMOE_DTYPE_BF16: return launch_product<__nv_bfloat16, true>(a, stream);
    case FMOE_DTYPE_F16: return launch_product<__half, true>(a, stream);
    default: return FMOE_ERR_BAD_ARG;
  }
}

}  // namespace fmoe
