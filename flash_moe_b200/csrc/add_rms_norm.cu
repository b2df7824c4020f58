// The pre-norm of a residual stack: s = T(x + r), n = s * rsqrt(mean(s^2) + eps) * w, with its gradient, and with an output in
// 8 bits.  No counterpart in the reference, which leaves normalisation and skip connection to its caller
// (flash_moe/modules/flash_moe.py:55-59).
//
// Memory-bound throughout: the forward moves 4 rows' worth of values per row (x, r in; s, n out), the backward 4 (dn, ds, s in;
// dx out).  32768 x 2048 bfloat16 take 80 us forward (6.7 TB/s, where a copy reaches 6.5) and 89 + 4 backward (6.0 TB/s), the
// 8-bit form 42 us at 16384 x 2048 with blocks of 128 columns (5.6 TB/s; 71 % of the issue slots).  A row stays in the registers
// of its group of warps between the sum of squares and the scaling, so each value is moved once.  Everything inside is float32; s
// is rounded to T before it is normalised, so that n belongs to the s that is stored and the backward finds the same s; n, dx and
// dw are rounded once.
#include <cuda_fp8.h>

#include <cstring>
#include <initializer_list>
#include <numeric>

#include "common.cuh"

namespace fmoe {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr float kE4m3Max = 448.f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: a zero group keeps a scale that can be divided by

// VEC values of T as they are loaded: 16 bytes, or one value where an array does not start at a multiple of 16 bytes
template <typename T, int VEC> struct Piece {
  uint4 q;
  __device__ __forceinline__ void load(const T* p) { q = ld16(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = q; }
  __device__ __forceinline__ void zero() { q = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&f)[VEC]) const { unpack16<T>(q, f); }
  __device__ __forceinline__ void set(const float (&f)[VEC]) { q = pack16<T>(f); }
};
template <typename T> struct Piece<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void zero() { v = from_f32<T>(0.f); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f32<T>(v); }
  __device__ __forceinline__ void set(const float (&f)[1]) { v = from_f32<T>(f[0]); }
};

// A group of WPG warps handles a batch of up to R rows at a time; thread i of a group holds the pieces i, i + 32 WPG, ... (C of
// them) of each row.
template <int WPG> struct Group {
  static constexpr int kThreads = 32 * WPG;
  static constexpr int kCta = WPG < 8 ? 256 : kThreads;
  static constexpr int kPerCta = kCta / kThreads;
};
template <int WPG> __device__ __forceinline__ void group_barrier() {
  if (WPG == 1) __syncwarp();
  else if (Group<WPG>::kPerCta == 1) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(static_cast<int>(threadIdx.x) / Group<WPG>::kThreads + 1), "n"(Group<WPG>::kThreads) : "memory");
}

// Values lo to hi - 1 of a piece, those that lie in its row.  Only a row's ends come here.
template <typename T, int VEC> __device__ __forceinline__ void load_part(Piece<T, VEC>& piece, const T* at, int lo, int hi) {
  T v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = i >= lo && i < hi ? at[i] : from_f32<T>(0.f);
  memcpy(&piece, v, sizeof(v));
}
// LOOP: unrolled, the stores take registers that a kernel with little else to hold gives to another CTA (32768 rows of 1001
// bfloat16: 60 us instead of 90); the 8-bit kernels are faster with them unrolled (106 us instead of 114).
template <bool LOOP, typename T, int VEC> __device__ __forceinline__ void store_part(const Piece<T, VEC>& piece, T* at, int lo, int hi) {
  if constexpr (VEC == 1) {
    if (lo < hi) piece.store(at);
  } else if constexpr (!LOOP) {
    T v[VEC];
    memcpy(v, &piece, sizeof(v));
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= lo && i < hi) at[i] = v[i];
  } else {
    constexpr int kBits = 8 * sizeof(T), kWord = 4 / sizeof(T);
#pragma unroll 1
    for (int i = lo; i < hi; ++i) {
      const int word = i / kWord;
      const uint32_t w = word == 0 ? piece.q.x : word == 1 ? piece.q.y : word == 2 ? piece.q.z : piece.q.w;
      const std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> bits = w >> (i % kWord * kBits % 32);
      memcpy(at + i, &bits, sizeof(T));
    }
  }
}
// zero outside [lo, hi)
template <typename T, int VEC> __device__ __forceinline__ void keep_part(Piece<T, VEC>& piece, int lo, int hi) {
  if constexpr (VEC > 1) {
    uint32_t w[4] = {piece.q.x, piece.q.y, piece.q.z, piece.q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (sizeof(T) == 4) {
        w[j] = j >= lo && j < hi ? w[j] : 0u;
      } else {
        const uint32_t low = 2 * j >= lo && 2 * j < hi ? 0x0000FFFFu : 0u, high = 2 * j + 1 >= lo && 2 * j + 1 < hi ? 0xFFFF0000u : 0u;
        w[j] &= low | high;
      }
    }
    piece.q = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// How a group walks over rows and a thread over a row's pieces.  Rows whose length is no multiple of a piece start at any value of
// one, but rows r, r + VEC, r + 2 VEC, ... all at the same: with SHIFT a group takes the rows of one remainder, and its pieces are
// the aligned ones of memory, of which a row's first and last lie in it in part.  A thread's columns, its weights and its part of
// dweight are the same for every row then.  Pieces are read whole, with the neighbours' values, which `mask` takes out where they
// are used (a wait inside the read would stop the reads behind it); only the last row's end is read value by value, so rows are not
// shorter than what a piece may reach into the next.
template <int VEC, int WPG, bool SHIFT> struct Walk {
  int64_t row, step, rows;
  int H, shift, pieces;
  __device__ __forceinline__ Walk(int64_t rows_, int H_, int batch) : rows(rows_), H(H_) {
    const int64_t group = static_cast<int64_t>(blockIdx.x) * (Group<WPG>::kPerCta) + threadIdx.x / Group<WPG>::kThreads;
    const int64_t groups = static_cast<int64_t>(gridDim.x) * Group<WPG>::kPerCta;
    if (SHIFT) {
      row = group;  // groups is a multiple of VEC: group + j * groups keeps the remainder
      step = groups;
      shift = static_cast<int>((group % VEC) * H % VEC);
    } else {
      row = group * batch;
      step = groups * batch;
      shift = 0;
    }
    pieces = (H + shift + VEC - 1) / VEC;
  }
  __device__ __forceinline__ int col(int piece) const { return piece * VEC - shift; }
  __device__ __forceinline__ bool whole(int piece) const {
    return !SHIFT ? piece < pieces : col(piece) >= 0 && col(piece) + VEC <= H;
  }
  // the part of a piece that lies in the row
  __device__ __forceinline__ int lo(int piece) const { return col(piece) < 0 ? -col(piece) : 0; }
  __device__ __forceinline__ int hi(int piece) const { return H - col(piece) < VEC ? H - col(piece) : VEC; }
  // the piece of row r of an array
  template <typename T> __device__ __forceinline__ void load(Piece<T, VEC>& p, const T* base, int64_t r, int piece) const {
    if (piece >= pieces) return;
    const T* at = base + r * H + col(piece);
    if (!SHIFT || r + 1 < rows || col(piece) + VEC <= H) p.load(at);
    else load_part<T, VEC>(p, at, lo(piece), hi(piece));
  }
  template <typename T> __device__ __forceinline__ void mask(Piece<T, VEC>& p, int piece) const {
    if (SHIFT && piece < pieces && !whole(piece)) keep_part<T, VEC>(p, lo(piece), hi(piece));
  }
  template <bool LOOP = true, typename T> __device__ __forceinline__ void store(const Piece<T, VEC>& p, T* row, int piece) const {
    if (whole(piece)) p.store(row + col(piece));
    else if (SHIFT && piece < pieces) store_part<LOOP, T, VEC>(p, row + col(piece), lo(piece), hi(piece));
  }
  // weights are not aligned like the rows
  template <typename T> __device__ __forceinline__ void weights(Piece<T, VEC>& p, const T* w, int piece) const {
    p.zero();
    if (w == nullptr || piece >= pieces) return;
    if (SHIFT) load_part<T, VEC>(p, w + col(piece), lo(piece), hi(piece));
    else p.load(w + col(piece));
  }
};

struct SumOp {
  static __device__ __forceinline__ float zero() { return 0.f; }
  static __device__ __forceinline__ float join(float a, float b) { return a + b; }
};
// of absolute values, by their bits: unlike fmaxf this keeps a NaN
struct MaxOp {
  static __device__ __forceinline__ float zero() { return 0.f; }
  static __device__ __forceinline__ float join(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
  }
};
template <typename Op> __device__ __forceinline__ float warp_join(float v, int lanes = 32) {
  for (int d = lanes >> 1; d > 0; d >>= 1) v = Op::join(v, __shfl_xor_sync(kFull, v, d));
  return v;
}

// Every thread of the group gets the join of v[i] over the group, in a fixed order.  `slot` [N][WPG]; the caller alternates
// between two of them, so one barrier is enough: a slot is written again two calls later, behind the barrier of the next call.
template <typename Op, int WPG, int N> __device__ __forceinline__ void group_join(float (&v)[N], float* slot) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Op::join(v[i], __shfl_xor_sync(kFull, v[i], d));
  if (WPG == 1) return;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WPG;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slot[i * WPG + warp] = v[i];
  }
  group_barrier<WPG>();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (WPG <= 8) {
      float a = slot[i * WPG];
#pragma unroll
      for (int j = 1; j < WPG; ++j) a = Op::join(a, slot[i * WPG + j]);
      v[i] = a;
    } else {
      v[i] = warp_join<Op>(lane < WPG ? slot[i * WPG + lane] : Op::zero());
    }
  }
}

enum { kNorm = 0, kFp8Row = 1, kFp8Block = 2 };

template <typename T> struct NormArgs {
  const T* x;
  const T* residual;  // nullable: x is normalised, summed is not written
  const T* weight;    // nullable
  T* summed;
  T* normed;
  __nv_fp8_storage_t* q;
  float* scales;
  int64_t rows;
  int H, batch;
  int group_shift, groups;  // kFp8Block: columns of a block, a power of two
  float eps;
};

template <typename T, int VEC, int WPG, int C, int R, bool SHIFT, int MODE>
__global__ void __launch_bounds__(Group<WPG>::kCta, Group<WPG>::kCta > 256 ? 1 : C > 2 ? 2 : 4)
add_rms_norm_kernel(const NormArgs<T> a) {
  constexpr int NT = Group<WPG>::kThreads;
  constexpr bool kTable = MODE == kFp8Block && (VEC == 1 || SHIFT);  // a piece may lie in two blocks, or a block in many warps
  const int g = threadIdx.x / NT, tid = threadIdx.x % NT;
  __shared__ float slots[Group<WPG>::kPerCta][3][R * WPG];
  extern __shared__ uint32_t block_max[];  // kTable: [kPerCta][groups]
  const Walk<VEC, WPG, SHIFT> walk(a.rows, a.H, a.batch);
  Piece<T, VEC> w[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    walk.weights(w[c], a.weight, c * NT + tid);
  }
  int turn = 0;
  for (int64_t r0 = walk.row; r0 < a.rows; r0 += walk.step, turn ^= 1) {
    Piece<T, VEC> s[R][C];
    float sq[R];
    auto row_live = [&](int r) { return R == 1 || (r < a.batch && r0 + r < a.rows); };
    {
      Piece<T, VEC> res[R][C];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          s[r][c].zero();
          res[r][c].zero();
          if (row_live(r)) {
            walk.load(s[r][c], a.x, r0 + r, c * NT + tid);
            if (a.residual != nullptr) walk.load(res[r][c], a.residual, r0 + r, c * NT + tid);
          }
        }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sq[r] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float f[VEC], v[VEC];
          s[r][c].get(f);
          if (a.residual != nullptr) {
            res[r][c].get(v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] += v[i];
            s[r][c].set(f);
          }
          walk.mask(s[r][c], c * NT + tid);
          s[r][c].get(f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) sq[r] = fmaf(f[i], f[i], sq[r]);
        }
      }
    }
    group_join<SumOp, WPG, R>(sq, slots[g][turn]);
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) rstd[r] = rsqrtf(sq[r] / static_cast<float>(a.H) + a.eps);
    auto value = [&](int r, int c, float (&y)[VEC]) {
      float wf[VEC];
      s[r][c].get(y);
      w[c].get(wf);
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] = y[i] * rstd[r] * (a.weight != nullptr ? wf[i] : 1.f);
    };
    auto magnitude = [&](int r, int c) {  // the largest |y| of a piece; what lies outside the row is 0 unless rstd is not finite
      float y[VEC], m = 0.f;
      if (c * NT + tid >= walk.pieces) return m;
      value(r, c, y);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int col = walk.col(c * NT + tid) + i;
        if (!SHIFT || (col >= 0 && col < a.H)) m = MaxOp::join(m, fabsf(y[i]));
      }
      return m;
    };
    if (MODE == kNorm) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (!row_live(r)) continue;
          if (a.residual != nullptr) walk.store(s[r][c], a.summed + (r0 + r) * a.H, c * NT + tid);
          float y[VEC];
          value(r, c, y);
          Piece<T, VEC> out;
          out.set(y);
          walk.store(out, a.normed + (r0 + r) * a.H, c * NT + tid);
        }
      continue;
    }
    // 8 bits: scale = max |y| / 448 over the row or the block of columns, q = e4m3(y / scale), both by products: the scale is within
    // 2^-23, the quotient within 2^-21, which decides only where it is that near to the middle between two values of 8 bits.
    // Rounding as divisions do costs 8 to 18 %: 41.3 -> 47.2 us for rows and 44.9 -> 49.4 for blocks of 128 at 16384 x 2048 bfloat16, 105 ->
    // 123 at 32768 x 1001, with both ends of an interval around the quotient rounded and a division only where they differ; a division
    // a value 53, 57 and 150.  The error against y stays what 8 bits make of it.
    float top[R];
    if (MODE == kFp8Row) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        top[r] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) top[r] = MaxOp::join(top[r], magnitude(r, c));
      }
      group_join<MaxOp, WPG, R>(top, slots[g][2]);
    }
    float most[R][C];
    if (kTable) {
      static_assert(!kTable || R == 1, "one table a group");
      uint32_t* m = block_max + g * a.groups;
      for (int i = tid; i < a.groups; i += NT) m[i] = 0;
      group_barrier<WPG>();
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float y[VEC];
        const int col = walk.col(c * NT + tid);
        if (c * NT + tid >= walk.pieces) continue;
        value(0, c, y);
        // a piece has values of one block, or of two
        const int block = (col > 0 ? col : 0) >> a.group_shift, next = (block + 1) << a.group_shift;
        float here = 0.f, there = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (col + i >= 0 && col + i < a.H) {
            if (col + i < next) here = MaxOp::join(here, fabsf(y[i]));
            else there = MaxOp::join(there, fabsf(y[i]));
          }
        atomicMax(m + block, __float_as_uint(here));
        if (VEC > 1 && next < a.H && col + VEC > next) atomicMax(m + block + 1, __float_as_uint(there));
      }
      group_barrier<WPG>();
    } else if (MODE == kFp8Block) {
      // a block is 4 to 32 neighbouring lanes
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) most[r][c] = magnitude(r, c);
      for (int d = (1 << a.group_shift) / (2 * VEC); d > 0; d >>= 1)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int c = 0; c < C; ++c) most[r][c] = MaxOp::join(most[r][c], __shfl_xor_sync(kFull, most[r][c], d));
    }
    auto scale_of = [&](float m) {
      m *= 1.f / kE4m3Max;
      return m < kMinScale ? kMinScale : m;  // a NaN stays
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int p = c * NT + tid, col = walk.col(p);
        if (!row_live(r) || p >= walk.pieces) continue;
        const int64_t row = r0 + r;
        const int block = (col > 0 ? col : 0) >> a.group_shift, next = (block + 1) << a.group_shift;
        float m0, m1 = 0.f;
        if (MODE == kFp8Row) m0 = top[r];
        else if (kTable) {
          m0 = __uint_as_float(block_max[g * a.groups + block]);
          if (VEC > 1 && next < a.H) m1 = __uint_as_float(block_max[g * a.groups + block + 1]);
        } else {
          m0 = most[r][c];
        }
        const float scale = scale_of(m0);
        // __fdividef: 2^-126 <= scale < 2^120, or infinite, where it gives 0
        const float inv = __fdividef(1.f, scale), inv1 = kTable && VEC > 1 ? __fdividef(1.f, scale_of(m1)) : inv;
        if (MODE == kFp8Row) {
          if (p == 0) a.scales[row] = scale;
        } else if (!kTable && (col & ((1 << a.group_shift) - 1)) == 0) {
          a.scales[row * a.groups + block] = scale;
        }
        if (a.residual != nullptr) walk.template store<false>(s[r][c], a.summed + row * a.H, p);
        float y[VEC];
        value(r, c, y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[i] *= !kTable || col + i < next ? inv : inv1;
        __nv_fp8_storage_t* q = a.q + row * a.H;
        if (VEC > 1 && walk.whole(p)) {
          uint32_t b[VEC > 1 ? VEC / 2 : 1];
#pragma unroll
          for (int i = 0; i + 1 < VEC; i += 2)
            b[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(y[i], y[i + 1]), __NV_SATFINITE, __NV_E4M3);
          if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q + col) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
          else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(q + col) = b[0] | (b[1] << 16);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (i >= walk.lo(p) && i < walk.hi(p)) q[col + i] = __nv_cvt_float_to_fp8(y[i], __NV_SATFINITE, __NV_E4M3);
        }
      }
    if (kTable) {
      for (int i = tid; i < a.groups; i += NT) a.scales[r0 * a.groups + i] = scale_of(__uint_as_float(block_max[g * a.groups + i]));
      group_barrier<WPG>();  // the table is cleared for the next row
    }
    if (MODE == kFp8Row && WPG > 1) group_barrier<WPG>();  // slots[g][2] is written again
  }
}

// dn, ds -> dx = ds + rstd (g - s rstd^2 mean(g s)), g = dn w;  part[group] = sum over its rows of dn s rstd.
// rstd comes from s once more: the second sum travels with the first, and the forward keeps nothing but s.
template <typename T> struct NormBackwardArgs {
  const T* dnormed;
  const T* dsummed;  // nullable
  const T* summed;
  const T* weight;  // nullable
  T* dx;
  float* part;  // nullable; [groups of the grid][H]
  int64_t rows;
  int H, batch;
  float eps;
};

template <typename T, int VEC, int WPG, int C, int R, bool SHIFT>
__global__ void __launch_bounds__(Group<WPG>::kCta, Group<WPG>::kCta > 256 || C > 2 ? 1 : 2) add_rms_norm_backward_kernel(const NormBackwardArgs<T> a) {
  constexpr int NT = Group<WPG>::kThreads;
  const int g = threadIdx.x / NT, tid = threadIdx.x % NT;
  __shared__ float slots[Group<WPG>::kPerCta][2][2 * R * WPG];
  const Walk<VEC, WPG, SHIFT> walk(a.rows, a.H, a.batch);
  Piece<T, VEC> w[C];
  float dw[C][VEC];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    walk.weights(w[c], a.weight, c * NT + tid);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[c][i] = 0.f;
  }
  int turn = 0;
  struct Batch {
    Piece<T, VEC> s[R][C], dn[R][C], ds[R][C];
  };
  auto fetch = [&](int64_t r0, Batch& b) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int p = c * NT + tid;
        b.s[r][c].zero();
        b.dn[r][c].zero();
        b.ds[r][c].zero();
        if (R == 1 || (r < a.batch && r0 + r < a.rows)) {
          walk.load(b.s[r][c], a.summed, r0 + r, p);
          walk.load(b.dn[r][c], a.dnormed, r0 + r, p);
          if (a.dsummed != nullptr) walk.load(b.ds[r][c], a.dsummed, r0 + r, p);
        }
      }
  };
  // the next batch is on the way while this one is worked on, where the registers of a CTA hold both
  constexpr bool kAhead = WPG * C * VEC <= 256;
  Batch now, next;
  if (walk.row < a.rows) fetch(walk.row, now);
  for (int64_t r0 = walk.row; r0 < a.rows; r0 += walk.step, turn ^= 1) {
    if (kAhead && r0 + walk.step < a.rows) fetch(r0 + walk.step, next);
    auto& s = now.s;
    auto& dn = now.dn;
    auto& ds = now.ds;
    float sum[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[2 * r] = sum[2 * r + 1] = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float f[VEC], d[VEC], wf[VEC];
        walk.mask(s[r][c], c * NT + tid);
        walk.mask(dn[r][c], c * NT + tid);
        s[r][c].get(f);
        dn[r][c].get(d);
        w[c].get(wf);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          sum[2 * r] = fmaf(f[i], f[i], sum[2 * r]);
          sum[2 * r + 1] = fmaf(a.weight != nullptr ? __fmul_rn(d[i], wf[i]) : d[i], f[i], sum[2 * r + 1]);
        }
      }
    }
    group_join<SumOp, WPG, 2 * R>(sum, slots[g][turn]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= a.batch || r0 + r >= a.rows) continue;
      const float inv_h = 1.f / static_cast<float>(a.H);
      const float rstd = rsqrtf(sum[2 * r] / static_cast<float>(a.H) + a.eps);
      const float k = rstd * rstd * (sum[2 * r + 1] * inv_h);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float f[VEC], d[VEC], e[VEC], wf[VEC], o[VEC];
        s[r][c].get(f);
        dn[r][c].get(d);
        ds[r][c].get(e);
        w[c].get(wf);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float gi = a.weight != nullptr ? __fmul_rn(d[i], wf[i]) : d[i];  // a weight of ones changes no bit
          o[i] = fmaf(rstd, fmaf(-f[i], k, gi), e[i]);
          dw[c][i] = fmaf(d[i], f[i] * rstd, dw[c][i]);
        }
        Piece<T, VEC> out;
        out.set(o);
        walk.store(out, a.dx + (r0 + r) * a.H, c * NT + tid);
      }
    }
    if (kAhead) now = next;
    else if (r0 + walk.step < a.rows) fetch(r0 + walk.step, now);
  }
  if (a.part != nullptr) {
    float* part = a.part + (static_cast<int64_t>(blockIdx.x) * Group<WPG>::kPerCta + g) * a.H;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = walk.col(c * NT + tid);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col + i >= 0 && col + i < a.H) part[col + i] = dw[c][i];
    }
  }
}

// dweight[c] = T(sum over the groups of part[group][c]), in a fixed order: a warp takes every 32nd group
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_dweight_kernel(const float* part, int groups, int H, T* dweight) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < H) {
#pragma unroll 8
    for (int i = w; i < groups; i += 32) v += part[static_cast<int64_t>(i) * H + c];
  }
  sums[w][lane] = v;
  __syncthreads();
  v = sums[lane][w];  // warp w adds up column w of the block
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  const int out = blockIdx.x * 32 + w;
  if (lane == 0 && out < H) dweight[out] = from_f32<T>(v);
}

constexpr int kMaxHidden = 16384;

// The shape of a call: how many warps share a row, how many pieces a thread holds of it, and how many rows at a time forward and
// backward take.  Measured with 2^25 bfloat16 values, of which four arrays take 41.5 us at the rate of a copy (forward / 8 bits with
// blocks of 128 columns / backward at one or two CTAs an SM, whichever is faster, us):
//   256 columns   1 warp,  1 piece,  4 rows 42 / 52 / 64, 2 rows 42 / 48 / 44, 1 row 46 / 52 / 54
//   1024          2 warps, 2 pieces 40 / 46 / 44;   4 warps, 1 piece  48 / 54 / 56;   1 warp,  4 pieces 42 / 48 / 46
//   2048          4 warps, 2 pieces 40 / 46 / 47;   8 warps, 1 piece  50 / 56 / 56;   2 warps, 4 pieces 42 / 50 / 46
//   4096          8 warps, 2 pieces 42 / 46 / 48;  16 warps, 1 piece  48 / 62 / 60;   4 warps, 4 pieces 44 / 50 / 50
//   8192          8 warps, 4 pieces 46 / 52 / 50;  16 warps, 2 pieces 44 / 71 / 51
//   16384        16 warps, 4 pieces 54 / 58 / 69;  32 warps, 2 pieces 60 / 64 / 73
// So one piece a thread is too little to keep in flight, and reductions across many warps cost what is left.
struct Shape {
  int wpg, c;
};
#define FMOE_VEC_SHAPES(X) X(0, 1, 1, 2, 2) X(1, 1, 2, 1, 1) X(2, 2, 2, 1, 1) X(3, 4, 2, 1, 1) X(4, 8, 2, 1, 1) X(5, 8, 4, 1, 1) \
  X(6, 16, 4, 1, 1) X(7, 32, 4, 1, 1)
#define FMOE_ONE_SHAPES(X) X(0, 1, 8, 1, 1) X(1, 8, 8, 1, 1) X(2, 16, 16, 1, 1) X(3, 32, 16, 1, 1)
#define FMOE_SHAPE(I_, W_, C_, RF_, RB_) {W_, C_},
constexpr Shape kVecShapes[] = {FMOE_VEC_SHAPES(FMOE_SHAPE)};
constexpr Shape kOneShapes[] = {FMOE_ONE_SHAPES(FMOE_SHAPE)};
#undef FMOE_SHAPE
template <int N> int smallest_shape(const Shape (&shapes)[N], int pieces) {
  int i = 0;
  while (i < N && shapes[i].wpg * 32 * shapes[i].c < pieces) ++i;
  return i;  // N, which no launch takes, where none holds that many
}
int shape_of(bool vec, int pieces) { return vec ? smallest_shape(kVecShapes, pieces) : smallest_shape(kOneShapes, pieces); }

// Groups that the grid of a backward has: all that its registers let run at once, and no more, since each group leaves a row of
// partial sums.  A multiple of eight, so that SHIFT keeps its remainders.  The device has no say: the workspace may have been sized
// while another was current.
int64_t backward_groups(Shape sh, int64_t rows) {
  const int cta = sh.wpg < 8 ? 256 : 32 * sh.wpg, per_cta = cta / (32 * sh.wpg);
  const int64_t cap = static_cast<int64_t>(kB200Sms) * (sh.wpg * sh.c <= 16 ? 2 : 1) * per_cta / 8 * 8;
  return rows < cap ? (rows + 7) / 8 * 8 : cap;
}

// rows a group takes at a time: as many as fit its registers once every SM has a group, fewer before
int batch_rows(int64_t rows, int most, int per_cta) {
  const int64_t each = rows / (static_cast<int64_t>(device_sm_count()) * per_cta);
  return static_cast<int>(each < 1 ? 1 : each < most ? each : most);
}

template <typename T, int VEC, int WPG, int C, int R, bool SHIFT>
int launch_forward(const NormArgs<T>& in, int mode, cudaStream_t stream) {
  NormArgs<T> a = in;
  constexpr int per_cta = Group<WPG>::kPerCta;
  a.batch = batch_rows(a.rows, R, per_cta);
  int64_t grid = (a.rows + static_cast<int64_t>(a.batch) * per_cta - 1) / (static_cast<int64_t>(a.batch) * per_cta);
  const int64_t cap = static_cast<int64_t>(device_sm_count()) * 8;
  if (grid > cap) grid = cap;
  if (SHIFT) grid = (grid + 7) / 8 * 8;
  const unsigned ctas = static_cast<unsigned>(grid);
  const int smem = mode == kFp8Block && (VEC == 1 || SHIFT) ? per_cta * a.groups * 4 : 0;
  if (mode == kNorm) add_rms_norm_kernel<T, VEC, WPG, C, R, SHIFT, kNorm><<<ctas, Group<WPG>::kCta, 0, stream>>>(a);
  else if (mode == kFp8Row) add_rms_norm_kernel<T, VEC, WPG, C, R, SHIFT, kFp8Row><<<ctas, Group<WPG>::kCta, 0, stream>>>(a);
  else add_rms_norm_kernel<T, VEC, WPG, C, R, SHIFT, kFp8Block><<<ctas, Group<WPG>::kCta, smem, stream>>>(a);
  FMOE_LAUNCH_CHECK();
  return FMOE_OK;
}

template <typename T, int VEC, int WPG, int C, int R, bool SHIFT>
int launch_backward(const NormBackwardArgs<T>& in, T* dweight, cudaStream_t stream) {
  NormBackwardArgs<T> a = in;
  constexpr int per_cta = Group<WPG>::kPerCta;
  a.batch = batch_rows(a.rows, R, per_cta);
  const int64_t groups = backward_groups({WPG, C}, a.rows);
  add_rms_norm_backward_kernel<T, VEC, WPG, C, R, SHIFT><<<static_cast<unsigned>(groups / per_cta), Group<WPG>::kCta, 0, stream>>>(a);
  FMOE_LAUNCH_CHECK();
  if (dweight != nullptr) {
    rms_norm_dweight_kernel<T><<<(a.H + 31) / 32, 1024, 0, stream>>>(a.part, static_cast<int>(groups), a.H, dweight);
    FMOE_LAUNCH_CHECK();
  }
  return FMOE_OK;
}

// kWhole: rows of aligned pieces; kShifted: rows of any length in memory that starts at a piece; kSingle: one value at a time
enum Form { kWhole, kShifted, kSingle };
constexpr int kMostPieces = 4096;  // of the widest shape
// pieces of a row, at most; rows of whole pieces have as many when their weights are read one by one (kShifted, no shift)
int pieces_of(Form form, int vec, int H) { return form == kSingle ? H : H % vec == 0 ? H / vec : (H + 2 * vec - 2) / vec; }
// A row's last piece reaches into what follows by up to vec - gcd(H, vec) values.  The row behind it has to cover them: rows of 1, 2, 3
// and 5 16-bit values, and of one float32, are too short.
bool may_shift(int vec, int H) { return pieces_of(kShifted, vec, H) <= kMostPieces && vec - std::gcd(H, vec) <= H; }
// kShifted reads weights one by one, so they may start anywhere
Form form_of(int vec, int H, const void* weight, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (!aligned16(p)) return kSingle;
  if (H % vec == 0 && aligned16(weight)) return kWhole;
  return may_shift(vec, H) ? kShifted : kSingle;
}

template <typename T>
int forward_typed(const void* x, const void* residual, const void* weight, void* summed, void* normed, void* q, float* scales,
                  int64_t rows, int H, int group, float eps, int mode, cudaStream_t stream) {
  constexpr int V = Vec16<T>::N;
  const Form form = form_of(V, H, weight, {x, residual, summed, normed, q});
  const NormArgs<T> a = {static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight),
                         static_cast<T*>(summed), static_cast<T*>(normed), static_cast<__nv_fp8_storage_t*>(q), scales, rows, H, 1,
                         group == 32 ? 5 : group == 64 ? 6 : 7, mode == kFp8Block ? (H + group - 1) / group : 1, eps};
  const int shape = shape_of(form != kSingle, pieces_of(form, V, H));
#define FMOE_VEC(I_, W_, C_, RF_, RB_)                                                                    \
  if (form == kWhole && shape == I_) return launch_forward<T, V, W_, C_, RF_, false>(a, mode, stream);    \
  if (form == kShifted && shape == I_) return launch_forward<T, V, W_, C_, 1, true>(a, mode, stream);
#define FMOE_ONE(I_, W_, C_, RF_, RB_) if (form == kSingle && shape == I_) return launch_forward<T, 1, W_, C_, RF_, false>(a, mode, stream);
  FMOE_VEC_SHAPES(FMOE_VEC)
  FMOE_ONE_SHAPES(FMOE_ONE)
#undef FMOE_VEC
#undef FMOE_ONE
  return FMOE_ERR_UNSUPPORTED;
}

template <typename T>
int backward_typed(const void* dnormed, const void* dsummed, const void* summed, const void* weight, void* dx, void* dweight,
                   float* part, int64_t rows, int H, float eps, cudaStream_t stream) {
  constexpr int V = Vec16<T>::N;
  const Form form = form_of(V, H, weight, {dnormed, dsummed, summed, dx});
  const NormBackwardArgs<T> a = {static_cast<const T*>(dnormed), static_cast<const T*>(dsummed), static_cast<const T*>(summed),
                                 static_cast<const T*>(weight), static_cast<T*>(dx), dweight != nullptr ? part : nullptr, rows, H, 1, eps};
  T* dw = static_cast<T*>(dweight);
  const int shape = shape_of(form != kSingle, pieces_of(form, V, H));
#define FMOE_VEC(I_, W_, C_, RF_, RB_)                                                                    \
  if (form == kWhole && shape == I_) return launch_backward<T, V, W_, C_, RB_, false>(a, dw, stream);     \
  if (form == kShifted && shape == I_) return launch_backward<T, V, W_, C_, 1, true>(a, dw, stream);
#define FMOE_ONE(I_, W_, C_, RF_, RB_) if (form == kSingle && shape == I_) return launch_backward<T, 1, W_, C_, RB_, false>(a, dw, stream);
  FMOE_VEC_SHAPES(FMOE_VEC)
  FMOE_ONE_SHAPES(FMOE_ONE)
#undef FMOE_VEC
#undef FMOE_ONE
  return FMOE_ERR_UNSUPPORTED;
}

}  // namespace

int launch_add_rms_norm(const void* x, const void* residual, const void* weight, void* summed, void* normed, void* q,
                        float* scales, int dtype, int64_t rows, int H, int group, float eps, cudaStream_t stream) {
  if (rows < 0 || H <= 0 || !(eps >= 0.f)) return FMOE_ERR_BAD_ARG;
  if (H > kMaxHidden) return FMOE_ERR_UNSUPPORTED;
  const bool fp8 = q != nullptr || scales != nullptr;
  if (fp8 && group != 0 && group != 32 && group != 64 && group != 128) return FMOE_ERR_BAD_ARG;
  if (rows == 0) return FMOE_OK;
  if (x == nullptr || (residual != nullptr) != (summed != nullptr)) return FMOE_ERR_BAD_ARG;
  if (fp8 ? (q == nullptr || scales == nullptr || normed != nullptr) : normed == nullptr) return FMOE_ERR_BAD_ARG;
  const int mode = !fp8 ? kNorm : group == 0 ? kFp8Row : kFp8Block;
  switch (dtype) {
    case FMOE_DTYPE_F32: return forward_typed<float>(x, residual, weight, summed, normed, q, scales, rows, H, group, eps, mode, stream);
    case FMOE_DTYPE_BF16: return forward_typed<__nv_bfloat16>(x, residual, weight, summed, normed, q, scales, rows, H, group, eps, mode, stream);
    case FMOE_DTYPE_F16: return forward_typed<__half>(x, residual, weight, summed, normed, q, scales, rows, H, group, eps, mode, stream);
    default: return FMOE_ERR_BAD_ARG;
  }
}

// the largest of what the forms of a call use
size_t add_rms_norm_backward_workspace_bytes(int64_t rows, int H, int dtype) {
  if (rows <= 0 || H <= 0 || H > kMaxHidden) return 0;
  const int n = 16 / dtype_size(dtype);
  int64_t groups = 0;
  for (const Form form : {kWhole, kShifted, kSingle}) {
    if (form != kSingle && !may_shift(n, H)) continue;  // H is at most kMostPieces whole ones, which may shift
    const Shape sh = form == kSingle ? kOneShapes[shape_of(false, H)] : kVecShapes[shape_of(true, pieces_of(form, n, H))];
    const int64_t g = backward_groups(sh, rows);
    groups = g > groups ? g : groups;
  }
  return static_cast<size_t>(groups) * H * sizeof(float);
}

int launch_add_rms_norm_backward(const void* dnormed, const void* dsummed, const void* summed, const void* weight, void* dx,
                                 void* dweight, int dtype, int64_t rows, int H, float eps, void* ws, size_t ws_bytes,
                                 cudaStream_t stream) {
  if (rows < 0 || H <= 0 || !(eps >= 0.f)) return FMOE_ERR_BAD_ARG;
  if (H > kMaxHidden) return FMOE_ERR_UNSUPPORTED;
  if (rows == 0) {
    if (dweight != nullptr) FMOE_CUDA_TRY(cudaMemsetAsync(dweight, 0, static_cast<size_t>(H) * dtype_size(dtype), stream));
    return FMOE_OK;
  }
  if (dnormed == nullptr || summed == nullptr || dx == nullptr) return FMOE_ERR_BAD_ARG;
  if (dweight != nullptr && (ws == nullptr || ws_bytes < add_rms_norm_backward_workspace_bytes(rows, H, dtype))) return FMOE_ERR_WORKSPACE;
  if (dweight != nullptr && !aligned16(ws)) return FMOE_ERR_ALIGNMENT;
  float* part = static_cast<float*>(ws);
  switch (dtype) {
    case FMOE_DTYPE_F32: return backward_typed<float>(dnormed, dsummed, summed, weight, dx, dweight, part, rows, H, eps, stream);
    case FMOE_DTYPE_BF16: return backward_typed<__nv_bfloat16>(dnormed, dsummed, summed, weight, dx, dweight, part, rows, H, eps, stream);
    case FMOE_DTYPE_F16: return backward_typed<__half>(dnormed, dsummed, summed, weight, dx, dweight, part, rows, H, eps, stream);
    default: return FMOE_ERR_BAD_ARG;
  }
}

}  // namespace fmoe
