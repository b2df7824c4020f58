// The pre-norm of a residual stack: s = T(x + r), n = s * rsqrt(mean(s^2) + eps) * w, with its gradient, and with an output in
// 8 bits.  No counterpart in the reference, which leaves normalisation and skip connection to its caller
// (flash_moe/modules/flash_moe.py:55-59).
//
// Memory-bound throughout: the forward moves 4 rows' worth of values per row (x, r in; s, n out), the backward 4 (dn, ds, s in;
// dx out).  A row stays in the registers of its group of warps between the sum of squares and the scaling, so each value is
// moved once.  Everything inside is float32; s is rounded to T before it is normalised, so that n belongs to the s that is
// stored and the backward finds the same s; n, dx and dw are rounded once.
#include <cuda_fp8.h>

#include "common.cuh"

namespace fmoe {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr float kE4m3Max = 448.f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: a zero group keeps a scale that can be divided by

// VEC values of T as they are loaded: 16 bytes, or one value where rows are not made of aligned 16-byte pieces
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
  int H, pieces, batch;
  int group_shift, groups;  // kFp8Block: columns of a block, a power of two
  float eps;
};

template <typename T, int VEC, int WPG, int C, int R, int MODE>
__global__ void __launch_bounds__(Group<WPG>::kCta) add_rms_norm_kernel(const NormArgs<T> a) {
  constexpr int NT = Group<WPG>::kThreads;
  const int g = threadIdx.x / NT, tid = threadIdx.x % NT;
  __shared__ float slots[Group<WPG>::kPerCta][3][R * WPG];
  extern __shared__ uint32_t block_max[];  // kFp8Block on single values: [kPerCta][groups]
  Piece<T, VEC> w[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = c * NT + tid;
    w[c].zero();
    if (a.weight != nullptr && p < a.pieces) w[c].load(a.weight + static_cast<int64_t>(p) * VEC);
  }
  int turn = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * Group<WPG>::kPerCta * a.batch;
  for (int64_t r0 = (static_cast<int64_t>(blockIdx.x) * Group<WPG>::kPerCta + g) * a.batch; r0 < a.rows; r0 += step, turn ^= 1) {
    Piece<T, VEC> s[R][C];
    float sq[R];
    {
      Piece<T, VEC> res[R][C];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int p = c * NT + tid;
          s[r][c].zero();
          res[r][c].zero();
          if (r < a.batch && r0 + r < a.rows && p < a.pieces) {
            const int64_t at = (r0 + r) * a.H + static_cast<int64_t>(p) * VEC;
            s[r][c].load(a.x + at);
            if (a.residual != nullptr) res[r][c].load(a.residual + at);
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
            s[r][c].get(f);
          }
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
    auto live = [&](int r, int p) { return r < a.batch && r0 + r < a.rows && p < a.pieces; };
    if (MODE == kNorm) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int p = c * NT + tid;
          if (!live(r, p)) continue;
          const int64_t at = (r0 + r) * a.H + static_cast<int64_t>(p) * VEC;
          if (a.residual != nullptr) s[r][c].store(a.summed + at);
          float y[VEC];
          value(r, c, y);
          Piece<T, VEC> out;
          out.set(y);
          out.store(a.normed + at);
        }
      continue;
    }
    // 8 bits: scale = max |y| / 448 over the row or the block of columns, q = e4m3(y / scale)
    float top[R];
    if (MODE == kFp8Row) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        top[r] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float y[VEC];
          if (!live(r, c * NT + tid)) continue;
          value(r, c, y);
#pragma unroll
          for (int i = 0; i < VEC; ++i) top[r] = MaxOp::join(top[r], fabsf(y[i]));
        }
      }
      group_join<MaxOp, WPG, R>(top, slots[g][2]);
    }
    if (MODE == kFp8Block && VEC == 1) {
      uint32_t* m = block_max + g * a.groups;
      for (int i = tid; i < a.groups; i += NT) m[i] = 0;
      group_barrier<WPG>();
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float y[VEC];
        const int p = c * NT + tid;
        if (!live(0, p)) continue;
        value(0, c, y);
        atomicMax(m + (p >> a.group_shift), __float_as_uint(fabsf(y[0])));
      }
      group_barrier<WPG>();
    }
    float most[R][C];
    if (MODE == kFp8Block && VEC > 1) {
      // a block is 4 to 32 neighbouring lanes
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float y[VEC];
          value(r, c, y);
          most[r][c] = 0.f;
#pragma unroll
          for (int i = 0; i < VEC; ++i) most[r][c] = MaxOp::join(most[r][c], fabsf(y[i]));
        }
      for (int d = (1 << a.group_shift) / (2 * VEC); d > 0; d >>= 1)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int c = 0; c < C; ++c) most[r][c] = MaxOp::join(most[r][c], __shfl_xor_sync(kFull, most[r][c], d));
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int p = c * NT + tid;
        const bool ok = live(r, p);
        float y[VEC], m;
        value(r, c, y);
        const int col = p * VEC;
        if (MODE == kFp8Row) m = top[r];
        else if (VEC == 1) m = ok ? __uint_as_float(block_max[g * a.groups + (p >> a.group_shift)]) : 0.f;
        else m = most[r][c];
        if (!ok) continue;
        m *= 1.f / kE4m3Max;
        const float scale = m < kMinScale ? kMinScale : m;  // a NaN stays
        const float inv = __fdividef(1.f, scale);           // 2^-126 <= scale < 2^120, or infinite: 0
        const int64_t at = (r0 + r) * a.H + col;
        if (MODE == kFp8Row) {
          if (p == 0) a.scales[r0 + r] = scale;
        } else if ((col & ((1 << a.group_shift) - 1)) == 0) {
          a.scales[(r0 + r) * a.groups + (col >> a.group_shift)] = scale;
        }
        if (a.residual != nullptr) s[r][c].store(a.summed + at);
        if (VEC == 1) {
          a.q[at] = __nv_cvt_float_to_fp8(y[0] * inv, __NV_SATFINITE, __NV_E4M3);
        } else {
          uint16_t b[VEC / 2 + 1];
#pragma unroll
          for (int i = 0; i < VEC; i += 2)
            b[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(y[i] * inv, y[i + (VEC > 1)] * inv), __NV_SATFINITE, __NV_E4M3);
          if (VEC == 8)
            *reinterpret_cast<uint2*>(a.q + at) = make_uint2(b[0] | (b[1] << 16), b[VEC / 4] | (b[3 * VEC / 8] << 16));
          else
            *reinterpret_cast<uint32_t*>(a.q + at) = b[0] | (b[1] << 16);
        }
      }
    if (MODE == kFp8Block && VEC == 1) group_barrier<WPG>();  // block_max is cleared for the next row
    if (MODE == kFp8Row && WPG > 1) group_barrier<WPG>();     // slots[g][2] is written again
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
  int H, pieces, batch;
  float eps;
};

template <typename T, int VEC, int WPG, int C, int R>
__global__ void __launch_bounds__(Group<WPG>::kCta) add_rms_norm_backward_kernel(const NormBackwardArgs<T> a) {
  constexpr int NT = Group<WPG>::kThreads;
  const int g = threadIdx.x / NT, tid = threadIdx.x % NT;
  __shared__ float slots[Group<WPG>::kPerCta][2][2 * R * WPG];
  Piece<T, VEC> w[C];
  float dw[C][VEC];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = c * NT + tid;
    w[c].zero();
    if (a.weight != nullptr && p < a.pieces) w[c].load(a.weight + static_cast<int64_t>(p) * VEC);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[c][i] = 0.f;
  }
  int turn = 0;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * Group<WPG>::kPerCta + g;
  const int64_t step = static_cast<int64_t>(gridDim.x) * Group<WPG>::kPerCta * a.batch;
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
        if (r < a.batch && r0 + r < a.rows && p < a.pieces) {
          const int64_t at = (r0 + r) * a.H + static_cast<int64_t>(p) * VEC;
          b.s[r][c].load(a.summed + at);
          b.dn[r][c].load(a.dnormed + at);
          if (a.dsummed != nullptr) b.ds[r][c].load(a.dsummed + at);
        }
      }
  };
  Batch now, next;
  if (slot * a.batch < a.rows) fetch(slot * a.batch, now);
  for (int64_t r0 = slot * a.batch; r0 < a.rows; r0 += step, turn ^= 1) {
    if (r0 + step < a.rows) fetch(r0 + step, next);  // on the way while this batch is worked on
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
        const int p = c * NT + tid;
        if (p >= a.pieces) continue;
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
        out.store(a.dx + (r0 + r) * a.H + static_cast<int64_t>(p) * VEC);
      }
    }
    now = next;
  }
  if (a.part != nullptr) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int p = c * NT + tid;
      if (p < a.pieces) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) a.part[slot * a.H + static_cast<int64_t>(p) * VEC + i] = dw[c][i];
      }
    }
  }
}

// dweight[c] = T(sum over the groups of part[group][c]), in a fixed order
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_dweight_kernel(const float* part, int groups, int H, T* dweight) {
  __shared__ float sums[8][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float v = 0.f;
  if (c < H)
    for (int i = w; i < groups; i += 8) v += part[static_cast<int64_t>(i) * H + c];
  sums[w][threadIdx.x & 31] = v;
  __syncthreads();
  if (w == 0 && c < H) {
    for (int i = 1; i < 8; ++i) v += sums[i][threadIdx.x];
    dweight[c] = from_f32<T>(v);
  }
}

constexpr int kMaxHidden = 16384;

// The shape of a call: how many warps share a row, how many pieces a thread holds of it, and how many rows at a time forward and
// backward take.  Few warps with two pieces a thread beat many with one: less of a row's time goes into reductions across warps.
struct Shape {
  int wpg, c;
};
#define FMOE_VEC_SHAPES(X) X(0, 1, 1, 4, 2) X(1, 1, 2, 1, 1) X(2, 2, 2, 1, 1) X(3, 4, 2, 1, 1) X(4, 8, 2, 1, 1) X(5, 8, 4, 1, 1) \
  X(6, 16, 4, 1, 1) X(7, 32, 4, 1, 1)
#define FMOE_ONE_SHAPES(X) X(0, 1, 8, 1, 1) X(1, 8, 8, 1, 1) X(2, 32, 16, 1, 1)
#define FMOE_SHAPE(I_, W_, C_, RF_, RB_) {W_, C_},
constexpr Shape kVecShapes[] = {FMOE_VEC_SHAPES(FMOE_SHAPE)};
constexpr Shape kOneShapes[] = {FMOE_ONE_SHAPES(FMOE_SHAPE)};
#undef FMOE_SHAPE
int shape_of(bool vec, int pieces) {
  int i = 0;
  if (vec) {
    while (kVecShapes[i].wpg * 32 * kVecShapes[i].c < pieces) ++i;
    return i;
  }
  while (kOneShapes[i].wpg * 32 * kOneShapes[i].c < pieces) ++i;
  return i;
}

// Groups that the grid of a backward has: all that its registers let run at once, and no more, since each group leaves a row of
// partial sums.
int64_t backward_groups(Shape sh, int64_t rows) {
  const int cta = sh.wpg < 8 ? 256 : 32 * sh.wpg, per_cta = cta / (32 * sh.wpg);
  const int64_t cap = static_cast<int64_t>(device_sm_count()) * (sh.wpg * sh.c <= 16 ? 2 : 1) * per_cta;
  return rows < cap ? (rows + per_cta - 1) / per_cta * per_cta : cap;
}

// rows a group takes at a time: as many as fit its registers once every SM has a group, fewer before
int batch_rows(int64_t rows, int most, int per_cta) {
  const int64_t each = rows / (static_cast<int64_t>(device_sm_count()) * per_cta);
  return static_cast<int>(each < 1 ? 1 : each < most ? each : most);
}

template <typename T, int VEC, int WPG, int C, int R>
int launch_forward(const NormArgs<T>& in, int mode, cudaStream_t stream) {
  NormArgs<T> a = in;
  constexpr int per_cta = Group<WPG>::kPerCta;
  a.batch = batch_rows(a.rows, R, per_cta);
  const int64_t want = (a.rows + static_cast<int64_t>(a.batch) * per_cta - 1) / (static_cast<int64_t>(a.batch) * per_cta);
  const int64_t cap = static_cast<int64_t>(device_sm_count()) * 8;
  const unsigned grid = static_cast<unsigned>(want < cap ? want : cap);
  const int smem = mode == kFp8Block && VEC == 1 ? per_cta * a.groups * 4 : 0;
  if (mode == kNorm) add_rms_norm_kernel<T, VEC, WPG, C, R, kNorm><<<grid, Group<WPG>::kCta, 0, stream>>>(a);
  else if (mode == kFp8Row) add_rms_norm_kernel<T, VEC, WPG, C, R, kFp8Row><<<grid, Group<WPG>::kCta, 0, stream>>>(a);
  else add_rms_norm_kernel<T, VEC, WPG, C, R, kFp8Block><<<grid, Group<WPG>::kCta, smem, stream>>>(a);
  FMOE_LAUNCH_CHECK();
  return FMOE_OK;
}

template <typename T, int VEC, int WPG, int C, int R>
int launch_backward(const NormBackwardArgs<T>& in, T* dweight, cudaStream_t stream) {
  NormBackwardArgs<T> a = in;
  constexpr int per_cta = Group<WPG>::kPerCta;
  a.batch = batch_rows(a.rows, R, per_cta);
  const int64_t groups = backward_groups({WPG, C}, a.rows);
  add_rms_norm_backward_kernel<T, VEC, WPG, C, R><<<static_cast<unsigned>(groups / per_cta), Group<WPG>::kCta, 0, stream>>>(a);
  FMOE_LAUNCH_CHECK();
  if (dweight != nullptr) {
    rms_norm_dweight_kernel<T><<<(a.H + 31) / 32, 256, 0, stream>>>(a.part, static_cast<int>(groups), a.H, dweight);
    FMOE_LAUNCH_CHECK();
  }
  return FMOE_OK;
}

template <typename T>
int forward_typed(const void* x, const void* residual, const void* weight, void* summed, void* normed, void* q, float* scales,
                  int64_t rows, int H, int group, float eps, int mode, cudaStream_t stream) {
  const bool vec = H % Vec16<T>::N == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(summed) &&
                   aligned16(normed) && aligned16(q);
  NormArgs<T> a = {static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight),
                   static_cast<T*>(summed), static_cast<T*>(normed), static_cast<__nv_fp8_storage_t*>(q), scales, rows, H,
                   vec ? H / Vec16<T>::N : H, 1, group == 32 ? 5 : group == 64 ? 6 : 7, mode == kFp8Block ? (H + group - 1) / group : 1, eps};
  const int shape = shape_of(vec, a.pieces);
#define FMOE_VEC(I_, W_, C_, RF_, RB_) if (vec && shape == I_) return launch_forward<T, Vec16<T>::N, W_, C_, RF_>(a, mode, stream);
#define FMOE_ONE(I_, W_, C_, RF_, RB_) if (!vec && shape == I_) return launch_forward<T, 1, W_, C_, RF_>(a, mode, stream);
  FMOE_VEC_SHAPES(FMOE_VEC)
  FMOE_ONE_SHAPES(FMOE_ONE)
#undef FMOE_VEC
#undef FMOE_ONE
  return FMOE_ERR_UNSUPPORTED;
}

bool backward_vec(int dtype, int H, const void* a, const void* b, const void* c, const void* d, const void* e) {
  return H % (16 / dtype_size(dtype)) == 0 && aligned16(a) && aligned16(b) && aligned16(c) && aligned16(d) && aligned16(e);
}

template <typename T>
int backward_typed(const void* dnormed, const void* dsummed, const void* summed, const void* weight, void* dx, void* dweight,
                   float* part, bool vec, int64_t rows, int H, float eps, cudaStream_t stream) {
  NormBackwardArgs<T> a = {static_cast<const T*>(dnormed), static_cast<const T*>(dsummed), static_cast<const T*>(summed),
                           static_cast<const T*>(weight), static_cast<T*>(dx), dweight != nullptr ? part : nullptr, rows, H,
                           vec ? H / Vec16<T>::N : H, 1, eps};
  T* dw = static_cast<T*>(dweight);
  const int shape = shape_of(vec, a.pieces);
#define FMOE_VEC(I_, W_, C_, RF_, RB_) if (vec && shape == I_) return launch_backward<T, Vec16<T>::N, W_, C_, RB_>(a, dw, stream);
#define FMOE_ONE(I_, W_, C_, RF_, RB_) if (!vec && shape == I_) return launch_backward<T, 1, W_, C_, RB_>(a, dw, stream);
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

// the larger of what the two forms of a call (16-byte pieces, single values) use
size_t add_rms_norm_backward_workspace_bytes(int64_t rows, int H, int dtype) {
  if (rows <= 0 || H <= 0 || H > kMaxHidden) return 0;
  const int n = 16 / dtype_size(dtype);
  int64_t groups = backward_groups(kOneShapes[shape_of(false, H)], rows);
  if (H % n == 0) {
    const int64_t v = backward_groups(kVecShapes[shape_of(true, H / n)], rows);
    groups = v > groups ? v : groups;
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
  const bool vec = backward_vec(dtype, H, dnormed, dsummed, summed, weight, dx);
  float* part = static_cast<float*>(ws);
  switch (dtype) {
    case FMOE_DTYPE_F32: return backward_typed<float>(dnormed, dsummed, summed, weight, dx, dweight, part, vec, rows, H, eps, stream);
    case FMOE_DTYPE_BF16: return backward_typed<__nv_bfloat16>(dnormed, dsummed, summed, weight, dx, dweight, part, vec, rows, H, eps, stream);
    case FMOE_DTYPE_F16: return backward_typed<__half>(dnormed, dsummed, summed, weight, dx, dweight, part, vec, rows, H, eps, stream);
    default: return FMOE_ERR_BAD_ARG;
  }
}

}  // namespace fmoe
