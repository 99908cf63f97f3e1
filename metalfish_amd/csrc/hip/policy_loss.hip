// Losses on rows of policy logits, with their gradients, for gfx950.
//
// With z_k = (x_k - max x) / T over a row's entries, S = sum exp(z_k) and
// p_k = exp(z_k) / S:
//   ln p_a = z_a - ln S,   H = ln S - E_p z,
//   KL(p || q) = ln E_p exp(-(d - E_p d)),   d_k = (x_k - y_k) / T,
// the last from ln(p_k / q_k) = d_k - E_p d + KL: no difference of two
// log-sum-exps of nearly equal rows is formed, and with u_k = d_k - E_p d
// (E_p u = 0) it is log1p(E_p (exp(-u) - 1 + u)), a sum of terms >= 0.
// The gradients follow without another statistic:
//   d ln p_a / dx_k = (1[k = a] - p_k) / T,
//   d KL / dx_k = p_k u_k / T,   dH / dx_k = -p_k (z_k - E_p z) / T.
//
// Every statistic is fp32.  The bound is memory: x (and y) are read once,
// held in registers in their own type, and the gradient is written from there
// (rows too long for that are read a second time).
#include "mfh_device.h"
#include "mfh_kernels.h"

namespace mfh {
namespace {

constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.69314718f;
constexpr int kMaxMoves = 256;

// 16 bytes of a row at any element's alignment (global memory takes
// unaligned vector accesses on gfx950).
typedef unsigned int u32x4_a4 __attribute__((ext_vector_type(4), aligned(4), may_alias));
typedef unsigned int u32x4_a2 __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <int DT> struct Elem;
template <> struct Elem<DT_F32> {
  using T = std::uint32_t;
  using V = u32x4_a4;
  static constexpr int kPerVec = 4;
  static constexpr std::uint32_t kNegInf = 0xFF800000u;
  static __device__ __forceinline__ float Get(u32x4 v, int i) { return __uint_as_float(v[i]); }
  static __device__ __forceinline__ float One(T v) { return __uint_as_float(v); }
  static __device__ __forceinline__ T Round(float f) { return __float_as_uint(f); }
  static __device__ __forceinline__ u32x4 Pack(const float *f) {
    return u32x4{Round(f[0]), Round(f[1]), Round(f[2]), Round(f[3])};
  }
};
template <> struct Elem<DT_BF16> {
  using T = std::uint16_t;
  using V = u32x4_a2;
  static constexpr int kPerVec = 8;
  static constexpr std::uint32_t kNegInf = 0xFF80FF80u;
  static __device__ __forceinline__ float Get(u32x4 v, int i) {
    return __uint_as_float(i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16);
  }
  static __device__ __forceinline__ float One(T v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ T Round(float f) { return f32_to_bf16(f); }
  static __device__ __forceinline__ u32x4 Pack(const float *f) {
    return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                 pack_bf16x2(f[6], f[7])};
  }
};
template <> struct Elem<DT_F16> {
  using T = std::uint16_t;
  using V = u32x4_a2;
  static constexpr int kPerVec = 8;
  static constexpr std::uint32_t kNegInf = 0xFC00FC00u;
  static __device__ __forceinline__ float One(T v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
  }
  static __device__ __forceinline__ float Get(u32x4 v, int i) {
    return One(static_cast<T>(i & 1 ? v[i >> 1] >> 16 : v[i >> 1] & 0xFFFFu));
  }
  static __device__ __forceinline__ T Round(float f) {
    return __builtin_bit_cast(T, static_cast<_Float16>(f));
  }
  static __device__ __forceinline__ u32x4 Pack(const float *f) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = Round(f[2 * i]) | static_cast<std::uint32_t>(Round(f[2 * i + 1])) << 16;
    return r;
  }
};

// Elements base .. base + kPerVec of a row of n; -inf beyond its end.
template <int DT>
__device__ __forceinline__ u32x4 LoadVec(const typename Elem<DT>::T *row, int base, int n) {
  using E = Elem<DT>;
  if (base + E::kPerVec <= n)
    return *reinterpret_cast<const typename E::V *>(row + base);
  u32x4 v = {E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf};
#pragma unroll
  for (int i = 0; i < E::kPerVec; ++i) {
    if (base + i < n) {
      if constexpr (DT == DT_F32) {
        v[i] = row[base + i];
      } else {
        const std::uint32_t b = row[base + i];
        v[i >> 1] = i & 1 ? (v[i >> 1] & 0xFFFFu) | b << 16 : (v[i >> 1] & 0xFFFF0000u) | b;
      }
    }
  }
  return v;
}

template <int DT>
__device__ __forceinline__ void StoreVec(typename Elem<DT>::T *row, int base, int n,
                                         const float *f) {
  using E = Elem<DT>;
  if (base + E::kPerVec <= n) {
    *reinterpret_cast<typename E::V *>(row + base) = E::Pack(f);
    return;
  }
#pragma unroll
  for (int i = 0; i < E::kPerVec; ++i)
    if (base + i < n)
      row[base + i] = E::Round(f[i]);
}

// exp2 on v_exp_f32: 1 ulp, results below 2^-126 are 0.
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// p (exp(-u) - 1 + u), the term of KL; exp(-u) p is exp2(ym c + shift) of the
// reference logit less the policy's maximum, ym.  Near 0 the series of u (its first
// term left out is 1.2e-8 of the sum at |u| = 1/4); far below, where exp(-u)
// may overflow against a tiny p, their product from the reference logit.
__device__ __forceinline__ float KlTerm(float p, float u, float ym, float c, float shift) {
  const bool far = !(u > -60.f);
  const float e = Exp2(far ? ym * c + shift : -u * kLog2e);
  const float series =
      u * u *
      (0.5f + u * (-1.f / 6 + u * (1.f / 24 + u * (-1.f / 120 + u * (1.f / 720 + u * (-1.f / 5040))))));
  const float phi = fabsf(u) < 0.25f ? series : e - 1.f + u;
  // p == 0: what is masked here adds nothing but its reference probability.
  return far ? (p == 0.f ? e : e - p * (1.f - u)) : (p == 0.f ? 0.f : p * phi);
}

// KL from the sum of its terms; infinite where the reference lacks what the
// policy plays (E_p d is, and no term then means anything).
__device__ __forceinline__ float KlOf(float terms, float mean_d) {
  return mean_d == __builtin_inff() ? mean_d : log1pf(terms);
}

// What a row's scalars come to, from its statistics.
struct RowStats {
  float m;        // maximum (0 where every entry is masked)
  float log_sum;  // ln S
  float inv_sum;  // 1 / S
  float mean_z;   // E_p z
  float mean_d;   // E_p d
  bool empty;     // no entry left
};

__device__ __forceinline__ RowStats Stats(float m, float s, float st, float sd, float inv_temp) {
  RowStats r;
  r.m = m;
  r.empty = s == 0.f;
  const float sum = r.empty ? 1.f : s;
  r.log_sum = logf(sum);
  r.inv_sum = 1.f / sum;
  r.mean_z = st * kLn2 * r.inv_sum;
  r.mean_d = sd * inv_temp * r.inv_sum;
  return r;
}

// The first term of the loss and its derivative by ln p_a.
struct Surrogate {
  float loss, slope;
};
__device__ __forceinline__ Surrogate Clipped(const RowLossParams &a, std::int64_t row, float logp) {
  const float adv = a.advantage[row];
  const float ratio = a.old_logp ? expf(logp - a.old_logp[row]) : 1.f;
  const float plain = ratio * adv;
  const float bounded = fminf(fmaxf(ratio, a.ratio_low), a.ratio_high) * adv;
  // The unclipped branch on ties and for NaN.
  return bounded < plain ? Surrogate{-bounded, 0.f} : Surrogate{-plain, -plain};
}

// Coefficients of one row's gradient
//   scale (slope 1[k = a] + p_k (kl u_k + entropy (z_k - E_p z) - slope)).
struct RowGrad {
  float scale, slope, kl, entropy;
};

template <bool REF>
__device__ __forceinline__ float GradTerm(const RowGrad &g, const RowStats &st, float x, float y,
                                          float inv_temp) {
  const float z = (x - st.m) * inv_temp;
  const float p = Exp2(z * kLog2e) * st.inv_sum;
  float v = g.entropy * (z - st.mean_z) - g.slope;
  if constexpr (REF)
    v += g.kl * ((x - y) * inv_temp - st.mean_d);
  return p == 0.f ? 0.f : p * v * g.scale;
}

// Writes the row's outputs; returns the coefficients of its gradient.
__device__ __forceinline__ RowGrad FinishRow(const RowLossParams &a, std::int64_t row, float w,
                                             const RowStats &st, bool acted, float za, float kl,
                                             bool writer) {
  acted = acted && !st.empty;
  const float logp = acted ? za - st.log_sum : 0.f;
  if (a.coef)
    return {w * a.inv_temp, acted ? 1.f : 0.f, 0.f, 0.f};
  if (a.mark) {
    if (writer)
      a.mark[row] = acted ? logp : kNoAction;
    return {0.f, 0.f, 0.f, 0.f};
  }
  Surrogate s{0.f, 0.f};
  if (acted && a.advantage)
    s = Clipped(a, row, logp);
  const float entropy = st.empty ? 0.f : st.log_sum - st.mean_z;
  if (writer) {
    float loss = s.loss;
    if (a.kl_coef != 0.f)
      loss += a.kl_coef * kl;
    if (a.entropy_coef != 0.f)
      loss -= a.entropy_coef * entropy;
    if (a.loss)
      a.loss[row] = w * loss;
    if (a.logp)
      a.logp[row] = logp;
    if (a.kl)
      a.kl[row] = kl;
    if (a.entropy)
      a.entropy[row] = entropy;
  }
  return {w * a.inv_temp, s.slope, a.kl_coef, a.entropy_coef};
}

__device__ __forceinline__ void ZeroOutputs(const RowLossParams &a, std::int64_t row) {
  if (a.loss)
    a.loss[row] = 0.f;
  if (a.logp)
    a.logp[row] = 0.f;
  if (a.kl)
    a.kl[row] = 0.f;
  if (a.entropy)
    a.entropy[row] = 0.f;
}

// Whether the divergence itself is asked for (its gradient needs no KL).
__device__ __forceinline__ bool WantsKl(const RowLossParams &a) {
  return a.kl || (a.loss && a.kl_coef != 0.f);
}

__device__ __forceinline__ bool OutsideSequences(const RowLossParams &a, std::int64_t row) {
  return a.seq_offsets && (row < a.seq_offsets[0] || row >= a.seq_offsets[a.n_seq]);
}

// The factor on a row's outputs; 0: the row is not read.
__device__ __forceinline__ float RowWeight(const RowLossParams &a, std::int64_t row) {
  return a.coef ? a.coef[row] : a.weight ? a.weight[row] : 1.f;
}

// Sums of N values over the W waves of a workgroup, the waves' in order.
template <int W, int N>
__device__ __forceinline__ void GroupSum(float (&v)[N], float (*red)[4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] = wave_sum(v[i]);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        red[wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w)
        s += red[w][i];
      v[i] = s;
    }
  }
}

template <int W>
__device__ __forceinline__ float GroupMax(float v, float (*red)[4]) {
  v = wave_max(v);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
      red[threadIdx.x >> 6][0] = v;
    __syncthreads();
    v = red[0][0];
#pragma unroll
    for (int w = 1; w < W; ++w)
      v = fmaxf(v, red[w][0]);
  }
  return v;
}

// A whole row in the registers of W waves, NV vectors of 16 bytes a lane.
template <int DT, int W, int NV, bool REF>
__global__ __launch_bounds__(64 * W) void DenseRowKernel(RowLossParams a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VE = E::kPerVec;
  __shared__ float red[W][4];
  const std::int64_t row = a.row0 + blockIdx.x;
  if (OutsideSequences(a, row))
    return;
  const int n = a.vocab;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *y = REF ? static_cast<const T *>(a.y) + row * a.ldy : nullptr;
  T *g = a.g ? static_cast<T *>(a.g) + row * a.ldg : nullptr;
  const bool writer = threadIdx.x == 0;
  const float w = RowWeight(a, row);
  if (w == 0.f) {
    if (writer)
      ZeroOutputs(a, row);
    const float zero[8] = {};
    if (g)
      for (int j = 0; j < NV; ++j)
        StoreVec<DT>(g, (j * 64 * W + threadIdx.x) * VE, n, zero);
    return;
  }
  u32x4 xr[NV], yr[REF ? NV : 1];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    xr[j] = LoadVec<DT>(x, (j * 64 * W + threadIdx.x) * VE, n);
  if constexpr (REF) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      yr[j] = LoadVec<DT>(y, (j * 64 * W + threadIdx.x) * VE, n);
  }
  const int act = a.actions ? a.actions[row] : -1;
  const bool acted = act >= 0 && act < n;
  const float xa = acted ? E::One(x[act]) : 0.f;

  float m = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i)
      m = fmaxf(m, E::Get(xr[j], i));
  m = GroupMax<W>(m, red);
  m = m == -__builtin_inff() ? 0.f : m;

  float sums[3] = {0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float xv = E::Get(xr[j], i);
      const float t = (xv - m) * a.inv_temp * kLog2e;
      const float e = Exp2(t);
      sums[0] += e;
      sums[1] += e == 0.f ? 0.f : e * t;
      if constexpr (REF)
        sums[2] += e == 0.f ? 0.f : e * (xv - E::Get(yr[j], i));
    }
  GroupSum<W>(sums, red);
  const RowStats st = Stats(m, sums[0], sums[1], sums[2], a.inv_temp);

  float kl = 0.f;
  if (REF && WantsKl(a)) {
    const float c = a.inv_temp * kLog2e;
    const float shift = (st.mean_d - st.log_sum) * kLog2e;
    float part[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float xv = E::Get(xr[j], i), yv = E::Get(yr[REF ? j : 0], i);
        const float p = Exp2((xv - m) * a.inv_temp * kLog2e) * st.inv_sum;
        part[0] += KlTerm(p, (xv - yv) * a.inv_temp - st.mean_d, yv - m, c, shift);
      }
    GroupSum<W>(part, red);
    kl = st.empty ? 0.f : KlOf(part[0], st.mean_d);
  }
  const RowGrad rg = FinishRow(a, row, w, st, acted, (xa - m) * a.inv_temp, kl, writer);
  if (!g)
    return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int base = (j * 64 * W + threadIdx.x) * VE;
    if (base >= n)
      break;
    float f[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      f[i] = st.empty ? 0.f
                      : GradTerm<REF>(rg, st, E::Get(xr[j], i), REF ? E::Get(yr[REF ? j : 0], i) : 0.f,
                                      a.inv_temp);
      if (base + i == act && !st.empty)
        f[i] += rg.scale * rg.slope;
    }
    StoreVec<DT>(g, base, n, f);
  }
}

// Rows longer than the registers hold: one pass for the statistics with a
// running maximum per lane, a second for KL and the gradient, from the end of
// the row backwards (its last part is nearest in the caches).
template <int DT, bool REF>
__global__ __launch_bounds__(1024) void LongRowKernel(RowLossParams a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VE = E::kPerVec, W = 16;
  __shared__ float red[W][4];
  const std::int64_t row = a.row0 + blockIdx.x;
  if (OutsideSequences(a, row))
    return;
  const int n = a.vocab;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *y = REF ? static_cast<const T *>(a.y) + row * a.ldy : nullptr;
  T *g = a.g ? static_cast<T *>(a.g) + row * a.ldg : nullptr;
  const bool writer = threadIdx.x == 0;
  const float w = RowWeight(a, row);
  constexpr int kStep = 1024 * VE;
  if (w == 0.f) {
    if (writer)
      ZeroOutputs(a, row);
    const float zero[8] = {};
    if (g)
      for (std::int64_t base = threadIdx.x * VE; base < n; base += kStep)
        StoreVec<DT>(g, static_cast<int>(base), n, zero);
    return;
  }
  const int act = a.actions ? a.actions[row] : -1;
  const bool acted = act >= 0 && act < n;
  const float xa = acted ? E::One(x[act]) : 0.f;

  const float c = a.inv_temp * kLog2e;
  float m = -__builtin_inff(), sums[3] = {0.f, 0.f, 0.f};
  for (std::int64_t b = threadIdx.x * VE; b < n; b += kStep) {
    const int base = static_cast<int>(b);
    const u32x4 xv = LoadVec<DT>(x, base, n);
    u32x4 yv;
    if constexpr (REF)
      yv = LoadVec<DT>(y, base, n);
    float top = m;
#pragma unroll
    for (int i = 0; i < VE; ++i)
      top = fmaxf(top, E::Get(xv, i));
    if (top > m) {
      // Sums over the old maximum as sums over the new: e and t of each term
      // fall by the same step.
      const float step = (m - top) * c, f = Exp2(step);
      if (sums[0] != 0.f)
        sums[1] = f == 0.f ? 0.f : f * (sums[1] + sums[0] * step);
      sums[0] *= f;
      sums[2] = f == 0.f ? 0.f : f * sums[2];
      m = top;
    }
    const float from = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float v = E::Get(xv, i);
      const float t = (v - from) * a.inv_temp * kLog2e;
      const float e = Exp2(t);
      sums[0] += e;
      sums[1] += e == 0.f ? 0.f : e * t;
      if constexpr (REF)
        sums[2] += e == 0.f ? 0.f : e * (v - E::Get(yv, i));
    }
  }
  float top = GroupMax<W>(m, red);
  top = top == -__builtin_inff() ? 0.f : top;
  if (sums[0] != 0.f) {
    const float step = (m - top) * c, f = Exp2(step);
    sums[1] = f == 0.f ? 0.f : f * (sums[1] + sums[0] * step);
    sums[0] *= f;
    sums[2] = f == 0.f ? 0.f : f * sums[2];
  }
  m = top;
  GroupSum<W>(sums, red);
  const RowStats st = Stats(m, sums[0], sums[1], sums[2], a.inv_temp);

  const bool want_kl = REF && WantsKl(a);
  const float za = (xa - m) * a.inv_temp;
  const RowGrad rg = FinishRow(a, row, w, st, acted, za, 0.f, writer && !want_kl);
  if (!g && !want_kl)
    return;
  const float shift = (st.mean_d - st.log_sum) * kLog2e;
  float part[1] = {0.f};
  const std::int64_t steps = (n + kStep - 1) / kStep;
  for (std::int64_t k = steps - 1; k >= 0; --k) {
    const std::int64_t b = k * kStep + threadIdx.x * VE;
    if (b >= n)
      continue;
    const int base = static_cast<int>(b);
    const u32x4 xv = LoadVec<DT>(x, base, n);
    u32x4 yv = {};
    if constexpr (REF)
      yv = LoadVec<DT>(y, base, n);
    float f[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float v = E::Get(xv, i), r = REF ? E::Get(yv, i) : 0.f;
      if constexpr (REF) {
        const float p = Exp2((v - m) * a.inv_temp * kLog2e) * st.inv_sum;
        part[0] += KlTerm(p, (v - r) * a.inv_temp - st.mean_d, r - m, c, shift);
      }
      f[i] = st.empty ? 0.f : GradTerm<REF>(rg, st, v, r, a.inv_temp);
      if (base + i == act && !st.empty)
        f[i] += rg.scale * rg.slope;
    }
    if (g)
      StoreVec<DT>(g, base, n, f);
  }
  if (want_kl) {
    GroupSum<W>(part, red);
    const float kl = st.empty ? 0.f : KlOf(part[0], st.mean_d);
    (void)FinishRow(a, row, w, st, acted, za, kl, writer);
  }
}

// A row's legal moves, one wave per row: at most four entries a lane.  The
// gradient row is put together in LDS, kPart columns at a time: zeros, then
// each entry's value added (moves listed twice add equal values, in any
// order), then the action's, then written out.
constexpr int kPart = 2048;
template <int DT, bool REF>
__global__ __launch_bounds__(64) void MovesRowKernel(RowLossParams a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VE = E::kPerVec, NE = kMaxMoves / 64;
  __shared__ float buf[kPart];
  const std::int64_t row = a.row0 + blockIdx.x;
  if (OutsideSequences(a, row))
    return;
  const int lane = threadIdx.x;
  const int n = a.vocab;
  T *g = a.g ? static_cast<T *>(a.g) + row * a.ldg : nullptr;
  const float w = RowWeight(a, row);
  if (w == 0.f) {
    if (lane == 0)
      ZeroOutputs(a, row);
    const float zero[8] = {};
    if (g)
      for (int base = lane * VE; base < n; base += 64 * VE)
        StoreVec<DT>(g, base, n, zero);
    return;
  }
  std::int64_t start = a.offsets[row], count = a.offsets[row + 1];
  start = start < 0 ? 0 : start > a.n_moves ? a.n_moves : start;
  count = (count > a.n_moves ? a.n_moves : count) - start;
  const int moves = count < 0 ? 0 : count > kMaxMoves ? kMaxMoves : static_cast<int>(count);
  const int act = a.actions ? a.actions[row] : -1;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *y = REF ? static_cast<const T *>(a.y) + row * a.ldy : nullptr;

  int col[NE];
  float xv[NE], yv[NE];
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    const int i = r * 64 + lane;
    col[r] = -1;
    xv[r] = yv[r] = -__builtin_inff();
    if (i < moves) {
      const int k = a.indices[start + i];
      const bool inside = k >= 0 && k < n;
      col[r] = inside ? k : -1;
      xv[r] = inside ? E::One(x[k]) : 0.f;
      if constexpr (REF)
        yv[r] = inside ? E::One(y[k]) : 0.f;
    }
  }
  // The entry of the action (the first of equal ones).
  bool acted = false;
  float xa = 0.f;
  float m = -__builtin_inff();
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    if (r * 64 >= moves)
      break;
    m = fmaxf(m, xv[r]);
    const unsigned long long hit = __ballot(act >= 0 && col[r] == act);
    if (hit && !acted) {
      acted = true;
      xa = __shfl(xv[r], __ffsll(hit) - 1);
    }
  }
  m = wave_max(m);
  m = m == -__builtin_inff() ? 0.f : m;
  float s = 0.f, sz = 0.f, sd = 0.f;
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    if (r * 64 >= moves)
      break;
    const float t = (xv[r] - m) * a.inv_temp * kLog2e;
    const float e = Exp2(t);
    s += e;
    sz += e == 0.f ? 0.f : e * t;
    if constexpr (REF)
      sd += e == 0.f ? 0.f : e * (xv[r] - yv[r]);
  }
  s = wave_sum(s);
  sz = wave_sum(sz);
  if constexpr (REF)
    sd = wave_sum(sd);
  const RowStats st = Stats(m, s, sz, sd, a.inv_temp);
  float kl = 0.f;
  if (REF && WantsKl(a)) {
    const float c = a.inv_temp * kLog2e;
    const float shift = (st.mean_d - st.log_sum) * kLog2e;
#pragma unroll
    for (int r = 0; r < NE; ++r) {
      if (r * 64 >= moves)
        break;
      const float p = Exp2((xv[r] - m) * a.inv_temp * kLog2e) * st.inv_sum;
      kl += KlTerm(p, (xv[r] - yv[r]) * a.inv_temp - st.mean_d, yv[r] - m, c, shift);
    }
    kl = wave_sum(kl);
    kl = st.empty ? 0.f : KlOf(kl, st.mean_d);
  }
  const RowGrad rg = FinishRow(a, row, w, st, acted, (xa - m) * a.inv_temp, kl, lane == 0);
  if (!g)
    return;
  for (int p0 = 0; p0 < n; p0 += kPart) {
    const int width = n - p0 < kPart ? n - p0 : kPart;
    for (int i = lane * 4; i < width; i += 256)
      *reinterpret_cast<f32x4 *>(buf + i) = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    if (!st.empty) {
#pragma unroll
      for (int r = 0; r < NE; ++r) {
        if (r * 64 >= moves)
          break;
        const int k = col[r] - p0;
        if (col[r] >= 0 && k >= 0 && k < width)
          unsafeAtomicAdd(buf + k, GradTerm<REF>(rg, st, xv[r], yv[r], a.inv_temp));
      }
      __syncthreads();
      if (acted && lane == 0 && act >= p0 && act < p0 + width)
        buf[act - p0] += rg.scale * rg.slope;
      __syncthreads();
    }
    for (int base = lane * VE; base < width; base += 64 * VE) {
      float f[VE];
#pragma unroll
      for (int i = 0; i < VE; i += 4)
        *reinterpret_cast<f32x4 *>(f + i) = *reinterpret_cast<const f32x4 *>(buf + base + i);
      StoreVec<DT>(g + p0, base, width, f);
    }
    __syncthreads();
  }
}

template <int DT, bool REF>
void LaunchRows(const RowLossParams &p, unsigned rows, hipStream_t s) {
  constexpr int VE = Elem<DT>::kPerVec;
  const int n = p.vocab;
  const dim3 grid(rows);
  if (p.offsets) {
    hipLaunchKernelGGL((MovesRowKernel<DT, REF>), grid, dim3(64), 0, s, p);
    return;
  }
  if (n <= 64 * VE * 1)
    hipLaunchKernelGGL((DenseRowKernel<DT, 1, 1, REF>), grid, dim3(64), 0, s, p);
  else if (n <= 64 * VE * 2)
    hipLaunchKernelGGL((DenseRowKernel<DT, 1, 2, REF>), grid, dim3(64), 0, s, p);
  else if (n <= 64 * VE * 4)
    hipLaunchKernelGGL((DenseRowKernel<DT, 1, 4, REF>), grid, dim3(64), 0, s, p);
  else if (n <= 256 * VE * 2)
    hipLaunchKernelGGL((DenseRowKernel<DT, 4, 2, REF>), grid, dim3(256), 0, s, p);
  else if (n <= 256 * VE * 4)
    hipLaunchKernelGGL((DenseRowKernel<DT, 4, 4, REF>), grid, dim3(256), 0, s, p);
  else if (n <= 1024 * VE * 4)
    hipLaunchKernelGGL((DenseRowKernel<DT, 16, 4, REF>), grid, dim3(1024), 0, s, p);
  else
    hipLaunchKernelGGL((LongRowKernel<DT, REF>), grid, dim3(1024), 0, s, p);
}

// Sum over the 256 threads of a workgroup, in a fixed order.
__device__ double GroupSum64(double v, double *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void PairLossKernel(PairLossParams a) {
  __shared__ double red[4];
  __shared__ float share[2];
  const std::int64_t pair = blockIdx.x;
  const float w = a.weight ? a.weight[pair] : 1.f;
  std::int64_t begin[2], end[2];
  double sum[2], count[2];
  for (int s = 0; s < 2; ++s) {
    std::int64_t b = a.seq_offsets[2 * pair + s], e = a.seq_offsets[2 * pair + s + 1];
    b = b < 0 ? 0 : b > a.rows ? a.rows : b;
    e = e < b ? b : e > a.rows ? a.rows : e;
    begin[s] = b;
    end[s] = e;
    double t = 0.0, c = 0.0;
    for (std::int64_t r = b + threadIdx.x; r < e; r += 256) {
      const float l = a.mark[r];
      if (l != kNoAction) {
        t += a.ref_logp ? static_cast<double>(l) - a.ref_logp[r] : static_cast<double>(l);
        c += 1.0;
      }
    }
    sum[s] = GroupSum64(t, red);
    count[s] = GroupSum64(c, red);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s)
      if (a.average && count[s] > 0.0)
        sum[s] /= count[s];
    const double beta = a.beta, diff = sum[0] - sum[1], h = beta * diff;
    double loss, slope;  // slope: by the difference of the two sums
    if (a.kind == 0) {
      // ln(1 + e^-h) and ln(1 + e^h) = ln(1 + e^-|h|) + max(0, -+h); sig(h)
      // from the same exponential.
      const double eps = a.smoothing, tail = exp(-fabs(h)), base = log1p(tail);
      const double sig = h >= 0.0 ? 1.0 / (1.0 + tail) : tail / (1.0 + tail);
      const double not_sig = h >= 0.0 ? tail / (1.0 + tail) : 1.0 / (1.0 + tail);
      loss = base + (1.0 - eps) * fmax(-h, 0.0) + eps * fmax(h, 0.0);
      if (h != h)
        loss = h;
      slope = beta * (eps * sig - (1.0 - eps) * not_sig);
    } else if (a.kind == 1) {
      loss = h < 1.0 ? 1.0 - h : h >= 1.0 ? 0.0 : h;
      slope = h < 1.0 ? -beta : h >= 1.0 ? 0.0 : h;
    } else {
      const double r = diff - 0.5 / beta;
      loss = r * r;
      slope = 2.0 * r;
    }
    if (a.loss)
      a.loss[pair] = w == 0.f ? 0.f : static_cast<float>(w * loss);
    if (a.margin)
      a.margin[pair] = w == 0.f ? 0.f : static_cast<float>(h);
    for (int s = 0; s < 2; ++s) {
      const double c = a.average && count[s] > 0.0 ? slope / count[s] : slope;
      share[s] = w == 0.f ? 0.f : static_cast<float>(w * (s == 0 ? c : -c));
    }
  }
  __syncthreads();
  for (int s = 0; s < 2; ++s)
    for (std::int64_t r = begin[s] + threadIdx.x; r < end[s]; r += 256) {
      const bool acted = a.mark[r] != kNoAction;
      if (a.coef)
        a.coef[r] = acted ? share[s] : 0.f;
      if (a.logp)
        a.logp[r] = acted ? a.mark[r] : 0.f;
    }
}

}  // namespace

hipError_t LaunchRowLoss(const RowLossParams &p, hipStream_t stream, std::string *err) {
  if (p.rows < 0 || p.vocab < 1 || (p.rows > 0 && !p.x) || (p.offsets && !p.indices && p.n_moves) ||
      p.vocab > (1 << 30) || (p.offsets && p.vocab > 32768)) {
    if (err)
      *err = "row_loss: needs rows >= 0, 1 <= vocab <= 2^30 (2^15 with move lists) and logits";
    return hipErrorInvalidValue;
  }
  RowLossParams q = p;
  // A launch holds fewer than 2^32 threads.
  constexpr std::int64_t kRows = std::int64_t(1) << 21;
  for (q.row0 = 0; q.row0 < p.rows; q.row0 += kRows) {
    const unsigned rows =
        static_cast<unsigned>(p.rows - q.row0 < kRows ? p.rows - q.row0 : kRows);
    switch (p.dtype * 2 + (p.y ? 1 : 0)) {
    case 2 * DT_F32: LaunchRows<DT_F32, false>(q, rows, stream); break;
    case 2 * DT_F32 + 1: LaunchRows<DT_F32, true>(q, rows, stream); break;
    case 2 * DT_BF16: LaunchRows<DT_BF16, false>(q, rows, stream); break;
    case 2 * DT_BF16 + 1: LaunchRows<DT_BF16, true>(q, rows, stream); break;
    case 2 * DT_F16: LaunchRows<DT_F16, false>(q, rows, stream); break;
    default: LaunchRows<DT_F16, true>(q, rows, stream); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return e;
  }
  return hipSuccess;
}

hipError_t LaunchPairLoss(const PairLossParams &p, hipStream_t stream, std::string *err) {
  if (p.pairs < 0 || p.pairs > (1 << 23) || (p.pairs > 0 && (!p.seq_offsets || (p.rows > 0 && !p.mark)))) {
    if (err)
      *err = "pair_loss: needs 0 <= pairs <= 2^23, offsets and log-probabilities";
    return hipErrorInvalidValue;
  }
  if (p.pairs > 0)
    hipLaunchKernelGGL(PairLossKernel, dim3(static_cast<unsigned>(p.pairs)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mfh
