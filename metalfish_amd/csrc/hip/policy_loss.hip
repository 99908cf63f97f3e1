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

// exp2 on v_exp_f32: 1 ulp, results below 2^-126 are 0.
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Reductions over a wave on the data-parallel paths of the vector unit (six
// dependent instructions; a shuffle through LDS is several times that), the
// result in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float Dpp(float old, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL,
                                                    ROWS, 0xF, false));
}
constexpr int kRowShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;
__device__ __forceinline__ float LastLane(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float WaveSum(float v) {
  v += Dpp<kRowShr + 1, 0xF>(0.f, v);
  v += Dpp<kRowShr + 2, 0xF>(0.f, v);
  v += Dpp<kRowShr + 4, 0xF>(0.f, v);
  v += Dpp<kRowShr + 8, 0xF>(0.f, v);
  v += Dpp<kBcast15, 0xA>(0.f, v);
  v += Dpp<kBcast31, 0xC>(0.f, v);
  return LastLane(v);
}
__device__ __forceinline__ float WaveMax(float v) {
  v = fmaxf(v, Dpp<kRowShr + 1, 0xF>(v, v));
  v = fmaxf(v, Dpp<kRowShr + 2, 0xF>(v, v));
  v = fmaxf(v, Dpp<kRowShr + 4, 0xF>(v, v));
  v = fmaxf(v, Dpp<kRowShr + 8, 0xF>(v, v));
  v = fmaxf(v, Dpp<kBcast15, 0xA>(v, v));
  v = fmaxf(v, Dpp<kBcast31, 0xC>(v, v));
  return LastLane(v);
}

// The same over the first W lanes (W = 4 or 16), which hold one value of each
// wave.
template <int W>
__device__ __forceinline__ float LanesSum(float v) {
  v += Dpp<kRowShr + 1, 0xF>(0.f, v);
  v += Dpp<kRowShr + 2, 0xF>(0.f, v);
  if constexpr (W == 16) {
    v += Dpp<kRowShr + 4, 0xF>(0.f, v);
    v += Dpp<kRowShr + 8, 0xF>(0.f, v);
  }
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), W - 1));
}
template <int W>
__device__ __forceinline__ float LanesMax(float v) {
  v = fmaxf(v, Dpp<kRowShr + 1, 0xF>(v, v));
  v = fmaxf(v, Dpp<kRowShr + 2, 0xF>(v, v));
  if constexpr (W == 16) {
    v = fmaxf(v, Dpp<kRowShr + 4, 0xF>(v, v));
    v = fmaxf(v, Dpp<kRowShr + 8, 0xF>(v, v));
  }
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), W - 1));
}

// Sums of N values over the W waves of a workgroup.
template <int W, int N>
__device__ __forceinline__ void GroupSum(float (&v)[N], float (*red)[4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] = WaveSum(v[i]);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        red[threadIdx.x >> 6][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = LanesSum<W>(red[threadIdx.x & (W - 1)][i]);
  }
}

template <int W>
__device__ __forceinline__ float GroupMax(float v, float (*red)[4]) {
  v = WaveMax(v);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
      red[threadIdx.x >> 6][0] = v;
    __syncthreads();
    v = LanesMax<W>(red[threadIdx.x & (W - 1)][0]);
  }
  return v;
}

// What a row's scalars come to, from its statistics.
struct RowStats {
  float m;         // maximum (0 where every entry is masked)
  float log_sum;   // ln S
  float log2_sum;  // log2 S
  float mean_z;    // E_p z
  float mean_d;    // E_p d
  bool empty;      // no entry left
};

// sums: of e, of e log2(e) and of e (x - y).
__device__ __forceinline__ RowStats Stats(float m, const float (&sums)[3], float inv_temp) {
  RowStats r;
  r.m = m;
  r.empty = sums[0] == 0.f;
  const float sum = r.empty ? 1.f : sums[0], inv = 1.f / sum;
  r.log_sum = logf(sum);
  r.log2_sum = r.log_sum * kLog2e;
  r.mean_z = sums[1] * kLn2 * inv;
  r.mean_d = sums[2] * inv_temp * inv;
  return r;
}

// One entry's part of the statistics, t = log2(e).  GUARD: an entry whose e is
// 0 adds nothing, also where its logits are infinite.  Rows without such
// entries are summed without the guard, and again with it if a sum comes out
// NaN (0 times infinity): it costs two of nine instructions.
template <bool REF, bool GUARD>
__device__ __forceinline__ void AddStats(float x, float y, float m, float c, float (&s)[3]) {
  const float t = (x - m) * c, e = Exp2(t);
  s[0] += e;
  s[1] += GUARD && e == 0.f ? 0.f : e * t;
  if constexpr (REF)
    s[2] += GUARD && e == 0.f ? 0.f : e * (x - y);
}

__device__ __forceinline__ bool NeedsGuard(const float (&s)[3]) {
  return s[1] != s[1] || s[2] != s[2];
}

// Coefficients of one row's gradient
//   scale (slope 1[k = a] + p_k (kl u_k + entropy (z_k - E_p z) - slope)).
struct RowGrad {
  float scale, slope, kl, entropy;
};

// The same for p_k (a (x_k - m) + b u_k + d), with what p and u need.
struct Coefs {
  float m, c, shift, inv_temp, mean_d, kl_shift, a, b, d;
};

__device__ __forceinline__ Coefs CoefsOf(const RowStats &st, const RowGrad &g, float inv_temp) {
  Coefs k;
  k.m = st.m;
  k.c = inv_temp * kLog2e;
  k.shift = -st.log2_sum;
  k.inv_temp = inv_temp;
  k.mean_d = st.mean_d;
  k.kl_shift = st.mean_d * kLog2e - st.log2_sum;
  k.a = g.scale * g.entropy * inv_temp;
  k.b = g.scale * g.kl;
  k.d = -g.scale * (g.slope + g.entropy * st.mean_z);
  return k;
}

// (exp(-u) - 1 + u) / u^2 for |u| <= 2: its interpolation of degree 8 in the
// Chebyshev nodes there, 1.6e-7 from it relative (3.0e-7 with the roundings).
__device__ __forceinline__ float KlSeries(float u) {
  float r = 0x1.3cbf98p-22f;
  r = r * u - 0x1.91528cp-19f;
  r = r * u + 0x1.9f1d2ap-16f;
  r = r * u - 0x1.9e9c00p-13f;
  r = r * u + 0x1.6c1b2ap-10f;
  r = r * u - 0x1.1117bcp-7f;
  r = r * u + 0x1.55554ap-5f;
  r = r * u - 0x1.555536p-3f;
  return r * u + 0x1.000000p-1f;
}

// p (exp(-u) - 1 + u), the term of KL, for any u; ym: the reference logit less
// the policy's maximum.  Far below 0, where exp(-u) may overflow against a
// tiny p, their product comes from ym; an entry that is masked here adds
// nothing but its reference probability.
__device__ __forceinline__ float KlTerm(const Coefs &k, float p, float u, float ym) {
  if (!(u > -60.f)) {
    const float q = Exp2(ym * k.c + k.kl_shift);
    return p == 0.f ? q : q - p * (1.f - u);
  }
  if (p == 0.f)
    return 0.f;
  return fabsf(u) <= 2.f ? p * u * u * KlSeries(u) : p * (Exp2(-u * kLog2e) - 1.f + u);
}

// KL from the sum of its terms; infinite where the reference lacks what the
// policy plays (E_p d is, and no term then means anything).
__device__ __forceinline__ float KlOf(float terms, float mean_d) {
  return mean_d == __builtin_inff() ? mean_d : log1pf(terms);
}

// The gradient of N entries without the action's own term, and their part of
// KL.  The terms of KL take the series unless an entry of the wave needs more.
template <int N, bool REF, bool GUARD>
__device__ __forceinline__ void FinishEntries(const Coefs &k, bool want_kl, const float (&x)[N],
                                              const float (&y)[N], float &kl, float (&f)[N]) {
  float p[N], u[N], top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float xm = x[i] - k.m;
    p[i] = Exp2(xm * k.c + k.shift);
    float v = k.a * xm + k.d;
    if constexpr (REF) {
      u[i] = (x[i] - y[i]) * k.inv_temp - k.mean_d;
      top = fmaxf(top, fabsf(u[i]));
      v = k.b * u[i] + v;
    }
    f[i] = GUARD && p[i] == 0.f ? 0.f : p[i] * v;
  }
  if (REF && want_kl) {
    if (GUARD || __any(!(top <= 2.f))) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        kl += KlTerm(k, p[i], u[i], y[i] - k.m);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        kl += p[i] * (u[i] * u[i]) * KlSeries(u[i]);
    }
  }
}

// Whether the divergence itself is asked for (its gradient needs no KL).
__device__ __forceinline__ bool WantsKl(const RowLossParams &a) {
  return a.kl || (a.loss && a.kl_coef != 0.f);
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

// A row's scalars once its statistics are there: the coefficients of its
// gradient, and what WriteRow needs.
struct RowResult {
  RowGrad grad;
  float logp, surrogate, entropy;
};
__device__ __forceinline__ RowResult Evaluate(const RowLossParams &a, std::int64_t row, float w,
                                              const RowStats &st, bool acted, float xa) {
  RowResult r{{w * a.inv_temp, 0.f, 0.f, 0.f}, 0.f, 0.f, 0.f};
  if (acted)
    r.logp = (xa - st.m) * a.inv_temp - st.log_sum;
  if (a.coef) {
    r.grad.slope = acted ? 1.f : 0.f;
    return r;
  }
  if (acted && a.advantage) {
    const Surrogate s = Clipped(a, row, r.logp);
    r.surrogate = s.loss;
    r.grad.slope = s.slope;
  }
  r.entropy = st.log_sum - st.mean_z;
  r.grad.kl = a.kl_coef;
  r.grad.entropy = a.entropy_coef;
  return r;
}

__device__ __forceinline__ void WriteRow(const RowLossParams &a, std::int64_t row, float w,
                                         bool acted, const RowResult &r, float kl) {
  if (a.coef)
    return;
  if (a.mark) {
    a.mark[row] = acted ? r.logp : kNoAction;
    return;
  }
  float loss = r.surrogate;
  if (a.kl_coef != 0.f)
    loss += a.kl_coef * kl;
  if (a.entropy_coef != 0.f)
    loss -= a.entropy_coef * r.entropy;
  if (a.loss)
    a.loss[row] = w * loss;
  if (a.logp)
    a.logp[row] = r.logp;
  if (a.kl)
    a.kl[row] = kl;
  if (a.entropy)
    a.entropy[row] = r.entropy;
}

// A row without an entry, or of weight 0.
__device__ __forceinline__ void WriteZeros(const RowLossParams &a, std::int64_t row) {
  if (a.mark)
    a.mark[row] = kNoAction;
  if (a.loss)
    a.loss[row] = 0.f;
  if (a.logp)
    a.logp[row] = 0.f;
  if (a.kl)
    a.kl[row] = 0.f;
  if (a.entropy)
    a.entropy[row] = 0.f;
}

__device__ __forceinline__ bool OutsideSequences(const RowLossParams &a, std::int64_t row) {
  return a.seq_offsets && (row < a.seq_offsets[0] || row >= a.seq_offsets[a.n_seq]);
}

// The factor on a row's outputs; 0: the row is not read.
__device__ __forceinline__ float RowWeight(const RowLossParams &a, std::int64_t row) {
  return a.coef ? a.coef[row] : a.weight ? a.weight[row] : 1.f;
}

// Zeros in a whole gradient row, by `threads` threads.
template <int DT>
__device__ __forceinline__ void ZeroRow(typename Elem<DT>::T *g, int n, int thread, int threads) {
  using E = Elem<DT>;
  const int vecs = n / E::kPerVec;
  for (int v = thread; v < vecs; v += threads)
    *reinterpret_cast<typename E::V *>(g + static_cast<std::int64_t>(v) * E::kPerVec) =
        u32x4{0, 0, 0, 0};
  const int t = vecs * E::kPerVec + thread;
  if (thread < E::kPerVec && t < n)
    g[t] = 0;
}

// Keeps the compiler from holding a register's elements unpacked from one
// pass over them to the next.
__device__ __forceinline__ void Repack(u32x4 &v) { asm volatile("" : "+v"(v)); }

template <int DT>
__device__ __forceinline__ void Unpack(u32x4 v, float (&x)[Elem<DT>::kPerVec]) {
#pragma unroll
  for (int i = 0; i < Elem<DT>::kPerVec; ++i)
    x[i] = Elem<DT>::Get(v, i);
}

// A whole row in the registers of W waves, NV vectors of 16 bytes a lane; the
// elements behind the last whole vector, one to a lane, in a register more.
// Three passes over the registers: maximum, sums, gradient with KL.  Four rows
// to a workgroup where a wave has one to itself.
template <int DT, int W, int NV, bool REF>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void DenseRowKernel(RowLossParams a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VE = E::kPerVec;
  __shared__ float red[W][4];
  const int tid = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  std::int64_t row = blockIdx.x;
  if constexpr (W == 1)
    row = row * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  row += a.row0;
  if (row >= a.rows || OutsideSequences(a, row))
    return;
  const int n = a.vocab, vecs = n / VE, rest = n - vecs * VE;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *y = REF ? static_cast<const T *>(a.y) + row * a.ldy : nullptr;
  T *g = a.g ? static_cast<T *>(a.g) + row * a.ldg : nullptr;
  const float w = RowWeight(a, row);
  if (w == 0.f) {
    if (tid == 0)
      WriteZeros(a, row);
    if (g)
      ZeroRow<DT>(g, n, tid, 64 * W);
    return;
  }
  const int act = a.actions ? a.actions[row] : -1;
  bool acted = act >= 0 && act < n;
  const float xa = acted ? E::One(x[act]) : 0.f;
  const float ya = REF && acted ? E::One(y[act]) : 0.f;
  u32x4 xr[NV], yr[REF ? NV : 1];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = j * 64 * W + tid;
    if (v < vecs)
      xr[j] = *reinterpret_cast<const typename E::V *>(x + v * VE);
  }
  if constexpr (REF) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = j * 64 * W + tid;
      if (v < vecs)
        yr[j] = *reinterpret_cast<const typename E::V *>(y + v * VE);
    }
  }
  const bool has_rest = tid < rest;
  const float xt[1] = {has_rest ? E::One(x[vecs * VE + tid]) : -__builtin_inff()};
  const float yt[1] = {REF && has_rest ? E::One(y[vecs * VE + tid]) : 0.f};

  float m = xt[0];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (j * 64 * W + tid < vecs) {
      float xs[VE];
      Unpack<DT>(xr[j], xs);
#pragma unroll
      for (int i = 0; i < VE; ++i)
        m = fmaxf(m, xs[i]);
    }
  m = GroupMax<W>(m, red);
  m = m == -__builtin_inff() ? 0.f : m;

  const float c = a.inv_temp * kLog2e;
  float sums[3];
  const auto sum = [&](auto guard) {
    constexpr bool GUARD = decltype(guard)::value;
    sums[0] = sums[1] = sums[2] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Repack(xr[j]);
      if (REF)
        Repack(yr[REF ? j : 0]);
      if (j * 64 * W + tid < vecs) {
        float xs[VE], ys[VE] = {};
        Unpack<DT>(xr[j], xs);
        if constexpr (REF)
          Unpack<DT>(yr[j], ys);
#pragma unroll
        for (int i = 0; i < VE; ++i)
          AddStats<REF, GUARD>(xs[i], ys[i], m, c, sums);
      }
    }
    if (has_rest)
      AddStats<REF, GUARD>(xt[0], yt[0], m, c, sums);
    GroupSum<W>(sums, red);
  };
  sum(std::false_type{});
  const bool guarded = NeedsGuard(sums);
  if (guarded)
    sum(std::true_type{});
  const RowStats st = Stats(m, sums, a.inv_temp);
  if (st.empty) {
    if (tid == 0)
      WriteZeros(a, row);
    if (g)
      ZeroRow<DT>(g, n, tid, 64 * W);
    return;
  }
  const RowResult res = Evaluate(a, row, w, st, acted, xa);
  const bool want_kl = REF && WantsKl(a);
  float kl[1] = {0.f};
  if (g || want_kl) {
    const Coefs k = CoefsOf(st, res.grad, a.inv_temp);
    const auto finish = [&](auto guard) {
      constexpr bool GUARD = decltype(guard)::value;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Repack(xr[j]);
        if (REF)
          Repack(yr[REF ? j : 0]);
        const int v = j * 64 * W + tid;
        if (v < vecs) {
          float xs[VE], ys[VE] = {}, f[VE];
          Unpack<DT>(xr[j], xs);
          if constexpr (REF)
            Unpack<DT>(yr[j], ys);
          FinishEntries<VE, REF, GUARD>(k, want_kl, xs, ys, kl[0], f);
          if (g)
            *reinterpret_cast<typename E::V *>(g + v * VE) = E::Pack(f);
        }
      }
      float ft[1];
      if (has_rest) {
        FinishEntries<1, REF, GUARD>(k, want_kl, xt, yt, kl[0], ft);
        if (g)
          g[vecs * VE + tid] = E::Round(ft[0]);
      }
      // The action's own term, by the thread that wrote its column.
      const int v = act / VE;
      if (g && acted && tid == (v < vecs ? v % (64 * W) : act - vecs * VE)) {
        float none = 0.f;
        const float xs[1] = {xa}, ys[1] = {ya};
        FinishEntries<1, REF, GUARD>(k, false, xs, ys, none, ft);
        g[act] = E::Round(ft[0] + res.grad.scale * res.grad.slope);
      }
    };
    if (guarded)
      finish(std::true_type{});
    else
      finish(std::false_type{});
    if (want_kl) {
      GroupSum<W>(kl, red);
      kl[0] = KlOf(kl[0], st.mean_d);
    }
  }
  if (tid == 0)
    WriteRow(a, row, w, acted, res, kl[0]);
}

// Rows longer than the registers hold: one pass for the statistics with a
// running maximum per lane, a second for KL and the gradient, from the end of
// the row backwards (its last part is nearest in the caches).
template <int DT, bool REF>
__global__ __launch_bounds__(1024) void LongRowKernel(RowLossParams a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VE = E::kPerVec, W = 16, kThreads = 64 * W;
  __shared__ float red[W][4];
  const std::int64_t row = a.row0 + blockIdx.x;
  if (OutsideSequences(a, row))
    return;
  const int tid = threadIdx.x;
  const int n = a.vocab, vecs = n / VE, rest = n - vecs * VE;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *y = REF ? static_cast<const T *>(a.y) + row * a.ldy : nullptr;
  T *g = a.g ? static_cast<T *>(a.g) + row * a.ldg : nullptr;
  const float w = RowWeight(a, row);
  if (w == 0.f) {
    if (tid == 0)
      WriteZeros(a, row);
    if (g)
      ZeroRow<DT>(g, n, tid, kThreads);
    return;
  }
  const int act = a.actions ? a.actions[row] : -1;
  const bool acted = act >= 0 && act < n;
  const float xa = acted ? E::One(x[act]) : 0.f;
  const float ya = REF && acted ? E::One(y[act]) : 0.f;
  const bool has_rest = tid < rest;
  const float xt[1] = {has_rest ? E::One(x[vecs * VE + tid]) : -__builtin_inff()};
  const float yt[1] = {REF && has_rest ? E::One(y[vecs * VE + tid]) : 0.f};

  const float c = a.inv_temp * kLog2e;
  float m = xt[0], sums[3] = {0.f, 0.f, 0.f};
  // Sums over the old maximum as sums over the new: e and t of each term fall
  // by the same step.
  const auto rescale = [&](float from, float to) {
    if (sums[0] == 0.f)
      return;
    const float step = (from - to) * c, f = Exp2(step);
    sums[1] = f == 0.f ? 0.f : f * (sums[1] + sums[0] * step);
    sums[0] *= f;
    sums[2] = f == 0.f ? 0.f : f * sums[2];
  };
  if (has_rest)
    AddStats<REF, true>(xt[0], yt[0], m == -__builtin_inff() ? 0.f : m, c, sums);
  for (int v = tid; v < vecs; v += kThreads) {
    float xs[VE], ys[VE] = {};
    Unpack<DT>(*reinterpret_cast<const typename E::V *>(x + static_cast<std::int64_t>(v) * VE), xs);
    if constexpr (REF)
      Unpack<DT>(*reinterpret_cast<const typename E::V *>(y + static_cast<std::int64_t>(v) * VE),
                 ys);
    float top = m;
#pragma unroll
    for (int i = 0; i < VE; ++i)
      top = fmaxf(top, xs[i]);
    if (top > m) {
      rescale(m, top);
      m = top;
    }
    const float from = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int i = 0; i < VE; ++i)
      AddStats<REF, true>(xs[i], ys[i], from, c, sums);
  }
  float top = GroupMax<W>(m, red);
  top = top == -__builtin_inff() ? 0.f : top;
  rescale(m, top);
  m = top;
  GroupSum<W>(sums, red);
  const RowStats st = Stats(m, sums, a.inv_temp);
  if (st.empty) {
    if (tid == 0)
      WriteZeros(a, row);
    if (g)
      ZeroRow<DT>(g, n, tid, kThreads);
    return;
  }
  const RowResult res = Evaluate(a, row, w, st, acted, xa);
  const bool want_kl = REF && WantsKl(a);
  float kl[1] = {0.f};
  if (g || want_kl) {
    const Coefs k = CoefsOf(st, res.grad, a.inv_temp);
    const int steps = (vecs + kThreads - 1) / kThreads;
    for (int j = steps - 1; j >= 0; --j) {
      const std::int64_t v = static_cast<std::int64_t>(j) * kThreads + tid;
      if (v >= vecs)
        continue;
      float xs[VE], ys[VE] = {}, f[VE];
      Unpack<DT>(*reinterpret_cast<const typename E::V *>(x + v * VE), xs);
      if constexpr (REF)
        Unpack<DT>(*reinterpret_cast<const typename E::V *>(y + v * VE), ys);
      FinishEntries<VE, REF, true>(k, want_kl, xs, ys, kl[0], f);
      if (g)
        *reinterpret_cast<typename E::V *>(g + v * VE) = E::Pack(f);
    }
    float ft[1];
    if (has_rest) {
      FinishEntries<1, REF, true>(k, want_kl, xt, yt, kl[0], ft);
      if (g)
        g[vecs * VE + tid] = E::Round(ft[0]);
    }
    const int v = act / VE;
    if (g && acted && tid == (v < vecs ? v % kThreads : act - vecs * VE)) {
      float none = 0.f;
      const float xs[1] = {xa}, ys[1] = {ya};
      FinishEntries<1, REF, true>(k, false, xs, ys, none, ft);
      g[act] = E::Round(ft[0] + res.grad.scale * res.grad.slope);
    }
    if (want_kl) {
      GroupSum<W>(kl, red);
      kl[0] = KlOf(kl[0], st.mean_d);
    }
  }
  if (tid == 0)
    WriteRow(a, row, w, acted, res, kl[0]);
}

// A row's legal moves, one wave per row and four rows per workgroup, at most
// four entries a lane.  The gradient row is zeros but for the entries: the
// zeros are written while the logits are on their way, the entries over them
// afterwards (a wave's stores reach an address in order).  A move listed twice
// adds up: a bit per column finds such rows, where the first of equal entries
// writes for all.
template <int DT, bool REF>
__global__ __launch_bounds__(256) void MovesRowKernel(RowLossParams a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int NE = kMaxMoves / 64;
  extern __shared__ std::uint32_t seen_all[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::int64_t row = a.row0 + static_cast<std::int64_t>(blockIdx.x) * 4 + wave;
  if (row >= a.rows || OutsideSequences(a, row))
    return;
  const int n = a.vocab, words = (n + 31) / 32;
  std::uint32_t *seen = seen_all + wave * words;
  T *g = a.g ? static_cast<T *>(a.g) + row * a.ldg : nullptr;
  const float w = RowWeight(a, row);
  if (w == 0.f) {
    if (lane == 0)
      WriteZeros(a, row);
    if (g)
      ZeroRow<DT>(g, n, lane, 64);
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
    if (i < moves) {
      const int k = a.indices[start + i];
      col[r] = k >= 0 && k < n ? k : -1;
    }
  }
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    const bool in = r * 64 + lane < moves, inside = col[r] >= 0;
    xv[r] = inside ? E::One(x[col[r]]) : in ? 0.f : -__builtin_inff();
    if constexpr (REF)
      yv[r] = inside ? E::One(y[col[r]]) : in ? 0.f : -__builtin_inff();
  }
  bool twice = false;
  if (g) {
    ZeroRow<DT>(g, n, lane, 64);
    for (int i = lane; i < words; i += 64)
      seen[i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int r = 0; r < NE; ++r) {
      if (r * 64 >= moves)
        break;
      bool again = false;
      if (col[r] >= 0) {
        const std::uint32_t bit = 1u << (col[r] & 31);
        again = atomicOr(seen + (col[r] >> 5), bit) & bit;
      }
      twice = twice || __any(again);
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
  m = WaveMax(m);
  m = m == -__builtin_inff() ? 0.f : m;
  const float c = a.inv_temp * kLog2e;
  float sums[3] = {0.f, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    if (r * 64 >= moves)
      break;
    AddStats<REF, true>(xv[r], REF ? yv[r] : 0.f, m, c, sums);
  }
  GroupSum<1>(sums, nullptr);
  const RowStats st = Stats(m, sums, a.inv_temp);
  if (st.empty) {
    if (lane == 0)
      WriteZeros(a, row);
    return;  // the gradient's zeros are written
  }
  const RowResult res = Evaluate(a, row, w, st, acted, xa);
  const bool want_kl = REF && WantsKl(a);
  float kl[1] = {0.f};
  if (g || want_kl) {
    const Coefs k = CoefsOf(st, res.grad, a.inv_temp);
    float f[NE];
#pragma unroll
    for (int r = 0; r < NE; ++r) {
      if (r * 64 >= moves)
        break;
      const float xs[1] = {xv[r]}, ys[1] = {REF ? yv[r] : 0.f};
      float ft[1];
      FinishEntries<1, REF, true>(k, want_kl, xs, ys, kl[0], ft);
      f[r] = ft[0];
    }
    if (g) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (!twice) {
#pragma unroll
        for (int r = 0; r < NE; ++r) {
          if (r * 64 >= moves)
            break;
          if (col[r] >= 0)
            g[col[r]] = E::Round(col[r] == act ? f[r] + res.grad.scale * res.grad.slope : f[r]);
        }
      } else {
        for (int r = 0; r * 64 < moves; ++r) {
          float times = 0.f;
          bool first = true;
          const int mine = r == 0 ? col[0] : r == 1 ? col[1] : r == 2 ? col[2] : col[3];
          const float value = r == 0 ? f[0] : r == 1 ? f[1] : r == 2 ? f[2] : f[3];
          for (int i = 0; i < moves; ++i) {
            const int q = i >> 6;
            const int other =
                __shfl(q == 0 ? col[0] : q == 1 ? col[1] : q == 2 ? col[2] : col[3], i & 63);
            if (other == mine) {
              times += 1.f;
              first = first && i >= r * 64 + lane;
            }
          }
          if (mine >= 0 && first)
            g[mine] = E::Round(mine == act ? times * value + res.grad.scale * res.grad.slope
                                           : times * value);
        }
      }
    }
    if (want_kl) {
      GroupSum<1>(kl, nullptr);
      kl[0] = KlOf(kl[0], st.mean_d);
    }
  }
  if (lane == 0)
    WriteRow(a, row, w, acted, res, kl[0]);
}

template <int DT, bool REF, int W, int NV>
void LaunchDense(const RowLossParams &p, unsigned rows, hipStream_t s) {
  if constexpr (W == 1)
    hipLaunchKernelGGL((DenseRowKernel<DT, 1, NV, REF>), dim3((rows + 3) / 4), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((DenseRowKernel<DT, W, NV, REF>), dim3(rows), dim3(64 * W), 0, s, p);
}

template <int DT, bool REF>
void LaunchRows(const RowLossParams &p, unsigned rows, hipStream_t s) {
  constexpr int VE = Elem<DT>::kPerVec;
  constexpr int WIDE = VE == 4 ? 8 : 4;  // vectors of a lane that hold 2048 columns
  if (p.offsets) {
    const unsigned bits = 4 * ((p.vocab + 31) / 32) * sizeof(std::uint32_t);
    hipLaunchKernelGGL((MovesRowKernel<DT, REF>), dim3((rows + 3) / 4), dim3(256), p.g ? bits : 0,
                       s, p);
    return;
  }
  const int vecs = p.vocab / VE;
  if (vecs <= 64)
    LaunchDense<DT, REF, 1, 1>(p, rows, s);
  else if (vecs <= 128)
    LaunchDense<DT, REF, 1, 2>(p, rows, s);
  else if (vecs <= 64 * WIDE / 2)
    LaunchDense<DT, REF, 1, WIDE / 2>(p, rows, s);
  else if (vecs <= 64 * WIDE)
    LaunchDense<DT, REF, 1, WIDE>(p, rows, s);
  else if (vecs <= 256 * 4)
    LaunchDense<DT, REF, 4, 4>(p, rows, s);
  else if (vecs <= 1024 * 4)
    LaunchDense<DT, REF, 16, 4>(p, rows, s);
  else if (vecs <= 1024 * 8)
    LaunchDense<DT, REF, 16, 8>(p, rows, s);
  else
    hipLaunchKernelGGL((LongRowKernel<DT, REF>), dim3(rows), dim3(1024), 0, s, p);
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
