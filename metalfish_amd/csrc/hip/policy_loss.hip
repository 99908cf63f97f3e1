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
// Every statistic is fp32; a gradient is rounded once, to its type.  x (and y)
// are read once, held in registers in their own type, and the gradient is
// written from there (rows longer than 8192 vectors of 16 bytes are read a
// second time).  What bounds it:
//  * fp32, or no reference: memory.  16384 x 1858 fp32 with a reference 60.4 us
//    (365 MB, 6.0 TB/s); 3588 x 32000 bf16: statistics 39.5 us (5.8 TB/s),
//    gradient 78 (5.9 TB/s).
//  * 16 bits with a reference and KL: the vector unit, about 44 instructions an
//    entry, three of them exponentials: 16384 x 1858 bf16 48 us (3.8 TB/s), 1500
//    x 50021 131 us (3.4 TB/s; the vector unit busy two thirds of it).
//  * move lists: the zeros around the entries, and lines of 128 bytes for
//    gathered logits: 20011 rows of 1858 bf16 20.8 us (74 MB written, about 50
//    MB of lines read).
//  * few rows: the launch and the loads that wait on one another, 5.0 us for 16
//    rows of moves.
#include "mfh_device.h"
#include "mfh_kernels.h"

namespace mfh {
namespace {

constexpr float kLog2e = 1.44269504f;
constexpr float kLog2eLow = 1.92596299e-8f;  // log2(e) - kLog2e
constexpr float kLn2 = 0.69314718f;
constexpr int kMaxMoves = 256;
constexpr unsigned kCus = 256;
// Whole rows of up to 256 vectors: four waves each up to this many rows, one
// each above.  1858 columns of bf16 with a reference: 64 rows 5.7 us on four
// waves, 7.2 on one; 512 rows 6.5 and 7.5; 2048 rows 14.1 and 12.4; 16384 rows
// 62.9 and 47.3.
constexpr unsigned kFewRows = 1024;
// Calls whose arrays hold more bytes than this go past the caches.  1858
// columns of fp32 with a reference: 512 rows (11 MB) 6.8 us through the caches,
// 7.1 past them; 1024 rows 9.9 and 9.2, 2048 rows 14.1 and 12.8; 20011 rows of
// moves in bf16 27.5 and 21, 3588 x 32000 bf16 (statistics, fastest runs)
// 57.7 and 48.7.
constexpr double kPastBytes = 16e6;

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

// Rows of an array of elements, in global memory.
template <int DT> using Row = MFH_GLOBAL typename Elem<DT>::T *;
template <int DT> using ConstRow = const MFH_GLOBAL typename Elem<DT>::T *;
template <int DT>
__device__ __forceinline__ ConstRow<DT> RowOf(const void *p, std::int64_t row, std::int64_t stride) {
  return (ConstRow<DT>)p + row * stride;
}
template <int DT>
__device__ __forceinline__ Row<DT> RowOf(void *p, std::int64_t row, std::int64_t stride) {
  return (Row<DT>)p + row * stride;
}

// A row's vectors, through the caches or (PAST, large calls) past them.
template <int DT, bool PAST>
__device__ __forceinline__ u32x4 LoadVec(ConstRow<DT> p) {
  const auto *v = (const MFH_GLOBAL typename Elem<DT>::V *)p;
  if constexpr (PAST)
    return __builtin_nontemporal_load(v);
  else
    return *v;
}
template <int DT, bool PAST>
__device__ __forceinline__ void StoreVec(Row<DT> p, u32x4 value) {
  auto *v = (MFH_GLOBAL typename Elem<DT>::V *)p;
  if constexpr (PAST)
    __builtin_nontemporal_store(static_cast<typename Elem<DT>::V>(value), v);
  else
    *v = value;
}

// Row scalars, on the vector unit's own exponential, logarithm and reciprocal
// (1 ulp each): every wave computes them for its one row, so their length
// counts.
__device__ __forceinline__ float Rcp(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float Log2(float x) { return __builtin_amdgcn_logf(x); }

// e^x: x log2(e) in two parts, the lower one applied to first order.
__device__ __forceinline__ float Exp(float x) {
  const float h = x * kLog2e;
  const float l = __builtin_fmaf(x, kLog2e, -h) + x * kLog2eLow;
  const float r = Exp2(h);
  // l is NaN where h is infinite, and r then is 0 or infinite.
  return r > 0.f && r < __builtin_inff() ? r + r * (l * kLn2) : r;
}

// ln(1 + z) for z >= 0: 2 atanh(s), s = z / (2 + z) <= 1/5, by its series below
// z = 1/2 (the first term left out is 3e-10 of the sum).
__device__ __forceinline__ float Log1p(float z) {
  if (!(z < 0.5f))
    return Log2(1.f + z) * kLn2;
  const float s = z * Rcp(2.f + z), q = s * s;
  return 2.f * s * (1.f + q * (1.f / 3 + q * (1.f / 5 + q * (1.f / 7 + q * (1.f / 9 + q / 11)))));
}

// A value that is the same in the whole wave, in a scalar register.
__device__ __forceinline__ float Scalar(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

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

// The same over the first W lanes (4, 8 or 16), which hold one value of each
// wave.
template <int W>
__device__ __forceinline__ float LanesSum(float v) {
  v += Dpp<kRowShr + 1, 0xF>(0.f, v);
  v += Dpp<kRowShr + 2, 0xF>(0.f, v);
  if constexpr (W >= 8)
    v += Dpp<kRowShr + 4, 0xF>(0.f, v);
  if constexpr (W >= 16)
    v += Dpp<kRowShr + 8, 0xF>(0.f, v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), W - 1));
}
template <int W>
__device__ __forceinline__ float LanesMax(float v) {
  v = fmaxf(v, Dpp<kRowShr + 1, 0xF>(v, v));
  v = fmaxf(v, Dpp<kRowShr + 2, 0xF>(v, v));
  if constexpr (W >= 8)
    v = fmaxf(v, Dpp<kRowShr + 4, 0xF>(v, v));
  if constexpr (W >= 16)
    v = fmaxf(v, Dpp<kRowShr + 8, 0xF>(v, v));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), W - 1));
}

// Sums of N values over the W waves of a workgroup.
template <int W, int N>
__device__ __forceinline__ void GroupSum(float (&v)[N], float (*red)[8]) {
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

// Sums over a row's entries: of e, of e log2(e), of e d with d = x - y; and the
// greatest |d|, or with the guards the greatest y.
struct Sums {
  float e, et, ed, far;
};
template <bool GUARD> __device__ __forceinline__ Sums NoSums() {
  return {0.f, 0.f, 0.f, GUARD ? -__builtin_inff() : 0.f};
}

// One entry's part, t = log2(e).  GUARD: an entry whose e is 0 adds nothing,
// also where its logits are infinite.  Rows without such entries are summed
// without the guard, and again with it if a sum comes out NaN (0 times
// infinity): it costs two of nine instructions.
template <bool REF, bool GUARD>
__device__ __forceinline__ void AddStats(float x, float y, float m, float c, Sums &s) {
  const float t = (x - m) * c, e = Exp2(t);
  s.e += e;
  s.et += GUARD && e == 0.f ? 0.f : e * t;
  if constexpr (REF) {
    const float d = x - y;
    s.ed += GUARD && e == 0.f ? 0.f : e * d;
    s.far = fmaxf(s.far, GUARD ? y : fabsf(d));
  }
}

// Over the W waves of a workgroup, each of which has summed relative to its own
// maximum `top` (0 where that is -inf): one exchange, and the sums relative to
// the row's maximum, which is returned (0 for -inf).  Relative to a maximum
// higher by `step` in log2 units every e falls by exp2(step) and every log2(e)
// by step.  A wave whose entries all vanish that way adds nothing, with the
// guard; without, it makes the sums NaN, which asks for it.
template <int W, bool REF, bool GUARD>
__device__ __forceinline__ float GroupSums(Sums &s, float top, float c, float (*red)[8]) {
  s.e = WaveSum(s.e);
  s.et = WaveSum(s.et);
  if constexpr (REF) {
    s.ed = WaveSum(s.ed);
    s.far = WaveMax(s.far);
  }
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      float *mine = red[threadIdx.x >> 6];
      *reinterpret_cast<f32x4 *>(mine) = f32x4{s.e, s.et, s.ed, s.far};
      mine[4] = top;
    }
    __syncthreads();
    const float *other = red[threadIdx.x & (W - 1)];
    const f32x4 v = *reinterpret_cast<const f32x4 *>(other);
    const float its = other[4];
    top = LanesMax<W>(its);
    top = top == -__builtin_inff() ? 0.f : top;
    const float step = (its - top) * c, f = Exp2(step);
    const float none = GUARD ? 0.f : __builtin_nanf("");
    s.e = LanesSum<W>(f * v[0]);
    s.et = LanesSum<W>(f == 0.f ? none : f * (v[1] + v[0] * step));
    if constexpr (REF) {
      s.ed = LanesSum<W>(f == 0.f ? none : f * v[2]);
      s.far = LanesMax<W>(v[3]);
    }
    return top;
  }
  return top == -__builtin_inff() ? 0.f : top;
}

// u below which a term of KL comes from the reference instead: there exp(-u)
// (up to 2^58 above it) may bring back a p that is below 2^-126 and 0.
constexpr float kFarBelow = -40.f;

// A NaN; an entry far from the reference on either side (-kFarBelow bounds |u|:
// below, KL's terms overflow, and above, u itself may: the lowest value in the
// reference against 1 / T above 1); or coefficients (Coefs a, b) above 1, whose
// product with a logit of the type's lowest value may overflow.
template <bool REF>
__device__ __forceinline__ bool NeedsGuard(const RowLossParams &a, float weight, const Sums &s) {
  return s.et != s.et || !(fabsf(weight * a.inv_temp) < 0x1p40f) ||
         !(fabsf(a.entropy_coef) * a.inv_temp <= 1.f) ||
         (REF && (!(fabsf(a.kl_coef) <= 1.f) ||
                  !((s.far + fabsf(s.ed * Rcp(s.e))) * a.inv_temp < -kFarBelow)));
}

// What a row's scalars come to, from its statistics.
struct RowStats {
  float m;         // maximum (0 where every entry is masked)
  float log_sum;   // ln S
  float log2_sum;  // log2 S
  float mean_z;    // E_p z
  float mean_d;    // E_p d, without 1 / T
  bool empty;      // no entry left
};

__device__ __forceinline__ RowStats Stats(float m, const Sums &sums) {
  RowStats r;
  r.m = m;
  r.empty = sums.e == 0.f;
  const float sum = r.empty ? 1.f : sums.e, inv = Rcp(sum);
  r.log2_sum = Log2(sum);
  r.log_sum = r.log2_sum * kLn2;
  r.mean_z = sums.et * kLn2 * inv;
  r.mean_d = sums.ed * inv;
  return r;
}

// A row with the guards whose E_p d is beyond kApart takes d from the two maxima,
// as (x - m) - (y - y_m): a constant between policy and reference (3.4e38 in a
// row whose reference is masked everywhere by the lowest value) would round the
// logits away.  Nearer, x - y is exact where it is small.  Sums of e d there are
// of e d kDown: several d of the lowest value would add up to infinity where
// their mean is finite.
constexpr float kApart = 64.f, kDown = 0x1p-32f, kUp = 0x1p32f;
__device__ __forceinline__ bool FarApart(const RowStats &st, float y_m) {
  return !(fabsf(st.mean_d) <= kApart) && fabsf(y_m) < __builtin_inff();
}
// One entry's part of that sum.
__device__ __forceinline__ float ApartPart(float x, float y, float m, float y_m, float c) {
  const float xm = x - m, e = Exp2(xm * c);
  return e == 0.f ? 0.f : e * ((xm - (y - y_m)) * kDown);
}
// E_p d from it: infinite only if the sum is.
__device__ __forceinline__ float ApartMean(float down, float e) {
  const float mean = down * Rcp(e) * kUp;
  return mean == __builtin_inff() && down < mean ? 0x1.fffffep127f : mean;
}

// Coefficients of one row's gradient
//   scale (slope 1[k = a] + p_k (kl u_k + entropy (z_k - E_p z) - slope)).
struct RowGrad {
  float scale, slope, kl, entropy;
};

// The same as P_k (a (x_k - m) + b u_k + d) with P = 2^power p, with what P and
// u need: a large scale's power of two is in P, so that a and b stay small
// whatever the row's weight (a loss scale of 2^16, say).  A small one's is not:
// the terms of KL, which no weight may change, are sums of P exp(-u), and a P
// smaller than p vanishes earlier.  Without the guards they are below 2^40
// times exp(40) = 2^58.
struct Coefs {
  float m, c, shift, inv_temp, mean_u, a, b, d;
  int power;
};
constexpr int kMostPower = 40;

__device__ __forceinline__ Coefs CoefsOf(const RowStats &st, const RowGrad &g, float inv_temp) {
  Coefs k;
  const int power = __builtin_amdgcn_frexp_expf(g.scale);
  k.power = power < 0 ? 0 : power > kMostPower ? kMostPower : power;
  const float scale = ldexpf(g.scale, -k.power);
  k.m = st.m;
  k.c = inv_temp * kLog2e;
  k.shift = static_cast<float>(k.power) - st.log2_sum;
  k.inv_temp = inv_temp;
  k.mean_u = st.mean_d * inv_temp;
  k.a = scale * g.entropy * inv_temp;
  k.b = scale * g.kl;
  k.d = -scale * (g.slope + g.entropy * st.mean_z);
  return k;
}

// And with the guards, in scalar registers: y_m the greatest reference logit,
// peak the greatest of ln(p_k exp(-u_k)) = (y_k - m) / T + E_p (x - y) / T - ln S.
// KL lies between peak and peak + ln(entries).  Above kWide it is taken as
// peak + ln sum exp((y_k - y_m) / T), which has no overflow; below, its terms
// in P are at most 2^40 exp(30) = 2^84 each.
struct FarCoefs {
  float mean_d, y_m, y_shift, peak;
  float steep, flat;     // b / T, as a factor of p from 1 on and of d - E_p d below: no
                         // step of a gradient leaves the range that it is in itself
  float above;           // u of more is infinite, or may be where p u is not (1 / T > 1)
  bool apart, wide, kl;  // d from the maxima; peak above kWide; KL in the gradient
};
constexpr float kWide = 30.f;
__device__ __forceinline__ FarCoefs FarCoefsOf(const RowStats &st, const Coefs &k, float y_m,
                                               bool apart) {
  FarCoefs f;
  f.peak = Scalar(k.mean_u + (apart ? 0.f : (y_m - st.m) * k.inv_temp) - st.log_sum);
  f.above = k.inv_temp > 1.f ? -kFarBelow : 0x1.fffffep127f;
  f.apart = __builtin_amdgcn_readfirstlane(apart);
  f.wide = __builtin_amdgcn_readfirstlane(f.peak > kWide);
  const float slope = k.b * k.inv_temp;
  f.steep = Scalar(fabsf(slope) < 1.f ? 1.f : slope);
  f.flat = Scalar(fabsf(slope) < 1.f ? slope : 1.f);
  f.kl = __builtin_amdgcn_readfirstlane(k.b != 0.f);
  f.y_shift = Scalar(f.wide ? 0.f : f.peak * kLog2e + static_cast<float>(k.power));
  f.mean_d = Scalar(st.mean_d);
  f.y_m = Scalar(y_m);
  return f;
}

// exp(-u) - 1 + u for u > kFarBelow: its series for |u| < 1/4 (the first term
// left out is 1.2e-8 of the sum), where the difference would cancel.
__device__ __forceinline__ float Phi(float u) {
  const float e = Exp2(-u * kLog2e);
  float r = -1.f / 5040;
  r = r * u + 1.f / 720;
  r = r * u - 1.f / 120;
  r = r * u + 1.f / 24;
  r = r * u - 1.f / 6;
  r = r * u + 0.5f;
  float near = u * u * r, far = (e - 1.f) + u;
  // Both, and a select: as a branch for each entry it took a fifth longer.
  asm volatile("" : "+v"(near), "+v"(far));
  return fabsf(u) < 0.25f ? near : far;
}

// P u from P and d less its mean, finite also where u is not.
__device__ __forceinline__ float TimesU(const Coefs &k, float p, float apart) {
  return p * k.inv_temp * apart;
}

// P (exp(-u) - 1 + u), the term of KL, for any u.  Far below 0, where exp(-u) is
// large against a tiny p, their product comes from the reference; an entry that
// is masked here adds nothing but its reference probability.  With f.wide,
// exp((y - y_m) / T) instead.
__device__ __forceinline__ float KlTerm(const Coefs &k, const FarCoefs &f, float p, float apart,
                                        float y) {
  const float u = apart * k.inv_temp;
  if (!f.wide && u > kFarBelow && u <= f.above)
    return p * Phi(u);
  const float q = u > 0.f && !f.wide ? 0.f : Exp2((y - f.y_m) * k.c + f.y_shift);
  return f.wide || p == 0.f ? q : q - p + TimesU(k, p, apart);
}

// KL from the sum of its terms; infinite where the reference lacks what the
// policy plays (E_p d is, and no term then means anything).
template <bool GUARD>
__device__ __forceinline__ float KlOf(float terms, const Coefs &k, const FarCoefs &f) {
  if constexpr (GUARD) {
    if (f.mean_d == __builtin_inff())
      return f.mean_d;
    if (f.wide)
      return f.peak + Log2(terms) * kLn2;
  }
  return Log1p(ldexpf(terms, -k.power));
}

// The gradient of N entries without the action's own term, and their part of
// KL.  GUARD: as for the sums, and any u.
template <int N, bool REF, bool GUARD>
__device__ __forceinline__ void FinishEntries(const Coefs &k, const FarCoefs &far, bool want_kl,
                                              const float (&x)[N], const float (&y)[N], float &kl,
                                              float (&f)[N]) {
  float p[N], u[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float xm = x[i] - k.m;
    p[i] = Exp2(xm * k.c + k.shift);
    float v = k.a * xm + k.d;
    if constexpr (REF && !GUARD) {
      u[i] = (x[i] - y[i]) * k.inv_temp - k.mean_u;
      v = k.b * u[i] + v;
    }
    f[i] = p[i] * v;
  }
  if constexpr (REF && GUARD) {
    float apart[N];
    if (far.apart) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        apart[i] = ((x[i] - k.m) - (y[i] - far.y_m)) - far.mean_d;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        apart[i] = (x[i] - y[i]) - far.mean_d;
    }
    // Without a coefficient KL is only watched: it may be infinite.
    if (far.kl) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[i] += (p[i] * far.steep) * (apart[i] * far.flat);
    }
    if (want_kl) {
      bool usual = !far.wide;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u[i] = apart[i] * k.inv_temp;
        usual = usual && u[i] > kFarBelow && u[i] <= far.above;
      }
      if (__all(usual)) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          kl += p[i] * Phi(u[i]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          kl += KlTerm(k, far, p[i], apart[i], y[i]);
      }
    }
  }
  if constexpr (GUARD) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      f[i] = p[i] == 0.f ? 0.f : f[i];
  }
  if (REF && !GUARD && want_kl) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      kl += p[i] * Phi(u[i]);
  }
}

// Whether the divergence itself is asked for (its gradient needs no KL).
__device__ __forceinline__ bool WantsKl(const RowLossParams &a) {
  return a.kl || (a.loss && a.kl_coef != 0.f);
}

// Element i of an input array, i the same in the whole wave, by a scalar load:
// a vector load would be waited for behind every row load and store that the
// wave has on its way.  No kernel writes the array while this one runs: an
// output that overlaps an input is refused.
template <class T> __device__ __forceinline__ T Uniform(const T *p, std::int64_t i) {
  return ((const MFH_CONSTANT T *)p)[i];
}

// A row's scalar inputs, loaded together before anything waits on one.
struct RowInputs {
  float weight;  // 0: the row is not read
  int action;
  float advantage, old_logp;
};
__device__ __forceinline__ RowInputs Inputs(const RowLossParams &a, std::int64_t row) {
  RowInputs r;
  r.weight = a.coef ? Uniform(a.coef, row) : a.weight ? Uniform(a.weight, row) : 1.f;
  r.action = a.actions ? Uniform(a.actions, row) : -1;
  r.advantage = a.advantage ? Uniform(a.advantage, row) : 0.f;
  r.old_logp = a.old_logp ? Uniform(a.old_logp, row) : 0.f;
  return r;
}

// The first term of the loss and its derivative by ln p_a.
struct Surrogate {
  float loss, slope;
};
__device__ __forceinline__ Surrogate Clipped(const RowLossParams &a, const RowInputs &in,
                                             float logp) {
  const float ratio = a.old_logp ? Exp(logp - in.old_logp) : 1.f;
  // The ratio may overflow: 0 times it is 0 (a NaN stays).
  if (in.advantage == 0.f && ratio == ratio)
    return {0.f, 0.f};
  const float plain = ratio * in.advantage;
  const float bounded = fminf(fmaxf(ratio, a.ratio_low), a.ratio_high) * in.advantage;
  // The unclipped branch on ties and for NaN.
  return bounded < plain ? Surrogate{-bounded, 0.f} : Surrogate{-plain, -plain};
}

// A row's scalars once its statistics are there: the coefficients of its
// gradient, and what WriteRow needs.
struct RowResult {
  RowGrad grad;
  float logp, surrogate, entropy;
};
__device__ __forceinline__ RowResult Evaluate(const RowLossParams &a, const RowInputs &in,
                                              const RowStats &st, bool acted, float xa) {
  RowResult r{{in.weight * a.inv_temp, 0.f, 0.f, 0.f}, 0.f, 0.f, 0.f};
  if (acted)
    r.logp = (xa - st.m) * a.inv_temp - st.log_sum;
  if (a.coef) {
    r.grad.slope = acted ? 1.f : 0.f;
    return r;
  }
  if (acted && a.advantage) {
    const Surrogate s = Clipped(a, in, r.logp);
    r.surrogate = s.loss;
    r.grad.slope = s.slope;
  }
  r.entropy = st.log_sum - st.mean_z;
  r.grad.kl = a.kl_coef;
  r.grad.entropy = a.entropy_coef;
  return r;
}

// What waits for the end of the row, out of the vector registers: with a
// reference three more decide the waves a SIMD holds (the shortest rows of bf16
// take 61 registers for eight waves, 65 with these).
template <bool REF> __device__ __forceinline__ void Park(RowResult &r) {
  if constexpr (REF) {
    r.logp = Scalar(r.logp);
    r.surrogate = Scalar(r.surrogate);
    r.entropy = Scalar(r.entropy);
  }
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
  // A coefficient may carry KL (up to 3e38 against masks of the lowest value) out
  // of the range that the weight brings it back to.
  const bool over = fabsf(loss) == __builtin_inff() && fabsf(w) < 1.f;
  if (a.loss)
    a.loss[row] = over ? w * (r.surrogate - a.entropy_coef * r.entropy) + w * a.kl_coef * kl
                       : w * loss;
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
  return a.seq_offsets &&
         (row < Uniform(a.seq_offsets, 0) || row >= Uniform(a.seq_offsets, a.n_seq));
}

// Zeros in a whole gradient row, by `threads` threads.
template <int DT>
__device__ __forceinline__ void ZeroRow(Row<DT> g, int n, int thread, int threads) {
  using E = Elem<DT>;
  const int vecs = n / E::kPerVec;
  for (int v = thread; v < vecs; v += threads)
    StoreVec<DT, false>(g + static_cast<std::int64_t>(v) * E::kPerVec, u32x4{0, 0, 0, 0});
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

template <int DT, bool REF, bool GUARD>
__device__ __forceinline__ void AddVec(u32x4 xr, u32x4 yr, float m, float c, Sums &sums) {
  constexpr int VE = Elem<DT>::kPerVec;
  float xs[VE], ys[VE] = {};
  Unpack<DT>(xr, xs);
  if constexpr (REF)
    Unpack<DT>(yr, ys);
#pragma unroll
  for (int i = 0; i < VE; ++i)
    AddStats<REF, GUARD>(xs[i], ys[i], m, c, sums);
}

template <int DT>
__device__ __forceinline__ void AddApart(u32x4 xr, u32x4 yr, float m, float y_m, float c,
                                         float &sum) {
  constexpr int VE = Elem<DT>::kPerVec;
  float xs[VE], ys[VE];
  Unpack<DT>(xr, xs);
  Unpack<DT>(yr, ys);
#pragma unroll
  for (int i = 0; i < VE; ++i)
    sum += ApartPart(xs[i], ys[i], m, y_m, c);
}

// Four entries at a time: eight would hold more registers.
template <int DT, bool REF, bool GUARD>
__device__ __forceinline__ u32x4 FinishVec(const Coefs &k, const FarCoefs &far, bool want_kl,
                                           u32x4 xr, u32x4 yr, float &kl) {
  using E = Elem<DT>;
  constexpr int VE = E::kPerVec;
  float f[VE];
#pragma unroll
  for (int h = 0; h < VE; h += 4) {
    float xs[4], ys[4] = {}, part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xs[i] = E::Get(xr, h + i);
      if constexpr (REF)
        ys[i] = E::Get(yr, h + i);
    }
    FinishEntries<4, REF, GUARD>(k, far, want_kl, xs, ys, kl, part);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[h + i] = part[i];
  }
  return E::Pack(f);
}

// The elements behind the last whole vector, and the action's own term, by the
// thread that wrote its column.
template <int DT, bool REF, bool GUARD>
__device__ __forceinline__ void FinishRest(const Coefs &k, const FarCoefs &far, bool want_kl,
                                           bool want_grad, Row<DT> g, const RowGrad &grad, int act,
                                           float xa, float ya, const float (&xt)[1],
                                           const float (&yt)[1], int vecs, bool has_rest,
                                           int threads, int tid, float &kl) {
  using E = Elem<DT>;
  constexpr int VE = E::kPerVec;
  float ft[1];
  if (has_rest) {
    FinishEntries<1, REF, GUARD>(k, far, want_kl, xt, yt, kl, ft);
    if (want_grad)
      g[vecs * VE + tid] = E::Round(ft[0]);
  }
  const int v = act / VE;
  if (want_grad && act >= 0 && tid == (v < vecs ? v % threads : act - vecs * VE)) {
    float none = 0.f;
    const float xs[1] = {xa}, ys[1] = {ya};
    FinishEntries<1, REF, GUARD>(k, far, false, xs, ys, none, ft);
    g[act] = E::Round(ft[0] + grad.scale * grad.slope);
  }
}

#define MFH_INLINE __attribute__((always_inline))

// A whole row in the registers of W waves, NV vectors of 16 bytes a lane; the
// elements behind the last whole vector, one to a lane, in a register more.
// Three passes over the registers: maximum, sums, gradient with KL.  Four rows
// to a workgroup where a wave has one to itself.
template <int DT, int W, int NV, bool REF, bool PAST>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void DenseRowKernel(RowLossParams a) {
  using E = Elem<DT>;
  constexpr int VE = E::kPerVec;
  __shared__ __align__(16) float red[W][8];
  const int tid = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  std::int64_t row = blockIdx.x;
  if constexpr (W == 1)
    row = row * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  row += a.row0;
  if (row >= a.end || OutsideSequences(a, row))
    return;
  const int n = a.vocab, vecs = n / VE, rest = n - vecs * VE;
  const ConstRow<DT> x = RowOf<DT>(a.x, row, a.ldx);
  const ConstRow<DT> y = RowOf<DT>(a.y, row, a.ldy);
  const Row<DT> g = RowOf<DT>(a.g, row, a.ldg);
  const bool want_grad = a.g != nullptr;
  const RowInputs in = Inputs(a, row);
  if (in.weight == 0.f) {
    if (tid == 0)
      WriteZeros(a, row);
    if (want_grad)
      ZeroRow<DT>(g, n, tid, 64 * W);
    return;
  }
  const int act = in.action;
  const bool listed = act >= 0 && act < n;
  const float xa = listed ? E::One(x[act]) : 0.f;
  const float ya = REF && listed ? E::One(y[act]) : 0.f;
  const bool acted = listed && xa != -__builtin_inff();
  u32x4 xr[NV], yr[REF ? NV : 1];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = j * 64 * W + tid;
    if (v < vecs)
      xr[j] = LoadVec<DT, PAST>(x + v * VE);
  }
  if constexpr (REF) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = j * 64 * W + tid;
      if (v < vecs)
        yr[j] = LoadVec<DT, PAST>(y + v * VE);
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
  const float top = WaveMax(m);

  const float c = a.inv_temp * kLog2e;
  Sums sums;
  const auto sum = [&](auto guard) MFH_INLINE {
    constexpr bool GUARD = decltype(guard)::value;
    sums = NoSums<GUARD>();
    m = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Repack(xr[j]);
      if (REF)
        Repack(yr[REF ? j : 0]);
      if (j * 64 * W + tid < vecs)
        AddVec<DT, REF, GUARD>(xr[j], yr[REF ? j : 0], m, c, sums);
    }
    if (has_rest)
      AddStats<REF, GUARD>(xt[0], yt[0], m, c, sums);
    m = GroupSums<W, REF, GUARD>(sums, top, c, red);
  };
  sum(std::false_type{});
  const bool guarded = NeedsGuard<REF>(a, in.weight, sums);
  if (guarded)
    sum(std::true_type{});
  RowStats st = Stats(m, sums);
  if (st.empty) {
    if (tid == 0)
      WriteZeros(a, row);
    if (want_grad)
      ZeroRow<DT>(g, n, tid, 64 * W);
    return;
  }
  const bool apart = REF && guarded && FarApart(st, sums.far);
  if (apart) {
    float part[1] = {has_rest ? ApartPart(xt[0], yt[0], m, sums.far, c) : 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Repack(xr[j]);
      Repack(yr[REF ? j : 0]);
      if (j * 64 * W + tid < vecs)
        AddApart<DT>(xr[j], yr[REF ? j : 0], m, sums.far, c, part[0]);
    }
    GroupSum<W>(part, red);
    st.mean_d = ApartMean(part[0], sums.e);
  }
  RowResult res = Evaluate(a, in, st, acted, xa);
  Park<REF>(res);
  const bool want_kl = REF && WantsKl(a);
  float kl[1] = {0.f};
  if (want_grad || want_kl) {
    const Coefs k = CoefsOf(st, res.grad, a.inv_temp);
    const auto finish = [&](auto guard) MFH_INLINE {
      constexpr bool GUARD = decltype(guard)::value;
      const FarCoefs far = GUARD ? FarCoefsOf(st, k, sums.far, apart) : FarCoefs{};
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Repack(xr[j]);
        if (REF)
          Repack(yr[REF ? j : 0]);
        const int v = j * 64 * W + tid;
        if (v < vecs) {
          const u32x4 f =
              FinishVec<DT, REF, GUARD>(k, far, want_kl, xr[j], yr[REF ? j : 0], kl[0]);
          if (want_grad)
            StoreVec<DT, PAST>(g + v * VE, f);
        }
      }
      FinishRest<DT, REF, GUARD>(k, far, want_kl, want_grad, g, res.grad, acted ? act : -1, xa, ya,
                                 xt, yt, vecs, has_rest, 64 * W, tid, kl[0]);
      if (want_kl) {
        GroupSum<W>(kl, red);
        kl[0] = KlOf<GUARD>(kl[0], k, far);
      }
    };
    if (guarded)
      finish(std::true_type{});
    else
      finish(std::false_type{});
  }
  if (tid == 0)
    WriteRow(a, row, in.weight, acted, res, kl[0]);
}

// A row that is not in registers, by a workgroup of 16 waves: one pass for the
// statistics with a running maximum per lane, a second for KL and the
// gradient, from the end of the row backwards (its last part is nearest in the
// caches).
template <int DT, bool REF>
__device__ __forceinline__ void StreamRow(const RowLossParams &a, std::int64_t row,
                                          const RowInputs &in, float (*red)[8]) {
  using E = Elem<DT>;
  constexpr int VE = E::kPerVec, W = 16, kThreads = 64 * W;
  const int tid = threadIdx.x;
  const int n = a.vocab, vecs = n / VE, rest = n - vecs * VE;
  const ConstRow<DT> x = RowOf<DT>(a.x, row, a.ldx);
  const ConstRow<DT> y = RowOf<DT>(a.y, row, a.ldy);
  const Row<DT> g = RowOf<DT>(a.g, row, a.ldg);
  const bool want_grad = a.g != nullptr;
  const int act = in.action;
  const bool listed = act >= 0 && act < n;
  const float xa = listed ? E::One(x[act]) : 0.f;
  const float ya = REF && listed ? E::One(y[act]) : 0.f;
  const bool acted = listed && xa != -__builtin_inff();
  const bool has_rest = tid < rest;
  const float xt[1] = {has_rest ? E::One(x[vecs * VE + tid]) : -__builtin_inff()};
  const float yt[1] = {REF && has_rest ? E::One(y[vecs * VE + tid]) : 0.f};

  const float c = a.inv_temp * kLog2e;
  float m = xt[0];
  Sums sums = NoSums<true>();
  // Sums over the old maximum as sums over the new: e and t of each term fall
  // by the same step.
  const auto rescale = [&](float from, float to) MFH_INLINE {
    if (sums.e == 0.f)
      return;
    const float step = (from - to) * c, f = Exp2(step);
    sums.et = f == 0.f ? 0.f : f * (sums.et + sums.e * step);
    sums.e *= f;
    sums.ed = f == 0.f ? 0.f : f * sums.ed;
  };
  if (has_rest)
    AddStats<REF, true>(xt[0], yt[0], m == -__builtin_inff() ? 0.f : m, c, sums);
  for (int v = tid; v < vecs; v += kThreads) {
    const u32x4 xr = LoadVec<DT, false>(x + static_cast<std::int64_t>(v) * VE);
    u32x4 yr = {};
    if constexpr (REF)
      yr = LoadVec<DT, false>(y + static_cast<std::int64_t>(v) * VE);
    float top = m;
#pragma unroll
    for (int i = 0; i < VE; ++i)
      top = fmaxf(top, E::Get(xr, i));
    if (top > m) {
      rescale(m, top);
      m = top;
    }
    AddVec<DT, REF, true>(xr, yr, m == -__builtin_inff() ? 0.f : m, c, sums);
  }
  const float top = WaveMax(m);
  rescale(m, top == -__builtin_inff() ? 0.f : top);
  m = GroupSums<W, REF, true>(sums, top, c, red);
  RowStats st = Stats(m, sums);
  if (st.empty) {
    if (tid == 0)
      WriteZeros(a, row);
    if (want_grad)
      ZeroRow<DT>(g, n, tid, kThreads);
    return;
  }
  const bool apart = REF && FarApart(st, sums.far);
  if (apart) {
    float part[1] = {has_rest ? ApartPart(xt[0], yt[0], m, sums.far, c) : 0.f};
    for (int v = tid; v < vecs; v += kThreads)
      AddApart<DT>(LoadVec<DT, false>(x + static_cast<std::int64_t>(v) * VE),
                   LoadVec<DT, false>(y + static_cast<std::int64_t>(v) * VE), m, sums.far, c,
                   part[0]);
    GroupSum<W>(part, red);
    st.mean_d = ApartMean(part[0], sums.e);
  }
  const RowResult res = Evaluate(a, in, st, acted, xa);
  const bool want_kl = REF && WantsKl(a);
  float kl[1] = {0.f};
  if (want_grad || want_kl) {
    const Coefs k = CoefsOf(st, res.grad, a.inv_temp);
    const FarCoefs far = FarCoefsOf(st, k, sums.far, apart);
    for (int j = (vecs - 1) / kThreads; j >= 0; --j) {
      const std::int64_t v = static_cast<std::int64_t>(j) * kThreads + tid;
      if (v >= vecs)
        continue;
      const u32x4 xr = LoadVec<DT, false>(x + v * VE);
      u32x4 yr = {};
      if constexpr (REF)
        yr = LoadVec<DT, false>(y + v * VE);
      const u32x4 f = FinishVec<DT, REF, true>(k, far, want_kl, xr, yr, kl[0]);
      if (want_grad)
        StoreVec<DT, true>(g + v * VE, f);
    }
    FinishRest<DT, REF, true>(k, far, want_kl, want_grad, g, res.grad, acted ? act : -1, xa, ya,
                              xt, yt, vecs, has_rest, kThreads, tid, kl[0]);
    if (want_kl) {
      GroupSum<W>(kl, red);
      kl[0] = KlOf<true>(kl[0], k, far);
    }
  }
  if (tid == 0)
    WriteRow(a, row, in.weight, acted, res, kl[0]);
}

// Rows longer than the registers hold, one workgroup a CU (each asks for half of
// the LDS, beside `red`): more rows at once push each other's first reading out
// of the last-level cache.  fp32 with a reference, one and two a CU: 2000 x
// 100003 605 and 684 us, 700 x 50021 101 and 110, 1818 x 33001 190 and 180;
// 1000 x 60000 without 91 and 97.
constexpr unsigned kHalfLds = 80 * 1024;
template <int DT, bool REF>
__global__ __launch_bounds__(1024) void StreamRowKernel(RowLossParams a) {
  __shared__ __align__(16) float red[16][8];
  const std::int64_t row = a.row0 + blockIdx.x;
  if (OutsideSequences(a, row))
    return;
  const RowInputs in = Inputs(a, row);
  if (in.weight != 0.f) {
    StreamRow<DT, REF>(a, row, in, red);
    return;
  }
  if (threadIdx.x == 0)
    WriteZeros(a, row);
  if (a.g)
    ZeroRow<DT>(RowOf<DT>(a.g, row, a.ldg), a.vocab, threadIdx.x, 1024);
}

// Rows that fill the registers of 16 waves, so that a CU holds one workgroup
// and its loads, passes and stores would follow one another.  A workgroup takes
// row after row (every gridDim.x-th), and as the last pass is done with a
// vector of the present row it loads the next row's into its registers.  All
// rows take the same way through the loop, so that there is one such place:
// rows of weight 0 compute nothing of use and store nothing.  NV: the vectors
// of a lane, the last one filled for some lane.  Takes rows from `row` on;
// returns the row that it leaves undone because it needs the guards (a.end or
// more: none).
template <int DT, int NV, bool REF, bool GUARD>
__device__ __forceinline__ std::int64_t LoopRows(const RowLossParams &a, std::int64_t row,
                                                 float (*red)[8]) {
  using E = Elem<DT>;
  constexpr int VE = E::kPerVec, W = 16, kThreads = 64 * W;
  const int tid = threadIdx.x;
  const int n = a.vocab, vecs = n / VE, rest = n - vecs * VE;
  const bool has_rest = tid < rest;
  const bool want_grad = a.g != nullptr;
  const bool want_kl = REF && WantsKl(a);
  const float c = a.inv_temp * kLog2e;

  u32x4 xr[NV], yr[REF ? NV : 1];
  // This lane's place among vectors j * kThreads on: NV is such that all are
  // there but for the last j, where the lanes behind the end share its last.
  // The same address arithmetic every time, from one register and the row's
  // uniform address (addresses kept for all j would be spilled, and the wait
  // for one to come back would be one for every load on its way).
  const auto place = [&](int j) MFH_INLINE {
    int lane = tid;
    asm volatile("" : "+v"(lane));
    const int end = vecs - j * kThreads - 1;
    return (j < NV - 1 || lane < end ? lane : end) * VE;
  };
  const auto filled = [&](int j) MFH_INLINE { return j < NV - 1 || j * kThreads + tid < vecs; };
  // Vector j of a row; the row's first ones where there is nothing to read.
  const auto load = [&](std::int64_t r, int j, bool live) MFH_INLINE {
    const int from = live ? j * kThreads * VE : 0, at = live ? place(j) : 0;
    xr[j] = LoadVec<DT, true>(RowOf<DT>(a.x, r, a.ldx) + from + at);
    if constexpr (REF)
      yr[j] = LoadVec<DT, true>(RowOf<DT>(a.y, r, a.ldy) + from + at);
  };
  const auto alive = [&](std::int64_t r) MFH_INLINE {
    return r < a.end && !OutsideSequences(a, r) && Inputs(a, r).weight != 0.f;
  };
  // The action's logits and the elements behind the last vector (some logit of
  // the row where there is none), as they are: a conversion would wait.
  struct Few {
    typename E::T xa, ya, xt, yt;
  };
  const auto load_few = [&](std::int64_t r, int act) MFH_INLINE {
    const ConstRow<DT> x = RowOf<DT>(a.x, r, a.ldx), y = RowOf<DT>(a.y, r, a.ldy);
    const int at = act >= 0 && act < n ? act : 0, last = has_rest ? vecs * VE + tid : 0;
    Few f{x[at], 0, x[last], 0};
    if constexpr (REF) {
      f.ya = y[at];
      f.yt = y[last];
    }
    return f;
  };
  bool live = alive(row);
  Few few = load_few(row, Inputs(a, row).action);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    load(row, j, live);
  while (row < a.end) {
    const std::int64_t next = row + gridDim.x;
    const bool next_live = alive(next);
    const std::int64_t next_row = next < a.end ? next : row;
    const Row<DT> g = RowOf<DT>(a.g, row, a.ldg);
    const RowInputs in = Inputs(a, row);
    const int act = in.action;
    const Few next_few = load_few(next_row, Inputs(a, next_row).action);
    const float xa = E::One(few.xa), ya = REF ? E::One(few.ya) : 0.f;
    const bool acted = act >= 0 && act < n && xa != -__builtin_inff();
    const float xt[1] = {has_rest ? E::One(few.xt) : -__builtin_inff()};
    const float yt[1] = {REF && has_rest ? E::One(few.yt) : 0.f};
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (filled(j)) {
        float xs[VE];
        Unpack<DT>(xr[j], xs);
#pragma unroll
        for (int i = 0; i < VE; ++i)
          m = fmaxf(m, xs[i]);
      }
    const float top = WaveMax(fmaxf(m, xt[0]));
    m = top == -__builtin_inff() ? 0.f : top;
    Sums sums = NoSums<GUARD>();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Repack(xr[j]);
      if (REF)
        Repack(yr[REF ? j : 0]);
      if (filled(j))
        AddVec<DT, REF, GUARD>(xr[j], yr[REF ? j : 0], m, c, sums);
    }
    if (has_rest)
      AddStats<REF, GUARD>(xt[0], yt[0], m, c, sums);
    m = GroupSums<W, REF, GUARD>(sums, top, c, red);
    // A row without an entry left needs them too (its sums hold 0 times -inf).
    if (!GUARD && live && NeedsGuard<REF>(a, in.weight, sums))
      return row;
    RowStats st = Stats(m, sums);
    const bool apart = REF && GUARD && FarApart(st, sums.far);
    if constexpr (REF && GUARD) {
      if (apart) {
        float part[1] = {has_rest ? ApartPart(xt[0], yt[0], m, sums.far, c) : 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          Repack(xr[j]);
          Repack(yr[j]);
          if (filled(j))
            AddApart<DT>(xr[j], yr[j], m, sums.far, c, part[0]);
        }
        GroupSum<W>(part, red);
        st.mean_d = ApartMean(part[0], sums.e);
      }
    }
    RowResult res = Evaluate(a, in, st, acted && !st.empty, xa);
    Park<REF>(res);
    const Coefs k = CoefsOf(st, res.grad, a.inv_temp);
    const FarCoefs far = GUARD ? FarCoefsOf(st, k, sums.far, apart) : FarCoefs{};
    float kl[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Repack(xr[j]);
      if (REF)
        Repack(yr[REF ? j : 0]);
      if (filled(j) && (want_grad || want_kl)) {
        const u32x4 f =
            FinishVec<DT, REF, GUARD>(k, far, want_kl, xr[j], yr[REF ? j : 0], kl[0]);
        if (want_grad && live)
          StoreVec<DT, true>(g + j * kThreads * VE + place(j), f);
      }
      // Not earlier: the present row's vector is in the registers.
      __builtin_amdgcn_sched_barrier(0);
      load(next_row, j, next_live);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (live && !st.empty) {
      FinishRest<DT, REF, GUARD>(k, far, want_kl, want_grad, g, res.grad, acted ? act : -1, xa, ya,
                                 xt, yt, vecs, has_rest, kThreads, tid, kl[0]);
      if (want_kl) {
        GroupSum<W>(kl, red);
        kl[0] = KlOf<GUARD>(kl[0], k, far);
      }
      if (tid == 0)
        WriteRow(a, row, in.weight, acted, res, kl[0]);
    } else if (live || !OutsideSequences(a, row)) {
      if (tid == 0)
        WriteZeros(a, row);
      if (want_grad)
        ZeroRow<DT>(g, n, tid, kThreads);
    }
    row = next;
    live = next_live;
    few = next_few;
  }
  return row;
}

template <int DT, int NV, bool REF>
__global__ __launch_bounds__(1024) void LoopRowKernel(RowLossParams a) {
  __shared__ __align__(16) float red[16][8];
  // From the first row that needs the guards on, all rows take them (columns
  // that only fill up a vocabulary are masked in every row).
  const std::int64_t row = LoopRows<DT, NV, REF, false>(a, a.row0 + blockIdx.x, red);
  if (row < a.end)
    (void)LoopRows<DT, NV, REF, true>(a, row, red);
}


// The entries of one row, NE a lane: columns (-1 outside the vocabulary, where
// the logit is 0, and behind the list) and logits.
template <int NE> struct Entries {
  int col[NE];
  float x[NE], y[NE];
};

template <int NE>
__device__ __forceinline__ void LoadColumns(const RowLossParams &a, std::int64_t start, int moves,
                                            Entries<NE> &e) {
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    const int i = r * 64 + (threadIdx.x & 63);
    e.col[r] = -1;
    if (i < moves) {
      const int k = a.indices[start + i];
      e.col[r] = k >= 0 && k < a.vocab ? k : -1;
    }
  }
}

template <int DT, bool REF, int NE>
__device__ __forceinline__ void LoadLogits(const RowLossParams &a, std::int64_t row, int moves,
                                           Entries<NE> &e) {
  using E = Elem<DT>;
  const ConstRow<DT> x = RowOf<DT>(a.x, row, a.ldx);
  const ConstRow<DT> y = RowOf<DT>(a.y, row, a.ldy);
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    const bool listed = r * 64 + static_cast<int>(threadIdx.x & 63) < moves;
    const bool inside = e.col[r] >= 0;
    e.x[r] = inside ? E::One(x[e.col[r]]) : listed ? 0.f : -__builtin_inff();
    e.y[r] = 0.f;
    if constexpr (REF)
      e.y[r] = inside ? E::One(y[e.col[r]]) : listed ? 0.f : -__builtin_inff();
  }
}

// One row's legal moves by one wave.  The gradient row is put together in LDS,
// part_cols columns at a time, and written once, in whole vectors: zeros, and
// each entry's value in its column.  A move listed twice adds up: each entry
// first leaves its number in its column, and where one finds another's, the
// first of equal entries counts them and writes for all.
template <int DT, bool REF, bool PAST, int NE>
__device__ __forceinline__ void MovesRow(const RowLossParams &a, std::int64_t row,
                                         const RowInputs &in, const Entries<NE> &entries,
                                         unsigned char *lds, int part_cols) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VE = E::kPerVec;
  const int lane = threadIdx.x & 63;
  const int n = a.vocab, act = in.action;
  const Row<DT> g = RowOf<DT>(a.g, row, a.ldg);
  const bool want_grad = a.g != nullptr;
  T *buf = reinterpret_cast<T *>(lds);
  const auto clear = [&](int cols) {
    for (int v = lane; v * VE < cols; v += 64)
      *reinterpret_cast<u32x4 *>(buf + v * VE) = u32x4{0, 0, 0, 0};
  };
  const int(&col)[NE] = entries.col;
  const float(&xv)[NE] = entries.x;
  const float(&yv)[NE] = entries.y;
  if (want_grad)
    clear(n < part_cols ? n : part_cols);
  // The entry of the action (the first of equal ones), if no mask took it out.
  bool acted = false;
  float xa = 0.f, m = xv[0];
#pragma unroll
  for (int r = 0; r < NE; ++r) {
    m = fmaxf(m, xv[r]);
    const unsigned long long hit =
        __ballot(act >= 0 && col[r] == act && xv[r] != -__builtin_inff());
    if (hit && !acted) {
      acted = true;
      xa = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(xv[r]), __ffsll(hit) - 1));
    }
  }
  const float top = WaveMax(m);
  m = top == -__builtin_inff() ? 0.f : top;
  const float c = a.inv_temp * kLog2e;
  Sums sums = NoSums<true>();
#pragma unroll
  for (int r = 0; r < NE; ++r)
    AddStats<REF, true>(xv[r], yv[r], m, c, sums);
  (void)GroupSums<1, REF, true>(sums, top, c, nullptr);
  RowStats st = Stats(m, sums);
  const bool apart = REF && FarApart(st, sums.far);
  if (apart) {
    float part = 0.f;
#pragma unroll
    for (int r = 0; r < NE; ++r)
      part += ApartPart(xv[r], yv[r], m, sums.far, c);
    st.mean_d = ApartMean(WaveSum(part), sums.e);
  }
  const RowResult res = Evaluate(a, in, st, acted, xa);
  const bool want_kl = REF && WantsKl(a);
  float kl = 0.f, f[NE] = {};
  if (!st.empty && (want_grad || want_kl)) {
    const Coefs k = CoefsOf(st, res.grad, a.inv_temp);
    const FarCoefs far = FarCoefsOf(st, k, sums.far, apart);
#pragma unroll
    for (int r = 0; r < NE; ++r) {
      const float xs[1] = {xv[r]}, ys[1] = {yv[r]};
      float ft[1];
      FinishEntries<1, REF, true>(k, far, want_kl, xs, ys, kl, ft);
      f[r] = ft[0];
    }
    if (want_kl)
      kl = KlOf<true>(WaveSum(kl), k, far);
  }
  if (lane == 0) {
    if (st.empty)
      WriteZeros(a, row);
    else
      WriteRow(a, row, in.weight, acted, res, kl);
  }
  if (!want_grad)
    return;
  for (int p0 = 0; p0 < n; p0 += part_cols) {
    const int cols = n - p0 < part_cols ? n - p0 : part_cols;
    if (p0 > 0)
      clear(cols);
    if (!st.empty) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      bool other = false;
#pragma unroll
      for (int r = 0; r < NE; ++r)
        if (col[r] >= p0 && col[r] < p0 + cols)
          buf[col[r] - p0] = static_cast<T>(r * 64 + lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int r = 0; r < NE; ++r)
        if (col[r] >= p0 && col[r] < p0 + cols)
          other = other || buf[col[r] - p0] != static_cast<T>(r * 64 + lane);
      const bool twice = __any(other);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int r = 0; r < NE; ++r) {
        float value = f[r];
        bool writes = col[r] >= p0 && col[r] < p0 + cols;
        if (twice) {
          float times = 0.f;
#pragma unroll
          for (int q = 0; q < NE; ++q)
#pragma unroll 1
            for (int i = 0; i < 64; ++i) {
              const int same = __builtin_amdgcn_readlane(col[q], i);
              if (same == col[r]) {
                times += 1.f;
                writes = writes && q * 64 + i >= r * 64 + lane;
              }
            }
          value *= times;
        }
        if (writes)
          buf[col[r] - p0] =
              E::Round(acted && col[r] == act ? value + res.grad.scale * res.grad.slope : value);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int vecs = cols / VE;
    for (int v = lane; v < vecs; v += 64)
      StoreVec<DT, PAST>(g + p0 + v * VE, *reinterpret_cast<const u32x4 *>(buf + v * VE));
    const int t = vecs * VE + lane;
    if (lane < VE && t < cols)
      g[p0 + t] = buf[t];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// A row by its list, by one wave.  Up to 64 moves, as nearly all rows have,
// take one entry a lane.
template <int DT, bool REF, bool PAST>
__device__ __forceinline__ void ListedRow(const RowLossParams &a, std::int64_t row,
                                          const RowInputs &in, unsigned char *lds, int part_cols) {
  std::int64_t start = Uniform(a.offsets, row), count = Uniform(a.offsets, row + 1);
  if (in.weight == 0.f) {
    if ((threadIdx.x & 63) == 0)
      WriteZeros(a, row);
    if (a.g)
      ZeroRow<DT>(RowOf<DT>(a.g, row, a.ldg), a.vocab, threadIdx.x & 63, 64);
    return;
  }
  start = start < 0 ? 0 : start > a.n_moves ? a.n_moves : start;
  count = (count > a.n_moves ? a.n_moves : count) - start;
  const int moves = count < 0 ? 0 : count > kMaxMoves ? kMaxMoves : static_cast<int>(count);
  if (moves <= 64) {
    Entries<1> e;
    LoadColumns(a, start, moves, e);
    LoadLogits<DT, REF>(a, row, moves, e);
    MovesRow<DT, REF, PAST>(a, row, in, e, lds, part_cols);
  } else {
    Entries<kMaxMoves / 64> e;
    LoadColumns(a, start, moves, e);
    LoadLogits<DT, REF>(a, row, moves, e);
    MovesRow<DT, REF, PAST>(a, row, in, e, lds, part_cols);
  }
}

// Four waves to a workgroup, each with a row of its own.  (Four rows a wave,
// their lists and logits loaded together, took 20 % longer at 20000 rows and
// 60 % at 1000: the waves hide each other's loads.)
constexpr int kPartBytes = 8192;  // of each wave's LDS
template <int DT, bool REF, bool PAST>
__global__ __launch_bounds__(256) void MovesRowKernel(RowLossParams a, int part_cols) {
  extern __shared__ u32x4 parts[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::int64_t row = a.row0 + static_cast<std::int64_t>(blockIdx.x) * 4 + wave;
  if (row >= a.end || OutsideSequences(a, row))
    return;
  ListedRow<DT, REF, PAST>(a, row, Inputs(a, row),
                           reinterpret_cast<unsigned char *>(parts) +
                               static_cast<size_t>(wave) * part_cols *
                                   sizeof(typename Elem<DT>::T),
                           part_cols);
}

// Columns of a part of a row in LDS: a whole number of vectors.
template <int DT> int PartCols(int vocab) {
  constexpr int VE = Elem<DT>::kPerVec, most = kPartBytes / (16 / VE);
  const int whole = (vocab + VE - 1) / VE * VE;
  return whole < most ? whole : most;
}

template <int DT, bool REF, bool PAST, int W, int NV>
void LaunchDense(const RowLossParams &p, unsigned rows, hipStream_t s) {
  hipLaunchKernelGGL((DenseRowKernel<DT, W, NV, REF, PAST>), dim3(W == 1 ? (rows + 3) / 4 : rows),
                     dim3(W == 1 ? 256 : 64 * W), 0, s, p);
}

template <int DT, bool REF, int NV>
void LaunchLoop(const RowLossParams &p, unsigned rows, hipStream_t s) {
  hipLaunchKernelGGL((LoopRowKernel<DT, NV, REF>), dim3(rows < kCus ? rows : kCus), dim3(1024), 0,
                     s, p);
}

// Which kernel takes rows of `vocab` columns.  Measured beside the choice:
//  * 465 vectors (1858 of fp32) on four waves 60.4 us at 16384 rows and 5.4 at
//    64, on one wave with eight vectors a lane 64.2 and 7.1;
//  * 1072 vectors (4288 of fp32) on eight waves, four vectors a lane 157 us at
//    16384 rows, eight a lane 185;
//  * 4000 vectors (32000 of bf16, 3588 rows) on eight waves 38 us, on sixteen
//    48.6 (statistics alone, fastest runs);
//  * 6253 vectors (50021 of bf16 with a reference, 1500 rows) in a loop 133 us,
//    one row a workgroup 145, streamed twice 173.
template <int DT, bool REF, bool PAST>
void LaunchRows(const RowLossParams &p, unsigned rows, hipStream_t s) {
  constexpr int VE = Elem<DT>::kPerVec;
  if (p.offsets) {
    const int part = PartCols<DT>(p.vocab);
    hipLaunchKernelGGL((MovesRowKernel<DT, REF, PAST>), dim3((rows + 3) / 4), dim3(256),
                       p.g ? 4 * part * sizeof(typename Elem<DT>::T) : 0, s, p, part);
    return;
  }
  const int vecs = p.vocab / VE;
  if (vecs <= 64)
    LaunchDense<DT, REF, PAST, 1, 1>(p, rows, s);
  else if (vecs <= 256 && rows <= kFewRows)
    LaunchDense<DT, REF, PAST, 4, 1>(p, rows, s);
  else if (vecs <= 128)
    LaunchDense<DT, REF, PAST, 1, 2>(p, rows, s);
  else if (vecs <= 256)
    LaunchDense<DT, REF, PAST, 1, 4>(p, rows, s);
  else if (vecs <= 512)
    LaunchDense<DT, REF, PAST, 4, 2>(p, rows, s);
  else if (vecs <= 1024)
    LaunchDense<DT, REF, PAST, 4, 4>(p, rows, s);
  else if (vecs <= 2048)
    LaunchDense<DT, REF, PAST, 8, 4>(p, rows, s);
  else if (vecs <= 4096)
    LaunchDense<DT, REF, PAST, 8, 8>(p, rows, s);
  else if (vecs <= 5120)
    LaunchLoop<DT, REF, 5>(p, rows, s);
  else if (vecs <= 6144)
    LaunchLoop<DT, REF, 6>(p, rows, s);
  else if (vecs <= 7168)
    LaunchLoop<DT, REF, 7>(p, rows, s);
  else if (vecs <= 8192)
    LaunchLoop<DT, REF, 8>(p, rows, s);
  else
    hipLaunchKernelGGL((StreamRowKernel<DT, REF>), dim3(rows), dim3(1024), kHalfLds, s, p);
}

template <int DT>
void LaunchRowsOf(const RowLossParams &p, bool past, unsigned rows, hipStream_t s) {
  if (p.y)
    past ? LaunchRows<DT, true, true>(p, rows, s) : LaunchRows<DT, true, false>(p, rows, s);
  else
    past ? LaunchRows<DT, false, true>(p, rows, s) : LaunchRows<DT, false, false>(p, rows, s);
}

// Sum over the W waves of a workgroup, in a fixed order.
template <int W> __device__ __forceinline__ double GroupSum64(double v, double *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v += __shfl_xor(v, o, 64);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
      red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < W; ++w)
      v += red[w];
  }
  return v;
}

// A pair's loss from the marks of its rows, by W waves; the coefficients of
// the gradients of its two sequences' rows.
struct PairResult {
  std::int64_t begin, middle, end;  // rows of the two sequences
  float share[2];
};
template <int W>
__device__ __forceinline__ PairResult PairLoss(const PairLossParams &a, std::int64_t pair,
                                               double *red) {
  PairResult r;
  const float w = a.weight ? Uniform(a.weight, pair) : 1.f;
  std::int64_t at[3];
#pragma unroll
  for (int s = 0; s < 3; ++s) {
    at[s] = Uniform(a.seq_offsets, 2 * pair + s);
    at[s] = at[s] < 0 ? 0 : at[s] > a.rows ? a.rows : at[s];
  }
  r.begin = at[0];
  r.middle = at[1] < at[0] ? at[0] : at[1];
  r.end = at[2] < r.middle ? r.middle : at[2];
  double sum[2] = {0.0, 0.0}, count[2] = {0.0, 0.0};
  for (std::int64_t i = r.begin + threadIdx.x; i < r.end; i += 64 * W) {
    const float l = a.mark[i];
    const double ref = a.ref_logp ? static_cast<double>(a.ref_logp[i]) : 0.0;
    const int s = i >= r.middle;
    if (l != kNoAction) {
      sum[s] += l - ref;
      count[s] += 1.0;
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    sum[s] = GroupSum64<W>(sum[s], red);
    if (a.average) {
      count[s] = GroupSum64<W>(count[s], red);
      if (count[s] > 0.0)
        sum[s] /= count[s];
    }
  }
  const double beta = a.beta, diff = sum[0] - sum[1], h = beta * diff;
  double loss, slope;  // slope: by the difference of the two sums
  if (a.kind == 0) {
    // ln(1 + e^-h) and ln(1 + e^h) = ln(1 + e^-|h|) + max(0, -+h); sig(h)
    // from the same exponential.  Without smoothing h may be +inf.
    const double eps = a.smoothing, tail = exp(-fabs(h)), base = log1p(tail);
    const double small = tail / (1.0 + tail), sig = h >= 0.0 ? 1.0 - small : small;
    loss = base + (1.0 - eps) * fmax(-h, 0.0) + (eps > 0.0 ? eps * fmax(h, 0.0) : 0.0);
    if (h != h)
      loss = h;
    slope = beta * (eps * sig - (1.0 - eps) * (h >= 0.0 ? small : 1.0 - small));
  } else if (a.kind == 1) {
    loss = h < 1.0 ? 1.0 - h : h >= 1.0 ? 0.0 : h;
    slope = h < 1.0 ? -beta : h >= 1.0 ? 0.0 : h;
  } else {
    const double off = diff - 0.5 / beta;
    loss = off * off;
    slope = 2.0 * off;
  }
  if (threadIdx.x == 0) {
    if (a.loss)
      a.loss[pair] = w == 0.f ? 0.f : static_cast<float>(w * loss);
    if (a.margin)
      a.margin[pair] = w == 0.f ? 0.f : static_cast<float>(h);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const double c = a.average && count[s] > 0.0 ? slope / count[s] : slope;
    r.share[s] = w == 0.f ? 0.f : static_cast<float>(w * (s == 0 ? c : -c));
  }
  return r;
}

template <int W> __global__ __launch_bounds__(64 * W) void PairLossKernel(PairLossParams a) {
  __shared__ double red[W];
  const PairResult r = PairLoss<W>(a, blockIdx.x, red);
  for (std::int64_t i = r.begin + threadIdx.x; i < r.end; i += 64 * W) {
    const float l = a.mark[i];
    const bool acted = l != kNoAction;
    if (a.coef)
      a.coef[i] = acted ? r.share[i >= r.middle] : 0.f;
    if (a.logp)
      a.logp[i] = acted ? l : 0.f;
  }
}

// A few short lines of moves in one launch: a workgroup takes a pair, its waves
// the pair's rows in turn; marks through the workspace as in the three
// launches.  Up to 8 rows a pair on average (one a wave) and 512 pairs: 16
// pairs of 2 rows 6.4 us (9.4 in three launches), 256 pairs of about 5 rows 8.1
// (11.3); 1024 pairs of 2 rows 15.1 (12.8), 128 pairs of 60 rows 50 (25).  The
// host does not know the lengths, and the longest pair is one workgroup's: 100
// pairs of 3 rows 7.0 (10.0), with one of 120 rows among them 44.5 (10.3), 512
// pairs of 4 with one of 2000 789 (27).
constexpr int kPairWaves = 8, kFewPairs = 512;
template <int DT>
__global__ __launch_bounds__(64 * kPairWaves) void PairMovesKernel(RowLossParams a,
                                                                   PairLossParams q,
                                                                   int part_cols) {
  extern __shared__ u32x4 parts[];
  __shared__ double red[kPairWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned char *lds = reinterpret_cast<unsigned char *>(parts) +
                       static_cast<size_t>(wave) * part_cols * sizeof(typename Elem<DT>::T);
  const std::int64_t pair = blockIdx.x;
  std::int64_t from = Uniform(q.seq_offsets, 2 * pair), to = Uniform(q.seq_offsets, 2 * pair + 2);
  from = from < 0 ? 0 : from;
  to = to > q.rows ? q.rows : to;
  RowLossParams marks = a;
  marks.g = nullptr;
  for (std::int64_t row = from + wave; row < to; row += kPairWaves) {
    RowInputs in = Inputs(marks, row);
    ListedRow<DT, false, false>(marks, row, in, lds, part_cols);
  }
  __syncthreads();
  const PairResult r = PairLoss<kPairWaves>(q, pair, red);
  RowLossParams grads = a;
  grads.mark = nullptr;
  grads.coef = q.mark;  // not read: the coefficient is at hand
  for (std::int64_t row = r.begin + wave; row < r.end; row += kPairWaves) {
    const float l = q.mark[row];
    const bool acted = l != kNoAction;
    if (q.logp && lane == 0)
      q.logp[row] = acted ? l : 0.f;
    if (!a.g)
      continue;
    RowInputs in{};
    in.weight = __int_as_float(__builtin_amdgcn_readfirstlane(
        __float_as_int(acted ? r.share[row >= r.middle] : 0.f)));
    in.action = a.actions ? Uniform(a.actions, row) : -1;
    ListedRow<DT, false, false>(grads, row, in, lds, part_cols);
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
  const double arrays = 1.0 + (p.y != nullptr) + (p.g != nullptr);
  const bool past = arrays * p.rows * p.vocab * DTypeBytes(p.dtype) > kPastBytes;
  // A launch holds fewer than 2^32 threads.
  constexpr std::int64_t kRows = std::int64_t(1) << 21;
  for (q.row0 = 0; q.row0 < p.rows; q.row0 += kRows) {
    q.end = p.rows - q.row0 < kRows ? p.rows : q.row0 + kRows;
    const unsigned rows = static_cast<unsigned>(q.end - q.row0);
    if (p.dtype == DT_F32)
      LaunchRowsOf<DT_F32>(q, past, rows, stream);
    else if (p.dtype == DT_BF16)
      LaunchRowsOf<DT_BF16>(q, past, rows, stream);
    else
      LaunchRowsOf<DT_F16>(q, past, rows, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return e;
  }
  return hipSuccess;
}

template <int DT>
static void LaunchPairMoves(const RowLossParams &p, const PairLossParams &q, hipStream_t s) {
  const int part = PartCols<DT>(p.vocab);
  hipLaunchKernelGGL(PairMovesKernel<DT>, dim3(static_cast<unsigned>(q.pairs)),
                     dim3(64 * kPairWaves),
                     p.g ? kPairWaves * part * sizeof(typename Elem<DT>::T) : 0, s, p, q, part);
}

hipError_t LaunchPreference(const RowLossParams &rows, const PairLossParams &pairs,
                            hipStream_t stream, std::string *err) {
  if (pairs.pairs < 0 || pairs.pairs > (1 << 23) ||
      (pairs.pairs > 0 && (!pairs.seq_offsets || (pairs.rows > 0 && !pairs.mark))) ||
      (pairs.rows > 0 && rows.g && !pairs.coef)) {
    if (err)
      *err = "preference: needs 0 <= pairs <= 2^23, offsets and a workspace";
    return hipErrorInvalidValue;
  }
  if (pairs.pairs == 0)
    return hipSuccess;
  if (rows.offsets && pairs.pairs <= kFewPairs && rows.rows <= kPairWaves * pairs.pairs) {
    RowLossParams p = rows;
    p.mark = pairs.mark;
    if (p.dtype == DT_F32)
      LaunchPairMoves<DT_F32>(p, pairs, stream);
    else if (p.dtype == DT_BF16)
      LaunchPairMoves<DT_BF16>(p, pairs, stream);
    else
      LaunchPairMoves<DT_F16>(p, pairs, stream);
    return hipGetLastError();
  }
  RowLossParams p = rows;
  p.g = nullptr;
  p.mark = pairs.mark;
  p.seq_offsets = pairs.seq_offsets;
  p.n_seq = 2 * pairs.pairs;
  hipError_t e = LaunchRowLoss(p, stream, err);
  if (e != hipSuccess)
    return e;
  const dim3 grid(static_cast<unsigned>(pairs.pairs));
  if (pairs.rows <= 256 * pairs.pairs)
    hipLaunchKernelGGL(PairLossKernel<1>, grid, dim3(64), 0, stream, pairs);
  else
    hipLaunchKernelGGL(PairLossKernel<4>, grid, dim3(256), 0, stream, pairs);
  e = hipGetLastError();
  if (e != hipSuccess || !rows.g)
    return e;
  p.g = rows.g;
  p.mark = nullptr;
  p.coef = pairs.coef;
  return LaunchRowLoss(p, stream, err);
}

}  // namespace mfh
