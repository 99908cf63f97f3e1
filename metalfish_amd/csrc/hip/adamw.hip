// AdamW over many tensors in one launch, for gfx950.
//
//   g = grad f,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   param = param (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: with states and gradients in 32 bits a weight costs 28
// bytes (159 M of them 753 us, 5.9 TB/s), with states in 8 bits, bf16 gradients
// and a bf16 copy 16 (427 to 436 us, 5.9 TB/s; the vector unit is busy four fifths of that).
// The tensors are cut into chunks of kAdamChunk values, listed once per set, and a
// workgroup takes whole chunks; every value is read and written once, in whole
// vectors.
//
// States in 8 bits are codes in blocks of kAdamBlock values with one fp32 scale
// each.  A block is four values a lane of one wave, so its largest value is one
// reduction over the wave and nothing leaves registers.  m is OCP e4m3
// (relative steps of 1/8 over 18 octaves below the block's largest), v has the
// sign's bit as a fifth one of exponent (34 octaves: a gradient 2^-17 of the
// block's largest still has its own v).  Products, sums and scales are rounded
// one by one (no contraction), so the codes are a function of the formulas
// alone.
#include "learn_device.h"
#include "mfh_device.h"
#include "mfh_kernels.h"

#include <algorithm>
#include <cmath>

namespace mfh {
namespace {

// A workgroup a chunk, up to this many: 159 M weights with a bf16 copy, bf16
// gradients and states in 8 bits 427 us, on 8192 workgroups that loop 470; all in
// 32 bits 753 and 801.
constexpr int kMaxGroups = 1 << 20;
constexpr int kPer = 4;                          // consecutive values of a lane
constexpr int kDeep = kAdamChunk / (256 * kPer);  // such runs of a lane in a chunk
static_assert(kAdamBlock == 64 * kPer, "a block is one run of a wave");

typedef unsigned int u32x2_a2 __attribute__((ext_vector_type(2), aligned(2), may_alias));
typedef unsigned int u32_a1 __attribute__((aligned(1), may_alias));

// How states are held: in 32 bits, or in 8 rounded to nearest or stochastically.
enum : int { kFull, kNearest, kStochastic };

// Uniform over the launch.
struct Step {
  double lr, size, grad_scale;  // size: lr / (1 - b1^t)
  double log_beta1, log_beta2;
  std::int64_t step;
  const float *d_lr;
  const std::int64_t *d_step;
  const double *sumsq;
  double max_norm;
  float b1, c1, b2, c2, eps, rbc2;  // c = 1 - b, rbc2 = 1 / sqrt(1 - b2^t)
  bool skip;
  std::uint64_t seed;
};

// A factor in 24 bits, as a product where it is below 2^-126.
struct Factor {
  float high, low;
};

// Vectors at any element's alignment, through the caches or (PAST) past them.
struct Vec16 {
  using V = u32x4_a4;
};
struct Vec8 {
  using V = u32x2_a2;
};
struct Vec4 {
  using V = u32_a1;
};
template <bool PAST, class K> __device__ __forceinline__ auto Load(const MFH_GLOBAL void *p) {
  const auto *v = (const MFH_GLOBAL typename K::V *)p;
  if constexpr (PAST)
    return __builtin_nontemporal_load(v);
  else
    return *v;
}
template <bool PAST, class K, class T>
__device__ __forceinline__ void Store(MFH_GLOBAL void *p, T value) {
  auto *v = (MFH_GLOBAL typename K::V *)p;
  if constexpr (PAST)
    __builtin_nontemporal_store(static_cast<typename K::V>(value), v);
  else
    *v = value;
}

// Four consecutive values from `at` on, of which `n` exist (FULL: all).
template <int DT, bool FULL, bool PAST>
__device__ __forceinline__ void Load4(const void *base, int at, int n, float *f) {
  const auto *p = (const MFH_GLOBAL typename Elem<DT>::T *)base + at;
  if (FULL || n >= 4) {
    if constexpr (DT == DT_F32) {
      const u32x4 v = Load<PAST, Vec16>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = __uint_as_float(v[e]);
    } else {
      const u32x2 v = Load<PAST, Vec8>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = Elem<DT>::One(static_cast<std::uint16_t>(v[e >> 1] >> (16 * (e & 1))));
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    f[e] = e < n ? Elem<DT>::One(p[e]) : 0.f;
}

template <int DT, bool FULL, bool PAST>
__device__ __forceinline__ void Store4(void *base, int at, int n, const float *f) {
  auto *p = (MFH_GLOBAL typename Elem<DT>::T *)base + at;
  if (FULL || n >= 4) {
    if constexpr (DT == DT_F32) {
      Store<PAST, Vec16>(p, Elem<DT>::Pack(f));
    } else {
      u32x2 v;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        v[i] = Elem<DT>::Round(f[2 * i]) |
               static_cast<std::uint32_t>(Elem<DT>::Round(f[2 * i + 1])) << 16;
      Store<PAST, Vec8>(p, v);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n)
      p[e] = Elem<DT>::Round(f[e]);
}

template <bool FULL, bool PAST>
__device__ __forceinline__ unsigned LoadCodes(const void *base, int at, int n) {
  const auto *p = (const MFH_GLOBAL std::uint8_t *)base + at;
  if (FULL || n >= 4)
    return Load<PAST, Vec4>(p);
  unsigned v = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n)
      v |= static_cast<unsigned>(p[e]) << (8 * e);
  return v;
}
template <bool FULL, bool PAST>
__device__ __forceinline__ void StoreCodes(void *base, int at, int n, unsigned v) {
  auto *p = (MFH_GLOBAL std::uint8_t *)base + at;
  if (FULL || n >= 4) {
    Store<PAST, Vec4>(p, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n)
      p[e] = static_cast<std::uint8_t>(v >> (8 * e));
}

// Largest of non-negative floats over a wave by their bits: NaN is above
// infinity, so neither is lost.
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned DppU(unsigned v) {
  return static_cast<unsigned>(__builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v),
                                                           CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float WaveMaxBits(unsigned v) {
  v = max(v, DppU<kRowShr + 1, 0xF>(v));
  v = max(v, DppU<kRowShr + 2, 0xF>(v));
  v = max(v, DppU<kRowShr + 4, 0xF>(v));
  v = max(v, DppU<kRowShr + 8, 0xF>(v));
  v = max(v, DppU<kBcast15, 0xA>(v));
  v = max(v, DppU<kBcast31, 0xC>(v));
  return __uint_as_float(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), 63)));
}

// Code of x >= 0 over its scale, already multiplied by the power of two that
// takes the code's smallest normal number to fp32's: exponent and three bits
// of mantissa are then the bits above 20, subnormal codes those of a subnormal
// number.  The twenty bits below are rounded to nearest, ties to even, or
// (STOCHASTIC) up by `up`.
template <bool STOCHASTIC>
__device__ __forceinline__ unsigned CodeOf(float y, unsigned up, unsigned most) {
  const unsigned bits = __float_as_uint(y);
  const unsigned add = STOCHASTIC ? up : 0x7FFFFu + ((bits >> 20) & 1u);
  return min((bits + add) >> 20, most);
}

// 32 bits that look random, from a value's place and the step's key: odd
// multipliers (the golden ratio, the square roots of 3 and 2) with shifts in
// between.  `x`: the place, with the key's low bits, times the first of them.
constexpr unsigned kGolden = 0x9E3779B1u;
__device__ __forceinline__ unsigned RandomBits(unsigned x, unsigned key_high) {
  x ^= x >> 15;
  x = x * 0xBB67AE85u + key_high;
  x ^= x >> 13;
  x *= 0x6A09E667u;
  return x ^ (x >> 16);
}

// Square root on the vector unit's own (1 ulp), which takes no subnormal
// numbers.
__device__ __forceinline__ float Sqrt(float v) {
  const bool small = v < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v);
  return small ? r * 0x1p-32f : r;
}

struct Uniform {
  Factor f;
  double lr, size;
  float b1, c1, b2, c2, eps, rbc2;
  unsigned key_low, key_high;
};

template <int PDT, int GDT, int STATE, bool FULL, bool PAST>
__device__ __forceinline__ void DoChunk(const AdamChunk &c, const Uniform &u) {
#pragma clang fp contract(off)
  constexpr bool EIGHT = STATE != kFull;
  const float size = static_cast<float>(u.size * c.lr_scale);
  const float keep = static_cast<float>(1.0 - u.lr * c.lr_scale * c.weight_decay);
  const int lane_at = threadIdx.x * kPer;
  float p[kDeep][4], g[kDeep][4], m[kDeep][4], v[kDeep][4];
  unsigned mc[kDeep], vc[kDeep];
  float ms[kDeep], vs[kDeep];
#pragma unroll
  for (int j = 0; j < kDeep; ++j) {
    const int at = j * 256 * kPer + lane_at, n = c.count - at;
    if (!FULL && j * 256 * kPer + (lane_at & ~(kAdamBlock - 1)) >= c.count)
      break;  // the whole wave
    Load4<PDT, FULL, PAST>(c.param, at, n, p[j]);
    Load4<GDT, FULL, PAST>(c.grad, at, n, g[j]);
    if constexpr (EIGHT) {
      const int block = at / kAdamBlock;
      mc[j] = LoadCodes<FULL, PAST>(c.m, at, n);
      vc[j] = LoadCodes<FULL, PAST>(c.v, at, n);
      ms[j] = ((const MFH_GLOBAL float *)c.m_scale)[block];
      vs[j] = ((const MFH_GLOBAL float *)c.v_scale)[block];
    } else {
      Load4<DT_F32, FULL, PAST>(c.m, at, n, m[j]);
      Load4<DT_F32, FULL, PAST>(c.v, at, n, v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kDeep; ++j) {
    const int at = j * 256 * kPer + lane_at, n = c.count - at;
    if (!FULL && j * 256 * kPer + (lane_at & ~(kAdamBlock - 1)) >= c.count)
      break;
    if constexpr (EIGHT) {
      m[j][0] = __builtin_amdgcn_cvt_f32_fp8(mc[j], 0) * ms[j];
      m[j][1] = __builtin_amdgcn_cvt_f32_fp8(mc[j], 1) * ms[j];
      m[j][2] = __builtin_amdgcn_cvt_f32_fp8(mc[j], 2) * ms[j];
      m[j][3] = __builtin_amdgcn_cvt_f32_fp8(mc[j], 3) * ms[j];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[j][e] = (__uint_as_float(((vc[j] >> (8 * e)) & 0xFFu) << 20) * 0x1p112f) * vs[j];
    }
    unsigned m_most = 0, v_most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gr = (g[j][e] * u.f.high) * u.f.low;
      m[j][e] = m[j][e] * u.b1 + gr * u.c1;
      v[j][e] = v[j][e] * u.b2 + (gr * gr) * u.c2;
      const float denom = __builtin_fmaf(Sqrt(v[j][e]), u.rbc2, u.eps);
      const float update = m[j][e] * __builtin_amdgcn_rcpf(denom);
      p[j][e] = __builtin_fmaf(-size, update, p[j][e] * keep);
      if constexpr (EIGHT) {
        if (FULL || e < n) {
          m_most = max(m_most, __float_as_uint(m[j][e]) & 0x7FFFFFFFu);
          v_most = max(v_most, __float_as_uint(v[j][e]));
        }
      }
    }
    Store4<PDT, FULL, PAST>(c.param, at, n, p[j]);
    if (c.copy) {
      // The copy of the weights as they are held, rounded from those.
      if constexpr (PDT != DT_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p[j][e] = Elem<PDT>::One(Elem<PDT>::Round(p[j][e]));
      }
      if (c.copy_dtype == DT_F32)
        Store4<DT_F32, FULL, PAST>(c.copy, at, n, p[j]);
      else if (c.copy_dtype == DT_BF16)
        Store4<DT_BF16, FULL, PAST>(c.copy, at, n, p[j]);
      else
        Store4<DT_F16, FULL, PAST>(c.copy, at, n, p[j]);
    }
    if constexpr (!EIGHT) {
      Store4<DT_F32, FULL, PAST>(c.m, at, n, m[j]);
      Store4<DT_F32, FULL, PAST>(c.v, at, n, v[j]);
    } else {
      const float m_scale = WaveMaxBits(m_most) * (1.f / 448.f);
      const float v_scale = WaveMaxBits(v_most) * (1.f / 122880.f);
      ms[j] = m_scale < 0x1p-100f ? 0x1p-100f : m_scale;  // NaN stays
      vs[j] = v_scale < 0x1p-120f ? 0x1p-120f : v_scale;
    }
  }
  if constexpr (EIGHT) {
    // The reciprocals of all the wave's scales in one division: lane 2 j has m's of
    // run j, lane 2 j + 1 v's.
    const int lane = threadIdx.x & 63;
    float scale = 1.f;
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      scale = lane == 2 * j ? ms[j] : scale;
      scale = lane == 2 * j + 1 ? vs[j] : scale;
    }
    const int inverse = __float_as_int(1.f / scale);
    // Places of a run differ in their two last bits, so their products with the
    // first multiplier differ by what the key's last bits say.
    unsigned steps[4];
#pragma unroll
    for (unsigned e = 0; e < 4; ++e)
      steps[e] = (((u.key_low ^ e) & 3u) - (u.key_low & 3u)) * kGolden;
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const int at = j * 256 * kPer + lane_at, n = c.count - at;
      if (!FULL && j * 256 * kPer + (lane_at & ~(kAdamBlock - 1)) >= c.count)
        break;
      const float m_inv = __int_as_float(__builtin_amdgcn_readlane(inverse, 2 * j)),
                  v_inv = __int_as_float(__builtin_amdgcn_readlane(inverse, 2 * j + 1));
      unsigned m_out = 0, v_out = 0, first = 0;
      if constexpr (STATE == kStochastic) {
        const std::uint64_t place = static_cast<std::uint64_t>(c.first_block) * kAdamBlock + at;
        const unsigned key = u.key_low ^ static_cast<unsigned>(place >> 32) * 0x6A09E664u;
        first = (static_cast<unsigned>(place) ^ key) * kGolden;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        unsigned r = 0;
        if constexpr (STATE == kStochastic)
          r = RandomBits(first + steps[e], u.key_high);
        const float x = m[j][e] * m_inv, y = v[j][e] * v_inv;
        unsigned a = CodeOf<STATE == kStochastic>(fabsf(x) * 0x1p-120f, (r & 0xFFFFu) << 4, 0x7Eu);
        a |= x < 0.f ? 0x80u : 0u;
        unsigned b = CodeOf<STATE == kStochastic>(y * 0x1p-112f, (r >> 16) << 4, 0xFFu);
        b = max(b, v[j][e] > 0.f ? 1u : 0u);
        m_out |= a << (8 * e);
        v_out |= b << (8 * e);
      }
      StoreCodes<FULL, PAST>(c.m, at, n, m_out);
      StoreCodes<FULL, PAST>(c.v, at, n, v_out);
      if (lane == 0) {
        ((MFH_GLOBAL float *)c.m_scale)[at / kAdamBlock] = ms[j];
        ((MFH_GLOBAL float *)c.v_scale)[at / kAdamBlock] = vs[j];
      }
    }
  }
}

template <int PDT, int GDT, int STATE, bool PAST>
__device__ __forceinline__ void AnyChunk(const AdamChunk &c, const Uniform &u) {
  if (c.count == kAdamChunk)
    DoChunk<PDT, GDT, STATE, true, PAST>(c, u);
  else
    DoChunk<PDT, GDT, STATE, false, PAST>(c, u);
}
template <int PDT, int STATE, bool PAST>
__device__ __forceinline__ void ByGrad(const AdamChunk &c, const Uniform &u) {
  if (c.grad_dtype == DT_F32)
    AnyChunk<PDT, DT_F32, STATE, PAST>(c, u);
  else if (c.grad_dtype == DT_BF16)
    AnyChunk<PDT, DT_BF16, STATE, PAST>(c, u);
  else
    AnyChunk<PDT, DT_F16, STATE, PAST>(c, u);
}

template <int STATE, bool PAST>
__global__ __launch_bounds__(256) void AdamWKernel(const AdamChunk *list, std::int64_t n, Step s) {
  const auto *chunks = (const MFH_CONSTANT AdamChunk *)list;
  Uniform u;
  double factor = s.grad_scale;
  if (s.sumsq) {
    const double sumsq = *s.sumsq;
    if (s.skip && !(sumsq < __builtin_inf()))
      return;
    const double norm = s.grad_scale * sqrt(sumsq);
    // NaN is not <= anything, and goes into every weight.
    if (!(norm <= s.max_norm))
      factor *= s.max_norm / norm;
  }
  const bool tiny = factor < 0x1p-126;
  u.f = {static_cast<float>(tiny ? factor * 0x1p64 : factor), tiny ? 0x1p-64f : 1.f};
  u.lr = s.lr;
  u.size = s.size;
  u.rbc2 = s.rbc2;
  std::int64_t step = s.step;
  if (s.d_lr || s.d_step) {
    if (s.d_lr)
      u.lr = *s.d_lr;
    if (s.d_step)
      step = *s.d_step < 1 ? 1 : *s.d_step;
    u.size = u.lr / -expm1(static_cast<double>(step) * s.log_beta1);
    u.rbc2 = static_cast<float>(1.0 / sqrt(-expm1(static_cast<double>(step) * s.log_beta2)));
  }
  u.b1 = s.b1;
  u.c1 = s.c1;
  u.b2 = s.b2;
  u.c2 = s.c2;
  u.eps = s.eps;
  std::uint64_t key = s.seed + static_cast<std::uint64_t>(step) * 0x9E3779B97F4A7C15ull;
  key ^= key >> 29;
  u.key_low = static_cast<unsigned>(key);
  u.key_high = static_cast<unsigned>(key >> 32);
  for (std::int64_t k = blockIdx.x; k < n; k += gridDim.x) {
    AdamChunk c;
    c.param = chunks[k].param;
    c.grad = chunks[k].grad;
    c.m = chunks[k].m;
    c.v = chunks[k].v;
    c.copy = chunks[k].copy;
    c.m_scale = chunks[k].m_scale;
    c.v_scale = chunks[k].v_scale;
    c.first_block = chunks[k].first_block;
    c.count = chunks[k].count;
    c.param_dtype = chunks[k].param_dtype;
    c.grad_dtype = chunks[k].grad_dtype;
    c.copy_dtype = chunks[k].copy_dtype;
    c.lr_scale = chunks[k].lr_scale;
    c.weight_decay = chunks[k].weight_decay;
    if (c.param_dtype == DT_F32)
      ByGrad<DT_F32, STATE, PAST>(c, u);
    else if (c.param_dtype == DT_BF16)
      ByGrad<DT_BF16, STATE, PAST>(c, u);
    else
      ByGrad<DT_F16, STATE, PAST>(c, u);
  }
}

}  // namespace

hipError_t LaunchAdamW(const AdamChunk *chunks, std::int64_t n_chunks, bool eight, bool past,
                       const AdamParams &p, hipStream_t stream, std::string *err) {
  if (n_chunks < 0 || (n_chunks > 0 && !chunks) || p.step < 1) {
    if (err)
      *err = "adamw: needs a chunk list and a step of at least 1";
    return hipErrorInvalidValue;
  }
  if (n_chunks == 0)
    return hipSuccess;
  Step s{};
  s.log_beta1 = std::log(p.beta1);
  s.log_beta2 = std::log(p.beta2);
  const double t = static_cast<double>(p.step);
  s.lr = p.lr;
  s.size = p.lr / -std::expm1(t * s.log_beta1);
  s.rbc2 = static_cast<float>(1.0 / std::sqrt(-std::expm1(t * s.log_beta2)));
  s.grad_scale = p.grad_scale;
  s.step = p.step;
  s.d_lr = p.d_lr;
  s.d_step = p.d_step;
  s.sumsq = p.sumsq;
  s.max_norm = p.max_norm;
  s.b1 = static_cast<float>(p.beta1);
  s.c1 = static_cast<float>(1.0 - p.beta1);
  s.b2 = static_cast<float>(p.beta2);
  s.c2 = static_cast<float>(1.0 - p.beta2);
  // The unit's reciprocal of less would be infinite, and 0 times it NaN.
  s.eps = p.eps > 0 ? std::max(static_cast<float>(p.eps), 0x1p-126f) : 0.f;
  s.skip = p.skip_nonfinite;
  s.seed = p.seed;
  const dim3 grid(static_cast<unsigned>(std::min<std::int64_t>(n_chunks, kMaxGroups)));
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, chunks, n_chunks, s);
  };
  if (!eight)
    past ? launch(AdamWKernel<kFull, true>) : launch(AdamWKernel<kFull, false>);
  else if (p.stochastic)
    past ? launch(AdamWKernel<kStochastic, true>) : launch(AdamWKernel<kStochastic, false>);
  else
    past ? launch(AdamWKernel<kNearest, true>) : launch(AdamWKernel<kNearest, false>);
  return hipGetLastError();
}

}  // namespace mfh
