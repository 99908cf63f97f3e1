// Rows of fp32, bf16 or fp16 elements and reductions over a wave, for the
// kernels of training (device code only).
#pragma once

#include "mfh_device.h"
#include "mfh_kernels.h"

namespace mfh {

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

}  // namespace mfh
