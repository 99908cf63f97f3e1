// The global norm of many gradient tensors and their scaling, for gfx950.
//
//   N = sqrt(sum over all tensors of g^2),  out = g min(1, max_norm / N).
//
// The tensors are cut into chunks of at most kGradChunk elements, listed once
// per set; a workgroup of 256 takes whole chunks.  Squares are summed in 64
// bits: a 32-bit sum would lose small gradients beside large ones and
// overflow from |g| = 2^64, and the card's 64-bit rate is far above what the
// memory delivers.  The norm has to be known before anything is written, so
// the gradients are read twice and written once.  The second reading goes
// backwards through the list, so that it starts with what the first one left
// in the last-level cache.
#include "mfh_device.h"
#include "mfh_kernels.h"

namespace mfh {
namespace {

typedef unsigned int u32x4_a4 __attribute__((ext_vector_type(4), aligned(4), may_alias));
typedef unsigned int u32x4_a2 __attribute__((ext_vector_type(4), aligned(2), may_alias));

constexpr int kMaxNormGroups = 1024;
constexpr int kMaxScaleGroups = 2048;

template <int DT>
__device__ __forceinline__ float One(std::uint32_t v) {
  if constexpr (DT == DT_F32)
    return __uint_as_float(v);
  else if constexpr (DT == DT_BF16)
    return __uint_as_float(v << 16);
  else
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<std::uint16_t>(v)));
}

template <int DT>
__device__ __forceinline__ std::uint32_t Round(float f) {
  if constexpr (DT == DT_F32)
    return __float_as_uint(f);
  else if constexpr (DT == DT_BF16)
    return f32_to_bf16(f);
  else
    return __builtin_bit_cast(std::uint16_t, static_cast<_Float16>(f));
}

template <int DT>
using Bits = std::conditional_t<DT == DT_F32, std::uint32_t, std::uint16_t>;
template <int DT>
using Vec = std::conditional_t<DT == DT_F32, u32x4_a4, u32x4_a2>;
template <int DT>
constexpr int kPerVec = DT == DT_F32 ? 4 : 8;

template <int DT>
__device__ __forceinline__ float Get(u32x4 v, int i) {
  if constexpr (DT == DT_F32)
    return One<DT>(v[i]);
  else
    return One<DT>(i & 1 ? v[i >> 1] >> 16 : v[i >> 1] & 0xFFFFu);
}

// Four loads are issued before the first is used.
constexpr int kDeep = 4;

template <int DT>
__device__ __forceinline__ double ChunkSumsq(const GradChunk &c) {
  constexpr int VE = kPerVec<DT>;
  const auto *src = static_cast<const Bits<DT> *>(c.src);
  const int vecs = c.count / VE;
  double sum = 0.0;
  for (int v0 = threadIdx.x; v0 < vecs; v0 += 256 * kDeep) {
    u32x4 r[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      r[j] = v0 + 256 * j < vecs
                 ? static_cast<u32x4>(
                       *reinterpret_cast<const Vec<DT> *>(src + (v0 + 256 * j) * VE))
                 : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const double g = Get<DT>(r[j], i);
        sum += g * g;
      }
  }
  const int t = vecs * VE + static_cast<int>(threadIdx.x);
  if (t < c.count) {
    const double g = One<DT>(src[t]);
    sum += g * g;
  }
  return sum;
}

// Sum over the 256 threads of a workgroup, in a fixed order.
__device__ __forceinline__ double GroupSum(double v, double *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0)
    red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void GradSumsqKernel(const GradChunk *chunks, std::int64_t n,
                                                       double *partials) {
  __shared__ double red[4];
  double sum = 0.0;
  for (std::int64_t k = blockIdx.x; k < n; k += gridDim.x) {
    const GradChunk c = chunks[k];
    if (c.dtype == DT_F32)
      sum += ChunkSumsq<DT_F32>(c);
    else if (c.dtype == DT_BF16)
      sum += ChunkSumsq<DT_BF16>(c);
    else
      sum += ChunkSumsq<DT_F16>(c);
  }
  sum = GroupSum(sum, red);
  if (threadIdx.x == 0)
    partials[blockIdx.x] = sum;
}

// The partials' sum, the same in every workgroup that forms it.
__device__ __forceinline__ double SumPartials(const double *partials, int n, double *red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += 256)
    v += partials[i];
  return GroupSum(v, red);
}

__global__ __launch_bounds__(256) void GradSumKernel(const double *partials, int n,
                                                     double *sumsq) {
  __shared__ double red[4];
  const double sum = SumPartials(partials, n, red);
  if (threadIdx.x == 0)
    *sumsq = sum;
}

template <int DT>
__device__ __forceinline__ void ScaleChunk(const GradChunk &c, float scale) {
  constexpr int VE = kPerVec<DT>;
  const auto *src = static_cast<const Bits<DT> *>(c.src);
  auto *dst = static_cast<Bits<DT> *>(c.dst);
  const int vecs = c.count / VE;
  for (int v0 = threadIdx.x; v0 < vecs; v0 += 256 * kDeep) {
    u32x4 r[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      if (v0 + 256 * j < vecs)
        r[j] = *reinterpret_cast<const Vec<DT> *>(src + (v0 + 256 * j) * VE);
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      if (v0 + 256 * j >= vecs)
        break;
      u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == DT_F32)
          o[i] = Round<DT>(Get<DT>(r[j], i) * scale);
        else if constexpr (DT == DT_BF16)
          o[i] = pack_bf16x2(Get<DT>(r[j], 2 * i) * scale, Get<DT>(r[j], 2 * i + 1) * scale);
        else
          o[i] = Round<DT>(Get<DT>(r[j], 2 * i) * scale) |
                 Round<DT>(Get<DT>(r[j], 2 * i + 1) * scale) << 16;
      }
      *reinterpret_cast<Vec<DT> *>(dst + (v0 + 256 * j) * VE) = o;
    }
  }
  const int t = vecs * VE + static_cast<int>(threadIdx.x);
  if (t < c.count)
    dst[t] = static_cast<Bits<DT>>(Round<DT>(One<DT>(src[t]) * scale));
}

__global__ __launch_bounds__(256) void GradScaleKernel(const GradChunk *chunks, std::int64_t n,
                                                       const double *partials, int parts,
                                                       float max_norm, float *norm) {
  __shared__ double red[4];
  const double total = sqrt(SumPartials(partials, parts, red));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0)
    *norm = static_cast<float>(total);
  // NaN is not <= anything, and goes into every gradient.
  const bool keep = total <= max_norm;
  const float scale = keep ? 1.f : static_cast<float>(max_norm / total);
  for (std::int64_t k = n - 1 - blockIdx.x; k >= 0; k -= gridDim.x) {
    const GradChunk c = chunks[k];
    if (!c.dst || (keep && c.dst == c.src))
      continue;
    if (c.dtype == DT_F32)
      ScaleChunk<DT_F32>(c, scale);
    else if (c.dtype == DT_BF16)
      ScaleChunk<DT_BF16>(c, scale);
    else
      ScaleChunk<DT_F16>(c, scale);
  }
}

}  // namespace

int GradNormGroups(std::int64_t chunks) {
  return static_cast<int>(chunks < 1 ? 1 : chunks < kMaxNormGroups ? chunks : kMaxNormGroups);
}

hipError_t LaunchGradSumsq(const GradChunk *chunks, std::int64_t n_chunks, double *partials,
                           hipStream_t stream, std::string *err) {
  if (n_chunks < 0 || (n_chunks > 0 && !chunks) || !partials) {
    if (err)
      *err = "grad_sumsq: needs a chunk list and partial sums";
    return hipErrorInvalidValue;
  }
  hipLaunchKernelGGL(GradSumsqKernel, dim3(GradNormGroups(n_chunks)), dim3(256), 0, stream, chunks,
                     n_chunks, partials);
  return hipGetLastError();
}

hipError_t LaunchGradSum(const double *partials, int n, double *sumsq, hipStream_t stream,
                         std::string *err) {
  if (n < 1 || !partials || !sumsq) {
    if (err)
      *err = "grad_sum: needs partial sums and a result";
    return hipErrorInvalidValue;
  }
  hipLaunchKernelGGL(GradSumKernel, dim3(1), dim3(256), 0, stream, partials, n, sumsq);
  return hipGetLastError();
}

hipError_t LaunchGradScale(const GradChunk *chunks, std::int64_t n_chunks, const double *partials,
                           int n, float max_norm, float *norm, hipStream_t stream,
                           std::string *err) {
  if (n_chunks < 0 || (n_chunks > 0 && !chunks) || n < 1 || !partials) {
    if (err)
      *err = "grad_scale: needs a chunk list and partial sums";
    return hipErrorInvalidValue;
  }
  const std::int64_t groups =
      n_chunks < 1 ? 1 : n_chunks < kMaxScaleGroups ? n_chunks : kMaxScaleGroups;
  hipLaunchKernelGGL(GradScaleKernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, stream,
                     chunks, n_chunks, partials, n, max_norm, norm);
  return hipGetLastError();
}

}  // namespace mfh
