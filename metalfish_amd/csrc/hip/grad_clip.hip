// The global norm of many gradient tensors and their scaling, for gfx950.
//
//   N = sqrt(sum over all tensors of g^2),  out = g min(1, max_norm / N).
//
// The tensors are cut into chunks of at most kGradChunkBytes, listed once per
// set; a workgroup of 256 takes whole chunks.  Squares are summed in 64
// bits: a 32-bit sum would lose small gradients beside large ones and
// overflow from |g| = 2^64, and the card's 64-bit rate is far above what the
// memory delivers.  The norm has to be known before anything is written, so
// the gradients are read twice and written once: three passes over the bytes,
// 304 us for 637 MB (norm 94, scaling 210: 6.3 TB/s), where a copy alone
// takes 207.  The last-level cache does not shorten the second reading:
// taking the chunks backwards, to begin with what the norm read last, took
// 310 to 325 us, and any share of them read through the cache instead of past
// it took no less.
#include "mfh_device.h"
#include "mfh_kernels.h"

namespace mfh {
namespace {

typedef unsigned int u32x4_a4 __attribute__((ext_vector_type(4), aligned(4), may_alias));
typedef unsigned int u32x4_a2 __attribute__((ext_vector_type(4), aligned(2), may_alias));

constexpr int kMaxNormGroups = 1024;
// Scaling past the caches: 210 us for 637 MB on 512 workgroups, 228 on 2048,
// 221 on 4096; 106, 113 and 110 for 318 MB.
constexpr int kMaxScaleGroups = 2048;
constexpr int kMaxScaleGroupsPast = 512;

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

// A whole chunk is four vectors a thread, all loaded before the first is used.
constexpr int kDeep = kGradChunkBytes / (16 * 256);

template <int DT, bool PAST>
__device__ __forceinline__ u32x4 Load(const MFH_GLOBAL Bits<DT> *p) {
  if constexpr (PAST)
    return __builtin_nontemporal_load((const MFH_GLOBAL Vec<DT> *)p);
  else
    return *(const MFH_GLOBAL Vec<DT> *)p;
}

template <int DT>
__device__ __forceinline__ void AddSquares(u32x4 v, double &sum) {
#pragma unroll
  for (int i = 0; i < kPerVec<DT>; ++i) {
    const double g = Get<DT>(v, i);
    sum += g * g;
  }
}

template <int DT, bool PAST>
__device__ __forceinline__ void ChunkSumsq(const GradChunk &c, double &sum) {
  constexpr int VE = kPerVec<DT>;
  const auto *src = (const MFH_GLOBAL Bits<DT> *)c.src;
  const int vecs = c.count / VE;
  if (vecs == 256 * kDeep) {
    u32x4 r[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      r[j] = Load<DT, PAST>(src + (256 * j + threadIdx.x) * VE);
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      AddSquares<DT>(r[j], sum);
    return;
  }
  for (int v = threadIdx.x; v < vecs; v += 256)
    AddSquares<DT>(Load<DT, PAST>(src + v * VE), sum);
  const int t = vecs * VE + static_cast<int>(threadIdx.x);
  if (t < c.count) {
    const double g = One<DT>(src[t]);
    sum += g * g;
  }
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

// Entry k of the list (an empty one of an empty list), by scalar loads: the
// list does not change while a kernel runs.
__device__ __forceinline__ GradChunk Entry(const MFH_CONSTANT GradChunk *chunks, std::int64_t k,
                                           std::int64_t n) {
  GradChunk c{};
  if (n > 0) {
    c.src = chunks[k].src;
    c.dst = chunks[k].dst;
    c.count = chunks[k].count;
    c.dtype = chunks[k].dtype;
  }
  return c;
}

template <bool PAST>
__global__ __launch_bounds__(256) void GradSumsqKernel(const GradChunk *list, std::int64_t n,
                                                       double *partials) {
  __shared__ double red[4];
  const auto *chunks = (const MFH_CONSTANT GradChunk *)list;
  double sum = 0.0;
  std::int64_t k = blockIdx.x;
  GradChunk c = Entry(chunks, k < n ? k : 0, n);
  while (k < n) {
    // The next chunk's entry is on its way while this one is read.
    const std::int64_t next = k + gridDim.x;
    const GradChunk ahead = Entry(chunks, next < n ? next : k, n);
    if (c.dtype == DT_F32)
      ChunkSumsq<DT_F32, PAST>(c, sum);
    else if (c.dtype == DT_BF16)
      ChunkSumsq<DT_BF16, PAST>(c, sum);
    else
      ChunkSumsq<DT_F16, PAST>(c, sum);
    k = next;
    c = ahead;
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

// A factor in 24 bits, as a product where it is below 2^-126 (gradients that
// have all but overflowed against a small norm): by itself it would keep only
// the bits of a denormal number.  fp16, of 2^16 at most, is 0 there either way
// and takes the factor as it is (31 M gradients, fp16 matrices: with both
// products 32.9 us, with one 32.0).
struct Factor {
  float high, low, whole;
};
__device__ __forceinline__ Factor FactorOf(double f) {
  const bool tiny = f < 0x1p-126;
  return {static_cast<float>(tiny ? f * 0x1p64 : f), tiny ? 0x1p-64f : 1.f,
          static_cast<float>(f)};
}
template <int DT> __device__ __forceinline__ float Times(float g, const Factor &f) {
  if constexpr (DT == DT_F16)
    return g * f.whole;
  else
    return (g * f.high) * f.low;
}

template <int DT, bool PAST>
__device__ __forceinline__ void ScaleVec(MFH_GLOBAL Bits<DT> *dst, u32x4 v, const Factor &scale) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == DT_F32)
      o[i] = Round<DT>(Times<DT>(Get<DT>(v, i), scale));
    else if constexpr (DT == DT_BF16)
      o[i] = pack_bf16x2(Times<DT>(Get<DT>(v, 2 * i), scale),
                         Times<DT>(Get<DT>(v, 2 * i + 1), scale));
    else
      o[i] = Round<DT>(Times<DT>(Get<DT>(v, 2 * i), scale)) |
             Round<DT>(Times<DT>(Get<DT>(v, 2 * i + 1), scale)) << 16;
  }
  if constexpr (PAST)
    __builtin_nontemporal_store(static_cast<Vec<DT>>(o), (MFH_GLOBAL Vec<DT> *)dst);
  else
    *(MFH_GLOBAL Vec<DT> *)dst = o;
}

template <int DT, bool PAST>
__device__ __forceinline__ void ScaleChunk(const GradChunk &c, const Factor &scale) {
  constexpr int VE = kPerVec<DT>;
  const auto *src = (const MFH_GLOBAL Bits<DT> *)c.src;
  auto *dst = (MFH_GLOBAL Bits<DT> *)c.dst;
  const int vecs = c.count / VE;
  if (vecs == 256 * kDeep) {
    u32x4 r[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      r[j] = Load<DT, PAST>(src + (256 * j + threadIdx.x) * VE);
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      ScaleVec<DT, PAST>(dst + (256 * j + threadIdx.x) * VE, r[j], scale);
    return;
  }
  for (int v = threadIdx.x; v < vecs; v += 256)
    ScaleVec<DT, PAST>(dst + v * VE, Load<DT, PAST>(src + v * VE), scale);
  const int t = vecs * VE + static_cast<int>(threadIdx.x);
  if (t < c.count)
    dst[t] = static_cast<Bits<DT>>(Round<DT>(Times<DT>(One<DT>(src[t]), scale)));
}

template <bool PAST>
__device__ __forceinline__ void ScaleChunk(const GradChunk &c, const Factor &scale) {
  if (c.dtype == DT_F32)
    ScaleChunk<DT_F32, PAST>(c, scale);
  else if (c.dtype == DT_BF16)
    ScaleChunk<DT_BF16, PAST>(c, scale);
  else
    ScaleChunk<DT_F16, PAST>(c, scale);
}

template <bool PAST>
__global__ __launch_bounds__(256) void GradScaleKernel(const GradChunk *list, std::int64_t n,
                                                       const double *partials, int parts,
                                                       float max_norm, float *norm) {
  __shared__ double red[4];
  const auto *chunks = (const MFH_CONSTANT GradChunk *)list;
  std::int64_t k = blockIdx.x;
  GradChunk c = Entry(chunks, k < n ? k : 0, n);
  const double total = sqrt(SumPartials(partials, parts, red));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0)
    *norm = static_cast<float>(total);
  // NaN is not <= anything, and goes into every gradient.
  const bool keep = total <= max_norm;
  const Factor scale = FactorOf(keep ? 1.0 : max_norm / total);
  while (k < n) {
    const std::int64_t next = k + gridDim.x;
    const GradChunk ahead = Entry(chunks, next < n ? next : k, n);
    if (c.dst && !(keep && c.dst == c.src))
      ScaleChunk<PAST>(c, scale);
    k = next;
    c = ahead;
  }
}

}  // namespace

int GradNormGroups(std::int64_t chunks) {
  return static_cast<int>(chunks < 1 ? 1 : chunks < kMaxNormGroups ? chunks : kMaxNormGroups);
}

hipError_t LaunchGradSumsq(const GradChunk *chunks, std::int64_t n_chunks,
                           bool past, double *partials, hipStream_t stream,
                           std::string *err) {
  if (n_chunks < 0 || (n_chunks > 0 && !chunks) || !partials) {
    if (err)
      *err = "grad_sumsq: needs a chunk list and partial sums";
    return hipErrorInvalidValue;
  }
  const dim3 grid(GradNormGroups(n_chunks));
  if (past)
    hipLaunchKernelGGL(GradSumsqKernel<true>, grid, dim3(256), 0, stream, chunks, n_chunks,
                       partials);
  else
    hipLaunchKernelGGL(GradSumsqKernel<false>, grid, dim3(256), 0, stream, chunks, n_chunks,
                       partials);
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

hipError_t LaunchGradScale(const GradChunk *chunks, std::int64_t n_chunks,
                           bool past, const double *partials, int n, float max_norm,
                           float *norm, hipStream_t stream, std::string *err) {
  if (n_chunks < 0 || (n_chunks > 0 && !chunks) || n < 1 || !partials) {
    if (err)
      *err = "grad_scale: needs a chunk list and partial sums";
    return hipErrorInvalidValue;
  }
  const std::int64_t most = past ? kMaxScaleGroupsPast : kMaxScaleGroups;
  const dim3 grid(static_cast<unsigned>(n_chunks < 1 ? 1 : n_chunks < most ? n_chunks : most));
  if (past)
    hipLaunchKernelGGL(GradScaleKernel<true>, grid, dim3(256), 0, stream, chunks, n_chunks,
                       partials, n, max_norm, norm);
  else
    hipLaunchKernelGGL(GradScaleKernel<false>, grid, dim3(256), 0, stream, chunks, n_chunks,
                       partials, n, max_norm, norm);
  return hipGetLastError();
}

}  // namespace mfh
