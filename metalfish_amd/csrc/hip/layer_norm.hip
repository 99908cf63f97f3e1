// Layer norm of rows h = residual + alpha x and its gradients, for gfx950.
//
//   y = n gamma + beta,  n = (h - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   dh = rstd (w - mean(w) - n mean(w n)),  w = dy gamma
//   dgamma = sum over rows of dy n,  dbeta = sum over rows of dy
//
// Bound by memory: the forward pass reads x (and the residual) and writes y,
// the backward pass reads dy, x (and the residual) and writes dx (and
// dresidual).  A row is held in the registers of 16, 64, 256 or 1024 lanes, so
// every pass over it after the first costs no memory; the variance is summed
// about the mean.  Workgroups loop over rows: gamma stays in registers, and in the
// backward pass each lane sums dy n and dy of its own columns over all rows of
// its workgroup.  Those partial sums (one row of 2 width a workgroup) are
// added up by a second kernel in a fixed order: no atomics, the same bits every
// run.
#include "learn_device.h"
#include "mfh_device.h"
#include "mfh_kernels.h"

namespace mfh {
namespace {

constexpr int kMaxHeld = 16384;   // columns of a row held in registers
constexpr int kMaxGroups = 512;   // workgroups of the backward pass

// Vector `c0` of a row of `width`, zeros behind its end.
template <int DT>
__device__ __forceinline__ u32x4 LoadPart(ConstRow<DT> p, int c0, int width) {
  constexpr int VE = Elem<DT>::kPerVec;
  if (c0 + VE <= width)
    return LoadVec<DT, false>(p + c0);
  u32x4 v{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (c0 + e < width) {
      const unsigned one = p[c0 + e];
      if constexpr (DT == DT_F32)
        v[e] = one;
      else
        v[e >> 1] |= one << (16 * (e & 1));
    }
  return v;
}

template <int DT>
__device__ __forceinline__ void StorePart(Row<DT> p, int c0, int width, const float *f) {
  constexpr int VE = Elem<DT>::kPerVec;
  if (c0 + VE <= width) {
    StoreVec<DT, false>(p + c0, Elem<DT>::Pack(f));
    return;
  }
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (c0 + e < width)
      p[c0 + e] = Elem<DT>::Round(f[e]);
}

__device__ __forceinline__ float WeightAt(const float *w, int c, int width, float none) {
  return w && c < width ? w[c] : none;
}

// Sum over the T lanes of a row, in every one of them.
template <int T>
__device__ __forceinline__ float RowSum(float v, float *red) {
  if constexpr (T == 16) {
    constexpr int kRor = 0x120;
    v += Dpp<kRor + 8, 0xF>(0.f, v);
    v += Dpp<kRor + 4, 0xF>(0.f, v);
    v += Dpp<kRor + 2, 0xF>(0.f, v);
    v += Dpp<kRor + 1, 0xF>(0.f, v);
    return v;
  } else {
    v = WaveSum(v);
    if constexpr (T > 64) {
      if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int w = 0; w < T / 64; ++w)
        v += red[w];
    }
    return v;
  }
}

// h of vector c0 of row `row`.
template <int DT>
__device__ __forceinline__ void LoadSum(const NormParams &p, std::int64_t row, int c0, float *h) {
  constexpr int VE = Elem<DT>::kPerVec;
  const u32x4 x = LoadPart<DT>(RowOf<DT>(p.x, row, p.ldx), c0, p.width);
  if (p.residual) {
    const u32x4 r = LoadPart<DT>(RowOf<DT>(p.residual, row, p.ldr), c0, p.width);
#pragma unroll
    for (int e = 0; e < VE; ++e)
      h[e] = Elem<DT>::Get(r, e) + p.alpha * Elem<DT>::Get(x, e);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      h[e] = p.alpha * Elem<DT>::Get(x, e);
  }
}

template <int T> constexpr int kBlock = T > 256 ? T : 256;

// T lanes a row, NV vectors a lane.
template <int DT, int T, int NV>
__global__ __launch_bounds__(kBlock<T>) void NormKernel(NormParams p) {
  constexpr int VE = Elem<DT>::kPerVec, kRows = kBlock<T> / T;
  constexpr bool kHold = NV * VE <= 16;
  __shared__ float red[2][16];
  const int t = threadIdx.x % T, width = p.width;
  // A quotient, so that a constant row has its value as its mean.
  const float n = static_cast<float>(width);
  float gamma[kHold ? NV * VE : 1], beta[kHold ? NV * VE : 1];
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < NV * VE; ++i) {
      const int c = ((i / VE) * T + t) * VE + i % VE;
      gamma[i] = WeightAt(p.gamma, c, width, 1.f);
      beta[i] = WeightAt(p.beta, c, width, 0.f);
    }
  }
  for (std::int64_t first = static_cast<std::int64_t>(blockIdx.x) * kRows; first < p.rows;
       first += static_cast<std::int64_t>(gridDim.x) * kRows) {
    const std::int64_t row = first + threadIdx.x / T;
    if (T < 256 && row >= p.rows)
      return;
    float h[NV * VE], sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      LoadSum<DT>(p, row, (i * T + t) * VE, h + i * VE);
#pragma unroll
    for (int i = 0; i < NV * VE; ++i)
      sum += h[i];  // zeros behind the row's end
    const float mean = RowSum<T>(sum, red[0]) / n;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV * VE; ++i) {
      const int c = ((i / VE) * T + t) * VE + i % VE;
      h[i] = c < width ? h[i] - mean : 0.f;
      sq += h[i] * h[i];
    }
    const float rstd = 1.f / sqrtf(RowSum<T>(sq, red[1]) / n + p.eps);
    if (t == 0) {
      if (p.mean)
        p.mean[row] = mean;
      if (p.rstd)
        p.rstd[row] = rstd;
    }
    if (p.y) {
      const Row<DT> y = RowOf<DT>(p.y, row, p.ldy);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c0 = (i * T + t) * VE;
        if (c0 >= width)
          continue;
        float out[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float g = kHold ? gamma[i * VE + e] : WeightAt(p.gamma, c0 + e, width, 1.f);
          const float b = kHold ? beta[i * VE + e] : WeightAt(p.beta, c0 + e, width, 0.f);
          out[e] = h[i * VE + e] * rstd * g + b;
        }
        StorePart<DT>(y, c0, width, out);
      }
    }
  }
}

// Rows too long for registers, read three times by 1024 lanes.
template <int DT>
__global__ __launch_bounds__(1024) void LongNormKernel(NormParams p) {
  constexpr int VE = Elem<DT>::kPerVec;
  __shared__ float red[2][16];
  const int width = p.width;
  const float n = static_cast<float>(width);
  for (std::int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float h[VE], sum = 0.f;
    for (int c0 = threadIdx.x * VE; c0 < width; c0 += 1024 * VE) {
      LoadSum<DT>(p, row, c0, h);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        sum += h[e];
    }
    const float mean = RowSum<1024>(sum, red[0]) / n;
    float sq = 0.f;
    for (int c0 = threadIdx.x * VE; c0 < width; c0 += 1024 * VE) {
      LoadSum<DT>(p, row, c0, h);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (c0 + e < width)
          sq += (h[e] - mean) * (h[e] - mean);
    }
    const float rstd = 1.f / sqrtf(RowSum<1024>(sq, red[1]) / n + p.eps);
    if (threadIdx.x == 0) {
      if (p.mean)
        p.mean[row] = mean;
      if (p.rstd)
        p.rstd[row] = rstd;
    }
    if (!p.y)
      continue;
    const Row<DT> y = RowOf<DT>(p.y, row, p.ldy);
    for (int c0 = threadIdx.x * VE; c0 < width; c0 += 1024 * VE) {
      LoadSum<DT>(p, row, c0, h);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        h[e] = (h[e] - mean) * rstd * WeightAt(p.gamma, c0 + e, width, 1.f) +
               WeightAt(p.beta, c0 + e, width, 0.f);
      StorePart<DT>(y, c0, width, h);
    }
  }
}


template <int DT>
__device__ __forceinline__ void StoreGrads(const NormParams &p, std::int64_t row, int c0,
                                           float *dh) {
  constexpr int VE = Elem<DT>::kPerVec;
  if (p.dresidual)
    StorePart<DT>(RowOf<DT>(p.dresidual, row, p.lddr), c0, p.width, dh);
  if (p.dx) {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      dh[e] *= p.alpha;
    StorePart<DT>(RowOf<DT>(p.dx, row, p.lddx), c0, p.width, dh);
  }
}

template <int DT, int T, int NV>
__global__ __launch_bounds__(kBlock<T>) void NormBackwardKernel(NormParams p) {
  constexpr int VE = Elem<DT>::kPerVec, kRows = kBlock<T> / T, N = NV * VE;
  __shared__ float red[2][2][16];
  __shared__ float sums[T * N * (T <= 256 ? 1 : 0) + 1];
  const int t = threadIdx.x % T, width = p.width;
  const float inv = 1.f / static_cast<float>(width);
  float gamma[N], dgamma[N], dbeta[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = ((i / VE) * T + t) * VE + i % VE;
    gamma[i] = WeightAt(p.gamma, c, width, 1.f);
    dgamma[i] = dbeta[i] = 0.f;
  }
  int turn = 0;
  for (std::int64_t first = static_cast<std::int64_t>(blockIdx.x) * kRows; first < p.rows;
       first += static_cast<std::int64_t>(gridDim.x) * kRows, turn ^= 1) {
    const std::int64_t row = first + threadIdx.x / T;
    if (T < 256 && row >= p.rows)
      break;
    float n[N], dy[N];
    const float mean = p.mean[row], rstd = p.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (i * T + t) * VE;
      LoadSum<DT>(p, row, c0, n + i * VE);
      const u32x4 v = LoadPart<DT>(RowOf<DT>(p.dy, row, p.lddy), c0, width);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        dy[i * VE + e] = Elem<DT>::Get(v, e);
    }
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      n[i] = (n[i] - mean) * rstd;
      const float w = dy[i] * gamma[i];  // 0 behind the row's end
      a += w;
      b += w * n[i];
      dgamma[i] += dy[i] * n[i];
      dbeta[i] += dy[i];
    }
    if constexpr (T > 64) {
      // Both sums in one exchange; two buffers, since a wave may be a row ahead.
      a = WaveSum(a);
      b = WaveSum(b);
      if ((threadIdx.x & 63) == 0) {
        red[turn][0][threadIdx.x >> 6] = a;
        red[turn][1][threadIdx.x >> 6] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < T / 64; ++w) {
        a += red[turn][0][w];
        b += red[turn][1][w];
      }
    } else {
      a = RowSum<T>(a, nullptr);
      b = RowSum<T>(b, nullptr);
    }
    a *= inv;
    b *= inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (i * T + t) * VE;
      if (c0 >= width)
        continue;
      float dh[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e)
        dh[e] = rstd * (dy[i * VE + e] * gamma[i * VE + e] - a - n[i * VE + e] * b);
      StoreGrads<DT>(p, row, c0, dh);
    }
  }
  if (!p.partials)
    return;
  // The workgroup's rows together, in the order of its row groups.
  float *out = p.partials + static_cast<std::int64_t>(blockIdx.x) * 2 * width;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    float *v = part ? dbeta : dgamma;
    if constexpr (T == 16) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] += __shfl_xor(v[i], 16, 64);
        v[i] += __shfl_xor(v[i], 32, 64);
      }
    }
    if constexpr (T <= 64) {
      const int lane = threadIdx.x & 63;
      for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x >> 6) == w && lane < T) {
#pragma unroll
          for (int i = 0; i < N; ++i)
            sums[i * T + lane] = w ? sums[i * T + lane] + v[i] : v[i];
        }
      }
      __syncthreads();
      for (int k = threadIdx.x; k < T * N; k += 256) {
        const int c = ((k / T / VE) * T + k % T) * VE + k / T % VE;
        if (c < width)
          out[part * width + c] = sums[k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = ((i / VE) * T + t) * VE + i % VE;
        if (c < width)
          out[part * width + c] = v[i];
      }
    }
  }
}

// Rows too long for registers: dh alone, read twice.
template <int DT>
__global__ __launch_bounds__(1024) void LongNormBackwardKernel(NormParams p) {
  constexpr int VE = Elem<DT>::kPerVec;
  __shared__ float red[2][16];
  const int width = p.width;
  const float inv = 1.f / static_cast<float>(width);
  for (std::int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    const ConstRow<DT> dy = RowOf<DT>(p.dy, row, p.lddy);
    float h[VE], a = 0.f, b = 0.f;
    for (int c0 = threadIdx.x * VE; c0 < width; c0 += 1024 * VE) {
      LoadSum<DT>(p, row, c0, h);
      const u32x4 v = LoadPart<DT>(dy, c0, width);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float w = Elem<DT>::Get(v, e) * WeightAt(p.gamma, c0 + e, width, 1.f);
        a += w;
        b += w * ((h[e] - mean) * rstd);
      }
    }
    a = RowSum<1024>(a, red[0]) * inv;
    b = RowSum<1024>(b, red[1]) * inv;
    for (int c0 = threadIdx.x * VE; c0 < width; c0 += 1024 * VE) {
      LoadSum<DT>(p, row, c0, h);
      const u32x4 v = LoadPart<DT>(dy, c0, width);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        h[e] = rstd * (Elem<DT>::Get(v, e) * WeightAt(p.gamma, c0 + e, width, 1.f) - a -
                       (h[e] - mean) * rstd * b);
      StoreGrads<DT>(p, row, c0, h);
    }
  }
}

// Their weights' partial sums: 256 lanes take a vector of columns each, a
// workgroup the rows blockIdx.y, blockIdx.y + gridDim.y, ...
template <int DT>
__global__ __launch_bounds__(256) void LongNormSumsKernel(NormParams p) {
  constexpr int VE = Elem<DT>::kPerVec;
  const int c0 = (blockIdx.x * 256 + threadIdx.x) * VE;
  if (c0 >= p.width)
    return;
  float dgamma[VE] = {}, dbeta[VE] = {};
  for (std::int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    float h[VE];
    LoadSum<DT>(p, row, c0, h);
    const u32x4 v = LoadPart<DT>(RowOf<DT>(p.dy, row, p.lddy), c0, p.width);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      dgamma[e] += Elem<DT>::Get(v, e) * ((h[e] - mean) * rstd);
      dbeta[e] += Elem<DT>::Get(v, e);
    }
  }
  float *out = p.partials + static_cast<std::int64_t>(blockIdx.y) * 2 * p.width;
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (c0 + e < p.width) {
      out[c0 + e] = dgamma[e];
      out[p.width + c0 + e] = dbeta[e];
    }
}

// Adds up `parts` rows of partial sums: 16 waves take every sixteenth row of
// 64 columns each.
__global__ __launch_bounds__(1024) void NormSumsKernel(const float *partials, int parts, int width,
                                                       float *dgamma, float *dbeta) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float *out = blockIdx.y ? dbeta : dgamma;
  if (!out)
    return;
  const float *in = partials + static_cast<std::int64_t>(blockIdx.y) * width + c;
  float sum = 0.f;
  if (c < width)
    for (int k = wave; k < parts; k += 16)
      sum += in[static_cast<std::int64_t>(k) * 2 * width];
  red[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < width) {
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w)
      sum += red[w][lane];
    out[c] = sum;
  }
}

// Lanes and vectors of a row of `width`: the fewest lanes that hold it in four
// vectors of fp32 or two of 16 bits.
struct Shape {
  int lanes, vectors;
};
Shape ShapeOf(int width, int dtype) {
  const int ve = dtype == DT_F32 ? 4 : 8;
  const int vectors = (width + ve - 1) / ve;
  if (vectors <= 16)
    return {16, 1};
  for (int lanes : {64, 256, 1024})
    for (int n = 1; n * ve <= 16; n *= 2)
      if (vectors <= lanes * n)
        return {lanes, n};
  return {0, 0};
}

int Groups(std::int64_t rows, int lanes) {
  const std::int64_t per = lanes >= 256 ? 1 : 256 / lanes;
  return static_cast<int>(std::min<std::int64_t>((rows + per - 1) / per, kMaxGroups));
}

template <int DT, int T, int NV>
void LaunchShape(const NormParams &p, bool backward, hipStream_t stream) {
  const int per = kBlock<T> / T;
  if (backward) {
    hipLaunchKernelGGL((NormBackwardKernel<DT, T, NV>), dim3(Groups(p.rows, T)), dim3(kBlock<T>),
                       0, stream, p);
  } else {
    const std::int64_t groups = std::min<std::int64_t>((p.rows + per - 1) / per, 2048);
    hipLaunchKernelGGL((NormKernel<DT, T, NV>), dim3(static_cast<unsigned>(groups)),
                       dim3(kBlock<T>), 0, stream, p);
  }
}

template <int DT> void LaunchType(const NormParams &p, bool backward, hipStream_t stream) {
  const Shape s = ShapeOf(p.width, DT);
  if (s.lanes == 16)
    LaunchShape<DT, 16, 1>(p, backward, stream);
  else if (s.lanes == 64 && s.vectors == 1)
    LaunchShape<DT, 64, 1>(p, backward, stream);
  else if (s.lanes == 64 && s.vectors == 2)
    LaunchShape<DT, 64, 2>(p, backward, stream);
  else if (s.lanes == 256 && s.vectors == 1)
    LaunchShape<DT, 256, 1>(p, backward, stream);
  else if (s.lanes == 256 && s.vectors == 2)
    LaunchShape<DT, 256, 2>(p, backward, stream);
  else if (s.lanes == 1024 && s.vectors == 1)
    LaunchShape<DT, 1024, 1>(p, backward, stream);
  else if (s.lanes == 1024 && s.vectors == 2)
    LaunchShape<DT, 1024, 2>(p, backward, stream);
  else if constexpr (DT == DT_F32) {
    if (s.lanes == 64)
      LaunchShape<DT, 64, 4>(p, backward, stream);
    else if (s.lanes == 256)
      LaunchShape<DT, 256, 4>(p, backward, stream);
    else
      LaunchShape<DT, 1024, 4>(p, backward, stream);
  }
}

template <int DT> void LaunchLong(const NormParams &p, bool backward, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(std::min<std::int64_t>(p.rows, 2048)));
  if (!backward) {
    hipLaunchKernelGGL(LongNormKernel<DT>, grid, dim3(1024), 0, stream, p);
    return;
  }
  // The weights' sums first: dx may be written over what they read.
  if (p.partials) {
    const int ve = Elem<DT>::kPerVec;
    const int across = (p.width + 256 * ve - 1) / (256 * ve);
    hipLaunchKernelGGL(LongNormSumsKernel<DT>, dim3(across, NormPartials(p.rows, p.width)),
                       dim3(256), 0, stream, p);
  }
  hipLaunchKernelGGL(LongNormBackwardKernel<DT>, grid, dim3(1024), 0, stream, p);
}

void Launch(const NormParams &p, bool backward, hipStream_t stream) {
  const bool held = p.width <= kMaxHeld;
  if (p.dtype == DT_F32)
    held ? LaunchType<DT_F32>(p, backward, stream) : LaunchLong<DT_F32>(p, backward, stream);
  else if (p.dtype == DT_BF16)
    held ? LaunchType<DT_BF16>(p, backward, stream) : LaunchLong<DT_BF16>(p, backward, stream);
  else
    held ? LaunchType<DT_F16>(p, backward, stream) : LaunchLong<DT_F16>(p, backward, stream);
}

bool Sound(const NormParams &p) {
  return p.rows >= 0 && p.width >= 1 && p.width <= (1 << 20) && (p.rows == 0 || p.x);
}

}  // namespace

int NormPartials(std::int64_t rows, int width) {
  if (width > kMaxHeld)
    return static_cast<int>(std::min<std::int64_t>(rows, 64));
  // As many for every type: that of the fewest lanes a row.
  const int lanes = std::min(ShapeOf(width, DT_F32).lanes, ShapeOf(width, DT_BF16).lanes);
  return Groups(rows, std::max(lanes, 256));
}

hipError_t LaunchNorm(const NormParams &p, hipStream_t stream, std::string *err) {
  if (!Sound(p)) {
    if (err)
      *err = "layer_norm: needs rows of 1 to 2^20 columns";
    return hipErrorInvalidValue;
  }
  if (p.rows > 0)
    Launch(p, false, stream);
  return hipGetLastError();
}

hipError_t LaunchNormBackward(const NormParams &p, hipStream_t stream, std::string *err) {
  if (!Sound(p) || (p.rows > 0 && (!p.dy || !p.mean || !p.rstd)) ||
      ((p.dgamma || p.dbeta) && p.rows > 0 && !p.partials)) {
    if (err)
      *err = "layer_norm_backward: needs rows of 1 to 2^20 columns, dy, statistics and workspace";
    return hipErrorInvalidValue;
  }
  if (p.rows > 0)
    Launch(p, true, stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && (p.dgamma || p.dbeta)) {
    const int parts =
        p.width > kMaxHeld ? NormPartials(p.rows, p.width) : Groups(p.rows, ShapeOf(p.width, p.dtype).lanes);
    hipLaunchKernelGGL(NormSumsKernel, dim3((p.width + 63) / 64, 2), dim3(1024), 0, stream,
                       p.partials, parts, p.width, p.dgamma, p.dbeta);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace mfh
