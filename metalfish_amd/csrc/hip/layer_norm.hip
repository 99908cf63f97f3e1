// Layer norm of rows h = residual + alpha x and its gradients, for gfx950.
//
//   y = n gamma + beta,  n = (h - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   dh = rstd (w - mean(w) - n mean(w n)),  w = dy gamma
//   dgamma = sum over rows of dy n,  dbeta = sum over rows of dy
//
// Bound by memory: the forward pass reads x (and the residual) and writes y,
// the backward pass reads dy, x (and the residual) and writes dx (and
// dresidual); 16384 x 1024 with a residual: bf16 18.0 us (5.6 TB/s) and 38.8 (4.3
// TB/s, the second kernel's 4.6 us with it), fp32 34.4 and 64.6.  A row of up to 32768
// columns (16384 in the fp32 backward pass, MaxHeld) is held in the registers of 16,
// 32, 64, 256 or 1024 lanes, so every pass over it after the first costs no memory, but
// for the weights' gradients of rows above 8192 columns; the variance is summed
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

// Columns of a row held in registers.
constexpr int MaxHeld(int dtype, bool backward) {
  return dtype == DT_F32 && backward ? 16384 : 32768;
}
constexpr int kMaxSummed = 8192;  // and of the weights' gradients beside it
constexpr int kColumnGroups = 64;  // workgroups down the rows of wider ones
constexpr int kMaxGroups = 256, kMoreGroups = 512;  // of the backward pass, up to 8 values a lane

// Sum over the T lanes of a row, in every one of them.
template <int T>
__device__ __forceinline__ float RowSum(float v, float *red) {
  if constexpr (T <= 32) {
    constexpr int kRor = 0x120;
    v += Dpp<kRor + 8, 0xF>(0.f, v);
    v += Dpp<kRor + 4, 0xF>(0.f, v);
    v += Dpp<kRor + 2, 0xF>(0.f, v);
    v += Dpp<kRor + 1, 0xF>(0.f, v);
    if constexpr (T == 32) {
      const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                      false);
      v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
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

__device__ __forceinline__ float WeightAt(const float *w, int c, float none) {
  return w ? w[c] : none;
}

template <int T> constexpr int kBlock = T > 256 ? T : 256;

// Which of a workgroup's rows a lane works on; in scalar registers where a wave
// has one, and its addresses with it.
template <int T> __device__ __forceinline__ int RowInGroup() {
  const int row = threadIdx.x / T;
  return T >= 64 ? __builtin_amdgcn_readfirstlane(row) : row;
}

// The vectors of a row that lane t of T has, NV of them: vector i begins at
// column (i T + t) VE.  A row's last vector, if it would reach behind the
// row's end, is the one that ends there: its first `skip` values are another lane's
// too, are worked on all the same (loads and stores stay whole vectors) and left
// out of sums.  Lanes behind the row's end (skip = VE) do that vector as well and
// store nothing.  Rows have at least one vector's columns.
template <int DT, int T, int NV, bool PAST> struct Lane {
  static constexpr int VE = Elem<DT>::kPerVec, N = NV * VE;
  int first[NV], skip[NV];
  __device__ __forceinline__ explicit Lane(int width) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = (i * T + static_cast<int>(threadIdx.x % T)) * VE;
      first[i] = min(c0, width - VE);
      skip[i] = min(c0 - first[i], VE);
    }
  }
  __device__ __forceinline__ void Load(const void *p, std::int64_t row, std::int64_t stride,
                                       u32x4 *v) const {
    const ConstRow<DT> r = RowOf<DT>(p, row, stride);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      v[i] = LoadVec<DT, PAST>(r + first[i]);
  }
  __device__ __forceinline__ void Store(void *p, std::int64_t row, std::int64_t stride, int i,
                                        const float *f) const {
    if (skip[i] < VE)
      StoreVec<DT, PAST>(RowOf<DT>(p, row, stride) + first[i], Elem<DT>::Pack(f));
  }
  // Weights of the lane's columns.
  __device__ __forceinline__ void Weights(const float *w, float none, float *f) const {
    if (!w) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[i] = none;
      return;
    }
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 v = LoadVec<DT_F32, false>((ConstRow<DT_F32>)w + first[i / VE] + i % VE);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[i + e] = __uint_as_float(v[e]);
    }
  }
  // The sum of a function of each value that is this lane's alone.
  template <class F> __device__ __forceinline__ float Sum(F f) const {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float part = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e)
        part += f(i * VE + e);
      if (skip[i] > 0) {
        part = 0.f;
#pragma unroll
        for (int e = 0; e < VE; ++e)
          part += e >= skip[i] ? f(i * VE + e) : 0.f;
      }
      sum += part;
    }
    return sum;
  }
};

// h = residual + alpha x from vectors of both.
template <int DT, int NV>
__device__ __forceinline__ void Sums(const NormParams &p, const u32x4 *x, const u32x4 *r, float *h) {
  constexpr int VE = Elem<DT>::kPerVec;
  if (p.residual) {
#pragma unroll
    for (int i = 0; i < NV * VE; ++i)
      h[i] = Elem<DT>::Get(r[i / VE], i % VE) + p.alpha * Elem<DT>::Get(x[i / VE], i % VE);
  } else {
#pragma unroll
    for (int i = 0; i < NV * VE; ++i)
      h[i] = p.alpha * Elem<DT>::Get(x[i / VE], i % VE);
  }
}

// T lanes a row, NV vectors a lane.  The next row is on its way while this one is
// summed; 4096 x 4096 bf16 with a residual 18.8 us (5.4 TB/s), 65536 x 256 13.6 (4.9).
template <int DT, int T, int NV, bool PAST>
__global__ __launch_bounds__(kBlock<T>) void NormKernel(NormParams p) {
  using L = Lane<DT, T, NV, PAST>;
  constexpr int N = L::N, kRows = kBlock<T> / T;
  constexpr bool kHold = N <= 16;  // the weights in registers
  __shared__ float red[2][16];
  const L lane(p.width);
  // A quotient, so that a constant row has its value as its mean.
  const float count = static_cast<float>(p.width);
  float gamma[N], beta[N];
  if constexpr (kHold) {
    lane.Weights(p.gamma, 1.f, gamma);
    lane.Weights(p.beta, 0.f, beta);
  }
  const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * kRows;
  std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * kRows + RowInGroup<T>();
  constexpr bool kAhead = T < 1024 || N <= 16;  // the next row's vectors in registers
  u32x4 x[NV], r[NV];
  const auto load = [&](std::int64_t at) {
    if (at >= p.rows)
      return;
    lane.Load(p.x, at, p.ldx, x);
    if (p.residual)
      lane.Load(p.residual, at, p.ldr, r);
  };
  if constexpr (kAhead)
    load(row);
  while (row < p.rows) {
    if constexpr (!kAhead)
      load(row);
    float h[N];
    Sums<DT, NV>(p, x, r, h);
    const std::int64_t next = row + step;
    if constexpr (kAhead)
      load(next);
    const float mean = RowSum<T>(lane.Sum([&](int i) { return h[i]; }), red[0]) / count;
#pragma unroll
    for (int i = 0; i < N; ++i)
      h[i] -= mean;
    const float var = RowSum<T>(lane.Sum([&](int i) { return h[i] * h[i]; }), red[1]) / count;
    const float rstd = 1.f / sqrtf(var + p.eps);
    if (threadIdx.x % T == 0) {
      if (p.mean)
        p.mean[row] = mean;
      if (p.rstd)
        p.rstd[row] = rstd;
    }
    if (p.y) {
      if constexpr (!kHold) {
        lane.Weights(p.gamma, 1.f, gamma);
        lane.Weights(p.beta, 0.f, beta);
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
        h[i] = h[i] * rstd * gamma[i] + beta[i];
#pragma unroll
      for (int i = 0; i < NV; ++i)
        lane.Store(p.y, row, p.ldy, i, h + i * L::VE);
    }
    row = next;
  }
}

// The backward pass has eight waves a workgroup and, of wide rows, one workgroup a
// CU: each leaves 8 bytes a column of partial sums, which more workgroups of fewer
// rows would let grow beside 2053 x 5003 fp16 (four waves, two workgroups a CU: 36
// us, so 27).
template <int T> constexpr int kBackBlock = T > 512 ? T : 512;

template <int DT, int T, int NV, bool PAST>
__global__ __launch_bounds__(kBackBlock<T>) void NormBackwardKernel(NormParams p) {
  using L = Lane<DT, T, NV, PAST>;
  constexpr int VE = L::VE, N = L::N, kRows = kBackBlock<T> / T, kWaves = T > 64 ? T / 64 : 1;
  constexpr bool kSums = T < 1024;                  // wider rows leave them to another kernel
  constexpr bool kHold = N <= (kSums ? 24 : 8);     // gamma in registers
  constexpr bool kAhead = T < 1024 && N <= 16;  // and the next row's vectors
  __shared__ float red[2][2][kRows][kWaves];
  __shared__ float sums[kSums ? T * N : 1];
  const int t = threadIdx.x % T, group = RowInGroup<T>(), width = p.width;
  const L lane(width);
  const float inv = 1.f / static_cast<float>(width);
  float gamma[N], dgamma[kSums ? N : 1], dbeta[kSums ? N : 1];
  if constexpr (kHold)
    lane.Weights(p.gamma, 1.f, gamma);
#pragma unroll
  for (int i = 0; i < (kSums ? N : 1); ++i)
    dgamma[i] = dbeta[i] = 0.f;
  struct Raw {
    u32x4 x[NV], r[NV], d[NV];
    float mean, rstd;
  };
  const auto load = [&](std::int64_t at, Raw *v) {
    if (at >= p.rows)
      return;
    lane.Load(p.x, at, p.ldx, v->x);
    lane.Load(p.dy, at, p.lddy, v->d);
    if (p.residual)
      lane.Load(p.residual, at, p.ldr, v->r);
    v->mean = p.mean[at];
    v->rstd = p.rstd[at];
  };
  const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * kRows;
  std::int64_t first = static_cast<std::int64_t>(blockIdx.x) * kRows;
  Raw now{}, ahead{};
  load(first + group, &now);
  // All rows of a workgroup go round together: they share barriers.
  for (int turn = 0; first < p.rows; turn ^= 1, first += step) {
    const std::int64_t row = first + group;
    const bool live = row < p.rows;
    if constexpr (kAhead)
      load(row + step, &ahead);
    if constexpr (!kHold)
      lane.Weights(p.gamma, 1.f, gamma);
    // Vectors stay as they are in memory and are unpacked again after the sums:
    // half the registers of 32-bit values in 16-bit rows.
    const auto unpack = [&](int i, float *n, float *dy) {
      Sums<DT, 1>(p, now.x + i, now.r + i, n);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        n[e] = (n[e] - now.mean) * now.rstd;
        dy[e] = Elem<DT>::Get(now.d[i], e);
      }
    };
    float a = 0.f, b = 0.f;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float n[VE], dy[VE], pa = 0.f, pb = 0.f;
        unpack(i, n, dy);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if constexpr (kSums) {
            dgamma[i * VE + e] += dy[e] * n[e];
            dbeta[i * VE + e] += dy[e];
          }
          dy[e] *= gamma[i * VE + e];
          pa += dy[e];
          pb += dy[e] * n[e];
        }
        if (lane.skip[i] > 0) {
          pa = pb = 0.f;
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (e >= lane.skip[i]) {
              pa += dy[e];
              pb += dy[e] * n[e];
            }
        }
        a += pa;
        b += pb;
      }
    }
    if constexpr (T > 64) {
      // Both sums in one exchange; two buffers, since a wave may be a row ahead.
      a = WaveSum(a);
      b = WaveSum(b);
      if ((threadIdx.x & 63) == 0) {
        red[turn][0][group][t >> 6] = a;
        red[turn][1][group][t >> 6] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        a += red[turn][0][group][w];
        b += red[turn][1][group][w];
      }
    } else {
      a = RowSum<T>(a, nullptr);
      b = RowSum<T>(b, nullptr);
    }
    a *= inv;
    b *= inv;
    if (live) {
      if constexpr (!kHold)
        lane.Weights(p.gamma, 1.f, gamma);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float n[VE], dh[VE];
        // Not the values unpacked above: those would stay in registers.
        asm("" : "+v"(now.x[i]), "+v"(now.r[i]), "+v"(now.d[i]));
        unpack(i, n, dh);
#pragma unroll
        for (int e = 0; e < VE; ++e)
          dh[e] = now.rstd * (dh[e] * gamma[i * VE + e] - a - n[e] * b);
        if (p.dresidual)
          lane.Store(p.dresidual, row, p.lddr, i, dh);
        if (p.dx) {
#pragma unroll
          for (int e = 0; e < VE; ++e)
            dh[e] *= p.alpha;
          lane.Store(p.dx, row, p.lddx, i, dh);
        }
      }
    }
    if constexpr (kAhead)
      now = ahead;
    else
      load(row + step, &now);
  }
  if constexpr (kSums) {
    if (!p.partials)
      return;
    // The workgroup's rows together, in the order of its row groups.
    float *out = p.partials + static_cast<std::int64_t>(blockIdx.x) * 2 * width;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      float *v = part ? dbeta : dgamma;
      if constexpr (T <= 32) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if constexpr (T == 16)
            v[i] += __shfl_xor(v[i], 16, 64);
          v[i] += __shfl_xor(v[i], 32, 64);
        }
      }
      {
        // A wave's rows are one by now; then those of the others, one after another.
        constexpr int kTeams = kBackBlock<T> / (T < 64 ? 64 : T), kTeam = kBackBlock<T> / kTeams;
        const int team = threadIdx.x / kTeam;
        const bool mine = threadIdx.x % kTeam < T;
        for (int w = 0; w < kTeams; ++w) {
          __syncthreads();
          if (team == w && mine) {
#pragma unroll
            for (int i = 0; i < N; ++i)
              sums[i * T + t] = w ? sums[i * T + t] + v[i] : v[i];
          }
        }
        if (team != kTeams - 1 || !mine)
          continue;
#pragma unroll
        for (int i = 0; i < N; ++i)
          v[i] = sums[i * T + t];
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i % VE >= lane.skip[i / VE])
          out[part * width + lane.first[i / VE] + i % VE] = v[i];
    }
  }
}

// Rows of less than a vector: one a thread, whose neighbours share its cache lines
// (1000000 x 5 fp32 55 us, backward 69).
template <int DT>
__device__ __forceinline__ float TinySum(const NormParams &p, std::int64_t row, int c) {
  const float x = p.alpha * Elem<DT>::One(RowOf<DT>(p.x, row, p.ldx)[c]);
  return p.residual ? Elem<DT>::One(RowOf<DT>(p.residual, row, p.ldr)[c]) + x : x;
}
template <int DT> __global__ __launch_bounds__(256) void TinyNormKernel(NormParams p) {
  const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (row >= p.rows)
    return;
  const float count = static_cast<float>(p.width);
  float h[8], sum = 0.f, sq = 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    h[c] = c < p.width ? TinySum<DT>(p, row, c) : 0.f;
    sum += h[c];
  }
  const float mean = sum / count;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    sq += c < p.width ? (h[c] - mean) * (h[c] - mean) : 0.f;
  const float rstd = 1.f / sqrtf(sq / count + p.eps);
  if (p.mean)
    p.mean[row] = mean;
  if (p.rstd)
    p.rstd[row] = rstd;
  if (!p.y)
    return;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (c < p.width)
      RowOf<DT>(p.y, row, p.ldy)[c] = Elem<DT>::Round(
          (h[c] - mean) * rstd * WeightAt(p.gamma, c, 1.f) + WeightAt(p.beta, c, 0.f));
}
// Their gradients; a workgroup's 256 threads loop over rows and add up their
// weights' gradients through LDS, in the order of the threads.
template <int DT> __global__ __launch_bounds__(256) void TinyNormBackwardKernel(NormParams p) {
  __shared__ float sums[2][8][256];
  const float inv = 1.f / static_cast<float>(p.width);
  float dgamma[8] = {}, dbeta[8] = {};
  for (std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * 256 + threadIdx.x; row < p.rows;
       row += static_cast<std::int64_t>(gridDim.x) * 256) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    float n[8], w[8], a = 0.f, b = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      n[c] = w[c] = 0.f;
      if (c < p.width) {
        n[c] = (TinySum<DT>(p, row, c) - mean) * rstd;
        const float dy = Elem<DT>::One(RowOf<DT>(p.dy, row, p.lddy)[c]);
        w[c] = dy * WeightAt(p.gamma, c, 1.f);
        dgamma[c] += dy * n[c];
        dbeta[c] += dy;
      }
      a += w[c];
      b += w[c] * n[c];
    }
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < p.width) {
        const float dh = rstd * (w[c] - a * inv - n[c] * (b * inv));
        if (p.dresidual)
          RowOf<DT>(p.dresidual, row, p.lddr)[c] = Elem<DT>::Round(dh);
        if (p.dx)
          RowOf<DT>(p.dx, row, p.lddx)[c] = Elem<DT>::Round(p.alpha * dh);
      }
  }
  if (!p.partials)
    return;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    sums[0][c][threadIdx.x] = dgamma[c];
    sums[1][c][threadIdx.x] = dbeta[c];
  }
  for (int half = 128; half > 0; half /= 2) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < half)
#pragma unroll
      for (int k = 0; k < 16; ++k)
        sums[k >> 3][k & 7][threadIdx.x] += sums[k >> 3][k & 7][threadIdx.x + half];
  }
  if (threadIdx.x == 0)
    for (int part = 0; part < 2; ++part)
      for (int c = 0; c < p.width; ++c)
        p.partials[(static_cast<std::int64_t>(blockIdx.x) * 2 + part) * p.width + c] =
            sums[part][c][0];
}

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
__device__ __forceinline__ float WeightIn(const float *w, int c, int width, float none) {
  return w && c < width ? w[c] : none;
}

// h of vector c0 of row `row`.
template <int DT>
__device__ __forceinline__ void LoadSum(const NormParams &p, std::int64_t row, int c0, float *h) {
  const u32x4 x = LoadPart<DT>(RowOf<DT>(p.x, row, p.ldx), c0, p.width);
  u32x4 r{0, 0, 0, 0};
  if (p.residual)
    r = LoadPart<DT>(RowOf<DT>(p.residual, row, p.ldr), c0, p.width);
  Sums<DT, 1>(p, &x, &r, h);
}

// Rows too long for registers, read three times by 1024 lanes, a vector of a lane on
// its way at a time, and the weights value by value once a row: 300 x 40000 bf16 with a
// residual 88 us (0.8 TB/s), backward 120.
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
        h[e] = (h[e] - mean) * rstd * WeightIn(p.gamma, c0 + e, width, 1.f) +
               WeightIn(p.beta, c0 + e, width, 0.f);
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

// Rows too long for registers: dh alone, read twice.  1000 x 16385 fp32 with a residual
// 138 us with the column sums; of 16384 columns, in registers, 90.
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
        const float w = Elem<DT>::Get(v, e) * WeightIn(p.gamma, c0 + e, width, 1.f);
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
        h[e] = rstd * (Elem<DT>::Get(v, e) * WeightIn(p.gamma, c0 + e, width, 1.f) - a -
                       (h[e] - mean) * rstd * b);
      StoreGrads<DT>(p, row, c0, h);
    }
  }
}

// The weights' partial sums of wide rows, which are read once more for them: 256
// lanes take a vector of columns each, a workgroup the rows blockIdx.y, blockIdx.y + gridDim.y, ...
template <int DT>
__global__ __launch_bounds__(256) void ColumnSumsKernel(NormParams p) {
  constexpr int VE = Elem<DT>::kPerVec;
  const int c0 = (blockIdx.x * 256 + threadIdx.x) * VE;
  if (c0 >= p.width)
    return;
  // The last vector ends with the row; its first columns are another lane's too.
  const int at = min(c0, p.width - VE);
  float dgamma[VE] = {}, dbeta[VE] = {};
#pragma unroll 4
  for (std::int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    const u32x4 x = LoadVec<DT, false>(RowOf<DT>(p.x, row, p.ldx) + at),
                d = LoadVec<DT, false>(RowOf<DT>(p.dy, row, p.lddy) + at);
    u32x4 r{0, 0, 0, 0};
    if (p.residual)
      r = LoadVec<DT, false>(RowOf<DT>(p.residual, row, p.ldr) + at);
    float h[VE];
    Sums<DT, 1>(p, &x, &r, h);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      dgamma[e] += Elem<DT>::Get(d, e) * ((h[e] - mean) * rstd);
      dbeta[e] += Elem<DT>::Get(d, e);
    }
  }
  float *out = p.partials + static_cast<std::int64_t>(blockIdx.y) * 2 * p.width + at;
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (e >= c0 - at) {
      out[e] = dgamma[e];
      out[p.width + e] = dbeta[e];
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
  const auto *in = (const MFH_GLOBAL float *)partials + static_cast<std::int64_t>(blockIdx.y) * width +
                   min(c, width - 1);
  float sum = 0.f;
  // Eight loads at a time.
  for (int k = wave; k < parts; k += 128) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = in[static_cast<std::int64_t>(min(k + 16 * i, parts - 1)) * 2 * width];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      sum += k + 16 * i < parts ? v[i] : 0.f;
  }
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

// Lanes and vectors of a row of `width` columns, at least a vector's and at most
// MaxHeld.
struct Shape {
  int lanes, vectors;
};
Shape ShapeOf(int width, int dtype) {
  const int ve = dtype == DT_F32 ? 4 : 8, most = 16 / ve;
  const int vectors = (width + ve - 1) / ve;
  if (vectors <= 32)
    return {vectors <= 16 ? 16 : 32, 1};
  for (int n = 1; n <= most; n *= 2)
    if (vectors <= 64 * n)
      return {64, n};
  // Four waves up to 32 values a lane, sixteen above.
  for (int n = 1; n <= 2 * most; n += n < most ? n : most / 2)
    if (vectors <= 256 * n)
      return {256, n};
  return {1024, vectors <= 1024 * most ? most : 2 * most};
}

// Workgroups of a backward pass: one a CU, or two where registers hold both (rows of
// up to 2048 values; 65536 x 256 bf16 27.7 us, with one 31.8; 200000 x 64 fp32 34.7 and
// 44.0; with 16 values a lane, 16384 x 1024 bf16 with a residual, 45.4 and 39.1).
int Groups(std::int64_t rows, int lanes, int values) {
  const std::int64_t per = lanes > 512 ? 1 : 512 / lanes;
  const std::int64_t most = lanes > 512 || values <= 8 ? kMoreGroups : kMaxGroups;
  return static_cast<int>(std::min<std::int64_t>((rows + per - 1) / per, most));
}

// Calls whose rows hold more bytes than this go past the caches, if every row
// begins on a whole cache line (lines that two rows share have to meet in one).
// 16384 x 1024 fp32 with a residual: 34.3 us past them, 39.1 through; backward 65.5
// and 70.7; 2053 x 5003 fp16 39.1 and 35.9.
constexpr double kPastBytes = 48e6;
bool Past(const NormParams &p, bool backward) {
  const struct {
    const void *p;
    std::int64_t stride;
  } arrays[] = {{p.x, p.ldx},
                {p.residual, p.ldr},
                {backward ? p.dy : p.y, backward ? p.lddy : p.ldy},
                {backward ? p.dx : nullptr, p.lddx},
                {backward ? p.dresidual : nullptr, p.lddr}};
  const std::int64_t es = DTypeBytes(p.dtype);
  int n = 0;
  for (const auto &a : arrays) {
    if (!a.p)
      continue;
    if (reinterpret_cast<std::uintptr_t>(a.p) % 128 != 0 || a.stride * es % 128 != 0)
      return false;
    ++n;
  }
  return static_cast<double>(p.rows) * p.width * es * n > kPastBytes;
}

template <int DT, int T, int NV, bool PAST>
void LaunchForward(const NormParams &p, hipStream_t stream) {
  constexpr int kPer = kBlock<T> / T;
  const std::int64_t groups =
      std::min<std::int64_t>((p.rows + kPer - 1) / kPer, T >= 1024 ? 512 : 1024);
  hipLaunchKernelGGL((NormKernel<DT, T, NV, PAST>), dim3(static_cast<unsigned>(groups)),
                     dim3(kBlock<T>), 0, stream, p);
}
template <int DT, int T, int NV, bool PAST>
void LaunchShape(const NormParams &p, bool backward, hipStream_t stream) {
  if (backward)
    hipLaunchKernelGGL((NormBackwardKernel<DT, T, NV, PAST>), dim3(Groups(p.rows, T, NV * Elem<DT>::kPerVec)),
                       dim3(kBackBlock<T>), 0, stream, p);
  else
    LaunchForward<DT, T, NV, PAST>(p, stream);
}
template <int DT, int T, int NV>
void LaunchShape(const NormParams &p, bool backward, hipStream_t stream) {
  if (Past(p, backward))
    LaunchShape<DT, T, NV, true>(p, backward, stream);
  else
    LaunchShape<DT, T, NV, false>(p, backward, stream);
}

template <int DT> void LaunchType(const NormParams &p, bool backward, hipStream_t stream) {
  constexpr int kMost = DT == DT_F32 ? 4 : 2;  // vectors of 16 values
  const Shape s = ShapeOf(p.width, DT);
  if (s.lanes == 16)
    return LaunchShape<DT, 16, 1>(p, backward, stream);
  if (s.lanes == 32)
    return LaunchShape<DT, 32, 1>(p, backward, stream);
  if (s.lanes == 64) {
    if (s.vectors == 1)
      return LaunchShape<DT, 64, 1>(p, backward, stream);
    if (s.vectors == kMost)
      return LaunchShape<DT, 64, kMost>(p, backward, stream);
    return LaunchShape<DT, 64, kMost / 2>(p, backward, stream);
  }
  if (s.lanes == 256) {
    if (s.vectors == 1)
      return LaunchShape<DT, 256, 1>(p, backward, stream);
    if (s.vectors == kMost / 2)
      return LaunchShape<DT, 256, kMost / 2>(p, backward, stream);
    if (s.vectors == kMost)
      return LaunchShape<DT, 256, kMost>(p, backward, stream);
    if (s.vectors == kMost * 3 / 2)
      return LaunchShape<DT, 256, kMost * 3 / 2>(p, backward, stream);
    return LaunchShape<DT, 256, kMost * 2>(p, backward, stream);
  }
  if (s.vectors == kMost)
    return LaunchShape<DT, 1024, kMost>(p, backward, stream);
  if constexpr (DT != DT_F32)
    return LaunchShape<DT, 1024, 2 * kMost>(p, backward, stream);
  else
    return LaunchForward<DT, 1024, 2 * kMost, false>(p, stream);
}

template <int DT> void LaunchTiny(const NormParams &p, bool backward, hipStream_t stream) {
  const std::int64_t groups = (p.rows + 255) / 256;
  if (backward) {
    hipLaunchKernelGGL(TinyNormBackwardKernel<DT>, dim3(Groups(groups, 512, 8)), dim3(256), 0, stream, p);
    return;
  }
  // Less than 2^32 threads a launch.
  constexpr std::int64_t kRows = std::int64_t(1) << 31;
  NormParams q = p;
  for (std::int64_t at = 0; at < p.rows; at += kRows) {
    const auto move = [&](const void *a, std::int64_t stride) -> void * {
      return a ? const_cast<char *>(static_cast<const char *>(a)) + at * stride * DTypeBytes(DT)
               : nullptr;
    };
    q.x = move(p.x, p.ldx);
    q.residual = move(p.residual, p.ldr);
    q.y = move(p.y, p.ldy);
    q.mean = p.mean ? p.mean + at : nullptr;
    q.rstd = p.rstd ? p.rstd + at : nullptr;
    q.rows = std::min(kRows, p.rows - at);
    hipLaunchKernelGGL(TinyNormKernel<DT>, dim3(static_cast<unsigned>((q.rows + 255) / 256)),
                       dim3(256), 0, stream, q);
  }
}

template <int DT> void LaunchLong(const NormParams &p, bool backward, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(std::min<std::int64_t>(p.rows, 2048)));
  if (!backward) {
    hipLaunchKernelGGL(LongNormKernel<DT>, grid, dim3(1024), 0, stream, p);
    return;
  }
  hipLaunchKernelGGL(LongNormBackwardKernel<DT>, grid, dim3(1024), 0, stream, p);
}

template <int DT> void LaunchOf(const NormParams &p, bool backward, hipStream_t stream) {
  constexpr int kPer = 256 * Elem<DT>::kPerVec;
  // The weights' sums first: dx may be written over what they read.
  if (backward && p.partials && p.width > kMaxSummed)
    hipLaunchKernelGGL(ColumnSumsKernel<DT>,
                       dim3((p.width + kPer - 1) / kPer, NormPartials(p.rows, p.width)), dim3(256), 0,
                       stream, p);
  if (p.width < Elem<DT>::kPerVec)
    LaunchTiny<DT>(p, backward, stream);
  else if (p.width <= MaxHeld(DT, backward))
    LaunchType<DT>(p, backward, stream);
  else
    LaunchLong<DT>(p, backward, stream);
}

void Launch(const NormParams &p, bool backward, hipStream_t stream) {
  if (p.dtype == DT_F32)
    LaunchOf<DT_F32>(p, backward, stream);
  else if (p.dtype == DT_BF16)
    LaunchOf<DT_BF16>(p, backward, stream);
  else
    LaunchOf<DT_F16>(p, backward, stream);
}

// Rows of partial sums that a backward pass leaves.
int PartsOf(const NormParams &p) {
  if (p.width > kMaxSummed)
    return NormPartials(p.rows, p.width);
  if (p.width < (p.dtype == DT_F32 ? 4 : 8))
    return Groups((p.rows + 255) / 256, 512, 8);
  const Shape s = ShapeOf(p.width, p.dtype);
  return Groups(p.rows, s.lanes, s.vectors * (p.dtype == DT_F32 ? 4 : 8));
}

bool Sound(const NormParams &p) {
  return p.rows >= 0 && p.width >= 1 && p.width <= (1 << 20) && (p.rows == 0 || p.x);
}

}  // namespace

int NormPartials(std::int64_t rows, int width) {
  // At least what Groups says of any type: 256 lanes of 8 values have 2048 columns.
  const int most = width > kMaxSummed ? kColumnGroups : width > 2048 ? kMaxGroups : kMoreGroups;
  return static_cast<int>(std::min<std::int64_t>(rows, most));
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
    hipLaunchKernelGGL(NormSumsKernel, dim3((p.width + 63) / 64, 2), dim3(1024), 0, stream,
                       p.partials, PartsOf(p), p.width, p.dgamma, p.dbeta);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace mfh
