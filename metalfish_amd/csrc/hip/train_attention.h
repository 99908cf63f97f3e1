// Attention with gradients: the pieces that its kernels share.
//
// The matrix instruction computes D[16 x 16] = A[16 x 32] B[32 x 16] from eight
// values a lane of A and of B: lane l holds row (column) l % 16 and eight of the
// 32 places summed over, and D leaves it with column l % 16, rows 4 (l / 16) ..
// + 3.  The sum does not care which places a lane holds as long as A and B
// agree, so two 16 x 16 results, eight values a lane, are one operand of the
// next product as they lie in registers: scores become probabilities and feed
// the product with V (or dout, Q, K) without passing through memory.  The other
// operand then takes its rows 4 (l / 16) .. + 3 of both tiles, column l % 16,
// from a row-major tile in LDS: two transposing reads of four values.
//
// fp32 runs the same code on the 16 x 16 x 4 instruction, eight times.
#pragma once

#include "learn_device.h"
#include "mfh_device.h"
#include "mfh_kernels.h"

namespace mfh {
namespace attend {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_a2 __attribute__((ext_vector_type(2), aligned(2), may_alias));

constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f;
constexpr int kTile = 64;  // rows of a workgroup (16 a wave), and keys of a step

// A row of a tile in LDS: 16 bytes of padding spread rows over the banks.
template <int DT, int DP> constexpr int kLd = DP + (DT == DT_F32 ? 4 : 8);

template <int DT> struct Mat;
template <class V> __device__ __forceinline__ V TwoReads(const std::uint16_t *a,
                                                         const std::uint16_t *b) {
  typedef __attribute__((address_space(3))) s16x4 *Lds;
  const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(a)),
              y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(b));
  const u32x2 p = __builtin_bit_cast(u32x2, x), q = __builtin_bit_cast(u32x2, y);
  return __builtin_bit_cast(V, (u32x4{p[0], p[1], q[0], q[1]}));
}
template <> struct Mat<DT_BF16> {
  using T = std::uint16_t;
  using E = __bf16;
  using Frag = bf16x8;
  static __device__ __forceinline__ f32x4 Mul(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ Frag Pack(f32x4 a, f32x4 b) {
    return __builtin_bit_cast(Frag, (u32x4{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]),
                                           pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])}));
  }
  static __device__ __forceinline__ float Get(Frag f, int i) { return static_cast<float>(f[i]); }
};
template <> struct Mat<DT_F16> {
  using T = std::uint16_t;
  using E = _Float16;
  using Frag = f16x8;
  static __device__ __forceinline__ f32x4 Mul(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ Frag Pack(f32x4 a, f32x4 b) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = static_cast<_Float16>(a[i]);
      f[4 + i] = static_cast<_Float16>(b[i]);
    }
    return f;
  }
  static __device__ __forceinline__ float Get(Frag f, int i) { return static_cast<float>(f[i]); }
};
template <> struct Mat<DT_F32> {
  using T = float;
  using E = float;
  using Frag = f32x8;
  static __device__ __forceinline__ f32x4 Mul(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag Pack(f32x4 a, f32x4 b) {
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  static __device__ __forceinline__ float Get(Frag f, int i) { return f[i]; }
};

// Eight consecutive values of a row in LDS.
template <int DT>
__device__ __forceinline__ typename Mat<DT>::Frag FromRow(const typename Mat<DT>::T *p) {
  if constexpr (DT == DT_F32) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  } else {
    return *reinterpret_cast<const typename Mat<DT>::Frag *>(p);
  }
}
template <int DT>
__device__ __forceinline__ void ToRow(typename Mat<DT>::T *p, typename Mat<DT>::Frag f) {
  if constexpr (DT == DT_F32) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<f32x4 *>(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
  } else {
    *reinterpret_cast<typename Mat<DT>::Frag *>(p) = f;
  }
}
// Column col0 + lane % 16 of rows row .. row + 3 and row + 16 .. row + 19 of a
// tile, row = row0 + 4 (lane / 16).
template <int DT, int LD>
__device__ __forceinline__ typename Mat<DT>::Frag FromColumns(const typename Mat<DT>::T *tile,
                                                              int row0, int col0, int lane) {
  const int fr = lane & 15, row = row0 + 4 * (lane >> 4);
  if constexpr (DT == DT_F32) {
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = tile[(row + j) * LD + col0 + fr];
      f[4 + j] = tile[(row + 16 + j) * LD + col0 + fr];
    }
    return f;
  } else {
    const std::uint16_t *p = tile + (row + (fr >> 2)) * LD + col0 + 4 * (fr & 3);
    return TwoReads<typename Mat<DT>::Frag>(p, p + 16 * LD);
  }
}

// Eight values from element d0 of a head's row in memory, zeros behind `dim`.
template <int DT>
__device__ __forceinline__ typename Mat<DT>::Frag FromMemory(ConstRow<DT> row, int d0, int dim) {
  using Frag = typename Mat<DT>::Frag;
  if (d0 + 8 <= dim) {
    if constexpr (DT == DT_F32) {
      const u32x4 a = *(const MFH_GLOBAL u32x4_a4 *)(row + d0),
                  b = *(const MFH_GLOBAL u32x4_a4 *)(row + d0 + 4);
      return __builtin_bit_cast(Frag, (__attribute__((ext_vector_type(8))) unsigned int){
                                          a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    } else {
      return __builtin_bit_cast(Frag, LoadVec<DT, false>(row + d0));
    }
  }
  Frag f{};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (d0 + e < dim) {
      if constexpr (DT == DT_F32)
        f[e] = __uint_as_float(row[d0 + e]);
      else
        f[e] = __builtin_bit_cast(typename Mat<DT>::E, row[d0 + e]);
    }
  return f;
}


// Stores four consecutive values from element d0 of a row.
template <int DT>
__device__ __forceinline__ void ToMemory(Row<DT> row, int d0, int dim, f32x4 v) {
  if (d0 + 4 <= dim) {
    if constexpr (DT == DT_F32) {
      *(MFH_GLOBAL u32x4_a4 *)(row + d0) = __builtin_bit_cast(u32x4, v);
    } else {
      u32x2 p;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        p[i] = Elem<DT>::Round(v[2 * i]) |
               static_cast<std::uint32_t>(Elem<DT>::Round(v[2 * i + 1])) << 16;
      *(MFH_GLOBAL u32x2_a2 *)(row + d0) = p;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d0 + e < dim)
      row[d0 + e] = Elem<DT>::Round(v[e]);
}

// Sum and maximum over the four lanes that hold one column of a result.
__device__ __forceinline__ float OverRows(float v, bool most) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = most ? fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]))
           : __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return most ? fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]))
              : __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// One launch's problem: a part of the work is (line and key head, tile, split
// of the axis that it loops over).
struct Args {
  TrainAttention a;
  int lines = 0;   // batch * kv_heads
  int rows = 0;    // group * q_len
  int tiles = 0;   // of the axis that workgroups share
  int steps = 0;   // tiles of the axis that they loop over
  int splits = 1;  // of that axis
  int dim4 = 0;    // dim rounded up to whole groups of four: a partial row
  std::int64_t work = 0;            // lines * tiles * splits
  std::int64_t first = 0, end = 0;  // the parts of one launch
  float *partials = nullptr;
  float *delta = nullptr;  // [lines][rows]
};

// Which part a workgroup does.  Workgroups go round the eight dies by their
// number; parts of one line stay on one, whose cache then holds its keys.
struct Part {
  int line, tile, split;
};
__device__ __forceinline__ bool PartOf(const Args &a, Part *p) {
  const std::int64_t per = (a.end - a.first + 7) / 8;
  const std::int64_t w = a.first + (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (w >= a.end)
    return false;
  const std::int64_t t = w / a.splits;
  p->split = static_cast<int>(w % a.splits);
  p->line = static_cast<int>(t / a.tiles);
  p->tile = static_cast<int>(t % a.tiles);
  return true;
}

__device__ __forceinline__ int LengthOf(const std::int32_t *lengths, int b, int most) {
  if (!lengths)
    return most;
  const int n = lengths[b];
  return n < 0 ? 0 : n > most ? most : n;
}

// A line's lengths, and the last key that query q of it sees (below 0: none).
struct Line {
  int b, kv, q_len, k_len;
  bool causal;
  __device__ __forceinline__ int Last(int q) const {
    if (q >= q_len)
      return -1;
    return causal ? min(k_len - 1, q + (k_len - q_len)) : k_len - 1;
  }
};
__device__ __forceinline__ Line LineOf(const Args &s, int line) {
  Line l;
  l.b = line / s.a.kv_heads;
  l.kv = line % s.a.kv_heads;
  l.q_len = LengthOf(s.a.q_lengths, l.b, s.a.q_len);
  l.k_len = LengthOf(s.a.k_lengths, l.b, s.a.k_len);
  l.causal = s.a.causal;
  return l;
}
// One more than the last key that any of rows first .. first + kTile - 1 sees.
__device__ __forceinline__ int KeysSeen(const Args &s, const Line &l, int first) {
  const int last = min(first + kTile, s.rows) - 1;
  const int h0 = first / s.a.q_len, h1 = last / s.a.q_len;
  int q = l.q_len - 1;
  if (h0 == h1) {
    if (first - h0 * s.a.q_len >= l.q_len)
      return 0;
    q = min(q, last - h0 * s.a.q_len);
  }
  return q < 0 ? 0 : max(0, l.Last(q) + 1);
}

// Address of a row of a view: row r of a line.
template <int DT, class P>
__device__ __forceinline__ P RowAt(const HeadsView &v, int b, int head, int token) {
  return (P)v.p + (static_cast<std::int64_t>(b) * v.batch + static_cast<std::int64_t>(token) * v.token +
                   static_cast<std::int64_t>(head) * v.head);
}
template <int DT>
__device__ __forceinline__ ConstRow<DT> In(const HeadsView &v, int b, int head, int token) {
  return RowAt<DT, ConstRow<DT>>(v, b, head, token);
}
template <int DT>
__device__ __forceinline__ Row<DT> Out(const HeadsView &v, int b, int head, int token) {
  return RowAt<DT, Row<DT>>(v, b, head, token);
}

__device__ __forceinline__ std::int64_t BiasAt(const TrainAttention &a, int b, int head, int q) {
  return static_cast<std::int64_t>(b) * a.bias_batch + static_cast<std::int64_t>(head) * a.bias_head +
         static_cast<std::int64_t>(q) * a.bias_query;
}
__device__ __forceinline__ float Bias1(const void *p, int dtype, std::int64_t at) {
  if (dtype == DT_F32)
    return ((const MFH_GLOBAL float *)p)[at];
  const std::uint16_t v = ((const MFH_GLOBAL std::uint16_t *)p)[at];
  return dtype == DT_BF16 ? Elem<DT_BF16>::One(v) : Elem<DT_F16>::One(v);
}
// Four consecutive values, of which n are in the array.
__device__ __forceinline__ f32x4 Bias4(const void *p, int dtype, std::int64_t at, int n) {
  f32x4 f{0.f, 0.f, 0.f, 0.f};
  if (n >= 4) {
    if (dtype == DT_F32)
      return __builtin_bit_cast(f32x4, *(const MFH_GLOBAL u32x4_a4 *)((const MFH_GLOBAL float *)p + at));
    const u32x2 v = *(const MFH_GLOBAL u32x2_a2 *)((const MFH_GLOBAL std::uint16_t *)p + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const auto one = static_cast<std::uint16_t>(v[e >> 1] >> (16 * (e & 1)));
      f[e] = dtype == DT_BF16 ? Elem<DT_BF16>::One(one) : Elem<DT_F16>::One(one);
    }
    return f;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n)
      f[e] = Bias1(p, dtype, at + e);
  return f;
}
__device__ __forceinline__ void StoreBias4(void *p, int dtype, std::int64_t at, int n, f32x4 f) {
  if (dtype == DT_F32)
    ToMemory<DT_F32>((Row<DT_F32>)p + at, 0, n, f);
  else if (dtype == DT_BF16)
    ToMemory<DT_BF16>((Row<DT_BF16>)p + at, 0, n, f);
  else
    ToMemory<DT_F16>((Row<DT_F16>)p + at, 0, n, f);
}

// kTile rows of a view as a row-major tile in LDS, 256 threads: chunk i of a
// thread is eight values of row RowOfChunk(i).
template <int DT, int DP> struct Stage {
  static constexpr int kChunks = kTile * DP / 8 / 256, kAcross = DP / 8;
  typename Mat<DT>::Frag f[kChunks];
  static __device__ __forceinline__ int RowOf(int i) { return (i * 256 + threadIdx.x) / kAcross; }
  static __device__ __forceinline__ int At(int i) { return (i * 256 + threadIdx.x) % kAcross * 8; }
  __device__ __forceinline__ void Store(typename Mat<DT>::T *tile) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      ToRow<DT>(tile + RowOf(i) * kLd<DT, DP> + At(i), f[i]);
  }
  // Keys first .. of a line: zeros from `end` on.
  __device__ __forceinline__ void Keys(const HeadsView &v, const Line &l, int first, int dim) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int j = first + RowOf(i);
      f[i] = typename Mat<DT>::Frag{};
      if (j < l.k_len)
        f[i] = FromMemory<DT>(In<DT>(v, l.b, l.kv, j), At(i), dim);
    }
  }
  // Rows first .. of a line: zeros where a row sees nothing.
  __device__ __forceinline__ void Rows(const Args &s, const HeadsView &v, const Line &l, int first) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int r = first + RowOf(i);
      f[i] = typename Mat<DT>::Frag{};
      if (r < s.rows) {
        const int h = r / s.a.q_len, q = r - h * s.a.q_len;
        if (l.Last(q) >= 0)
          f[i] = FromMemory<DT>(In<DT>(v, l.b, l.kv * s.a.group + h, q), At(i), s.a.dim);
      }
    }
  }
};

// Scores of a key tile against the 16 rows of a wave, keys down: lane l has
// row l % 16 and keys 16 t + 4 (l / 16) + e.
template <int DT, int DP>
__device__ __forceinline__ void Scores(const typename Mat<DT>::T *tile,
                                       const typename Mat<DT>::Frag *rows, int lane, f32x4 *out) {
  const int fr = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    out[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
      out[t] = Mat<DT>::Mul(FromRow<DT>(tile + (16 * t + fr) * kLd<DT, DP> + 32 * c + 8 * g),
                            rows[c], out[t]);
  }
}

template <int DT, int DP>
__global__ __launch_bounds__(256) void ForwardKernel(Args s) {
  using M = Mat<DT>;
  constexpr int LD = kLd<DT, DP>;
  __shared__ __attribute__((aligned(16))) typename M::T ks[kTile * LD], vs[kTile * LD];
  Part part;
  if (!PartOf(s, &part))
    return;
  const TrainAttention &a = s.a;
  const Line l = LineOf(s, part.line);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int first = part.tile * kTile, r = first + 16 * wave + fr;
  const bool live = r < s.rows;
  const int h = live ? r / a.q_len : 0, q = live ? r - h * a.q_len : 0, head = l.kv * a.group + h;
  const int last = live ? l.Last(q) : -1;
  typename M::Frag qf[DP / 32];
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) {
    qf[c] = typename M::Frag{};
    if (last >= 0)
      qf[c] = FromMemory<DT>(In<DT>(a.q, l.b, head, q), 32 * c + 8 * g, a.dim);
  }
  const std::int64_t bias_at = a.bias ? BiasAt(a, l.b, head, q) : 0;
  const int seen = KeysSeen(s, l, first);
  const int per = (s.steps + s.splits - 1) / s.splits;
  const int begin = part.split * per, end = min(begin + per, (seen + kTile - 1) / kTile);
  f32x4 acc[DP / 16];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float most = -__builtin_inff(), total = 0.f;
  Stage<DT, DP> kt, vt;
  if (begin < end) {
    kt.Keys(a.k, l, begin * kTile, a.dim);
    vt.Keys(a.v, l, begin * kTile, a.dim);
  }
  for (int step = begin; step < end; ++step) {
    kt.Store(ks);
    vt.Store(vs);
    __syncthreads();
    if (step + 1 < end) {
      kt.Keys(a.k, l, (step + 1) * kTile, a.dim);
      vt.Keys(a.v, l, (step + 1) * kTile, a.dim);
    }
    f32x4 x[4];
    Scores<DT, DP>(ks, qf, lane, x);
    const int j0 = step * kTile + 4 * g;
    float top = most;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int j = j0 + 16 * t;
      f32x4 bias{0.f, 0.f, 0.f, 0.f};
      if (a.bias && j <= last)
        bias = Bias4(a.bias, a.bias_dtype, bias_at + j, a.k_len - j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[t][e] = j + e <= last ? x[t][e] * a.scale + bias[e] : -__builtin_inff();
        top = fmaxf(top, x[t][e]);
      }
    }
    top = OverRows(top, true);
    const float base = top == -__builtin_inff() ? 0.f : top;
    const float old = Exp2((most - base) * kLog2e);
    most = top;
    total *= old;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[t][e] = Exp2((x[t][e] - base) * kLog2e);
        total += x[t][e];
      }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
      acc[i] *= old;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const typename M::Frag p = M::Pack(x[2 * u], x[2 * u + 1]);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        acc[i] = M::Mul(FromColumns<DT, LD>(vs, 32 * u, 16 * i, lane), p, acc[i]);
    }
    __syncthreads();
  }
  total = OverRows(total, false);
  if (!live)
    return;
  const std::int64_t flat = static_cast<std::int64_t>(part.line) * s.rows + r;
  if (s.splits > 1) {
    const std::int64_t n = static_cast<std::int64_t>(s.lines) * s.rows;
    float *o = s.partials + (part.split * n + flat) * s.dim4;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
      if (16 * i + 4 * g < s.dim4)
        *reinterpret_cast<f32x4 *>(o + 16 * i + 4 * g) = acc[i];
    if (g == 0) {
      float *st = s.partials + s.splits * n * s.dim4 + (part.split * n + flat) * 2;
      st[0] = most;
      st[1] = total;
    }
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const Row<DT> out = Out<DT>(a.out, l.b, head, q);
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
    ToMemory<DT>(out, 16 * i + 4 * g, a.dim, acc[i] * inv);
  if (a.lse && g == 0)
    a.lse[flat] = total == 0.f ? -__builtin_inff() : most + kLn2 * __builtin_amdgcn_logf(total);
}

// Joins the splits of a forward pass: one wave a row.
template <int DT>
__global__ __launch_bounds__(256) void JoinForwardKernel(Args s) {
  const std::int64_t n = static_cast<std::int64_t>(s.lines) * s.rows;
  const std::int64_t flat = static_cast<std::int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (flat >= n)
    return;
  const int lane = threadIdx.x & 63;
  const float *st = s.partials + s.splits * n * s.dim4;
  float most = -__builtin_inff();
  for (int k = 0; k < s.splits; ++k)
    most = fmaxf(most, st[(k * n + flat) * 2]);
  const float base = most == -__builtin_inff() ? 0.f : most;
  float total = 0.f;
  f32x2 o{0.f, 0.f};
  for (int k = 0; k < s.splits; ++k) {
    const float w = Exp2((st[(k * n + flat) * 2] - base) * kLog2e);
    total += w * st[(k * n + flat) * 2 + 1];
    if (2 * lane < s.dim4) {
      const f32x2 v = *reinterpret_cast<const f32x2 *>(s.partials + (k * n + flat) * s.dim4 + 2 * lane);
      // An empty split of a row holds zeros.
      o[0] += w * v[0];
      o[1] += w * v[1];
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int line = static_cast<int>(flat / s.rows), r = static_cast<int>(flat % s.rows);
  const int b = line / s.a.kv_heads, head = line % s.a.kv_heads * s.a.group + r / s.a.q_len;
  const Row<DT> out = Out<DT>(s.a.out, b, head, r % s.a.q_len);
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (2 * lane + e < s.a.dim)
      out[2 * lane + e] = Elem<DT>::Round(o[e] * inv);
  if (s.a.lse && lane == 0)
    s.a.lse[flat] = total == 0.f ? -__builtin_inff() : most + kLn2 * __builtin_amdgcn_logf(total);
}

// A row's log-sum-exp as what its scores are taken off: +inf where it sees
// nothing, so that every probability is 0.
__device__ __forceinline__ float Lse(float v) { return v == -__builtin_inff() ? __builtin_inff() : v; }

// delta = dout . out of each row, then dq (and dbias) of a tile of rows over the
// keys.
template <int DT, int DP>
__global__ __launch_bounds__(256) void BackwardRowsKernel(Args s) {
  using M = Mat<DT>;
  constexpr int LD = kLd<DT, DP>;
  __shared__ __attribute__((aligned(16))) typename M::T ks[kTile * LD], vs[kTile * LD];
  Part part;
  if (!PartOf(s, &part))
    return;
  const TrainAttention &a = s.a;
  const Line l = LineOf(s, part.line);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int first = part.tile * kTile, r = first + 16 * wave + fr;
  const bool live = r < s.rows;
  const int h = live ? r / a.q_len : 0, q = live ? r - h * a.q_len : 0, head = l.kv * a.group + h;
  const int last = live ? l.Last(q) : -1;
  const std::int64_t flat = static_cast<std::int64_t>(part.line) * s.rows + r;
  typename M::Frag qf[DP / 32], df[DP / 32];
  float delta = 0.f;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) {
    qf[c] = df[c] = typename M::Frag{};
    if (last >= 0) {
      const int d0 = 32 * c + 8 * g;
      qf[c] = FromMemory<DT>(In<DT>(a.q, l.b, head, q), d0, a.dim);
      df[c] = FromMemory<DT>(In<DT>(a.dout, l.b, head, q), d0, a.dim);
      const typename M::Frag o = FromMemory<DT>(In<DT>(a.out, l.b, head, q), d0, a.dim);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        delta += M::Get(o, e) * M::Get(df[c], e);
    }
  }
  delta = OverRows(delta, false);
  if (live && g == 0 && part.split == 0)
    s.delta[flat] = delta;
  if (!a.dq.p && !a.dbias)
    return;
  const float lse = last >= 0 ? Lse(a.lse[flat]) : __builtin_inff();
  const std::int64_t bias_at = a.bias ? BiasAt(a, l.b, head, q) : 0;
  // Every element of the bias's gradient is written, so no key is left out.
  const int seen = a.dbias ? a.k_len : KeysSeen(s, l, first);
  const int per = (s.steps + s.splits - 1) / s.splits;
  const int begin = part.split * per, end = min(begin + per, (seen + kTile - 1) / kTile);
  f32x4 acc[DP / 16];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  Stage<DT, DP> kt, vt;
  if (begin < end) {
    kt.Keys(a.k, l, begin * kTile, a.dim);
    vt.Keys(a.v, l, begin * kTile, a.dim);
  }
  for (int step = begin; step < end; ++step) {
    kt.Store(ks);
    vt.Store(vs);
    __syncthreads();
    if (step + 1 < end) {
      kt.Keys(a.k, l, (step + 1) * kTile, a.dim);
      vt.Keys(a.v, l, (step + 1) * kTile, a.dim);
    }
    f32x4 x[4], dp[4];
    Scores<DT, DP>(ks, qf, lane, x);
    Scores<DT, DP>(vs, df, lane, dp);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int j = step * kTile + 4 * g + 16 * t;
      f32x4 bias{0.f, 0.f, 0.f, 0.f};
      if (a.bias && j <= last)
        bias = Bias4(a.bias, a.bias_dtype, bias_at + j, a.k_len - j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = Exp2((x[t][e] * a.scale + bias[e] - lse) * kLog2e);
        x[t][e] = j + e <= last ? p * (dp[t][e] - delta) : 0.f;
      }
      if (a.dbias && live && j < a.k_len)
        StoreBias4(a.dbias, a.bias_dtype, bias_at + j, a.k_len - j, x[t]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const typename M::Frag ds = M::Pack(x[2 * u], x[2 * u + 1]);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        acc[i] = M::Mul(FromColumns<DT, LD>(ks, 32 * u, 16 * i, lane), ds, acc[i]);
    }
    __syncthreads();
  }
  if (!live || !a.dq.p)
    return;
  if (s.splits > 1) {
    const std::int64_t n = static_cast<std::int64_t>(s.lines) * s.rows;
    float *o = s.partials + (part.split * n + flat) * s.dim4;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
      if (16 * i + 4 * g < s.dim4)
        *reinterpret_cast<f32x4 *>(o + 16 * i + 4 * g) = acc[i];
    return;
  }
  const Row<DT> out = Out<DT>(a.dq, l.b, head, q);
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
    ToMemory<DT>(out, 16 * i + 4 * g, a.dim, acc[i] * a.scale);
}

// dk and dv of a tile of keys over the rows that share them; each wave has 16
// keys and holds them, and rows go through LDS.
template <int DT, int DP>
__global__ __launch_bounds__(256) void BackwardKeysKernel(Args s) {
  using M = Mat<DT>;
  constexpr int LD = kLd<DT, DP>;
  __shared__ __attribute__((aligned(16))) typename M::T qs[kTile * LD], dos[kTile * LD];
  __shared__ __attribute__((aligned(16))) int lasts[kTile];
  __shared__ __attribute__((aligned(16))) float lses[kTile], deltas[kTile];
  __shared__ std::int64_t biases[kTile];
  Part part;
  if (!PartOf(s, &part))
    return;
  const TrainAttention &a = s.a;
  const Line l = LineOf(s, part.line);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int key0 = part.tile * kTile, j = key0 + 16 * wave + fr;
  typename M::Frag kf[DP / 32], vf[DP / 32];
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) {
    kf[c] = vf[c] = typename M::Frag{};
    if (j < l.k_len) {
      kf[c] = FromMemory<DT>(In<DT>(a.k, l.b, l.kv, j), 32 * c + 8 * g, a.dim);
      vf[c] = FromMemory<DT>(In<DT>(a.v, l.b, l.kv, j), 32 * c + 8 * g, a.dim);
    }
  }
  f32x4 dk[DP / 16], dv[DP / 16];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
    dk[i] = dv[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int per = (s.steps + s.splits - 1) / s.splits;
  const int begin = part.split * per, end = min(begin + per, s.steps);
  for (int step = begin; step < end; ++step) {
    const int first = step * kTile;
    if (KeysSeen(s, l, first) <= key0)
      continue;  // the same in the whole workgroup
    Stage<DT, DP> qt, dt;
    qt.Rows(s, a.q, l, first);
    dt.Rows(s, a.dout, l, first);
    qt.Store(qs);
    dt.Store(dos);
    if (threadIdx.x < kTile) {
      const int r = first + threadIdx.x;
      int last = -1;
      float lse = __builtin_inff(), delta = 0.f;
      if (r < s.rows) {
        const int h = r / a.q_len, q = r - h * a.q_len;
        const std::int64_t flat = static_cast<std::int64_t>(part.line) * s.rows + r;
        last = l.Last(q);
        if (last >= 0) {
          lse = Lse(a.lse[flat]);
          delta = s.delta[flat];
        }
        biases[threadIdx.x] = a.bias ? BiasAt(a, l.b, l.kv * a.group + h, q) : 0;
      }
      lasts[threadIdx.x] = last;
      lses[threadIdx.x] = lse;
      deltas[threadIdx.x] = delta;
    }
    __syncthreads();
    f32x4 x[4], dp[4];
    Scores<DT, DP>(qs, kf, lane, x);
    Scores<DT, DP>(dos, vf, lane, dp);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int at = 16 * t + 4 * g;
      const f32x4 lse = *reinterpret_cast<const f32x4 *>(lses + at),
                  delta = *reinterpret_cast<const f32x4 *>(deltas + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool sees = j <= lasts[at + e];
        const float bias = a.bias && sees ? Bias1(a.bias, a.bias_dtype, biases[at + e] + j) : 0.f;
        const float p = Exp2((x[t][e] * a.scale + bias - lse[e]) * kLog2e);
        x[t][e] = sees ? p : 0.f;
        dp[t][e] = sees ? p * (dp[t][e] - delta[e]) : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const typename M::Frag p = M::Pack(x[2 * u], x[2 * u + 1]),
                             ds = M::Pack(dp[2 * u], dp[2 * u + 1]);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        dv[i] = M::Mul(FromColumns<DT, LD>(dos, 32 * u, 16 * i, lane), p, dv[i]);
        dk[i] = M::Mul(FromColumns<DT, LD>(qs, 32 * u, 16 * i, lane), ds, dk[i]);
      }
    }
    __syncthreads();
  }
  if (j >= a.k_len)
    return;
  if (s.splits > 1) {
    const std::int64_t n = static_cast<std::int64_t>(s.lines) * a.k_len;
    const std::int64_t flat = static_cast<std::int64_t>(part.line) * a.k_len + j;
    float *o = s.partials + (2 * part.split * n + flat) * s.dim4;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
      if (16 * i + 4 * g < s.dim4) {
        *reinterpret_cast<f32x4 *>(o + 16 * i + 4 * g) = dk[i];
        *reinterpret_cast<f32x4 *>(o + n * s.dim4 + 16 * i + 4 * g) = dv[i];
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    if (a.dk.p)
      ToMemory<DT>(Out<DT>(a.dk, l.b, l.kv, j), 16 * i + 4 * g, a.dim, dk[i] * a.scale);
    if (a.dv.p)
      ToMemory<DT>(Out<DT>(a.dv, l.b, l.kv, j), 16 * i + 4 * g, a.dim, dv[i]);
  }
}

// Adds up the splits of dq (KEYS false) or of dk and dv: one wave a row.
template <int DT, bool KEYS>
__global__ __launch_bounds__(256) void JoinBackwardKernel(Args s) {
  const int per = KEYS ? s.a.k_len : s.rows;
  const std::int64_t n = static_cast<std::int64_t>(s.lines) * per;
  const std::int64_t all = KEYS ? 2 * n : n;
  const std::int64_t at = static_cast<std::int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (at >= all || 2 * lane >= s.dim4)
    return;
  f32x2 o{0.f, 0.f};
  for (int k = 0; k < s.splits; ++k) {
    const f32x2 v = *reinterpret_cast<const f32x2 *>(s.partials + (k * all + at) * s.dim4 + 2 * lane);
    o[0] += v[0];
    o[1] += v[1];
  }
  const bool second = KEYS && at >= n;
  const std::int64_t flat = second ? at - n : at;
  const int line = static_cast<int>(flat / per), r = static_cast<int>(flat % per);
  const int b = line / s.a.kv_heads, kv = line % s.a.kv_heads;
  Row<DT> out;
  if constexpr (KEYS) {
    const HeadsView &v = second ? s.a.dv : s.a.dk;
    if (!v.p)
      return;
    out = Out<DT>(v, b, kv, r);
  } else {
    out = Out<DT>(s.a.dq, b, kv * s.a.group + r / s.a.q_len, r % s.a.q_len);
  }
  const float scale = second ? 1.f : s.a.scale;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (2 * lane + e < s.a.dim)
      out[2 * lane + e] = Elem<DT>::Round(o[e] * scale);
}

// The gradient of a bias that lines or heads share: a workgroup has 64 queries
// and 64 keys of one of its planes and loops over what shares it.
template <int DT, int DP>
__global__ __launch_bounds__(256) void BiasGradKernel(Args s, int plane_heads) {
  using M = Mat<DT>;
  const TrainAttention &a = s.a;
  const int k_tiles = (a.k_len + kTile - 1) / kTile, q_tiles = (a.q_len + kTile - 1) / kTile;
  const std::int64_t id = s.first + blockIdx.x;
  const int kt = static_cast<int>(id % k_tiles), qt = static_cast<int>(id / k_tiles % q_tiles);
  const int plane = static_cast<int>(id / k_tiles / q_tiles);
  const int b_plane = plane / plane_heads, h_plane = plane % plane_heads;
  const int b0 = a.bias_batch ? b_plane : 0, b1 = a.bias_batch ? b_plane + 1 : a.batch;
  const int h0 = a.bias_head ? h_plane : 0, h1 = a.bias_head ? h_plane + 1 : a.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int q = qt * kTile + 16 * wave + fr;
  const bool live = q < a.q_len;
  const std::int64_t bias_at = BiasAt(a, b_plane, h_plane, live ? q : 0);
  f32x4 acc[4], bias[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int j = kt * kTile + 16 * t + 4 * g;
    acc[t] = bias[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (live && j < a.k_len)
      bias[t] = Bias4(a.bias, a.bias_dtype, bias_at + j, a.k_len - j);
  }
  for (int b = b0; b < b1; ++b)
    for (int head = h0; head < h1; ++head) {
      const int kv = head / a.group;
      const Line l = LineOf(s, b * a.kv_heads + kv);
      const int last = live ? l.Last(q) : -1;
      const std::int64_t flat = (static_cast<std::int64_t>(b) * a.heads + head) * a.q_len + q;
      typename M::Frag qf[DP / 32], df[DP / 32];
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        qf[c] = df[c] = typename M::Frag{};
        if (last >= 0) {
          qf[c] = FromMemory<DT>(In<DT>(a.q, b, head, q), 32 * c + 8 * g, a.dim);
          df[c] = FromMemory<DT>(In<DT>(a.dout, b, head, q), 32 * c + 8 * g, a.dim);
        }
      }
      const float lse = last >= 0 ? Lse(a.lse[flat]) : __builtin_inff();
      const float delta = last >= 0 ? s.delta[flat] : 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 x{0.f, 0.f, 0.f, 0.f}, dp{0.f, 0.f, 0.f, 0.f};
        const int key = kt * kTile + 16 * t + fr, j = kt * kTile + 16 * t + 4 * g;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          typename M::Frag kf{}, vf{};
          if (key < l.k_len) {
            kf = FromMemory<DT>(In<DT>(a.k, b, kv, key), 32 * c + 8 * g, a.dim);
            vf = FromMemory<DT>(In<DT>(a.v, b, kv, key), 32 * c + 8 * g, a.dim);
          }
          x = M::Mul(kf, qf[c], x);
          dp = M::Mul(vf, df[c], dp);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = Exp2((x[e] * a.scale + bias[t][e] - lse) * kLog2e);
          acc[t][e] += j + e <= last ? p * (dp[e] - delta) : 0.f;
        }
      }
    }
  if (!live)
    return;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int j = kt * kTile + 16 * t + 4 * g;
    if (j < a.k_len)
      StoreBias4(a.dbias, a.bias_dtype, bias_at + j, a.k_len - j, acc[t]);
  }
}

// Workgroups that fill the card twice; a split loops over two tiles at least.
inline int SplitsOf(std::int64_t groups, int steps) {
  const std::int64_t want = 512 / std::max<std::int64_t>(groups, 1);
  return static_cast<int>(std::max<std::int64_t>(1, std::min<std::int64_t>(want, steps / 2)));
}
inline int Tiles(int n) { return (n + kTile - 1) / kTile; }

// Shapes of the three launches, and the workspace that they share.
inline Args ArgsOf(const TrainAttention &a, bool keys) {
  Args s;
  s.a = a;
  s.lines = a.batch * a.kv_heads;
  s.rows = a.group * a.q_len;
  s.dim4 = (a.dim + 3) & ~3;
  s.tiles = keys ? Tiles(a.k_len) : Tiles(s.rows);
  s.steps = keys ? Tiles(s.rows) : Tiles(a.k_len);
  s.splits = SplitsOf(static_cast<std::int64_t>(s.lines) * s.tiles, s.steps);
  s.work = static_cast<std::int64_t>(s.lines) * s.tiles * s.splits;
  return s;
}
// Whether the bias is shared by lines or heads.
inline bool SharedBias(const TrainAttention &a) {
  return a.dbias && ((a.bias_batch == 0 && a.batch > 1) || (a.bias_head == 0 && a.heads > 1));
}
inline std::uint64_t DeltaBytes(const Args &s) {
  return (static_cast<std::uint64_t>(s.lines) * s.rows * 4 + 15) & ~std::uint64_t(15);
}
inline std::uint64_t ForwardBytes(const Args &s) {
  return s.splits == 1 ? 0
                       : static_cast<std::uint64_t>(s.splits) * s.lines * s.rows * (s.dim4 + 2) * 4;
}
inline std::uint64_t RowsBytes(const Args &s) {
  return s.splits == 1 ? 0 : static_cast<std::uint64_t>(s.splits) * s.lines * s.rows * s.dim4 * 4;
}
inline std::uint64_t KeysBytes(const Args &s) {
  return s.splits == 1
             ? 0
             : static_cast<std::uint64_t>(s.splits) * 2 * s.lines * s.a.k_len * s.dim4 * 4;
}

// A launch has less than 2^32 threads; more work takes several.
constexpr std::int64_t kMostGroups = std::int64_t(1) << 23;
template <class K> hipError_t Run(K kernel, Args s, hipStream_t stream) {
  hipError_t e = hipSuccess;
  for (s.first = 0; e == hipSuccess && s.first < s.work; s.first = s.end) {
    s.end = std::min(s.work, s.first + kMostGroups);
    const auto groups = static_cast<unsigned>((s.end - s.first + 7) / 8 * 8);
    hipLaunchKernelGGL(kernel, dim3(groups), dim3(256), 0, stream, s);
    e = hipGetLastError();
  }
  return e;
}
// Four rows a workgroup; splits have few.
template <class K> hipError_t RunJoin(K kernel, const Args &s, std::int64_t n, hipStream_t stream) {
  if (n == 0)
    return hipSuccess;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n + 3) / 4)), dim3(256), 0, stream, s);
  return hipGetLastError();
}

template <int DT, int DP> hipError_t Forward(const TrainAttention &a, hipStream_t stream) {
  Args s = ArgsOf(a, false);
  s.partials = static_cast<float *>(a.workspace);
  hipError_t e = Run(ForwardKernel<DT, DP>, s, stream);
  if (e == hipSuccess && s.splits > 1)
    e = RunJoin(JoinForwardKernel<DT>, s, static_cast<std::int64_t>(s.lines) * s.rows, stream);
  return e;
}

template <int DT, int DP> hipError_t Backward(const TrainAttention &a, hipStream_t stream) {
  Args s = ArgsOf(a, false);
  s.delta = static_cast<float *>(a.workspace);
  s.partials = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + DeltaBytes(s));
  const bool shared = SharedBias(a);
  if (shared)
    s.a.dbias = nullptr;
  hipError_t e = Run(BackwardRowsKernel<DT, DP>, s, stream);
  if (e == hipSuccess && s.splits > 1 && a.dq.p)
    e = RunJoin(JoinBackwardKernel<DT, false>, s, static_cast<std::int64_t>(s.lines) * s.rows,
                stream);
  if (e == hipSuccess && (a.dk.p || a.dv.p)) {
    Args k = ArgsOf(a, true);
    k.delta = s.delta;
    k.partials = s.partials;
    e = Run(BackwardKeysKernel<DT, DP>, k, stream);
    if (e == hipSuccess && k.splits > 1)
      e = RunJoin(JoinBackwardKernel<DT, true>, k, 2 * static_cast<std::int64_t>(k.lines) * a.k_len,
                  stream);
  }
  if (e == hipSuccess && shared) {
    s.a.dbias = a.dbias;
    const int planes_b = a.bias_batch ? a.batch : 1, planes_h = a.bias_head ? a.heads : 1;
    s.work = static_cast<std::int64_t>(Tiles(a.q_len)) * Tiles(a.k_len) * planes_b * planes_h;
    for (s.first = 0; e == hipSuccess && s.first < s.work; s.first += kMostGroups) {
      const auto groups = static_cast<unsigned>(std::min(s.work - s.first, kMostGroups));
      hipLaunchKernelGGL((BiasGradKernel<DT, DP>), dim3(groups), dim3(256), 0, stream, s, planes_h);
      e = hipGetLastError();
    }
  }
  return e;
}

// By head size: a tile's columns are padded to 32, 64 or 128.
template <int DT>
hipError_t ByDim(const TrainAttention &a, bool backward, hipStream_t stream) {
  if (a.dim <= 32)
    return backward ? Backward<DT, 32>(a, stream) : Forward<DT, 32>(a, stream);
  if (a.dim <= 64)
    return backward ? Backward<DT, 64>(a, stream) : Forward<DT, 64>(a, stream);
  return backward ? Backward<DT, 128>(a, stream) : Forward<DT, 128>(a, stream);
}

// One source a type.
hipError_t AttentionF32(const TrainAttention &a, bool backward, hipStream_t stream);
hipError_t AttentionBf16(const TrainAttention &a, bool backward, hipStream_t stream);
hipError_t AttentionF16(const TrainAttention &a, bool backward, hipStream_t stream);

}  // namespace attend
}  // namespace mfh
