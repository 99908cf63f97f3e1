// Attention with gradients: the kernels, and the pieces that they share.
//
// The matrix instruction computes D[16 x 16] = A[16 x 32] B[32 x 16] from eight
// values a lane of A and of B: lane l holds row (column) l % 16 and eight of the
// 32 places summed over, and D leaves it with column l % 16, rows 4 (l / 16) ..
// + 3.  The sum does not care which places a lane holds as long as A and B
// agree, and rows may be taken in any order.  Results of four instructions over
// the rows RowOf(t, i) of a tile of 64 leave lane l, for one column, with rows
// 8 (l / 16) .. + 7 and the same 32 further: two operands of eight values for the
// next product as they lie in registers.  Scores become probabilities and feed
// the products with V (or dout, Q, K) without passing through memory, and a bias
// comes in vectors of eight.  The other operand takes those eight rows of one
// column from a row-major tile in LDS: two transposing reads of four values.
// Columns are taken in such an order too that a lane ends with consecutive
// elements of a head.
//
// fp32 runs the same code on the 16 x 16 x 4 instruction, eight times.
//
// With 16-bit inputs probabilities and dS are rounded to the inputs' type where they
// become operands (Mat::Pack): the instruction takes no wider ones beside them, and
// the fp32 one has an eighth of the rate that products reach (154 of 1216 TFLOP/s).
// That is at most 2^-8 (bf16) or 2^-11 (fp16) of each; scores, maxima, sums, delta and
// every accumulator are fp32.
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
// The row of a 64-row tile that row i of result t stands for, and the element
// of a head that row i of result t of a transposed product does.
__device__ __forceinline__ constexpr int RowOf64(int t, int i) {
  return 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
}
// Eight rows from row0 + 8 (lane / 16) on of a tile, at the element of a head of
// DP that row lane % 16 of result t of a transposed product stands for, or
// (DP = 64, t = 0 .. 3, keys) plainly column col0 + lane % 16.
template <int DT, int LD>
__device__ __forceinline__ typename Mat<DT>::Frag Columns(const typename Mat<DT>::T *tile, int row0,
                                                          int quad_step, int col0, int lane) {
  const int fr = lane & 15, row = row0 + 8 * (lane >> 4);
  if constexpr (DT == DT_F32) {
    const float *p = tile + row * LD + col0 + quad_step * (fr >> 2) + (fr & 3);
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f[j] = p[j * LD];
    return f;
  } else {
    const std::uint16_t *p = tile + (row + (fr >> 2)) * LD + col0 + quad_step * (fr & 3);
    return TwoReads<typename Mat<DT>::Frag>(p, p + 4 * LD);
  }
}
// Element (DP / 4) (i / 4) + 4 t + i % 4 of a head: a lane of the result then has
// the DP / 4 elements from (DP / 4) (lane / 16) on.
template <int DT, int DP, int LD>
__device__ __forceinline__ typename Mat<DT>::Frag HeadColumns(const typename Mat<DT>::T *tile,
                                                              int row0, int t, int lane) {
  return Columns<DT, LD>(tile, row0, DP / 4, 4 * t, lane);
}

// Eight values of a head's row in memory.
template <int DT>
__device__ __forceinline__ typename Mat<DT>::Frag FromMemory(ConstRow<DT> p) {
  if constexpr (DT == DT_F32) {
    const f32x4 a = __builtin_bit_cast(f32x4, LoadVec<DT, false>(p)),
                b = __builtin_bit_cast(f32x4, LoadVec<DT, false>(p + 4));
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  } else {
    return __builtin_bit_cast(typename Mat<DT>::Frag, LoadVec<DT, false>(p));
  }
}

// Stores four consecutive values, with eight: the next four too.
template <int DT>
__device__ __forceinline__ void ToMemory(Row<DT> p, f32x4 v) {
  if constexpr (DT == DT_F32) {
    StoreVec<DT, false>(p, __builtin_bit_cast(u32x4, v));
  } else {
    u32x2 o;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      o[i] = Elem<DT>::Round(v[2 * i]) |
             static_cast<std::uint32_t>(Elem<DT>::Round(v[2 * i + 1])) << 16;
    *(MFH_GLOBAL u32x2_a2 *)p = o;
  }
}
template <int DT>
__device__ __forceinline__ void ToMemory(Row<DT> p, f32x4 v, f32x4 w) {
  const float f[8] = {v[0], v[1], v[2], v[3], w[0], w[1], w[2], w[3]};
  StoreVec<DT, false>(p, Elem<DT>::Pack(f));
  if constexpr (DT == DT_F32)
    StoreVec<DT, false>(p + 4, Elem<DT>::Pack(f + 4));
}

// A lane's elements of a head, DP / 4 of them from (DP / 4) (lane / 16) on.
template <int DT, int DP>
__device__ __forceinline__ void StoreHead(Row<DT> row, int lane, int dim, const f32x4 *v,
                                          float scale) {
  const int d0 = DP / 4 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < DP / 16; i += 2)
    if (d0 + 4 * i < dim)
      ToMemory<DT>(row + d0 + 4 * i, v[i] * scale, v[i + 1] * scale);
}
// The same to a row of partial sums.
template <int DP>
__device__ __forceinline__ void StorePartial(float *row, int lane, int dim, const f32x4 *v) {
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    const int d = DP / 4 * (lane >> 4) + 4 * i;
    if (d < dim)
      *reinterpret_cast<f32x4 *>(row + d) = v[i];
  }
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

// One launch's problem: a part of the work is (line and key head, tile, split
// of the axis that it loops over).
struct Args {
  TrainAttention a;
  int lines = 0;   // batch * kv_heads
  int rows = 0;    // group * q_len
  int tiles = 0;   // of the axis that workgroups share
  int steps = 0;   // tiles of the axis that they loop over
  int splits = 1;  // of that axis
  int wide = 1;    // 16-column sets of a wave: a tile has 64 times as many
  int line0 = 0, lines_now = 0, tile0 = 0;  // the part of one launch
  bool spread = false, turn = false;        // the order of workgroups
  int across = 0;                           // of them along x, in a launch of both passes
  int down = 0;    // tiles from the last to the first, in so many interleaved runs
  float *partials = nullptr;
  float *delta = nullptr;  // [lines][rows]
  float *rest = nullptr;   // [lines][rows], with a bias (Coarse)
};

__device__ __forceinline__ int Uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Causal rows' tiles from the last to the first, in interleaved runs of tiles, one a
// head where heads have tiles of their own.  More runs than tiles would launch workgroups
// for nothing (1024 lines of one query of 128 heads over one key head, 64 keys of 64, bf16:
// 128 a line, 76 us and backward 158; so 2, 11.7 and 46).  The tile at place `at`; behind
// the last tile there is none.
inline int RunsDown(int tiles, int heads) {
  const int each = (tiles + heads - 1) / heads;
  return each > 0 ? (tiles + each - 1) / each : 0;
}
inline int PlacesDown(int tiles, int runs) {
  return runs ? (tiles + runs - 1) / runs * runs : tiles;
}
__host__ __device__ inline int TileDown(int at, int tiles, int runs) {
  const int each = (tiles + runs - 1) / runs;
  return at % runs * each + (each - 1 - at / runs);
}

// Which part a workgroup does.  Workgroups go round the eight dies by their
// number, and round a die's CUs.  Without splits blockIdx.x is the line and y the
// tile; with many lines (spread) x is a multiple of eight, so that the parts of one
// line share a die's cache and neighbouring heads, which share memory lines, do
// too; where the last tiles have most to do (causal rows), they come first.  With
// splits (few lines) each die takes an eighth of them in the order of memory: 3
// queries over 20011 keys, four lines, 10.9 us; one line after another along x, 18.4.
// Few lines that may differ in length take turns with the tiles, or a long one's
// parts meet on the same CUs: backward of four lines of up to 1021 tokens with four
// key heads, rows and keys launched apart, 67 us, 87 without.  Equal lines stay where they are, for the cache: 2 x 16
// heads of 128 over 2048 tokens forward 58 us, 77 in turns.
struct Part {
  int line, tile, split;
};
__device__ __forceinline__ bool PartOf(const Args &s, int x, int across, int down, Part *p) {
  const int at = s.spread ? (x & 7) * (across >> 3) + (x >> 3) : x;
  // y counts a line's parts.
  int line = at, y = s.tile0 + down, tile = y;
  bool mine = at < s.lines_now;
  p->split = 0;
  if (s.splits > 1) {
    const int parts = s.tiles * s.splits;
    if (s.turn) {
      y = at / s.lines;
      line = at - y * s.lines;
    } else {
      line = at / parts;
      y = at - line * parts;
    }
    tile = y / s.splits;
    p->split = y - tile * s.splits;
    mine = line < s.lines;
  }
  if (s.turn) {
    // One further a tile, and a step aside after each 256 workgroups (the CUs): 67
    // us in that case; one further a tile alone, 72.
    const unsigned aside = (static_cast<unsigned>(y) * s.lines_now >> 8) * (s.a.kv_heads + 1);
    line = static_cast<int>((line + y + aside) % static_cast<unsigned>(s.lines_now));
  }
  if (s.down)
    tile = TileDown(tile, s.tiles, s.down);
  p->line = s.line0 + line;
  p->tile = tile;
  return mine && tile < s.tiles;
}

__device__ __forceinline__ bool PartOf(const Args &s, Part *p) {
  return PartOf(s, blockIdx.x, gridDim.x, blockIdx.y, p);
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
  l.b = s.a.kv_heads == 1 ? line : line / s.a.kv_heads;
  l.kv = line - l.b * s.a.kv_heads;
  l.q_len = Uniform(LengthOf(s.a.q_lengths, l.b, s.a.q_len));
  l.k_len = Uniform(LengthOf(s.a.k_lengths, l.b, s.a.k_len));
  l.causal = s.a.causal;
  return l;
}
// `count` rows of a line from `first` on: the head and query of the first, and
// whether all are that head's.
struct Span64 {
  int h, q;
  bool same;
};
__device__ __forceinline__ Span64 SpanOf(const Args &s, int first, int count) {
  if (s.a.group == 1)
    return {0, first, true};
  const int h = first / s.a.q_len, q = first - h * s.a.q_len;
  return {h, q, q + count <= s.a.q_len};
}
// One more than the last key that any of them sees.
__device__ __forceinline__ int KeysSeen(const Line &l, const Span64 &t, int count) {
  int q = l.q_len - 1;
  if (t.same) {
    if (t.q >= l.q_len)
      return 0;
    q = min(q, t.q + count - 1);
  }
  return q < 0 ? 0 : max(0, l.Last(q) + 1);
}

// A token's offset: strides of tokens are below 2^32.
__device__ __forceinline__ std::uint64_t Tokens(const HeadsView &v, int token) {
  return static_cast<std::uint64_t>(static_cast<std::uint32_t>(token)) *
         static_cast<std::uint32_t>(v.token);
}
template <int DT, class P>
__device__ __forceinline__ P RowAt(const HeadsView &v, int b, int head, int token) {
  return (P)v.p +
         (static_cast<std::int64_t>(b) * v.batch + static_cast<std::int64_t>(head) * v.head) +
         Tokens(v, token);
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
__device__ __forceinline__ float OfHalf(int dtype, std::uint16_t v) {
  return dtype == DT_BF16 ? Elem<DT_BF16>::One(v) : Elem<DT_F16>::One(v);
}
// How a bias is read: not at all, in vectors of eight of 16 or of 32 bits a value,
// or (rows of less than eight keys) value by value.  A vector that would reach
// behind its row is the one that ends there, moved down: value by value, bf16 heads
// of 64 with a bias, 4 x 16 over 1001 tokens, took 168 us forward and 612 backward,
// so 71 and 247.
enum : int { kNoBias, kHalves, kVectors, kValues };
// The values from number `skip` (below 8) on, any behind them.
__device__ __forceinline__ u32x4 MovedDown(u32x4 v, int skip) {
  std::uint64_t low = v[0] | static_cast<std::uint64_t>(v[1]) << 32,
                high = v[2] | static_cast<std::uint64_t>(v[3]) << 32;
  if (skip & 4)
    low = high;
  const int bits = 16 * (skip & 3);
  if (bits) {
    low = low >> bits | high << (64 - bits);
    high >>= bits;
  }
  return u32x4{static_cast<std::uint32_t>(low), static_cast<std::uint32_t>(low >> 32),
               static_cast<std::uint32_t>(high), static_cast<std::uint32_t>(high >> 32)};
}
__device__ __forceinline__ u32x4 Halves8(const TrainAttention &a, std::int64_t row, int j) {
  const int from = min(j, a.k_len - 8), skip = min(j - from, 7);
  const u32x4 v = LoadVec<DT_BF16, false>((ConstRow<DT_BF16>)a.bias + row + from);
  return skip > 0 ? MovedDown(v, skip) : v;
}
// Eight consecutive values from key j on (any of the row's where there are less).
template <int BIAS>
__device__ __forceinline__ void Bias8(const TrainAttention &a, std::int64_t row, int j, f32x4 *f) {
  if constexpr (BIAS == kVectors) {
    const int from = min(j, a.k_len - 8), skip = min(j - from, 7);
    const auto *p = (ConstRow<DT_F32>)a.bias + row + from;
    f[0] = __builtin_bit_cast(f32x4, LoadVec<DT_F32, false>(p));
    f[1] = __builtin_bit_cast(f32x4, LoadVec<DT_F32, false>(p + 4));
    if (skip > 0) {
#pragma unroll
      for (int by = 4; by > 0; by /= 2)
        if (skip & by) {
#pragma unroll
          for (int e = 0; e + by < 8; ++e)
            f[e >> 2][e & 3] = f[(e + by) >> 2][(e + by) & 3];
        }
    }
  } else if constexpr (BIAS == kHalves) {
    const u32x4 v = Halves8(a, row, j);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      f[e >> 2][e & 3] =
          a.bias_dtype == DT_BF16 ? Elem<DT_BF16>::Get(v, e) : Elem<DT_F16>::Get(v, e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const std::int64_t at = row + min(j + e, a.k_len - 1);
      f[e >> 2][e & 3] = a.bias_dtype == DT_F32
                             ? ((const MFH_GLOBAL float *)a.bias)[at]
                             : OfHalf(a.bias_dtype, ((const MFH_GLOBAL std::uint16_t *)a.bias)[at]);
    }
  }
}
template <int BIAS, int DT>
__device__ __forceinline__ void Store8(Row<DT> p, int n, const f32x4 *f) {
  if (BIAS != kValues && n >= 8) {
    ToMemory<DT>(p, f[0], f[1]);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n)
      p[e] = Elem<DT>::Round(f[e >> 2][e & 3]);
}
// The gradient of as many as there are.
template <int BIAS>
__device__ __forceinline__ void StoreBias8(const TrainAttention &a, std::int64_t row, int j,
                                           const f32x4 *f) {
  const int n = a.k_len - j;
  if (n <= 0)
    return;
  if (BIAS == kVectors || (BIAS == kValues && a.bias_dtype == DT_F32))
    Store8<BIAS, DT_F32>((Row<DT_F32>)a.dbias + row + j, n, f);
  else if (a.bias_dtype == DT_BF16)
    Store8<BIAS, DT_BF16>((Row<DT_BF16>)a.dbias + row + j, n, f);
  else
    Store8<BIAS, DT_F16>((Row<DT_F16>)a.dbias + row + j, n, f);
}

// kTile rows of a view as a row-major tile in LDS, 256 threads: chunk i of a
// thread is eight values of row RowIn(i).
template <int DT, int DP> struct Stage {
  static constexpr int kChunks = kTile * DP / 8 / 256, kAcross = DP / 8;
  typename Mat<DT>::Frag f[kChunks];
  static __device__ __forceinline__ int RowIn(int i) { return (i * 256 + threadIdx.x) / kAcross; }
  static __device__ __forceinline__ int At(int i) { return (i * 256 + threadIdx.x) % kAcross * 8; }
  __device__ __forceinline__ void Store(typename Mat<DT>::T *tile) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      ToRow<DT>(tile + RowIn(i) * kLd<DT, DP> + At(i), f[i]);
  }
  // Keys first .. of a line: zeros from its end on.
  __device__ __forceinline__ void Keys(const HeadsView &v, const Line &l, int first, int dim) {
    const ConstRow<DT> base = In<DT>(v, l.b, l.kv, 0);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int j = first + RowIn(i);
      f[i] = typename Mat<DT>::Frag{};
      if (j < l.k_len && At(i) < dim)
        f[i] = FromMemory<DT>(base + Tokens(v, j) + At(i));
    }
  }
  // Less the products of each row with another's: lanes beside each other hold a row.
  __device__ __forceinline__ void StoreDots(const Stage &with, float *dots) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float v = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v += Mat<DT>::Get(f[i], e) * Mat<DT>::Get(with.f[i], e);
      v += Dpp<0xB1, 0xF>(0.f, v);  // its neighbour's, the pair's, the four's, the eight's
      v += Dpp<0x4E, 0xF>(0.f, v);
      if constexpr (kAcross >= 8)
        v += Dpp<0x141, 0xF>(0.f, v);
      if constexpr (kAcross >= 16)
        v += Dpp<0x140, 0xF>(0.f, v);
      if (At(i) == 0)
        dots[RowIn(i)] = -v;
    }
  }
  // Rows first .. of a line: zeros where a row sees nothing.
  __device__ __forceinline__ void Rows(const Args &s, const HeadsView &v, const Line &l,
                                       const Span64 &t, int first) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      int h = t.h, q = t.q + RowIn(i);
      f[i] = typename Mat<DT>::Frag{};
      if (!t.same) {
        const int r = first + RowIn(i);
        h = r / s.a.q_len;
        q = h < s.a.group ? r - h * s.a.q_len : s.a.q_len;
      }
      if (l.Last(q) >= 0 && At(i) < s.a.dim)
        f[i] = FromMemory<DT>(In<DT>(v, l.b, l.kv * s.a.group + h, q) + At(i));
    }
  }
};

// A bias of 16-bit values beside kTile rows and ACROSS keys in LDS, in whole
// vectors (kHalves); rows that are not the line's and keys behind its end hold
// anything.
template <int ACROSS> struct BiasStage {
  static constexpr int kLd = ACROSS + 8, kChunks = kTile * ACROSS / 8 / 256;
  u32x4 f[kChunks];
  static __device__ __forceinline__ int RowIn(int i) {
    return (i * 256 + static_cast<int>(threadIdx.x)) / (ACROSS / 8);
  }
  static __device__ __forceinline__ int At(int i) {
    return (i * 256 + static_cast<int>(threadIdx.x)) % (ACROSS / 8) * 8;
  }
  __device__ __forceinline__ void Load(const Args &s, const Line &l, const Span64 &t, int first,
                                       int key0) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      int h = t.h, q = t.q + RowIn(i);
      if (!t.same) {
        const int r = first + RowIn(i);
        h = r / s.a.q_len;
        q = h < s.a.group ? r - h * s.a.q_len : s.a.q_len;
      }
      f[i] = u32x4{0, 0, 0, 0};
      if (q < s.a.q_len && key0 + At(i) < s.a.k_len)
        f[i] = Halves8(s.a, BiasAt(s.a, l.b, l.kv * s.a.group + h, q), key0 + At(i));
    }
  }
  __device__ __forceinline__ void Store(std::uint16_t *tile) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      *reinterpret_cast<u32x4 *>(tile + RowIn(i) * kLd + At(i)) = f[i];
  }
  // Four rows from `row` on of the key col0 + lane % 16.
  static __device__ __forceinline__ f32x4 Four(const std::uint16_t *tile, int row, int col0, int lane,
                                               int dtype) {
    const int fr = lane & 15;
    typedef __attribute__((address_space(3))) s16x4 *Lds;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (Lds)(tile + (row + (fr >> 2)) * kLd + col0 + 4 * (fr & 3)));
    f32x4 f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      f[e] = OfHalf(dtype, static_cast<std::uint16_t>(x[e]));
    return f;
  }
};

// Products of a tile of 64 rows in LDS with N times 16 columns of a wave (ADD:
// added to `out`): lane l has column l % 16 of each, rows RowOf64.
template <int DT, int DP, int N, bool ADD>
__device__ __forceinline__ void Products(const typename Mat<DT>::T *tile,
                                         const typename Mat<DT>::Frag (*cols)[DP / 32], int lane,
                                         f32x4 (*out)[4]) {
  const int fr = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      const typename Mat<DT>::Frag f =
          FromRow<DT>(tile + RowOf64(t, fr) * kLd<DT, DP> + 32 * c + 8 * g);
#pragma unroll
      for (int n = 0; n < N; ++n)
        out[n][t] =
            Mat<DT>::Mul(f, cols[n][c], ADD || c > 0 ? out[n][t] : f32x4{0.f, 0.f, 0.f, 0.f});
    }
}
__device__ __forceinline__ void Fill(f32x4 *v, int n, float f) {
#pragma unroll
  for (int i = 0; i < n; ++i)
    v[i] = f32x4{f, f, f, f};
}

// A row of a workgroup's tile as a lane has it.
struct RowOfWave {
  int r, q, head, last;
  bool live;
};
__device__ __forceinline__ RowOfWave RowFor(const Args &s, const Line &l, int r) {
  RowOfWave w;
  w.r = r;
  w.live = r < s.rows;
  int h = 0;
  w.q = w.live ? r : 0;
  if (s.a.group > 1) {
    h = w.live ? r / s.a.q_len : 0;
    w.q = w.live ? r - h * s.a.q_len : 0;
  }
  w.head = l.kv * s.a.group + h;
  w.last = w.live ? l.Last(w.q) : -1;
  return w;
}
template <int DT, int DP>
__device__ __forceinline__ void LoadRow(const Args &s, const HeadsView &v, const Line &l,
                                        const RowOfWave &w, int lane, typename Mat<DT>::Frag *f) {
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
    f[c] = typename Mat<DT>::Frag{};
  if (w.last < 0)
    return;
  const int d0 = 8 * (lane >> 4);
  const ConstRow<DT> row = In<DT>(v, l.b, s.a.group == 1 ? l.kv : w.head, w.q) + d0;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
    if (32 * c + d0 < s.a.dim)
      f[c] = FromMemory<DT>(row + 32 * c);
}
// The same of a key.
template <int DT, int DP>
__device__ __forceinline__ void LoadKey(const Args &s, const HeadsView &v, const Line &l, int j,
                                        int lane, typename Mat<DT>::Frag *f) {
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
    f[c] = typename Mat<DT>::Frag{};
  if (j >= l.k_len)
    return;
  const int d0 = 8 * (lane >> 4);
  const ConstRow<DT> row = In<DT>(v, l.b, l.kv, j) + d0;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
    if (32 * c + d0 < s.a.dim)
      f[c] = FromMemory<DT>(row + 32 * c);
}

// Scores less `off`, whatever is not seen at -inf, from products.  Without a
// bias in units of ln 2, ready for the exponential; a bias of the type's lowest value
// would overflow in those, so with one they are natural and the differences are
// multiplied (Exp).
template <int BIAS> __device__ __forceinline__ float Exp(float x) {
  return Exp2(BIAS ? x * kLog2e : x);
}
template <int BIAS>
__device__ __forceinline__ void ToScores(const TrainAttention &a, std::int64_t bias_at, int j0,
                                         int last, float off, f32x4 *x) {
  if constexpr (BIAS != kNoBias) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4 bias[2];
      Bias8<BIAS>(a, bias_at, j0 + 32 * u, bias);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[2 * u + (e >> 2)][e & 3] =
            (x[2 * u + (e >> 2)][e & 3] * a.scale + bias[e >> 2][e & 3]) - off;
    }
  } else {
    const float scale = a.scale * kLog2e;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[t][e] = x[t][e] * scale - off;
  }
  if (j0 + 39 > last) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j0 + 32 * (t >> 1) + 4 * (t & 1) + e > last)
          x[t][e] = -__builtin_inff();
  }
}

// Waves a SIMD that registers have to allow.
template <int DT, int DP> constexpr int kWaves = DT == DT_F32 && DP == 128 ? 1 : 2;

// The forward pass: a wave has N sets of 16 rows and goes over tiles of 64 keys with
// the running maximum and sum of its rows; out is scaled once at the end.  ONE: all
// keys in one tile.  Squares are bound by memory (256 x 32 heads of 64 x 64 x 32, bf16
// with a bias 43.7 us, 4.7 TB/s), long lines by LDS reads, exponentials and matrix
// instructions together (4 x 32 x 2048 x 64 bf16 202 us, 681 TFLOP/s; causal 4 x 16 66,
// 519; fp32, where products reach 154 TFLOP/s, 2 x 16 causal 184, 93).
template <int DT, int DP, int N, int BIAS, bool ONE>
__global__ __launch_bounds__(256, (kWaves<DT, DP>)) void ForwardKernel(Args s) {
  using M = Mat<DT>;
  constexpr int LD = kLd<DT, DP>;
  __shared__ __attribute__((aligned(16))) typename M::T ks[kTile * LD], vs[kTile * LD];
  Part part;
  if (!PartOf(s, &part))
    return;
  const TrainAttention &a = s.a;
  const Line l = LineOf(s, part.line);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int first = part.tile * kTile * N;
  const int seen = KeysSeen(l, SpanOf(s, first, kTile * N), kTile * N);
  const int per = ONE ? 1 : (s.steps + s.splits - 1) / s.splits;
  const int begin = ONE ? 0 : part.split * per, end = min(begin + per, (seen + kTile - 1) / kTile);
  Stage<DT, DP> kt, vt;
  if (begin < end) {
    kt.Keys(a.k, l, begin * kTile, a.dim);
    vt.Keys(a.v, l, begin * kTile, a.dim);
  }
  RowOfWave w[N];
  typename M::Frag qf[N][DP / 32];
  std::int64_t bias_at[N];
  f32x4 acc[N][DP / 16];
  float most[N], total[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    w[n] = RowFor(s, l, first + 16 * (N * wave + n) + fr);
    LoadRow<DT, DP>(s, a.q, l, w[n], lane, qf[n]);
    bias_at[n] = BIAS ? BiasAt(a, l.b, w[n].head, w[n].q) : 0;
    Fill(acc[n], DP / 16, 0.f);
    most[n] = -__builtin_inff();
    total[n] = 0.f;
  }
  for (int step = begin; step < end; ++step) {
    kt.Store(ks);
    vt.Store(vs);
    __syncthreads();
    if (!ONE && step + 1 < end) {
      kt.Keys(a.k, l, (step + 1) * kTile, a.dim);
      vt.Keys(a.v, l, (step + 1) * kTile, a.dim);
    }
    f32x4 x[N][4];
    Products<DT, DP, N, false>(ks, qf, lane, x);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      ToScores<BIAS>(a, bias_at[n], step * kTile + 8 * g, w[n].last, 0.f, x[n]);
      float top = most[n];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top = fmaxf(top, x[n][t][e]);
      top = OverRows(top, true);
      const float base = top == -__builtin_inff() ? 0.f : top;
      const float old = Exp<BIAS>(most[n] - base);
      most[n] = top;
      total[n] *= old;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[n][t][e] = Exp<BIAS>(x[n][t][e] - base);
          total[n] += x[n][t][e];
        }
      if constexpr (!ONE) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
          acc[n][i] *= old;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      typename M::Frag p[N];
#pragma unroll
      for (int n = 0; n < N; ++n)
        p[n] = M::Pack(x[n][2 * u], x[n][2 * u + 1]);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const typename M::Frag v = HeadColumns<DT, DP, LD>(vs, 32 * u, i, lane);
#pragma unroll
        for (int n = 0; n < N; ++n)
          acc[n][i] = M::Mul(v, p[n], acc[n][i]);
      }
    }
    if constexpr (!ONE)
      __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    total[n] = OverRows(total[n], false);
    if (!w[n].live)
      continue;
    const std::int64_t flat = static_cast<std::int64_t>(part.line) * s.rows + w[n].r;
    // Natural units from here on.
    most[n] *= BIAS ? 1.f : kLn2;
    if (!ONE && s.splits > 1) {
      const std::int64_t all = static_cast<std::int64_t>(s.lines) * s.rows;
      StorePartial<DP>(s.partials + (part.split * all + flat) * s.a.dim, lane, s.a.dim, acc[n]);
      if (g == 0) {
        float *st = s.partials + s.splits * all * s.a.dim + (part.split * all + flat) * 2;
        st[0] = most[n];
        st[1] = total[n];
      }
      continue;
    }
    // A row that sees nothing has 0 times every value, which may be infinite.
    if (total[n] == 0.f)
      Fill(acc[n], DP / 16, 0.f);
    StoreHead<DT, DP>(Out<DT>(a.out, l.b, w[n].head, w[n].q), lane, a.dim, acc[n],
                      total[n] == 0.f ? 0.f : 1.f / total[n]);
    if (a.lse && g == 0)
      a.lse[flat] = total[n] == 0.f ? -__builtin_inff()
                                    : most[n] + kLn2 * __builtin_amdgcn_logf(total[n]);
  }
}

constexpr int kMostSplits = 256;
constexpr int kFewSplits = 8;

// Joins up to kFewSplits splits of a forward pass: four elements a thread, each
// of which forms its row's weights.
template <int DT>
__global__ __launch_bounds__(256) void JoinFewKernel(Args s) {
  const std::int64_t n = static_cast<std::int64_t>(s.lines) * s.rows;
  const std::int64_t id = static_cast<std::int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int across = s.a.dim / 4;
  const std::int64_t flat = id / across;
  const int c = static_cast<int>(id % across);
  if (flat >= n)
    return;
  const float *st = s.partials + s.splits * n * s.a.dim;
  f32x4 v[kFewSplits];
  float most[kFewSplits], total[kFewSplits], top = -__builtin_inff();
#pragma unroll
  for (int k = 0; k < kFewSplits; ++k) {
    const int i = min(k, s.splits - 1);
    most[k] = st[(i * n + flat) * 2];
    total[k] = st[(i * n + flat) * 2 + 1];
    v[k] = *reinterpret_cast<const f32x4 *>(s.partials + (i * n + flat) * s.a.dim + 4 * c);
    top = fmaxf(top, most[k]);
  }
  const float base = top == -__builtin_inff() ? 0.f : top;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kFewSplits; ++k)
    if (k < s.splits) {
      const float w = Exp2((most[k] - base) * kLog2e);
      sum += total[k] * w;
      o += v[k] * w;
    }
  const int line = static_cast<int>(flat / s.rows), r = static_cast<int>(flat % s.rows);
  const int b = line / s.a.kv_heads, head = line % s.a.kv_heads * s.a.group + r / s.a.q_len;
  ToMemory<DT>(Out<DT>(s.a.out, b, head, r % s.a.q_len) + 4 * c,
               sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o * (1.f / sum));
  if (s.a.lse && c == 0)
    s.a.lse[flat] = sum == 0.f ? -__builtin_inff() : top + kLn2 * __builtin_amdgcn_logf(sum);
}

// Joins the splits of a forward pass: a workgroup a row.  All lanes form the
// splits' weights, then groups of lanes that hold a row add every so many splits.
template <int DT>
__global__ __launch_bounds__(256) void JoinForwardKernel(Args s) {
  __shared__ float red[2][4], weight[kMostSplits];
  __shared__ f32x4 sums[256];
  const std::int64_t n = static_cast<std::int64_t>(s.lines) * s.rows, flat = blockIdx.x;
  const float *st = s.partials + s.splits * n * s.a.dim;
  const int k = threadIdx.x;
  float most = -__builtin_inff(), total = 0.f;
  if (k < s.splits) {
    most = st[(k * n + flat) * 2];
    total = st[(k * n + flat) * 2 + 1];
  }
  const float mine = most;
  most = WaveMax(most);
  if ((k & 63) == 0)
    red[0][k >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float base = most == -__builtin_inff() ? 0.f : most;
  const float w = Exp2((mine - base) * kLog2e);
  weight[k] = w;
  total = WaveSum(total * w);
  if ((k & 63) == 0)
    red[1][k >> 6] = total;
  __syncthreads();
  total = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int across = s.a.dim / 4, groups = 256 / across, group = k / across, c = k % across;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  if (group < groups) {
#pragma unroll 4
    for (int i = group; i < s.splits; i += groups) {
      // A split that saw nothing holds zeros.
      const f32x4 v = *reinterpret_cast<const f32x4 *>(s.partials + (i * n + flat) * s.a.dim + 4 * c);
      o += v * weight[i];
    }
  }
  sums[k] = o;
  __syncthreads();
  if (k >= across)
    return;
  for (int i = 1; i < groups; ++i)
    o += sums[i * across + k];
  const int line = static_cast<int>(flat / s.rows), r = static_cast<int>(flat % s.rows);
  const int b = line / s.a.kv_heads, head = line % s.a.kv_heads * s.a.group + r / s.a.q_len;
  ToMemory<DT>(Out<DT>(s.a.out, b, head, r % s.a.q_len) + 4 * k,
               total == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o * (1.f / total));
  if (s.a.lse && k == 0)
    s.a.lse[flat] = total == 0.f ? -__builtin_inff() : most + kLn2 * __builtin_amdgcn_logf(total);
}

// A row's log-sum-exp in the units of its scores, as what they are taken off:
// +inf where it sees nothing, so that every probability is 0.
template <int BIAS> __device__ __forceinline__ float Lse(float v) {
  if (v == -__builtin_inff())
    return __builtin_inff();
  return BIAS ? v : v * kLog2e;
}
// Such a row's gradients are stored as 0: 0 times a key or value that is not finite
// is not.
__device__ __forceinline__ bool SeesNothing(float lse) { return lse == __builtin_inff(); }
// A row's probabilities from a bias as large as this are too coarse by its
// log-sum-exp alone: ln(sum) is below a rounding of it, and where a mask of the
// type's lowest value takes every key, each would have probability 1.  Such rows
// are divided by their own sum: the exponent of 2 gets `rest` = -log2 of that
// added, 0 in all others.
__device__ __forceinline__ bool Coarse(float lse) {
  return fabsf(lse) > 256.f && fabsf(lse) < __builtin_inff();
}
template <int BIAS> __device__ __forceinline__ float Probability(float x, float rest) {
  return Exp2(BIAS ? __builtin_fmaf(x, kLog2e, rest) : x);
}
// delta = dout . out of a row, over the four lanes that share it.
template <int DT, int DP>
__device__ __forceinline__ float Delta(const typename Mat<DT>::Frag *out,
                                       const typename Mat<DT>::Frag *dout) {
  float delta = 0.f;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      delta += Mat<DT>::Get(out[c], e) * Mat<DT>::Get(dout[c], e);
  return OverRows(delta, false);
}

// delta of each row, then dq (and dbias) of a tile of rows over the keys: three
// products a step, and with the keys' kernel seven where five would do, but each sum
// stays in the registers of one wave.  4 x 32 x 2048 x 64 bf16 559 us for both (615
// TFLOP/s of the five).
template <int DT, int DP, int N, int BIAS>
__device__ __forceinline__ void BackwardRows(const Args &s, const Part &part,
                                             typename Mat<DT>::T *ks, typename Mat<DT>::T *vs) {
  using M = Mat<DT>;
  constexpr int LD = kLd<DT, DP>;
  const TrainAttention &a = s.a;
  const Line l = LineOf(s, part.line);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int first = part.tile * kTile * N;
  // Every element of the bias's gradient is written, so no key is left out.
  const int seen = a.dbias ? a.k_len : KeysSeen(l, SpanOf(s, first, kTile * N), kTile * N);
  const int per = (s.steps + s.splits - 1) / s.splits;
  const int begin = part.split * per, end = min(begin + per, (seen + kTile - 1) / kTile);
  Stage<DT, DP> kt, vt;
  if (begin < end && (a.dq.p || a.dbias)) {
    kt.Keys(a.k, l, begin * kTile, a.dim);
    vt.Keys(a.v, l, begin * kTile, a.dim);
  }
  RowOfWave w[N];
  typename M::Frag qf[N][DP / 32], df[N][DP / 32];
  float delta[N], lse[N], rest[N];
  std::int64_t bias_at[N];
  f32x4 acc[N][DP / 16];
  bool coarse = false;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    w[n] = RowFor(s, l, first + 16 * (N * wave + n) + fr);
    const std::int64_t flat = static_cast<std::int64_t>(part.line) * s.rows + w[n].r;
    LoadRow<DT, DP>(s, a.q, l, w[n], lane, qf[n]);
    LoadRow<DT, DP>(s, a.dout, l, w[n], lane, df[n]);
    typename M::Frag of[DP / 32];
    LoadRow<DT, DP>(s, a.out, l, w[n], lane, of);
    delta[n] = Delta<DT, DP>(of, df[n]);
    if (s.delta && w[n].live && g == 0 && part.split == 0)
      s.delta[flat] = delta[n];
    lse[n] = w[n].last >= 0 ? Lse<BIAS>(a.lse[flat]) : __builtin_inff();
    rest[n] = 0.f;
    coarse = coarse || Coarse(lse[n]);
    bias_at[n] = BIAS ? BiasAt(a, l.b, w[n].head, w[n].q) : 0;
    Fill(acc[n], DP / 16, 0.f);
  }
  if constexpr (BIAS != kNoBias) {
    if (__syncthreads_or(coarse)) {
      // Rare: all keys once more beforehand, for their sum.
      float sum[N] = {};
      for (int step = 0; step < s.steps; ++step) {
        kt.Keys(a.k, l, step * kTile, a.dim);
        __syncthreads();
        kt.Store(ks);
        __syncthreads();
        f32x4 x[N][4];
        Products<DT, DP, N, false>(ks, qf, lane, x);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          ToScores<BIAS>(a, bias_at[n], step * kTile + 8 * g, w[n].last, lse[n], x[n]);
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sum[n] += Exp<BIAS>(x[n][t][e]);
        }
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float all = OverRows(sum[n], false);
        rest[n] = Coarse(lse[n]) ? -__builtin_amdgcn_logf(all) : 0.f;
      }
      __syncthreads();
      if (begin < end)
        kt.Keys(a.k, l, begin * kTile, a.dim);
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (w[n].live && g == 0 && part.split == 0)
        s.rest[static_cast<std::int64_t>(part.line) * s.rows + w[n].r] = rest[n];
  }
  if (!a.dq.p && !a.dbias)
    return;
  for (int step = begin; step < end; ++step) {
    kt.Store(ks);
    vt.Store(vs);
    __syncthreads();
    if (step + 1 < end) {
      kt.Keys(a.k, l, (step + 1) * kTile, a.dim);
      vt.Keys(a.v, l, (step + 1) * kTile, a.dim);
    }
    f32x4 x[N][4], dp[N][4];
#pragma unroll
    for (int n = 0; n < N; ++n)
      Fill(dp[n], 4, -delta[n]);
    Products<DT, DP, N, false>(ks, qf, lane, x);
    Products<DT, DP, N, true>(vs, df, lane, dp);
    const int j0 = step * kTile + 8 * g;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      ToScores<BIAS>(a, bias_at[n], j0, w[n].last, lse[n], x[n]);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[n][t][e] = Probability<BIAS>(x[n][t][e], rest[n]) * dp[n][t][e];
      if (BIAS && a.dbias && w[n].live) {
        if (SeesNothing(lse[n]))
          Fill(x[n], 4, 0.f);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          StoreBias8<BIAS>(a, bias_at[n], j0 + 32 * u, x[n] + 2 * u);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      typename M::Frag ds[N];
#pragma unroll
      for (int n = 0; n < N; ++n)
        ds[n] = M::Pack(x[n][2 * u], x[n][2 * u + 1]);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const typename M::Frag k = HeadColumns<DT, DP, LD>(ks, 32 * u, i, lane);
#pragma unroll
        for (int n = 0; n < N; ++n)
          acc[n][i] = M::Mul(k, ds[n], acc[n][i]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!w[n].live || !a.dq.p)
      continue;
    if (SeesNothing(lse[n]))
      Fill(acc[n], DP / 16, 0.f);
    if (s.splits > 1) {
      if (w[n].last < 0)
        continue;
      const std::int64_t all = static_cast<std::int64_t>(s.lines) * s.rows,
                         flat = static_cast<std::int64_t>(part.line) * s.rows + w[n].r;
      StorePartial<DP>(s.partials + (part.split * all + flat) * s.a.dim, lane, s.a.dim, acc[n]);
    } else {
      StoreHead<DT, DP>(Out<DT>(a.dq, l.b, w[n].head, w[n].q), lane, a.dim, acc[n], a.scale);
    }
  }
}

template <int DT, int DP, int N, int BIAS>
__global__ __launch_bounds__(256, (kWaves<DT, DP>)) void BackwardRowsKernel(Args s) {
  __shared__ __attribute__((aligned(16))) typename Mat<DT>::T tiles[2][kTile * kLd<DT, DP>];
  Part part;
  if (PartOf(s, &part))
    BackwardRows<DT, DP, N, BIAS>(s, part, tiles[0], tiles[1]);
}

// What a workgroup of the keys' kernel holds of its 64 rows, next to the tiles.
struct RowInfo {
  __attribute__((aligned(16))) int last[kTile];
  __attribute__((aligned(16))) float lse[kTile], delta[kTile], rest[kTile];  // delta negated
  std::int64_t bias[kTile];
};

// dk and dv of a tile of keys over the rows that share them; each wave has N
// times 16 keys and holds them, and rows go through LDS.  Bound by LDS: a step of 64
// rows of 64 elements reads 32 KB a wave, for 32 matrix instructions at N = 1 and 64 at
// N = 2 (four lines of up to 1021 tokens, 16 heads over 4: 38 us, with the rows' beside it
// 50).
template <int DT, int DP, int N, int BIAS, bool ALONE>
__device__ __forceinline__ void BackwardKeys(const Args &s, const Part &part,
                                             typename Mat<DT>::T *qs, typename Mat<DT>::T *dos,
                                             RowInfo &info, std::uint16_t *bs) {
  using M = Mat<DT>;
  constexpr int LD = kLd<DT, DP>;
  using Biases = BiasStage<kTile * N>;
  const TrainAttention &a = s.a;
  const Line l = LineOf(s, part.line);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int key0 = part.tile * kTile * N;
  int j[N];
  typename M::Frag kf[N][DP / 32], vf[N][DP / 32];
  f32x4 dk[N][DP / 16], dv[N][DP / 16];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    j[n] = key0 + 16 * (N * wave + n) + fr;
    LoadKey<DT, DP>(s, a.k, l, j[n], lane, kf[n]);
    LoadKey<DT, DP>(s, a.v, l, j[n], lane, vf[n]);
    Fill(dk[n], DP / 16, 0.f);
    Fill(dv[n], DP / 16, 0.f);
  }
  const float scale = BIAS ? a.scale : a.scale * kLog2e;
  const int per = (s.steps + s.splits - 1) / s.splits;
  const int end = min((part.split + 1) * per, s.steps);
  // The next tile from `step` on of which a row sees one of these keys.
  Span64 span{};
  const auto next = [&](int step) {
    for (; step < end; ++step) {
      span = SpanOf(s, step * kTile, kTile);
      if (KeysSeen(l, span, kTile) > key0)
        break;
    }
    return step;
  };
  Stage<DT, DP> qt, dt, ot;
  Biases bt;
  int my_last = -1;
  float my_lse = 0.f, my_delta = 0.f, my_rest = 0.f;
  std::int64_t my_bias = 0;
  bool all_see = false;
  const auto load = [&](int step) {
    qt.Rows(s, a.q, l, span, step * kTile);
    dt.Rows(s, a.dout, l, span, step * kTile);
    if constexpr (ALONE)
      ot.Rows(s, a.out, l, span, step * kTile);
    if constexpr (BIAS == kHalves)
      bt.Load(s, l, span, step * kTile, key0);
    all_see = span.same && span.q + kTile <= l.q_len && l.Last(span.q) >= key0 + kTile * N - 1;
    if (threadIdx.x < kTile) {
      const RowOfWave w = RowFor(s, l, step * kTile + threadIdx.x);
      const std::int64_t flat = static_cast<std::int64_t>(part.line) * s.rows + w.r;
      my_last = w.last;
      my_lse = __builtin_inff();
      my_delta = 0.f;
      if (w.last >= 0) {
        my_lse = Lse<BIAS>(a.lse[flat]);
        if constexpr (!ALONE)
          my_delta = -s.delta[flat];
        if constexpr (BIAS != kNoBias)
          my_rest = s.rest[flat];
      }
      my_bias = BIAS ? BiasAt(a, l.b, w.head, w.q) : 0;
    }
  };
  int step = next(part.split * per);
  if (step < end)
    load(step);
  while (step < end) {
    qt.Store(qs);
    dt.Store(dos);
    if constexpr (ALONE)
      dt.StoreDots(ot, info.delta);
    if constexpr (BIAS == kHalves)
      bt.Store(bs);
    if (threadIdx.x < kTile) {
      info.last[threadIdx.x] = my_last;
      info.lse[threadIdx.x] = my_lse;
      if constexpr (!ALONE)
        info.delta[threadIdx.x] = my_delta;
      info.rest[threadIdx.x] = my_rest;
      info.bias[threadIdx.x] = my_bias;
    }
    __syncthreads();
    const bool plain = all_see;
    step = next(step + 1);
    if (step < end)
      load(step);
    f32x4 x[N][4], dp[N][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      dp[0][t] = *reinterpret_cast<const f32x4 *>(info.delta + RowOf64(t, 4 * g));
#pragma unroll
      for (int n = 1; n < N; ++n)
        dp[n][t] = dp[0][t];
    }
    // All of the step's biases at once: rows apart, keys side by side in lanes.
    constexpr bool kEach = BIAS == kVectors || BIAS == kValues;
    f32x4 bias[kEach ? N : 1][4];
    if constexpr (kEach) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const std::int64_t at = info.bias[RowOf64(t, 4 * g + e)] + min(j[n], a.k_len - 1);
            bias[n][t][e] =
                BIAS == kVectors || a.bias_dtype == DT_F32
                    ? ((const MFH_GLOBAL float *)a.bias)[at]
                    : OfHalf(a.bias_dtype, ((const MFH_GLOBAL std::uint16_t *)a.bias)[at]);
          }
    }
    Products<DT, DP, N, false>(qs, kf, lane, x);
    Products<DT, DP, N, true>(dos, vf, lane, dp);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int at = RowOf64(t, 4 * g);
      const f32x4 lse = *reinterpret_cast<const f32x4 *>(info.lse + at);
      f32x4 rest{0.f, 0.f, 0.f, 0.f};
      if constexpr (BIAS != kNoBias)
        rest = *reinterpret_cast<const f32x4 *>(info.rest + at);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        f32x4 b{0.f, 0.f, 0.f, 0.f};
        if constexpr (kEach)
          b = bias[n][t];
        else if constexpr (BIAS == kHalves)
          b = Biases::Four(bs, at, 16 * (N * wave + n), lane, a.bias_dtype);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BIAS != kNoBias)
            x[n][t][e] = Probability<BIAS>(x[n][t][e] * scale + b[e] - lse[e], rest[e]);
          else
            x[n][t][e] = Exp2(x[n][t][e] * scale - lse[e]);
        }
      }
      if (!plain) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[n][t][e] = j[n] <= info.last[at + e] ? x[n][t][e] : 0.f;
      }
#pragma unroll
      for (int n = 0; n < N; ++n)
        dp[n][t] *= x[n][t];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      typename M::Frag p[N], ds[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        p[n] = M::Pack(x[n][2 * u], x[n][2 * u + 1]);
        ds[n] = M::Pack(dp[n][2 * u], dp[n][2 * u + 1]);
      }
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const typename M::Frag d = HeadColumns<DT, DP, LD>(dos, 32 * u, i, lane),
                               q = HeadColumns<DT, DP, LD>(qs, 32 * u, i, lane);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          dv[n][i] = M::Mul(d, p[n], dv[n][i]);
          dk[n][i] = M::Mul(q, ds[n], dk[n][i]);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (j[n] >= a.k_len)
      continue;
    if (s.splits > 1) {
      if (j[n] >= l.k_len)
        continue;  // zeros that the join knows of
      const std::int64_t all = static_cast<std::int64_t>(s.lines) * a.k_len,
                         flat = static_cast<std::int64_t>(part.line) * a.k_len + j[n];
      float *o = s.partials + (2 * part.split * all + flat) * s.a.dim;
      StorePartial<DP>(o, lane, s.a.dim, dk[n]);
      StorePartial<DP>(o + all * s.a.dim, lane, s.a.dim, dv[n]);
      continue;
    }
    if (j[n] >= l.k_len) {
      Fill(dk[n], DP / 16, 0.f);
      Fill(dv[n], DP / 16, 0.f);
    }
    if (a.dk.p)
      StoreHead<DT, DP>(Out<DT>(a.dk, l.b, l.kv, j[n]), lane, a.dim, dk[n], a.scale);
    if (a.dv.p)
      StoreHead<DT, DP>(Out<DT>(a.dv, l.b, l.kv, j[n]), lane, a.dim, dv[n], 1.f);
  }
}
template <int DT, int DP, int N, int BIAS>
__global__ __launch_bounds__(256, (kWaves<DT, DP>)) void BackwardKeysKernel(Args s) {
  __shared__ __attribute__((aligned(16))) typename Mat<DT>::T tiles[2][kTile * kLd<DT, DP>];
  __shared__ RowInfo info;
  // A bias of 16 bits goes through LDS too: read from memory value by value, a key a
  // lane, the backward pass of 4 x 16 bf16 heads of 64 over 1024 tokens took 295 us,
  // so 198.
  __shared__ __attribute__((aligned(16)))
  std::uint16_t bs[BIAS == kHalves ? kTile * BiasStage<kTile * N>::kLd : 1];
  Part part;
  if (PartOf(s, &part))
    BackwardKeys<DT, DP, N, BIAS, false>(s, part, tiles[0], tiles[1], info, bs);
}

// Both in one launch (BothAtOnce): the first key_groups workgroups have keys and
// form delta themselves from out, the others rows.
template <int DT, int DP>
__global__ __launch_bounds__(256, (kWaves<DT, DP>)) void BackwardBothKernel(Args rows, Args keys,
                                                                            int key_groups) {
  __shared__ __attribute__((aligned(16))) typename Mat<DT>::T tiles[2][kTile * kLd<DT, DP>];
  __shared__ RowInfo info;
  Part part;
  const int id = static_cast<int>(blockIdx.x);
  if (id < key_groups) {
    if (PartOf(keys, id % keys.across, keys.across, id / keys.across, &part))
      BackwardKeys<DT, DP, 1, kNoBias, true>(keys, part, tiles[0], tiles[1], info, nullptr);
  } else {
    const int at = id - key_groups;
    if (PartOf(rows, at % rows.across, rows.across, at / rows.across, &part))
      BackwardRows<DT, DP, 1, kNoBias>(rows, part, tiles[0], tiles[1]);
  }
}

// Adds up the splits of dq (KEYS false) or of dk and dv: four elements a thread.
// What no split holds is 0: keys behind a line's end, rows that see nothing.
template <int DT, bool KEYS>
__global__ __launch_bounds__(256) void JoinBackwardKernel(Args s) {
  const int per = KEYS ? s.a.k_len : s.rows, across = s.a.dim / 4;
  const std::int64_t n = static_cast<std::int64_t>(s.lines) * per;
  const std::int64_t all = KEYS ? 2 * n : n;
  const std::int64_t id = static_cast<std::int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const std::int64_t at = id / across;
  const int c = static_cast<int>(id % across);
  if (at >= all)
    return;
  const bool second = KEYS && at >= n;
  const std::int64_t flat = second ? at - n : at;
  const int line = static_cast<int>(flat / per), r = static_cast<int>(flat % per);
  const int b = line / s.a.kv_heads, kv = line % s.a.kv_heads;
  const Line l{b, kv, LengthOf(s.a.q_lengths, b, s.a.q_len), LengthOf(s.a.k_lengths, b, s.a.k_len),
               s.a.causal};
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  if (KEYS ? r < l.k_len : l.Last(r % s.a.q_len) >= 0) {
#pragma unroll 8
    for (int k = 0; k < s.splits; ++k)
      o += *reinterpret_cast<const f32x4 *>(s.partials + (k * all + at) * s.a.dim + 4 * c);
  }
  Row<DT> out;
  if constexpr (KEYS) {
    const HeadsView &v = second ? s.a.dv : s.a.dk;
    if (!v.p)
      return;
    out = Out<DT>(v, b, kv, r);
  } else {
    out = Out<DT>(s.a.dq, b, kv * s.a.group + r / s.a.q_len, r % s.a.q_len);
  }
  ToMemory<DT>(out + 4 * c, o * (second ? 1.f : s.a.scale));
}

// The whole backward pass of a head of up to 64 queries and 64 keys, none of
// them shared: one workgroup, each input read once.  Bound by the latency of memory,
// since a workgroup loads, waits, computes and stores once, with nothing of another
// head on its way: 256 x 32 heads of 32 elements, bf16 with a bias, 88.3 us (4.2 TB/s,
// the vector unit a third busy); 256 x 16 of 64 elements, whose rows are whole cache
// lines, 72.6 (4.2 too).  delta is the sum of p dp over
// the keys, which are all here: out is not read, and a query that sees one key has
// gradients of exactly 0.  A wave has 16 queries while
// scores, probabilities, dS and dq are formed, and 16 keys for dk and dv; P and
// then dS change hands through a tile of LDS that held V before (256 x 16 heads of
// 64 elements: 75 us; with tiles of their own, and so two workgroups a CU instead
// of four, 5 more).
template <int DT, int DP, int BIAS>
__global__ __launch_bounds__(256, 2) void SquareBackwardKernel(Args s) {
  using M = Mat<DT>;
  constexpr int LD = kLd<DT, DP>, LP = kLd<DT, kTile>;
  __shared__ __attribute__((aligned(16))) typename M::T ks[kTile * LD], qs[kTile * LD],
      dos[kTile * LD], ps[kTile * (LP > LD ? LP : LD)];
  typename M::T *vs = ps;  // until the products with V are done
  Part part;
  if (!PartOf(s, &part))
    return;
  const TrainAttention &a = s.a;
  const Line l = LineOf(s, part.line);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int mine = 16 * wave + fr;  // a query, and later a key
  const RowOfWave w = RowFor(s, l, mine);
  const std::int64_t flat = static_cast<std::int64_t>(part.line) * s.rows + mine;
  typename M::Frag qf[1][DP / 32], df[1][DP / 32];
  {
    typename M::Frag kf[DP / 32], vf[DP / 32];
    LoadKey<DT, DP>(s, a.k, l, mine, lane, kf);
    LoadRow<DT, DP>(s, a.q, l, w, lane, qf[0]);
    LoadKey<DT, DP>(s, a.v, l, mine, lane, vf);
    LoadRow<DT, DP>(s, a.dout, l, w, lane, df[0]);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      const int at = mine * LD + 32 * c + 8 * g;
      ToRow<DT>(ks + at, kf[c]);
      ToRow<DT>(qs + at, qf[0][c]);
      ToRow<DT>(vs + at, vf[c]);
      ToRow<DT>(dos + at, df[0][c]);
    }
  }
  const float lse = w.last >= 0 ? Lse<BIAS>(a.lse[flat]) : __builtin_inff();
  const std::int64_t bias_at = BIAS ? BiasAt(a, l.b, w.head, w.q) : 0;
  __syncthreads();
  f32x4 xs[1][4], dps[1][4], *x = xs[0], *dp = dps[0];
  Products<DT, DP, 1, false>(ks, qf, lane, xs);
  Products<DT, DP, 1, false>(vs, df, lane, dps);
  ToScores<BIAS>(a, bias_at, 8 * g, w.last, lse, x);
  // dp of the key that has more than half of the row, if one has: delta is summed
  // about it.
  float rest = 0.f, delta = 0.f, near = -__builtin_inff();
  if constexpr (BIAS != kNoBias) {
    if (__any(Coarse(lse))) {
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum += Exp<BIAS>(x[t][e]);
      sum = OverRows(sum, false);
      rest = Coarse(lse) ? -__builtin_amdgcn_logf(sum) : 0.f;
    }
    if (w.live && g == 0)
      s.rest[flat] = rest;
  }
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[t][e] = Probability<BIAS>(x[t][e], rest);
      near = x[t][e] > 0.5f ? dp[t][e] : near;
    }
  near = OverRows(near, true);
  near = near == -__builtin_inff() ? 0.f : near;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      delta += x[t][e] * (dp[t][e] - near);
  delta = near + OverRows(delta, false);
  if (w.live && g == 0)
    s.delta[flat] = delta;
#pragma unroll
  for (int t = 0; t < 4; ++t)
    dp[t] = (dp[t] - delta) * x[t];
  if (SeesNothing(lse))
    Fill(dp, 4, 0.f);
  if (BIAS && a.dbias && w.live) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      StoreBias8<BIAS>(a, bias_at, 8 * g + 32 * u, dp + 2 * u);
  }
  f32x4 acc[DP / 16];
  Fill(acc, DP / 16, 0.f);
  typename M::Frag ds[2];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    ds[u] = M::Pack(dp[2 * u], dp[2 * u + 1]);
    ToRow<DT>(ps + mine * LP + 32 * u + 8 * g, M::Pack(x[2 * u], x[2 * u + 1]));
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
      acc[i] = M::Mul(HeadColumns<DT, DP, LD>(ks, 32 * u, i, lane), ds[u], acc[i]);
  }
  if (SeesNothing(lse))
    Fill(acc, DP / 16, 0.f);
  if (w.live && a.dq.p)
    StoreHead<DT, DP>(Out<DT>(a.dq, l.b, w.head, w.q), lane, a.dim, acc, a.scale);
  if (!a.dk.p && !a.dv.p)
    return;
  // The wave's 16 keys' column sums of P and then of dS, each times a tile.
  const auto over_rows = [&](const typename M::T *tile, const HeadsView &out, float scale) {
    __syncthreads();
    Fill(acc, DP / 16, 0.f);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const typename M::Frag p = Columns<DT, LP>(ps, 32 * u, 4, 16 * wave, lane);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        acc[i] = M::Mul(HeadColumns<DT, DP, LD>(tile, 32 * u, i, lane), p, acc[i]);
    }
    if (mine >= l.k_len)
      Fill(acc, DP / 16, 0.f);
    if (mine < a.k_len && out.p)
      StoreHead<DT, DP>(Out<DT>(out, l.b, l.kv, mine), lane, a.dim, acc, scale);
  };
  over_rows(dos, a.dv, 1.f);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u)
    ToRow<DT>(ps + mine * LP + 32 * u + 8 * g, ds[u]);
  over_rows(qs, a.dk, a.scale);
}

// The gradient of a bias that lines or heads share: a workgroup has 64 queries
// and 64 keys of one of its planes and loops over what shares it, so a small plane
// that much shares leaves most of the card idle: 256 x 32 heads of 64 x 64 x 32, bf16,
// backward 741 us with a bias shared by the lines (32 workgroups of 256 rounds, 2.6 us
// each) and 17400 shared by the heads too (one of 8192); 88 with one of its own.
template <int DT, int DP, int BIAS>
__global__ __launch_bounds__(256) void BiasGradKernel(Args s, int plane_heads, std::int64_t first) {
  using M = Mat<DT>;
  const TrainAttention &a = s.a;
  const int k_tiles = (a.k_len + kTile - 1) / kTile, q_tiles = (a.q_len + kTile - 1) / kTile;
  const std::int64_t id = first + blockIdx.x;
  const int kt = static_cast<int>(id % k_tiles), qt = static_cast<int>(id / k_tiles % q_tiles);
  const int plane = static_cast<int>(id / k_tiles / q_tiles);
  const int b_plane = plane / plane_heads, h_plane = plane % plane_heads;
  const int b0 = a.bias_batch ? b_plane : 0, b1 = a.bias_batch ? b_plane + 1 : a.batch;
  const int h0 = a.bias_head ? h_plane : 0, h1 = a.bias_head ? h_plane + 1 : a.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, g = lane >> 4;
  const int q = qt * kTile + 16 * wave + fr, j0 = kt * kTile + 8 * g;
  const bool live = q < a.q_len;
  const std::int64_t bias_at = BiasAt(a, b_plane, h_plane, live ? q : 0);
  f32x4 acc[4], bias[4];
  Fill(acc, 4, 0.f);
  Fill(bias, 4, 0.f);
#pragma unroll
  for (int u = 0; u < 2; ++u)
    Bias8<BIAS>(a, bias_at, j0 + 32 * u, bias + 2 * u);
  for (int b = b0; b < b1; ++b)
    for (int head = h0; head < h1; ++head) {
      const int kv = head / a.group;
      const Line l = LineOf(s, b * a.kv_heads + kv);
      RowOfWave w{q, q, head, live ? l.Last(q) : -1, live};
      const std::int64_t flat = (static_cast<std::int64_t>(b) * a.heads + head) * a.q_len + q;
      typename M::Frag qf[DP / 32], df[DP / 32];
      LoadRow<DT, DP>(s, a.q, l, w, lane, qf);
      LoadRow<DT, DP>(s, a.dout, l, w, lane, df);
      const float lse = w.last >= 0 ? Lse<BIAS>(a.lse[flat]) : __builtin_inff();
      const float delta = w.last >= 0 ? s.delta[flat] : 0.f, rest = w.last >= 0 ? s.rest[flat] : 0.f;
      const int last = SeesNothing(lse) ? -1 : w.last;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 x{0.f, 0.f, 0.f, 0.f}, dp{-delta, -delta, -delta, -delta};
        const int key = kt * kTile + RowOf64(t, fr), j = kt * kTile + RowOf64(t, 4 * g);
        typename M::Frag kf[DP / 32], vf[DP / 32];
        LoadKey<DT, DP>(s, a.k, l, key, lane, kf);
        LoadKey<DT, DP>(s, a.v, l, key, lane, vf);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          x = M::Mul(kf[c], qf[c], x);
          dp = M::Mul(vf[c], df[c], dp);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = Probability<BIAS>(x[e] * a.scale + bias[t][e] - lse, rest);
          acc[t][e] += j + e <= last ? p * dp[e] : 0.f;
        }
      }
    }
  if (!live)
    return;
#pragma unroll
  for (int u = 0; u < 2; ++u)
    StoreBias8<BIAS>(a, bias_at, j0 + 32 * u, acc + 2 * u);
}

// Workgroups that fill the card twice, a split of two tiles at least; six times where
// each still loops over ten: causal bf16, 8 heads of 64 over 2048 tokens 24 us and
// backward 54.5 (four times, over sixteen: 27.5 and 56.8), 8 heads of 128 over 2 and 4000
// tokens 89 and 364 (107 and 381); some lines lose (8 x 4 over 1, up to 2000 tokens,
// backward 103 and 95).  Eight times, over eight, lost everywhere.
inline int SplitsOf(std::int64_t groups, int steps) {
  const std::int64_t g = std::max<std::int64_t>(groups, 1);
  const std::int64_t want = std::min<std::int64_t>(
      std::max<std::int64_t>(512 / g, std::min<std::int64_t>(1536 / g, steps / 10)), kMostSplits);
  return static_cast<int>(std::max<std::int64_t>(1, std::min<std::int64_t>(want, steps / 2)));
}
inline int Tiles(int n, int wide = 1) {
  return static_cast<int>((static_cast<std::int64_t>(n) + kTile * wide - 1) / (kTile * wide));
}

inline int HowBias(const TrainAttention &a) {
  if (!a.bias || a.k_len == 0)
    return kNoBias;
  if (a.k_len < 8)
    return kValues;
  return a.bias_dtype == DT_F32 ? kVectors : kHalves;
}

// Shapes of the launches, and the workspace that they share.
inline Args ArgsOf(const TrainAttention &a, bool keys) {
  Args s;
  s.a = a;
  s.lines = a.batch * a.kv_heads;
  s.rows = a.group * a.q_len;
  const int across = keys ? a.k_len : s.rows;
  // Two sets of columns a wave halve the reads of LDS per product, where enough
  // workgroups are left and registers hold them.  Keys with a bias gain from
  // fewer: bf16 heads of 64, 4 x 16 over 1024 tokens (512 workgroups) 198 us, with one
  // set 220; 2 x 8 (128) 73.9 and 73.1.
  const bool fits =
      (a.dim <= 32 || (a.dim <= 64 && a.dtype != DT_F32)) && HowBias(a) != kValues;
  const std::int64_t enough = keys && a.bias ? 512 : 1024;
  s.wide = fits && static_cast<std::int64_t>(s.lines) * Tiles(across, 2) >= enough ? 2 : 1;
  s.tiles = Tiles(across, s.wide);
  s.steps = keys ? Tiles(s.rows) : Tiles(a.k_len);
  s.splits = SplitsOf(static_cast<std::int64_t>(s.lines) * s.tiles, s.steps);
  if (!keys && a.causal)
    s.down = RunsDown(s.tiles, s.a.group);
  return s;
}
// Whether the bias is shared by lines or heads.
inline bool SharedBias(const TrainAttention &a) {
  return a.dbias && ((a.bias_batch == 0 && a.batch > 1) || (a.bias_head == 0 && a.heads > 1));
}
inline std::uint64_t DeltaBytes(const Args &s) {
  return (static_cast<std::uint64_t>(s.lines) * s.rows * 4 + 15) & ~std::uint64_t(15);
}
// delta, and with a bias `rest`.
inline std::uint64_t RowValuesBytes(const Args &s) { return DeltaBytes(s) * (s.a.bias ? 2 : 1); }
inline std::uint64_t ForwardBytes(const Args &s) {
  return s.splits == 1 ? 0
                       : static_cast<std::uint64_t>(s.splits) * s.lines * s.rows * (s.a.dim + 2) * 4;
}
inline std::uint64_t RowsBytes(const Args &s) {
  return s.splits == 1 ? 0 : static_cast<std::uint64_t>(s.splits) * s.lines * s.rows * s.a.dim * 4;
}
inline std::uint64_t KeysBytes(const Args &s) {
  return s.splits == 1
             ? 0
             : static_cast<std::uint64_t>(s.splits) * 2 * s.lines * s.a.k_len * s.a.dim * 4;
}

// A launch has less than 2^32 threads, and less than 2^16 workgroups along y;
// more work takes several.
constexpr std::int64_t kMostGroups = std::int64_t(1) << 23;
template <class K> hipError_t Run(K kernel, Args s, hipStream_t stream) {
  if (s.lines == 0 || s.tiles == 0)
    return hipSuccess;
  const bool ragged = s.a.q_lengths || s.a.k_lengths;
  if (s.splits > 1) {
    const std::int64_t parts = static_cast<std::int64_t>(s.lines) * s.tiles * s.splits;
    s.turn = ragged;
    s.spread = !ragged;
    s.lines_now = s.lines;
    s.down = 0;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((parts + 7) / 8 * 8)), dim3(256), 0, stream,
                       s);
    return hipGetLastError();
  }
  const std::int64_t tiles = PlacesDown(s.tiles, s.down);
  const std::int64_t most_tiles = std::min<std::int64_t>(tiles, 65535);
  const std::int64_t most_lines = std::max<std::int64_t>(8, kMostGroups / most_tiles / 8 * 8);
  hipError_t e = hipSuccess;
  for (std::int64_t line = 0; e == hipSuccess && line < s.lines; line += most_lines)
    for (std::int64_t tile = 0; e == hipSuccess && tile < tiles; tile += most_tiles) {
      s.line0 = static_cast<int>(line);
      s.lines_now = static_cast<int>(std::min<std::int64_t>(most_lines, s.lines - line));
      s.tile0 = static_cast<int>(tile);
      s.spread = s.lines_now >= 64;
      s.turn = ragged && !s.spread;
      const dim3 grid(s.spread ? (s.lines_now + 7) / 8 * 8 : s.lines_now,
                      static_cast<unsigned>(std::min<std::int64_t>(most_tiles, tiles - tile)));
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, s);
      e = hipGetLastError();
    }
  return e;
}
// A pass's workgroups as a part of one launch along x.
inline std::int64_t GroupsOf(Args *s) {
  const bool ragged = s->a.q_lengths || s->a.k_lengths;
  s->lines_now = s->lines;
  if (s->splits > 1) {
    s->turn = ragged;
    s->spread = !ragged;
    s->down = 0;
    s->across = (s->lines * s->tiles * s->splits + 7) / 8 * 8;
    return s->across;
  }
  s->spread = s->lines >= 64;
  s->turn = ragged && !s->spread;
  s->across = s->spread ? (s->lines + 7) / 8 * 8 : s->lines;
  return static_cast<std::int64_t>(s->across) * PlacesDown(s->tiles, s->down);
}
// Whether a backward pass does rows and keys in one launch: the one's last workgroups
// run beside the other's, and a launch is saved.  bf16, causal: 1 x 4 over 4096 tokens of
// 64 99 us, apart 120; four lines of up to 1021, 16 heads over 4, 57.8 and 64.4; 2 x 4 over
// 116 8.5 and 13.2.  Heads of 128 leave a SIMD two waves and gain less: 37 x 8 over 2, 66
// tokens (700 workgroups) 28 and 37, 2 x 16 over 2048 (2048) 221 and 214.  With a bias the
// keys need what the rows find out (Coarse).
inline bool BothAtOnce(const Args &rows, const Args &keys) {
  const std::int64_t most = rows.a.dim > 64 ? 1024 : 4096;
  return !rows.a.bias && rows.wide == 1 && keys.wide == 1 && rows.a.q_len > 0 && rows.a.k_len > 0 &&
         (static_cast<std::int64_t>(rows.tiles) * rows.splits +
          static_cast<std::int64_t>(keys.tiles) * keys.splits) * rows.lines <= most;
}
// Splits have few rows.
template <class K> hipError_t RunJoin(K kernel, const Args &s, std::int64_t groups, hipStream_t stream) {
  if (groups == 0)
    return hipSuccess;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, stream, s);
  return hipGetLastError();
}

// Where ArgsOf may ask for two sets of columns.
template <int DT, int DP> constexpr bool kTwo = DP == 32 || (DP == 64 && DT != DT_F32);

template <int DT, int DP, int BIAS>
hipError_t Forward(const TrainAttention &a, hipStream_t stream) {
  constexpr int kWide = kTwo<DT, DP> && BIAS != kValues ? 2 : 1;
  Args s = ArgsOf(a, false);
  s.partials = static_cast<float *>(a.workspace);
  hipError_t e;
  if (s.steps <= 1) {
    s.wide = 1;
    s.tiles = Tiles(s.rows);
    s.down = s.down ? RunsDown(s.tiles, a.group) : 0;
    e = Run(ForwardKernel<DT, DP, 1, BIAS, true>, s, stream);
  } else if (s.wide == 2) {
    e = Run(ForwardKernel<DT, DP, kWide, BIAS, false>, s, stream);
  } else {
    e = Run(ForwardKernel<DT, DP, 1, BIAS, false>, s, stream);
  }
  const std::int64_t rows = static_cast<std::int64_t>(s.lines) * s.rows;
  if (e == hipSuccess && s.splits > kFewSplits)
    e = RunJoin(JoinForwardKernel<DT>, s, rows, stream);
  else if (e == hipSuccess && s.splits > 1)
    e = RunJoin(JoinFewKernel<DT>, s, (rows * (a.dim / 4) + 255) / 256, stream);
  return e;
}

template <int DT, int DP, int BIAS>
hipError_t Backward(const TrainAttention &a, hipStream_t stream) {
  constexpr int kWide = kTwo<DT, DP> && BIAS != kValues ? 2 : 1;
  constexpr bool kSquare = DT != DT_F32 || DP < 128;  // four tiles in LDS, two workgroups a CU
  Args s = ArgsOf(a, false);
  s.delta = static_cast<float *>(a.workspace);
  s.rest = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + DeltaBytes(s));
  s.partials = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + RowValuesBytes(s));
  const bool shared = SharedBias(a);
  if (shared)
    s.a.dbias = nullptr;
  const bool square = kSquare && a.group == 1 && a.q_len <= kTile && a.k_len <= kTile && a.q_len > 0 &&
                      a.k_len > 0;
  const auto joins = [&](std::int64_t rows) { return (rows * (a.dim / 4) + 255) / 256; };
  hipError_t e = hipSuccess;
  if constexpr (kSquare) {
    if (square) {
      s.tiles = 1;
      e = Run(SquareBackwardKernel<DT, DP, BIAS>, s, stream);
    }
  }
  if constexpr (BIAS == kNoBias) {
    Args k = ArgsOf(a, true);
    if (!square && BothAtOnce(s, k) && (a.dk.p || a.dv.p)) {
      s.delta = nullptr;
      k.partials = s.partials + RowsBytes(s) / sizeof(float);
      // Whole rounds of the dies, so that the rows' workgroups begin on the first; what
      // is added is behind the last tile of keys.
      const std::int64_t key_groups = (GroupsOf(&k) + 7) / 8 * 8,
                         row_groups = a.dq.p ? GroupsOf(&s) : 0;
      hipLaunchKernelGGL((BackwardBothKernel<DT, DP>),
                         dim3(static_cast<unsigned>(key_groups + row_groups)), dim3(256), 0, stream, s,
                         k, static_cast<int>(key_groups));
      e = hipGetLastError();
      if (e == hipSuccess && s.splits > 1 && a.dq.p)
        e = RunJoin(JoinBackwardKernel<DT, false>, s,
                    joins(static_cast<std::int64_t>(s.lines) * s.rows), stream);
      if (e == hipSuccess && k.splits > 1)
        e = RunJoin(JoinBackwardKernel<DT, true>, k,
                    joins(2 * static_cast<std::int64_t>(k.lines) * a.k_len), stream);
      return e;
    }
  }
  if (!square)
    e = s.wide == 2 ? Run(BackwardRowsKernel<DT, DP, kWide, BIAS>, s, stream)
                    : Run(BackwardRowsKernel<DT, DP, 1, BIAS>, s, stream);
  if (e == hipSuccess && s.splits > 1 && a.dq.p)
    e = RunJoin(JoinBackwardKernel<DT, false>, s, joins(static_cast<std::int64_t>(s.lines) * s.rows),
                stream);
  if (e == hipSuccess && (a.dk.p || a.dv.p) && !square) {
    Args k = ArgsOf(a, true);
    k.delta = s.delta;
    k.rest = s.rest;
    k.partials = s.partials;
    e = k.wide == 2 ? Run(BackwardKeysKernel<DT, DP, kWide, BIAS>, k, stream)
                    : Run(BackwardKeysKernel<DT, DP, 1, BIAS>, k, stream);
    if (e == hipSuccess && k.splits > 1)
      e = RunJoin(JoinBackwardKernel<DT, true>, k,
                  joins(2 * static_cast<std::int64_t>(k.lines) * a.k_len), stream);
  }
  if constexpr (BIAS != kNoBias) {
    if (e == hipSuccess && shared) {
      s.a.dbias = a.dbias;
      const int planes_b = a.bias_batch ? a.batch : 1, planes_h = a.bias_head ? a.heads : 1;
      const std::int64_t work =
          static_cast<std::int64_t>(Tiles(a.q_len)) * Tiles(a.k_len) * planes_b * planes_h;
      for (std::int64_t first = 0; e == hipSuccess && first < work; first += kMostGroups) {
        const auto groups = static_cast<unsigned>(std::min(work - first, kMostGroups));
        hipLaunchKernelGGL((BiasGradKernel<DT, DP, BIAS>), dim3(groups), dim3(256), 0, stream, s,
                           planes_h, first);
        e = hipGetLastError();
      }
    }
  }
  return e;
}

template <int DT, int DP>
hipError_t ByBias(const TrainAttention &a, bool backward, hipStream_t stream) {
  const int how = HowBias(a);
  if (how == kNoBias)
    return backward ? Backward<DT, DP, kNoBias>(a, stream) : Forward<DT, DP, kNoBias>(a, stream);
  if (how == kHalves)
    return backward ? Backward<DT, DP, kHalves>(a, stream) : Forward<DT, DP, kHalves>(a, stream);
  if (how == kVectors)
    return backward ? Backward<DT, DP, kVectors>(a, stream) : Forward<DT, DP, kVectors>(a, stream);
  return backward ? Backward<DT, DP, kValues>(a, stream) : Forward<DT, DP, kValues>(a, stream);
}

// By head size: a tile's columns are padded to 32, 64 or 128.
template <int DT>
hipError_t ByDim(const TrainAttention &a, bool backward, hipStream_t stream) {
  if (a.dim <= 32)
    return ByBias<DT, 32>(a, backward, stream);
  return a.dim <= 64 ? ByBias<DT, 64>(a, backward, stream) : ByBias<DT, 128>(a, backward, stream);
}

// One source a type.
hipError_t AttentionF32(const TrainAttention &a, bool backward, hipStream_t stream);
hipError_t AttentionBf16(const TrainAttention &a, bool backward, hipStream_t stream);
hipError_t AttentionF16(const TrainAttention &a, bool backward, hipStream_t stream);

}  // namespace attend
}  // namespace mfh
