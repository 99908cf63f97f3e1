// Which bytes the arrays of a call hold, and whether two of them share any
// (host only; learn_api.cpp, train_api.cpp).
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <vector>

namespace mfh {

// `rows` rows of `row_bytes`, `stride` bytes from one to the next; one row for
// an array without gaps.  logits: of the logits' shape.
struct Span {
  const char *name;
  const void *p;
  std::int64_t rows, row_bytes, stride;
  bool written, logits;
};

inline std::uintptr_t Address(const void *p) { return reinterpret_cast<std::uintptr_t>(p); }

// Whether [begin, begin + bytes) shares a byte with a row of `s`.
inline bool Touches(const Span &s, std::uintptr_t begin, std::int64_t bytes) {
  if (s.rows <= 0 || s.row_bytes <= 0 || bytes <= 0)
    return false;
  const std::uintptr_t first = Address(s.p), size = static_cast<std::uintptr_t>(s.row_bytes),
                       stride = static_cast<std::uintptr_t>(s.stride),
                       end = begin + static_cast<std::uintptr_t>(bytes);
  if (end <= first)
    return false;
  // The last row that begins before `end` ends last of those that do.
  std::uintptr_t row = s.rows > 1 ? (end - 1 - first) / stride : 0;
  row = std::min(row, static_cast<std::uintptr_t>(s.rows - 1));
  return first + row * stride + size > begin;
}

// Whether two sets of `rows` rows of `row_bytes`, strides in bytes, share a
// byte in any other way than being the same rows.
inline bool RowsClash(const void *p, std::int64_t p_stride, const void *q, std::int64_t q_stride,
                      std::int64_t rows, std::int64_t row_bytes) {
  const std::uintptr_t a = Address(p), b = Address(q);
  if (a == b && (p_stride == q_stride || rows <= 1))
    return false;
  const std::uintptr_t a_end = a + (rows - 1) * p_stride + row_bytes,
                       b_end = b + (rows - 1) * q_stride + row_bytes;
  if (a_end <= b || b_end <= a)
    return false;
  if (p_stride != q_stride || rows <= 1)
    return true;
  // Equal strides: interleaved rows are apart if they are within one stride.
  const std::uintptr_t apart = (a > b ? a - b : b - a) % static_cast<std::uintptr_t>(p_stride);
  return apart < static_cast<std::uintptr_t>(row_bytes) ||
         static_cast<std::uintptr_t>(p_stride) - apart < static_cast<std::uintptr_t>(row_bytes);
}

// The first pair of arrays, one of them written, that share a byte: its places
// in `a` and `b`.  Arrays of the logits' shape are compared by RowsClash, since
// a gradient may be the logits; of two others, or one of each, at most one has
// gaps.
template <size_t N> bool FindOverlap(const Span (&spans)[N], size_t *a, size_t *b) {
  for (size_t i = 0; i < N; ++i)
    for (size_t j = 0; j < i; ++j) {
      const Span &x = spans[i], &y = spans[j];
      if (!x.p || !y.p || !(x.written || y.written) || (x.logits && y.logits))
        continue;
      const Span &rows = x.logits ? x : y, &flat = x.logits ? y : x;
      if (Touches(rows, Address(flat.p), flat.rows > 0 ? flat.row_bytes : 0)) {
        *a = x.written ? i : j;
        *b = x.written ? j : i;
        return true;
      }
    }
  return false;
}

// Byte ranges in order, those that meet joined.
struct ByteRange {
  std::uintptr_t begin, end;
};
inline std::vector<ByteRange> Joined(std::vector<ByteRange> ranges) {
  std::sort(ranges.begin(), ranges.end(),
            [](const ByteRange &x, const ByteRange &y) { return x.begin < y.begin; });
  std::vector<ByteRange> out;
  for (const ByteRange &r : ranges) {
    if (!out.empty() && r.begin <= out.back().end)
      out.back().end = std::max(out.back().end, r.end);
    else
      out.push_back(r);
  }
  return out;
}
inline bool Meets(const std::vector<ByteRange> &joined, const void *p, std::uint64_t bytes) {
  const std::uintptr_t begin = Address(p), end = begin + bytes;
  // The first range that ends behind `begin`.
  const auto it = std::upper_bound(joined.begin(), joined.end(), begin,
                                   [](std::uintptr_t v, const ByteRange &r) { return v < r.end; });
  return bytes > 0 && it != joined.end() && it->begin < end;
}

// An array of up to three dimensions of strided runs of `inner` bytes; strides
// in bytes, not negative.
struct Region {
  struct Dim {
    std::int64_t n, stride;
  };
  const char *name;
  const void *p;
  std::int64_t inner;
  bool written;
  Dim dims[3];
};
inline Region RegionOf(const char *name, const void *p, std::int64_t inner, bool written,
                       const std::vector<Region::Dim> &dims) {
  Region r{name, p, inner, written, {{1, 0}, {1, 0}, {1, 0}}};
  for (size_t i = 0; i < dims.size() && i < 3; ++i)
    r.dims[i] = dims[i];
  return r;
}
inline bool Empty(const Region &r) {
  return r.inner <= 0 || r.dims[0].n <= 0 || r.dims[1].n <= 0 || r.dims[2].n <= 0;
}
// Bytes from the first to behind the last, of the dimensions whose stride is
// no multiple of `s` (0: of all).
inline std::int64_t Reach(const Region &r, std::int64_t s) {
  std::int64_t n = r.inner;
  for (const Region::Dim &d : r.dims)
    if (d.n > 1 && (s == 0 || d.stride % s != 0))
      n += (d.n - 1) * d.stride;
  return n;
}

// Whether each dimension steps over all that the narrower ones reach: then no
// two runs share a byte.
inline bool Nested(const Region &r) {
  Region::Dim d[3] = {r.dims[0], r.dims[1], r.dims[2]};
  std::sort(d, d + 3, [](const Region::Dim &x, const Region::Dim &y) { return x.stride < y.stride; });
  std::int64_t reach = r.inner;
  for (const Region::Dim &x : d)
    if (x.n > 1) {
      if (x.stride < reach)
        return false;
      reach += (x.n - 1) * x.stride;
    }
  return true;
}

// Whether two arrays share no byte, as far as this can tell: they lie behind
// one another, or, with respect to one of their strides s, every other stride
// is a multiple of s or stays inside a part of s that the other array leaves
// free (columns of one array, say, or heads between heads).
inline bool Apart(const Region &x, const Region &y) {
  if (Empty(x) || Empty(y))
    return true;
  const std::uintptr_t a = Address(x.p), b = Address(y.p);
  if (a + static_cast<std::uintptr_t>(Reach(x, 0)) <= b ||
      b + static_cast<std::uintptr_t>(Reach(y, 0)) <= a)
    return true;
  for (const Region *r : {&x, &y})
    for (const Region::Dim &d : r->dims) {
      if (d.n <= 1 || d.stride <= 0)
        continue;
      const std::int64_t s = d.stride, wide = Reach(x, s), other = Reach(y, s);
      if (wide > s || other > s)
        continue;
      const auto us = static_cast<std::uintptr_t>(s);
      // From x's run on to y's, round the period.
      const auto gap = static_cast<std::int64_t>((b % us + us - a % us) % us);
      if (gap >= wide && gap + other <= s)
        return true;
    }
  return false;
}

}  // namespace mfh
