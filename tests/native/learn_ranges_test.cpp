// The overlap checks of the losses against sets of bytes, on random small
// layouts (no device).
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>

#include "learn_ranges.h"

using mfh::ByteRange;
using mfh::Span;

namespace {

std::set<std::uintptr_t> Bytes(const Span &s) {
  std::set<std::uintptr_t> out;
  for (std::int64_t r = 0; r < s.rows; ++r)
    for (std::int64_t b = 0; b < s.row_bytes; ++b)
      out.insert(mfh::Address(s.p) + static_cast<std::uintptr_t>(r * s.stride + b));
  return out;
}

bool Share(const std::set<std::uintptr_t> &a, const std::set<std::uintptr_t> &b) {
  for (const std::uintptr_t v : a)
    if (b.count(v))
      return true;
  return false;
}

void Need(bool ok, const char *what, int trial) {
  if (ok)
    return;
  std::printf("%s differs in trial %d\n", what, trial);
  std::exit(1);
}

}  // namespace

int main() {
  std::mt19937 rng(1);
  const auto pick = [&](int low, int high) {
    return std::uniform_int_distribution<int>(low, high)(rng);
  };
  const auto at = [&](int low, int high) {
    return reinterpret_cast<const void *>(static_cast<std::uintptr_t>(1000 + pick(low, high)));
  };
  for (int trial = 0; trial < 200000; ++trial) {
    const std::int64_t bytes = pick(1, 6), stride = bytes + pick(0, 8), rows = pick(0, 5);
    const Span grad{"grad", at(0, 60), rows, bytes, stride, true, true};
    const Span flat{"flat", at(-20, 80), 1, pick(0, 12), 1, trial % 2 == 0, false};
    const Span other{"other", at(-20, 80), 1, pick(0, 12), 1, trial % 3 == 0, false};
    const auto g = Bytes(grad), f = Bytes(flat), o = Bytes(other);
    Need(mfh::Touches(grad, mfh::Address(flat.p), flat.row_bytes) == Share(g, f), "Touches", trial);
    const bool want = Share(g, f) || Share(g, o) || ((flat.written || other.written) && Share(f, o));
    size_t a = 9, b = 9;
    const Span spans[] = {flat, grad, other};
    Need(mfh::FindOverlap(spans, &a, &b) == want, "FindOverlap", trial);
    if (want)
      Need(spans[a].written && a != b && Share(Bytes(spans[a]), Bytes(spans[b])), "the pair found",
           trial);
    // Equal strides and shapes: the same rows, or no byte in common.
    const Span rows2{"logits", at(0, 60), rows, bytes, stride, false, true};
    if (rows > 0 && rows2.p != grad.p) {
      const bool clash = mfh::RowsClash(rows2.p, stride, grad.p, stride, rows, bytes);
      Need(clash || !Share(g, Bytes(rows2)), "RowsClash", trial);
    }
    std::vector<ByteRange> ranges;
    std::set<std::uintptr_t> held;
    for (int i = pick(0, 5); i > 0; --i) {
      const std::uintptr_t begin = static_cast<std::uintptr_t>(pick(0, 60)), size = pick(1, 9);
      ranges.push_back({begin, begin + size});
      for (std::uintptr_t v = begin; v < begin + size; ++v)
        held.insert(v);
    }
    const auto joined = mfh::Joined(ranges);
    for (size_t i = 1; i < joined.size(); ++i)
      Need(joined[i - 1].end < joined[i].begin, "Joined", trial);
    const std::uintptr_t begin = static_cast<std::uintptr_t>(pick(0, 70)), size = pick(0, 9);
    bool meets = false;
    for (std::uintptr_t v = begin; v < begin + size; ++v)
      meets = meets || held.count(v);
    Need(mfh::Meets(joined, reinterpret_cast<const void *>(begin), size) == meets, "Meets", trial);
  }
  // Past 2 GiB: rows 3 GiB apart, an array in a gap, one that reaches a row.
  const std::int64_t gib = std::int64_t(1) << 30;
  const Span far{"far", reinterpret_cast<const void *>(std::uintptr_t(4096)), 100, 512, 3 * gib, true,
                 true};
  const std::uintptr_t row = 4096 + 57 * 3 * static_cast<std::uintptr_t>(gib);
  Need(!mfh::Touches(far, row + 512, 3 * gib - 512), "a whole gap", -1);
  Need(mfh::Touches(far, row + 512, 3 * gib - 511), "a gap and a byte", -1);
  Need(mfh::Touches(far, row + 511, 1) && !mfh::Touches(far, row - 1, 1), "a row's ends", -1);
  std::printf("learn ranges ok\n");
  return 0;
}
