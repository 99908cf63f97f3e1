// Apart and Nested of learn_ranges.h against sets of bytes: Apart may miss
// that two arrays are apart, never that they are not.
#include "learn_ranges.h"

#include <cstdio>
#include <random>
#include <set>

using namespace mfh;

static std::multiset<std::uintptr_t> Bytes(const Region &r) {
  std::multiset<std::uintptr_t> out;
  for (std::int64_t i = 0; i < r.dims[0].n; ++i)
    for (std::int64_t j = 0; j < r.dims[1].n; ++j)
      for (std::int64_t k = 0; k < r.dims[2].n; ++k)
        for (std::int64_t b = 0; b < r.inner; ++b)
          out.insert(Address(r.p) + i * r.dims[0].stride + j * r.dims[1].stride +
                     k * r.dims[2].stride + b);
  return out;
}

static bool Share(const Region &x, const Region &y) {
  const auto a = Bytes(x), b = Bytes(y);
  for (auto v : a)
    if (b.count(v))
      return true;
  return false;
}

static int Fail(const char *what) {
  std::printf("FAILED: %s\n", what);
  return 1;
}

int main() {
  std::mt19937 rng(7);
  const auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const auto any = [&]() {
    return RegionOf("x", reinterpret_cast<void *>(std::uintptr_t(4096 + pick(0, 90))), pick(0, 6),
                    true, {{pick(0, 3), pick(0, 40)}, {pick(1, 4), pick(0, 24)}, {pick(1, 3), pick(0, 12)}});
  };
  int apart = 0, found = 0;
  for (int i = 0; i < 200000; ++i) {
    const Region x = any(), y = any();
    const bool share = Share(x, y);
    if (Apart(x, y)) {
      ++found;
      if (share)
        return Fail("apart, but they share a byte");
    }
    apart += !share;
    if (Apart(x, y) != Apart(y, x))
      return Fail("not the same both ways");
    if (Nested(x) && !Empty(x)) {
      const auto b = Bytes(x);
      if (std::set<std::uintptr_t>(b.begin(), b.end()).size() != b.size())
        return Fail("nested, but two runs share a byte");
    }
  }
  if (found * 2 < apart)
    return Fail("half of the arrays that are apart are not found so");
  // q, k and v in one array [line, token, 3, head, dim]; heads between heads.
  const auto at = [](std::uintptr_t p) { return reinterpret_cast<void *>(p); };
  const std::int64_t d = 64, h = 8, t = 100;
  const auto part = [&](int i) {
    return RegionOf("x", at(1 << 20 | i * h * d), d, true,
                    {{4, t * 3 * h * d}, {t, 3 * h * d}, {h, d}});
  };
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j)
      if (Apart(part(i), part(j)) != (i != j))
        return Fail("parts of one array");
  const auto mixed = [&](int i) {
    return RegionOf("x", at(1 << 20 | i * d), d, true, {{4, t * 3 * h * d}, {t, 3 * d}, {h, t * 3 * d}});
  };
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j)
      if (Apart(mixed(i), mixed(j)) != (i != j))
        return Fail("parts of one array, heads first");
  if (!Nested(part(0)) || !Nested(mixed(1)))
    return Fail("arrays without shared elements");
  std::printf("learn regions ok\n");
  return 0;
}
