// How the paged attention's work is cut among warps: plain integer
// arithmetic, the same on host and device (the CPU tests build it alone).
//
// A tile is 16 or 32 consecutive positions of one sequence for one block of
// query heads that share a key head. Tiles are numbered sequence by sequence, head
// block by head block, along the positions; warp w of n takes the tiles
// [w * total / n, (w + 1) * total / n). So every warp reads the same amount
// whatever the lengths are, and a (sequence, head block) is cut only where two
// warps' shares meet.
#pragma once

#include <stdint.h>

#if defined(__CUDACC__)
#define PAGED_HD __host__ __device__ __forceinline__
#else
#define PAGED_HD inline
#endif

namespace inferc_dev {
namespace paged {

// Unsigned division by a constant of the launch, exact for every 32-bit n:
// q = (((n * mul) >> 32) + n) >> shift with shift = ceil(log2 d) and
// mul = floor(2^32 (2^shift - d) / d) + 1, the sum formed in 64 bits.
struct FastDiv {
  uint32_t d = 1, mul = 1, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t d_) : d(d_) {
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  PAGED_HD uint32_t div(uint32_t n) const {
    const uint64_t hi = ((uint64_t)n * mul) >> 32;
    return (uint32_t)((hi + n) >> shift);
  }
  PAGED_HD uint32_t mod(uint32_t n) const { return n - div(n) * d; }
};

// a / b for a >= 0, b > 0; in 32 bits where they fit (a quarter of the time).
PAGED_HD int64_t divide(int64_t a, int64_t b) {
  if (((uint64_t)a | (uint64_t)b) >> 32 == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// Warps that get work: no more than there are tiles.
PAGED_HD int64_t warps_used(int64_t total, int64_t warps) {
  return warps < total ? warps : total;
}

PAGED_HD int64_t first_tile(int64_t w, int64_t total, int64_t warps) {
  return divide(w * total, warps);
}

// The warp whose share holds tile t (warps <= total).
PAGED_HD int64_t owner_of(int64_t t, int64_t total, int64_t warps) {
  return divide((t + 1) * warps - 1, total);
}

// The parts of one (sequence, head block): warp `first`'s second slot, then
// the first slots of the warps behind it.
struct Parts {
  int64_t first;
  int count;
  PAGED_HD int64_t slot(int i) const { return i == 0 ? 2 * first + 1 : 2 * (first + i); }
};

// `count` parts from warp `first` on. Of the `warps` there are, whatever the numbers:
// lengths that change while they are read must not name a slot that is none.
PAGED_HD Parts parts_within(int64_t first, int64_t count, int64_t warps) {
  if (first > warps - 1) first = warps - 1;
  if (first < 0) first = 0;
  if (count > warps - first) count = warps - first;
  return {first, count > 1 ? (int)count : 1};
}

// Those of tiles t0 .. t0 + tiles - 1 of `total`, which `used` warps share.
PAGED_HD Parts parts_of(int64_t t0, int64_t tiles, int64_t total, int64_t used) {
  if (total < 1) return {0, 1};
  const int64_t first = owner_of(t0, total, used);
  return parts_within(first, owner_of(t0 + tiles - 1, total, used) - first + 1, used);
}

// Rows of `length` elements at base + i * step[0].stride + j * step[1].stride.
struct Step {
  int64_t count, stride;
};
struct Rows2 {
  int64_t base, length;
  Step step[2];
};

// Whether two sets of rows share an element; b's own rows do not. A look at the extents
// decides where those are apart; else each of a's rows is looked up among b's.
inline bool rows_meet(Rows2 a, Rows2 b) {
  auto extent = [](Rows2& r) {
    int64_t n = r.length;
    for (Step& s : r.step) {
      if (s.count <= 0) return (int64_t)0;
      if (s.count == 1) s.stride = 0;
      if (s.stride < 0) {  // the same rows, from the other end
        r.base += s.stride * (s.count - 1);
        s.stride = -s.stride;
      }
      n += s.stride * (s.count - 1);
    }
    return r.length > 0 ? n : 0;
  };
  const int64_t n = extent(a), m = extent(b);
  if (n == 0 || m == 0 || a.base + n <= b.base || b.base + m <= a.base) return false;
  const bool first = b.step[0].stride >= b.step[1].stride;
  const Step outer = b.step[first ? 0 : 1], inner = b.step[first ? 1 : 0];
  const int64_t block = b.length + inner.stride * (inner.count - 1);
  // indexes m of rows [m * stride, m * stride + size) that [x, x + a.length) meets
  struct Range {
    int64_t from, to;
  };
  auto meets = [&](int64_t x, Step s, int64_t size) {
    if (s.count == 1) return Range{0, x < size && x + a.length > 0 ? 1 : 0};
    auto floor_div = [](int64_t n, int64_t d) { return n >= 0 ? n / d : -((-n + d - 1) / d); };
    int64_t from = floor_div(x - size, s.stride) + 1, to = floor_div(x + a.length - 1, s.stride) + 1;
    if (from < 0) from = 0;
    if (to > s.count) to = s.count;
    return Range{from, to};
  };
  for (int64_t i = 0; i < a.step[0].count; ++i)
    for (int64_t j = 0; j < a.step[1].count; ++j) {
      const int64_t x = a.base + i * a.step[0].stride + j * a.step[1].stride - b.base;
      const Range blocks = meets(x, outer, block);
      for (int64_t k = blocks.from; k < blocks.to; ++k) {
        const Range rows = meets(x - k * outer.stride, inner, b.length);
        if (rows.from < rows.to) return true;
      }
    }
  return false;
}

// Slots of a warp's ring that were filled, for the keys and values of `tiles` tiles and
// the keys of one more (`keys`), and not taken yet: the ones a warp that gives up waits for.
PAGED_HD int fills_in_flight(int tiles, bool keys, int taken) {
  return 2 * tiles + (keys ? 1 : 0) - taken;
}

}  // namespace paged
}  // namespace inferc_dev
