// Attention of one new token per sequence over the paged cache: the kernel
// that reads the cache. paged_attention.cu has the entry point, the join of
// cut sequences and the running sums; one file per element type instantiates
// this one.
//
// Mathematics. For a key head and the query heads that share it (a block of 8
// or 16), every warp walks its tiles of positions with the running maximum m and
// sum l of the softmax:
//   S^T = K Q^T   (16 positions x heads),   m' = max(m, S),  P = 2^(S - m')
//   O^T = 2^(m - m') O^T + V^T P            (head_dim x heads)
// with scores in the log2 domain. The positions are the matrix instruction's
// rows and the heads its 8 columns, so the whole width is used from 8 heads
// per key head on, and one head per key head still costs only 1 / 2 of what
// 16 rows of queries would.
//
// What bounds it: every byte of K and V is read once and used for 2 flops per
// query head, so HBM: 0.92 of the measured copy rate for 1.07 GB in 64 sequences
// (177 us), 0.86 for one sequence of 131k positions and 8 key heads (95 us), and
// latency below some 20 MB. mma.sync is enough (at 8 heads, 0.1 PFLOP/s of it at
// full bandwidth); tcgen05 tiles would need 64 rows and a trip through tensor
// memory for each 16 positions.
//
// Measured and not taken (same cases): shares of half or a third per warp, so
// that late warps find work (16 x 8 heads of 128: 33 -> 37 and 43 us, for the
// parts that more cuts leave); three or four blocks per SM with smaller rings
// (33 -> 39 us).
//
// Layout. Each warp owns a ring of kSlots shared-memory slots, each a tile of K
// or of V in 128-byte columns with the 128-byte swizzle (free of bank conflicts
// for ldmatrix and for fp32's 16-byte loads). One lane fills them by TMA, boxes
// of 16 rows of 128 bytes, some tiles ahead and across the boundaries of heads
// and sequences, so that warps never wait for each other and the loads never
// drain. A box never leaves its page when the page size is a multiple of 16;
// for other page sizes, or strides a tensor map cannot carry, the slots are
// filled by 16-byte cp.async, row by row. Rows past a sequence's end, or on a
// page that does not exist, are scored -inf and their values cleared before
// they are used, whatever the page holds there.
//
// A tile is 32 positions where a row has up to 256 bytes and 16 above: the
// cost of a tile that does not depend on its rows (maximum over the warp,
// bookkeeping, waits) was most of its instructions at 16 (779 MB of fp16 heads
// of 64: 233 us, at 32 positions 128 us).
//
// Numbers. 16-bit products are exact in fp32. P goes into the second product
// as two 16-bit pieces, P = hi + lo, so that rounding it adds less than the
// result's own rounding; fp16 P carries a factor 2^10 (in m), which keeps
// weights down to 2^-34 of the largest. fp32 operands are taken as two tf32
// pieces each, three products (big big, big small, small big), so that at most
// 2^-20 of a product is lost (cut operands lose 3 * 2^-23, rounded ones 2^-22,
// small * small is below 2^-21).
//
// Pieces of an infinity are an infinity and a NaN or a zero, whose products are
// NaN where the definition has a weight of 0 or an infinite result. So a share
// whose sums come out infinite or NaN is walked again in plain fp32 operations
// (walk_again); the others pay one look at the sums per share.
#pragma once

#include <atomic>

#include "paged.cuh"
#include "tc_ptx.cuh"

namespace inferc_dev {
namespace paged {

struct AttendArgs {
  Args a;
  const void* q;
  int64_t q_batch, q_head;
  void* out;
  int64_t o_batch, o_head;
  float scale;      // times log2(e)
  int group;        // query heads per key head
  int block;        // query heads per block (at most 16)
  int blocks;       // blocks per key head
  int tile;         // positions per tile
  bool whole;       // one block of the grid reads one (sequence, key head), see attend_kernel
  int64_t warps;    // in the grid
  int4* jobs;       // [warps] (sequence or -1, head block, parts) whose first part this warp left
  int4* starts;     // [warps] (sequence, head block, tile) where a warp's share begins
  float* part_ml;   // [2 warps, block, 2] maximum and sum of a part
  float* part_o;    // [2 warps, block, head_dim]
  float* scores;    // [batch, q_heads, capacity] or nullptr
  float* stats;     // [batch, q_heads, 2] maximum and 1 / sum (with scores)
  int64_t capacity;
  float* w;
  int64_t w_batch, w_head;
};

constexpr int kWarps = 4;  // per block

constexpr int kBox = 16;  // rows that TMA fetches at once, and of one matrix instruction

// Shared memory of a warp: kSlots slots of kColumns columns of kTile rows of
// 128 bytes, then a barrier and a row mask for each slot.
template <typename T, int kDim>
struct Layout {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kTile = kDim * (int)sizeof(T) <= 256 ? 32 : 16;  // positions
  static constexpr int kElems = 128 / sizeof(T);                       // per column
  static constexpr int kColumns = (kDim + kElems - 1) / kElems;
  static constexpr int kColumn = kTile * 128;
  static constexpr int kSlot = kColumns * kColumn;
  // Two blocks (8 warps) per SM with as many slots as their shares of the
  // 227 KB allow, one block where that would leave fewer than three.
  static constexpr int kTwo = 110 * 1024 / (kWarps * (kSlot + 16));
  static constexpr int kBlocks = kTwo >= 3 ? 2 : 1;
  static constexpr int kFit = kBlocks == 2 ? kTwo : 220 * 1024 / (kWarps * (kSlot + 16));
  static constexpr int kSlots = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kWarps * kSlots * (kSlot + 16) + 1024;  // + alignment slack
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  const int bytes = ok ? 16 : 0;  // the rest of the 16 is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = big + small, each to tf32's 11 bits (nearest; the instruction drops the
// 13 low bits, so half a step is added to what it drops).
__device__ __forceinline__ void split_tf32(float x, uint32_t& big, uint32_t& small) {
  big = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  small = __float_as_uint(x - __uint_as_float(big)) + 0x1000u;
}

// The same by cutting instead of rounding, in half the instructions: big keeps
// 11 bits, small the other 13, of which the instruction uses at least 11.
__device__ __forceinline__ void cut_tf32(uint32_t x, uint32_t& big, uint32_t& small) {
  big = x & 0xffffe000u;
  small = __float_as_uint(__uint_as_float(x) - __uint_as_float(big));
}

// P in [0, 1] (fp16: [0, 2^10]) as two 16-bit pieces, two values packed.
template <typename T>
__device__ __forceinline__ void split_pair16(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
}

// A place in the numbering of tiles.
template <int kTile>
struct Cursor {
  int b, hk, block, tile, tiles, len;

  // Goes to sequence `first` or the first one after it that holds something.
  __device__ __forceinline__ void open(const AttendArgs& g, int first) {
    b = first;
    hk = block = tile = tiles = 0;
    for (; b < (int)g.a.kv.batch; ++b) {
      len = seq_len(g.a, b);
      tiles = (len + kTile - 1) / kTile;
      if (tiles) return;
    }
  }
  __device__ __forceinline__ void next(const AttendArgs& g) {
    if (++tile < tiles) return;
    tile = 0;
    if (++block < g.blocks) return;
    block = 0;
    if (++hk < (int)g.a.kv.kv_heads) return;
    open(g, b + 1);
  }
};

// Everything that one warp holds of a (sequence, head block) between tiles, on
// tensor instructions: S^T = K Q^T, softmax, O^T += V^T P for kCols blocks of 8
// query heads. `d` and the place of rows in a slot are as in Layout.
template <typename T, int kDim, int kCols>
struct TensorHeads {
  using L = Layout<T, kDim>;
  static constexpr bool kWide = L::kWide;
  static constexpr int kSubs = L::kTile / kBox;
  static constexpr int kKSteps = kWide ? kDim / 8 : kDim / 16;  // steps along head_dim
  static constexpr int kMTiles = kDim / 16;                     // blocks of 16 columns of V
  static constexpr int kPartFloats = kCols * 8 * kDim;
  static constexpr float kLift = std::is_same_v<T, __half> ? 10.f : 0.f;
  static constexpr bool kPieces = true;  // operands enter as sums of pieces
  // fp32 queries are split once where their pieces fit the registers
  static constexpr bool kSplitOnce = kWide && kDim * kCols <= 128;
  uint32_t qf[kCols][kKSteps][kSplitOnce ? 4 : 2];
  float o[kCols][kMTiles][4];
  float m[kCols][2], l[kCols][2];
  float sc[kSubs][kCols][4];  // of 16 positions gid and gid + 8, of 8 heads 2 tig and 2 tig + 1

  __device__ __forceinline__ static int gid() { return (threadIdx.x & 31) >> 2; }
  __device__ __forceinline__ static int tig() { return threadIdx.x & 3; }

  __device__ __forceinline__ void begin(const T* q, int64_t q_head, int cols, int d) {
    bool odd = false;  // fp32: infinities and NaN, some of which split_tf32 makes zeros of
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int h = c * 8 + gid();
      const T* row = q + (int64_t)h * q_head;
#pragma unroll
      for (int s = 0; s < kKSteps; ++s) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = kWide ? s * 8 + tig() + 4 * i : s * 16 + tig() * 2 + 8 * i;
          const bool in = h < cols && col < d;
          uint32_t x = 0;
          if (in) x = *reinterpret_cast<const uint32_t*>(row + col);
          if constexpr (kWide) odd |= (x & 0x7f800000u) == 0x7f800000u;
          if constexpr (kSplitOnce) split_tf32(__uint_as_float(x), qf[c][s][i], qf[c][s][2 + i]);
          else qf[c][s][i] = x;
        }
      }
      m[c][0] = m[c][1] = -INFINITY;
      l[c][0] = l[c][1] = 0.f;
#pragma unroll
      for (int i = 0; i < kMTiles; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
    }
    if (kWide && __any_sync(0xffffffffu, odd))
#pragma unroll
      for (int c = 0; c < kCols; ++c) l[c][0] = l[c][1] = NAN;
  }

  // Whether a sum of the warp's is infinite or NaN.
  __device__ __forceinline__ bool odd() const {
    float x[4] = {};  // NaN once anything infinite or NaN was multiplied by 0
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      x[0] = fmaf(l[c][0], 0.f, x[0]);
      x[1] = fmaf(l[c][1], 0.f, x[1]);
#pragma unroll
      for (int i = 0; i < kMTiles; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fmaf(o[c][i][j], 0.f, x[j]);
    }
    const float any = (x[0] + x[1]) + (x[2] + x[3]);
    return __any_sync(0xffffffffu, any != any);
  }

  __device__ __forceinline__ void scores(const unsigned char* slot, float scale) {
    const int lane = threadIdx.x & 31;
    // ldmatrix: row and 16-byte piece of this lane, swizzled; the step's bits of the piece are
    // xored in
    const uint32_t k_addr = smem_addr(slot) + ((lane & 7) + ((lane >> 3) & 1) * 8) * 128 +
                            (((lane >> 4) ^ (lane & 7)) << 4);
    // two chains of products, so that one need not wait for the one before
    float acc[kSubs][kCols][2][4] = {}, sum[kSubs][kCols][4] = {};
#pragma unroll
    for (int s = 0; s < kKSteps; ++s) {
      uint32_t qs[kCols][4];
      if constexpr (kWide) {
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if constexpr (kSplitOnce) {
              qs[c][i] = qf[c][s][i];
              qs[c][2 + i] = qf[c][s][2 + i];
            } else {
              split_tf32(__uint_as_float(qf[c][s][i]), qs[c][i], qs[c][2 + i]);
            }
          }
      }
#pragma unroll
      for (int u = 0; u < kSubs; ++u) {
        uint32_t a[4];
        ldmatrix4((k_addr ^ ((s & 3) << 5)) + (s >> 2) * L::kColumn + u * kBox * 128, a);
        if constexpr (!kWide) {
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            mma16<T>(acc[u][c][s & 1], a, qf[c][s][0], qf[c][s][1]);
        } else {
          uint32_t big[4], small[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) cut_tf32(a[i], big[i], small[i]);
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            mma_tf32(acc[u][c][1], small, qs[c][0], qs[c][1]);
            mma_tf32(acc[u][c][0], big, qs[c][0], qs[c][1]);
            mma_tf32(acc[u][c][1], big, qs[c][2], qs[c][3]);
            if ((s & 3) == 3 || s + 1 == kKSteps) settle(sum[u][c], acc[u][c][0]);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kSubs; ++u)
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sc[u][c][i] = ((kWide ? sum[u][c][i] : acc[u][c][0][i]) + acc[u][c][1][i]) * scale;
  }

  // The instruction adds to its accumulator by cutting, always towards zero: over many steps
  // that would cost fp32 results a digit (2e-6 of an output of 1000 positions of 256 columns) and
  // bias 16-bit ones (262144 positions in one warp's share: 1.7e-3 too small, 3.5 half steps of
  // fp16). So fp32 scores take four steps of the large products, and values those of one tile,
  // then join a sum that is rounded.
  __device__ __forceinline__ static void settle(float (&sum)[4], float (&acc)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[i] += acc[i];
      acc[i] = 0.f;
    }
  }

  // Rows without a bit in the mask are left out.
  __device__ __forceinline__ void leave_out(uint32_t mask) {
#pragma unroll
    for (int u = 0; u < kSubs; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(mask >> (u * kBox + gid() + (i >> 1) * 8) & 1))
#pragma unroll
          for (int c = 0; c < kCols; ++c) sc[u][c][i] = -INFINITY;
  }

  // The scores of `left` positions to `to` (row of the first head), `stride` apart.
  __device__ __forceinline__ void write_scores(float* to0, int64_t stride, int cols, int left) {
    to0 += tig() * 2 * stride + gid();
    left -= gid();
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (c * 8 + tig() * 2 + i >= cols) continue;
        float* to = to0 + (c * 8 + i) * stride;
#pragma unroll
        for (int u = 0; u < kSubs; ++u) {
          if (left > u * kBox) to[u * kBox] = sc[u][c][i];
          if (left > u * kBox + 8) to[u * kBox + 8] = sc[u][c][i + 2];
        }
      }
  }

  __device__ __forceinline__ void softmax() {
    float top[kCols][2];
    bool grew = false;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(sc[0][c][i], sc[0][c][i + 2]);
#pragma unroll
        for (int u = 1; u < kSubs; ++u) x = fmaxf(x, fmaxf(sc[u][c][i], sc[u][c][i + 2]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        top[c][i] = x - kLift;
        grew |= top[c][i] > m[c][i];
      }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        float keep[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float to = fmaxf(m[c][i], top[c][i]);
          keep[i] = to == -INFINITY ? 1.f : ex2(m[c][i] - to);
          m[c][i] = to;
          l[c][i] *= keep[i];
        }
#pragma unroll
        for (int i = 0; i < kMTiles; ++i) {
          o[c][i][0] *= keep[0];
          o[c][i][1] *= keep[1];
          o[c][i][2] *= keep[0];
          o[c][i][3] *= keep[1];
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float base = m[c][i] == -INFINITY ? 0.f : m[c][i];
#pragma unroll
        for (int u = 0; u < kSubs; ++u) {
          sc[u][c][i] = ex2(sc[u][c][i] - base);
          sc[u][c][i + 2] = ex2(sc[u][c][i + 2] - base);
          l[c][i] += sc[u][c][i] + sc[u][c][i + 2];
        }
      }
  }

  __device__ __forceinline__ void values(const unsigned char* slot) {
    const int lane = threadIdx.x & 31;
    if constexpr (!kWide) {
      const uint32_t v_addr = smem_addr(slot) + ((lane & 7) + (lane >> 4) * 8) * 128 +
                              ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
      uint32_t hi[kSubs][kCols][2], lo[kSubs][kCols][2];
#pragma unroll
      for (int u = 0; u < kSubs; ++u)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            split_pair16<T>(sc[u][c][2 * i], sc[u][c][2 * i + 1], hi[u][c][i], lo[u][c][i]);
            hi[u][c][i] = transpose8x8(hi[u][c][i]);
            lo[u][c][i] = transpose8x8(lo[u][c][i]);
          }
#pragma unroll
      for (int i = 0; i < kMTiles; ++i) {
        float fresh[kCols][4] = {};
#pragma unroll
        for (int u = 0; u < kSubs; ++u) {
          uint32_t a[4];
          ldmatrix4_trans((v_addr ^ ((i & 3) << 5)) + (i >> 2) * L::kColumn + u * kBox * 128, a);
#pragma unroll
          for (int c = 0; c < kCols; ++c) mma16<T>(fresh[c], a, lo[u][c][0], lo[u][c][1]);
#pragma unroll
          for (int c = 0; c < kCols; ++c) mma16<T>(fresh[c], a, hi[u][c][0], hi[u][c][1]);
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) settle(o[c][i], fresh[c]);
      }
    } else {
      constexpr int kEights = kSubs * 2;  // eight positions each
      // P of positions (2 tig, 2 tig + 1) of each eight, head gid, from the lanes that hold them
      uint32_t big_p[kEights][kCols][2], small_p[kEights][kCols][2];
#pragma unroll
      for (int e = 0; e < kEights; ++e)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int src = (tig() * 2 + i) * 4 + (gid() >> 1);
            const float x = __shfl_sync(0xffffffffu, sc[e >> 1][c][2 * (e & 1)], src);
            const float y = __shfl_sync(0xffffffffu, sc[e >> 1][c][2 * (e & 1) + 1], src);
            split_tf32(gid() & 1 ? y : x, big_p[e][c][i], small_p[e][c][i]);
          }
      const unsigned char* r0 = slot + tig() * 2 * 128 + ((gid() ^ (tig() * 2)) << 4);
      const unsigned char* r1 = slot + (tig() * 2 + 1) * 128 + ((gid() ^ (tig() * 2 + 1)) << 4);
#pragma unroll
      for (int i = 0; i < kMTiles; i += 2) {
        float fresh[2][kCols][4] = {};
#pragma unroll
        for (int e = 0; e < kEights; ++e) {
          const int at = (i >> 1) * L::kColumn + e * 8 * 128;
          const uint4 x = *reinterpret_cast<const uint4*>(r0 + at);
          const uint4 y = *reinterpret_cast<const uint4*>(r1 + at);
          uint32_t big[2][4], small[2][4];
          cut_tf32(x.x, big[0][0], small[0][0]);
          cut_tf32(x.y, big[0][1], small[0][1]);
          cut_tf32(y.x, big[0][2], small[0][2]);
          cut_tf32(y.y, big[0][3], small[0][3]);
          cut_tf32(x.z, big[1][0], small[1][0]);
          cut_tf32(x.w, big[1][1], small[1][1]);
          cut_tf32(y.z, big[1][2], small[1][2]);
          cut_tf32(y.w, big[1][3], small[1][3]);
#pragma unroll
          for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              mma_tf32(fresh[v][c], small[v], big_p[e][c][0], big_p[e][c][1]);
              mma_tf32(fresh[v][c], big[v], small_p[e][c][0], small_p[e][c][1]);
              mma_tf32(fresh[v][c], big[v], big_p[e][c][0], big_p[e][c][1]);
            }
        }
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int c = 0; c < kCols; ++c) settle(o[c][i + v], fresh[v][c]);
      }
    }
  }

  // Passes (head, maximum, sum) once per head, then (head, column, value) of the
  // lane's unnormalised output; the sums are the warp's.
  template <typename Head, typename Value>
  __device__ __forceinline__ void end(int cols, int d, Head&& head, Value&& value) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = l[c][i];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int h = c * 8 + tig() * 2 + i;
        if (h >= cols) continue;
        if (gid() == 0) head(h, m[c][i], x);
        const float inv = x == 0.f ? 0.f : 1.f / x;  // 0: every page was bad
#pragma unroll
        for (int j = 0; j < kMTiles; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int col = kWide ? (j >> 1) * 32 + gid() * 4 + (j & 1) * 2 + half
                                  : j * 16 + half * 8 + gid();
            if (col < d) value(h, col, o[c][j][2 * half + i], inv);
          }
      }
  }
};

// The same for one fp32 query head per key head, on the CUDA cores: the matrix
// instruction would use one of its 8 columns, and three of them per product with
// the splitting of K and V are over twice the instructions (32 x 12 heads of 64,
// 100 MB and their running sums: 31 us against 36 us, both with kTmaKeep). A lane
// takes a position of the tile (half of its columns where the tile has 16
// positions) for the scores, and kDim / 32 columns for the values; P passes through shared memory. Two fp32 operations per
// instruction (fma.rn.f32x2).
template <int kDim>
struct OneHead {
  using L = Layout<float, kDim>;
  static constexpr int kTile = L::kTile, kSplit = 32 / kTile;
  static constexpr int kQuads = kDim / kSplit / 4;  // float4s of a row that a lane multiplies
  static constexpr int kMine = kDim / 32;           // output columns of a lane: 2 or 4
  static constexpr int kPartFloats = kDim;
  static constexpr bool kPieces = false;
  unsigned long long q[kQuads][2], o[kMine / 2];
  float m, l, s;

  __device__ __forceinline__ static unsigned long long pack(float a, float b) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
  }
  __device__ __forceinline__ static float2 unpack(unsigned long long v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
  __device__ __forceinline__ static unsigned long long fma2(unsigned long long a,
                                                            unsigned long long b,
                                                            unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
  }

  __device__ __forceinline__ void begin(const float* row, int64_t, int, int d) {
    const int first = (threadIdx.x & 31) / kTile * (kDim / kSplit);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (first + 4 * i < d) x = *reinterpret_cast<const float4*>(row + first + 4 * i);
      q[i][0] = pack(x.x, x.y);
      q[i][1] = pack(x.z, x.w);
    }
#pragma unroll
    for (int i = 0; i < kMine / 2; ++i) o[i] = 0;
    m = -INFINITY;
    l = 0.f;
  }

  __device__ __forceinline__ void scores(const unsigned char* slot, float scale) {
    const int lane = threadIdx.x & 31, row = lane % kTile;
    const int first = lane / kTile * kQuads;  // 16-byte piece of the row
    unsigned long long a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int piece = first + i;
      const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(
          slot + (piece >> 3) * L::kColumn + row * 128 + (((piece ^ row) & 7) << 4));
      a = fma2(q[i][0], k.x, a);
      b = fma2(q[i][1], k.y, b);
    }
    const float2 x = unpack(a), y = unpack(b);
    s = (x.x + x.y) + (y.x + y.y);
    if constexpr (kSplit == 2) s += __shfl_xor_sync(0xffffffffu, s, 16);
    s *= scale;
  }

  __device__ __forceinline__ void leave_out(uint32_t mask) {
    if (!(mask >> (threadIdx.x % kTile) & 1)) s = -INFINITY;
  }

  __device__ __forceinline__ void write_scores(float* to, int64_t, int, int left) {
    const int lane = threadIdx.x & 31;
    if (lane < kTile && lane < left) to[lane] = s;
  }

  __device__ __forceinline__ void softmax() {
    const float top = fmaxf(m, warp_max(s));
    if (top > m) {  // the same in every lane
      const float keep = ex2(m - top);
      m = top;
      l *= keep;
      const unsigned long long k2 = pack(keep, keep);
#pragma unroll
      for (int i = 0; i < kMine / 2; ++i) o[i] = fma2(o[i], k2, 0);
    }
    s = ex2(s - (m == -INFINITY ? 0.f : m));
    if ((threadIdx.x & 31) < kTile) l += s;
  }

  __device__ __forceinline__ void values(const unsigned char* slot) {
    __shared__ __align__(16) float2 s_p[kWarps][kTile];
    const int lane = threadIdx.x & 31;
    float2* p = s_p[threadIdx.x >> 5];
    if (lane < kTile) p[lane] = make_float2(s, s);
    __syncwarp();
    const int piece = lane * kMine / 4, inside = lane * kMine % 4 * 4;
    const unsigned char* column = slot + (piece >> 3) * L::kColumn + inside;
#pragma unroll
    for (int j = 0; j < kTile; j += 2) {
      const ulonglong2 pp = *reinterpret_cast<const ulonglong2*>(p + j);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned char* at = column + (j + u) * 128 + (((piece ^ (j + u)) & 7) << 4);
        const unsigned long long w = u ? pp.y : pp.x;
        if constexpr (kMine == 4) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(at);
          o[0] = fma2(w, v.x, o[0]);
          o[kMine / 2 - 1] = fma2(w, v.y, o[kMine / 2 - 1]);
        } else {
          o[0] = fma2(w, *reinterpret_cast<const unsigned long long*>(at), o[0]);
        }
      }
    }
  }

  template <typename Head, typename Value>
  __device__ __forceinline__ void end(int, int d, Head&& head, Value&& value) {
    const int lane = threadIdx.x & 31;
    const float x = warp_sum(l), inv = x == 0.f ? 0.f : 1.f / x;  // 0: every page was bad
    if (lane == 0) head(0, m, x);
#pragma unroll
    for (int i = 0; i < kMine / 2; ++i) {
      const float2 v = unpack(o[i]);
      const int col = lane * kMine + 2 * i;
      if (col < d) value(0, col, v.x, inv);
      if (col + 1 < d) value(0, col + 1, v.y, inv);
    }
  }
};

template <typename T>
__device__ __forceinline__ void zero_heads(const AttendArgs& g, int64_t b, int h0, int h1) {
  const int pieces = g.a.kv.head_dim / 8;
  const float zero[8] = {};
  for (int i = threadIdx.x; i < (h1 - h0) * pieces; i += blockDim.x)
    store8(reinterpret_cast<T*>(g.out) + b * g.o_batch + (h0 + i / pieces) * g.o_head +
               (i % pieces) * 8,
           zero);
}

// What a whole block left in shared memory (one part per warp), joined: the
// output of one (sequence, key head) and, where they are kept, its weights.
template <typename T>
__device__ __forceinline__ void join_whole(const AttendArgs& g, int b, int hk, int len,
                                           const float2* ml, const float* o, int part) {
  const InfercPagedKv& kv = g.a.kv;
  const int d = kv.head_dim, quads = d / 4, cols = g.group;
  for (int i = threadIdx.x; i < cols * quads; i += kWarps * 32) {
    const int h = i / quads, quad = i - h * quads;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int p = 0; p < kWarps; ++p) m = fmaxf(m, ml[p * 16 + h].x);
    const float to = m == -INFINITY ? 0.f : m;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < kWarps; ++p) {
      const float2 x = ml[p * 16 + h];
      if (x.y == 0.f) continue;  // a warp without tiles left nothing
      const float f = ex2(x.x - to);
      const float4 v = reinterpret_cast<const float4*>(o + p * part + h * d)[quad];
      l += f * x.y;
      sum.x += f * v.x;
      sum.y += f * v.y;
      sum.z += f * v.z;
      sum.w += f * v.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: every page was bad
    T* out = reinterpret_cast<T*>(g.out) + b * g.o_batch + (hk * g.group + h) * g.o_head + quad * 4;
    out[0] = T(sum.x * inv);
    out[1] = T(sum.y * inv);
    out[2] = T(sum.z * inv);
    out[3] = T(sum.w * inv);
  }
  if (!g.w) return;
  const float* s = g.scores + (b * (int64_t)(kv.kv_heads * g.group) + hk * g.group) * g.capacity;
  float* w = g.w + b * g.w_batch + hk * g.w_head;
  for (int j = threadIdx.x; j < len; j += kWarps * 32) {
    float sum = 0.f;
    for (int h = 0; h < cols; ++h) {
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int p = 0; p < kWarps; ++p) m = fmaxf(m, ml[p * 16 + h].x);
      const float to = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int p = 0; p < kWarps; ++p) {
        const float2 x = ml[p * 16 + h];
        l += x.y == 0.f ? 0.f : ex2(x.x - to) * x.y;
      }
      sum += ex2(s[h * g.capacity + j] - to) * (l == 0.f ? 0.f : 1.f / l);
    }
    w[j] += sum;
  }
}

// Positions [j0, j1) of query heads q0 .. q0 + cols - 1 of a sequence once more, in
// plain fp32 operations and from global memory, and what the warp's share leaves of
// them; for operands with infinities or NaN, so simple: a head at a time, a lane for a
// position's score and for every 32nd column of the values.
template <typename T>
__device__ __forceinline__ void walk_heads(const AttendArgs& g, int b, int hk, int q0, int cols,
                                           int j0, int j1, bool whole, int64_t part, float2* ml,
                                           float* po) {
  const InfercPagedKv& kv = g.a.kv;
  const int lane = threadIdx.x & 31, d = kv.head_dim;
  constexpr int kMine = 256 / 32;
  for (int h = 0; h < cols; ++h) {
    const T* q = reinterpret_cast<const T*>(g.q) + b * g.q_batch + (q0 + h) * g.q_head;
    const int64_t row = b * (kv.kv_heads * g.group) + q0 + h;
    float m = -INFINITY, l = 0.f, o[kMine] = {};
    for (int first = j0; first < j1; first += 32) {
      const int j = first + lane;
      int64_t off_v = -1;
      float s = -INFINITY;
      if (j < j1) {
        const uint32_t index = g.a.page.div(j), slot = j - index * g.a.page.d;
        const int id = page_of(g.a, kv.page_table + b * kv.table_stride, index);
        if (id >= 0) {
          const T* k = reinterpret_cast<const T*>(kv.k) + id * kv.k_page_stride +
                       slot * kv.k_token_stride + hk * kv.k_head_stride;
          off_v = id * kv.v_page_stride + slot * kv.v_token_stride + hk * kv.v_head_stride;
          float sum = 0.f;
          for (int c = 0; c < d; c += 8) {
            float x[8], y[8];
            load8(q + c, x);
            load8(k + c, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(x[i], y[i], sum);
          }
          s = sum * g.scale;
        }
        if (g.scores) g.scores[row * g.capacity + j] = s;
      }
      const float top = fmaxf(m, warp_max(s)), to = top == -INFINITY ? 0.f : top;
      const float keep = ex2(m - to), p = ex2(s - to);
      m = top;
      l = l * keep + p;
#pragma unroll
      for (int i = 0; i < kMine; ++i) o[i] *= keep;
      if (__any_sync(0xffffffffu, p != p)) {  // the head's sum is NaN, and all of its results
        l = NAN;
        break;
      }
      for (int r = 0; r < 32; ++r) {
        const int64_t off = __shfl_sync(0xffffffffu, off_v, r);
        const float w = __shfl_sync(0xffffffffu, p, r);
        if (off < 0) continue;
        const T* v = reinterpret_cast<const T*>(kv.v) + off;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (lane + 32 * i < d) o[i] = fmaf(w, static_cast<float>(v[lane + 32 * i]), o[i]);
      }
    }
    const float sum = warp_sum(l), inv = sum == 0.f ? 0.f : 1.f / sum;
    if (lane == 0) {
      if (g.whole) {
        ml[h] = make_float2(m, sum);
      } else if (!whole) {
        reinterpret_cast<float2*>(g.part_ml)[part * g.block + h] = make_float2(m, sum);
      } else if (g.stats) {
        reinterpret_cast<float2*>(g.stats)[row] = make_float2(m == -INFINITY ? 0.f : m, inv);
      }
    }
    T* out = reinterpret_cast<T*>(g.out) + b * g.o_batch + (q0 + h) * g.o_head;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int col = lane + 32 * i;
      if (col >= d) continue;
      if (whole) out[col] = T(o[i] * inv);
      else po[h * d + col] = o[i];
    }
  }
}

// The head blocks of a warp's share, `count` tiles from (sequence, head block, tile) =
// `first` on, that have a bit in `bits` (number them through, modulo 64). Behind the
// kernel's loop and a function of its own, so that it takes none of the loop's
// registers (called within it, 16 x 32/4 heads of 256 took 46 us instead of 40).
template <typename T, int kTile>
__device__ __noinline__ void walk_again(const AttendArgs& g, int3 first, int count, int64_t w,
                                        unsigned long long bits, float2* ml, float* ring) {
  const InfercPagedKv& kv = g.a.kv;
  __syncwarp();  // what is written over is other lanes'
  Cursor<kTile> at;
  at.open(g, first.x);
  at.hk = first.y / g.blocks;
  at.block = first.y - at.hk * g.blocks;
  at.tile = first.z;
  while (count > 0 && at.b < (int)kv.batch) {
    const int n = min(count, at.tiles - at.tile);
    const bool begins = at.tile == 0, ends = at.tile + n == at.tiles;
    const int head = at.hk * g.blocks + at.block;
    if (bits >> ((at.b * (int64_t)(kv.kv_heads * g.blocks) + head) & 63) & 1) {
      const int q0 = at.hk * g.group + at.block * g.block;
      const int64_t part = 2 * w + (begins ? 1 : 0);
      walk_heads<T>(g, at.b, at.hk, q0, min(g.block, (at.hk + 1) * g.group - q0),
                    at.tile * kTile, min(at.len, (at.tile + n) * kTile),
                    begins && ends && !g.whole, part, ml,
                    g.whole ? ring : g.part_o + part * g.block * kv.head_dim);
    }
    count -= n;
    at.tile = at.tiles - 1;
    at.next(g);
  }
}

// How tiles are fetched: by cp.async, by TMA, or by TMA where the scores that the
// kernel writes are read again by the kernel behind it, so that keys and values are to
// leave L2 first (64 sequences, 50 MB of scores: 214 -> 209 us; fp32, 32 x 12 heads:
// 31 -> 28 us). A kernel of its own: chosen at every load it took the calls
// without scores 0.2 to 0.6 us.
enum Fetch : int { kCopy, kTmaKeep, kTmaOnce };

template <typename T, int kDim, typename Heads, int kFetch>
__global__ void __launch_bounds__(kWarps * 32, Layout<T, kDim>::kBlocks)
    attend_kernel(const __grid_constant__ AttendArgs g, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map) {
  using L = Layout<T, kDim>;
  constexpr int kElem = sizeof(T), kThreads = kWarps * 32, kTile = L::kTile;
  constexpr int kSubs = kTile / kBox;
  constexpr bool kTma = kFetch != kCopy;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int64_t s_before[kThreads];
  __shared__ int64_t s_warp[kWarps];
  __shared__ float2 s_ml[kWarps * 16];  // g.whole: each warp's maxima and sums
  __shared__ int3 s_first[kWarps];      // where a warp's share begins,
  __shared__ unsigned long long s_odd[kWarps];  // its head blocks to be walked again
  const InfercPagedKv& kv = g.a.kv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = (int)kv.kv_heads * g.blocks;
  const int batch = (int)kv.batch;
  const int d = kv.head_dim;
  unsigned char* ring = smem + warp * L::kSlots * L::kSlot;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kWarps * L::kSlots * L::kSlot) +
                   warp * L::kSlots;
  uint32_t* masks = reinterpret_cast<uint32_t*>(smem + kWarps * L::kSlots * (L::kSlot + 8)) +
                    warp * L::kSlots;
  const uint32_t ring_addr = smem_addr(ring);
  if constexpr (kTma) {
    if (lane == 0) {
      for (int i = 0; i < L::kSlots; ++i) tc::mbar_init(&full[i], 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      tc::fence_proxy_async();
    }
  } else if (d < kDim) {  // what no copy fills
    for (int i = lane * 16; i < L::kSlots * L::kSlot; i += 32 * 16)
      *reinterpret_cast<uint4*>(ring + i) = make_uint4(0, 0, 0, 0);
  }
  __syncwarp();
  if constexpr (kTma)
    if (tid == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&k_map)));
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)));
    }

  pdl_wait();  // lengths, tables, queries and caches may come from the kernel before
  // (finish_kernel reads the lengths as soon as every block has passed here)
  pdl_launch_dependents();

  int64_t w = (int64_t)blockIdx.x * kWarps + warp;
  int64_t total = 0, used = 0, t0 = 0;  // tiles, warps that share them, this warp's first
  int count = 0;
  Cursor<kTile> load;
  if (g.whole) {
    // Short sequences, few heads: the block's four warps share one (sequence, key head) and
    // join their parts in shared memory, which spares the search and a second kernel.
    load.b = blockIdx.x / (int)kv.kv_heads;
    load.hk = blockIdx.x - load.b * (int)kv.kv_heads;
    load.block = 0;
    load.len = seq_len(g.a, load.b);
    load.tiles = (load.len + kTile - 1) / kTile;
    load.tile = load.tiles * warp / kWarps;
    count = load.tiles * (warp + 1) / kWarps - load.tile;
  } else {
    // Tiles before each thread's run of sequences, and in all.
    const int run = (batch + kThreads - 1) / kThreads;
    const int run0 = min(tid * run, batch), run1 = min(run0 + run, batch);
    int64_t mine = 0;
    for (int b = run0; b < run1; ++b)
      mine += (int64_t)((seq_len(g.a, b) + kTile - 1) / kTile) * heads;
    int64_t scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += x;
    }
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    int64_t ahead = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) ahead += s_warp[i];
      total += s_warp[i];
    }
    s_before[tid] = ahead + scan - mine;
    // A sequence of length 0 gives zeros.
    for (int64_t b = blockIdx.x; b < batch; b += gridDim.x)
      if (seq_len(g.a, b) == 0)
        zero_heads<T>(g, b, 0, (int)kv.kv_heads * g.group);
    __syncthreads();

    if (g.jobs && lane == 0 && w < g.warps) g.jobs[w] = make_int4(-1, 0, 0, 0);
    used = warps_used(total, g.warps);
    if (w >= used) return;
    t0 = first_tile(w, total, used);
    count = (int)(first_tile(w + 1, total, used) - t0);

    // The tile t0: the thread whose run holds it, then the sequence, then the head.
    int lo = -1;  // runs that begin at t0 or before it, less one
#pragma unroll
    for (int i = 0; i < kThreads; i += 32)
      lo += __popc(__ballot_sync(0xffffffffu, s_before[i + lane] <= t0));
    int64_t left = t0 - s_before[lo];
    load.open(g, min(lo * run, batch));
    while (load.b < batch && left >= (int64_t)load.tiles * heads) {
      left -= (int64_t)load.tiles * heads;
      load.open(g, load.b + 1);
    }
    if (load.b >= batch) {  // only if the lengths change under the kernel
      if (g.starts && lane == 0) g.starts[w] = make_int4(batch, 0, 0, 0);
      return;
    }
    const int head = (int)divide(left, load.tiles);
    load.hk = head / g.blocks;
    load.block = head - load.hk * g.blocks;
    load.tile = (int)(left - (int64_t)head * load.tiles);
    if (g.starts && lane == 0) g.starts[w] = make_int4(load.b, head, load.tile, 0);
  }
  Cursor<kTile> use = load;
  const int whole_len = load.len;
  if (Heads::kPieces && lane == 0) {
    s_first[warp] = make_int3(load.b, load.hk * g.blocks + load.block, load.tile);
    s_odd[warp] = 0;
  }

  // ---- loads: one slot at a time, the keys of a tile, then its values.
  // Kept from a tile's keys to its values:
  int tiles_in = 0, slot_in = 0;  // tiles whose values are on their way; next slot
  bool fetched = false;           // the keys of one more are
  uint32_t mask_in = 0;           // rows that exist
  // kTma: pages of the tile's boxes (those of the next tile are read one ahead) and the
  // first row's place in its page
  int page_next[kSubs], page[kSubs];
  uint32_t at[kSubs];
  // else: this lane's row of the tile, in V
  int64_t off_v = 0;
  bool row_ok = false;

  auto look_up = [&]() {
    if constexpr (kTma) {
      const int32_t* row = kv.page_table + load.b * kv.table_stride;
#pragma unroll
      for (int i = 0; i < kSubs; ++i) {
        const int j = load.tile * kTile + i * kBox;
        page_next[i] = -1;
        if (load.b < batch && j < load.len) page_next[i] = row[g.a.page.div(j)];
      }
    }
  };
  auto boxes = [&](const CUtensorMap* map) {
    const uint32_t bar = tc::smem_u32(&full[slot_in]);
    const uint32_t dst = ring_addr + slot_in * L::kSlot;
    [[maybe_unused]] uint64_t policy = 0;
    if constexpr (kFetch == kTmaOnce)
      asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
#pragma unroll
    for (int s = 0; s < kSubs; ++s)
      if (mask_in >> (s * kBox) & 1) {
#pragma unroll
        for (int i = 0; i < L::kColumns; ++i) {
          if constexpr (kFetch == kTmaOnce)
            asm volatile(
                "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                ".L2::cache_hint [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(
                    dst + i * L::kColumn + s * kBox * 128),
                "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(i * L::kElems), "r"(at[s]),
                "r"(load.hk), "r"(page[s]), "l"(policy)
                : "memory");
          else
            asm volatile(
                "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst + i * L::kColumn +
                                                             s * kBox * 128),
                "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(i * L::kElems), "r"(at[s]),
                "r"(load.hk), "r"(page[s])
                : "memory");
        }
      }
  };
  auto expect = [&]() {
    uint32_t bytes = 0;
#pragma unroll
    for (int s = 0; s < kSubs; ++s)
      if (mask_in >> (s * kBox) & 1) bytes += L::kColumns * kBox * 128;
    if (bytes) tc::mbar_expect_tx(&full[slot_in], bytes);
    else tc::mbar_arrive(&full[slot_in]);
  };
  // kLanes lanes share a row, 16 bytes each.
  auto copy_rows = [&](const void* cache, int64_t off) {
    constexpr int kPieces = kDim * kElem / 16;
    constexpr int kLanes = kPieces <= 8 ? 8 : kPieces <= 16 ? 16 : 32;
    constexpr int kRowsAt = 32 / kLanes, kTurns = (kPieces + 31) / 32;
    const int pieces = d * kElem / 16, piece0 = lane % kLanes;
    const uint32_t dst = ring_addr + slot_in * L::kSlot;
#pragma unroll
    for (int i = 0; i < kTile / kRowsAt; ++i) {
      const int row = i * kRowsAt + lane / kLanes;
      const int64_t from = __shfl_sync(0xffffffffu, off, row);
      const bool ok = __shfl_sync(0xffffffffu, (int)row_ok, row);
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int piece = piece0 + 32 * t;
        if (piece < pieces)
          copy16(dst + (piece >> 3) * L::kColumn + row * 128 + (((piece & 7) ^ (row & 7)) << 4),
                 static_cast<const char*>(cache) + from + piece * 16, ok);
      }
    }
  };
  auto filled = [&]() {
    if constexpr (!kTma) asm volatile("cp.async.commit_group;" ::: "memory");
    slot_in = slot_in + 1 == L::kSlots ? 0 : slot_in + 1;
  };
  auto fill_k = [&]() {
    if (tiles_in < count && load.b < batch) {
      fetched = true;
      if constexpr (kTma) {
        mask_in = 0;
#pragma unroll
        for (int s = 0; s < kSubs; ++s) {
          const int j = load.tile * kTile + s * kBox;
          page[s] = page_next[s];
          at[s] = g.a.page.mod(j);
          const int rows = min(load.len - j, kBox);
          if (rows > 0) {
            if (page[s] >= 0 && page[s] < kv.num_pages) mask_in |= ((1u << rows) - 1) << (s * kBox);
            else *g.a.flag = 1;
          }
        }
        if (lane == 0) {
          masks[slot_in] = mask_in;
          expect();
          boxes(&k_map);
        }
      } else {
        const int j = load.tile * kTile + (lane & (kTile - 1));
        row_ok = j < load.len;
        int id = 0;
        uint32_t slot = 0;
        if (row_ok) {
          const uint32_t index = g.a.page.div(j);
          slot = j - index * g.a.page.d;
          id = page_of(g.a, kv.page_table + load.b * kv.table_stride, index);
          row_ok = id >= 0;
        }
        const int64_t off_k = row_ok ? (id * kv.k_page_stride + slot * kv.k_token_stride +
                                        load.hk * kv.k_head_stride) * kElem
                                     : 0;
        off_v = row_ok ? (id * kv.v_page_stride + slot * kv.v_token_stride +
                          load.hk * kv.v_head_stride) * kElem
                       : 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, row_ok);
        if (lane == 0) masks[slot_in] = mask;
        copy_rows(kv.k, off_k);
      }
    }
    filled();
  };
  auto fill_v = [&]() {
    if (fetched) {
      fetched = false;
      ++tiles_in;
      if constexpr (kTma) {
        if (lane == 0) {
          expect();
          boxes(&v_map);
        }
      } else {
        copy_rows(kv.v, off_v);
      }
      load.next(g);
      look_up();
    }
    filled();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < L::kSlots; ++i) {
    if (i & 1) fill_v();
    else fill_k();
  }

  int slot_out = 0;
  uint32_t phase = 0;
  // Waits for the slot's rows; false, in every lane, after the time limit.
  auto wait = [&]() {
    bool done = true;
    if constexpr (kTma) {
      done = tc::warp_wait(&full[slot_out], phase);
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::kSlots - 1) : "memory");
      __syncwarp();
    }
    return done;
  };
  auto released = [&]() {
    if (++slot_out == L::kSlots) {
      slot_out = 0;
      phase ^= 1;
    }
  };
  // Gives up behind `taken` slots: no copy into this block's memory may be in flight when it
  // leaves.
  auto give_up = [&](int taken) {
    if (lane == 0) atomicExch(g.a.flag + 1, 1);
    for (int i = fills_in_flight(tiles_in, fetched, taken); i > 0; --i) {
      tc::mbar_wait(&full[slot_out], phase);
      released();
    }
  };

  // g.whole: a warp's part, [head][head_dim], takes its ring's memory once all loads have arrived
  constexpr int kPart = L::kSlots * L::kSlot / 4;
  static_assert(kPart >= Heads::kPartFloats, "a part fits a ring");

  Heads heads_of;  // the state of one (sequence, head block)
  bool begins = false;
  int q0 = 0, cols = 0;
  constexpr uint32_t kAll = kTile == 32 ? 0xffffffffu : (1u << (kTile & 31)) - 1;

  int t = 0, keys_taken = 0;  // of a tile whose values did not come
#pragma unroll 1
  for (; t < count && use.b < batch; ++t) {
    if (t == 0 || use.tile == 0) {
      begins = use.tile == 0;
      q0 = use.hk * g.group + use.block * g.block;
      cols = min(g.block, (use.hk + 1) * g.group - q0);
      heads_of.begin(reinterpret_cast<const T*>(g.q) + use.b * g.q_batch + q0 * g.q_head, g.q_head,
                     cols, d);
    }

    if (!wait()) break;
    const uint32_t mask = masks[slot_out];
    heads_of.scores(ring + slot_out * L::kSlot, g.scale);
    __syncwarp();
    if constexpr (L::kSlots % 2 == 0) fill_k();
    else fill_v();
    released();

    if (mask != kAll) heads_of.leave_out(mask);
    if (g.scores)
      heads_of.write_scores(
          g.scores + (use.b * (int64_t)(kv.kv_heads * g.group) + q0) * g.capacity +
              use.tile * kTile,
          g.capacity, cols, use.len - use.tile * kTile);
    heads_of.softmax();

    if (!wait()) {
      keys_taken = 1;
      break;
    }
    unsigned char* v_ptr = ring + slot_out * L::kSlot;
    if (kTma && mask != kAll) {  // rows that do not exist
#pragma unroll
      for (int i = 0; i < L::kSlot / 512; ++i) {
        const int to = i * 512 + lane * 16;
        if (!(mask >> ((to % L::kColumn) >> 7) & 1))
          *reinterpret_cast<uint4*>(v_ptr + to) = make_uint4(0, 0, 0, 0);
      }
      tc::fence_proxy_async();  // before TMA writes here again
      __syncwarp();
    }
    heads_of.values(v_ptr);
    __syncwarp();
    if constexpr (L::kSlots % 2 == 0) fill_v();
    else fill_k();
    released();

    // the end of the sequence's head block, or of this warp's share
    const bool ends = use.tile + 1 == use.tiles;
    if (ends || t + 1 == count) {
      const bool whole = begins && ends && !g.whole;
      const int64_t part = 2 * w + (begins ? 1 : 0);
      if (begins && !ends && g.jobs && lane == 0) {
        const int64_t last = t0 + t + use.tiles - use.tile - 1;
        g.jobs[w] = make_int4(use.b, use.hk * g.blocks + use.block,
                              (int)(owner_of(last, total, used) - w) + 1, 0);
      }
      T* out = reinterpret_cast<T*>(g.out) + use.b * g.o_batch + q0 * g.o_head;
      float* po = g.whole ? reinterpret_cast<float*>(ring) : g.part_o + part * g.block * d;
      bool odd = false;
      if constexpr (Heads::kPieces) odd = heads_of.odd();
      if (odd) {  // leaves nothing yet: the queries are read again, and out may be where they are
        if (lane == 0)
          s_odd[warp] |= 1ull << ((use.b * (int64_t)heads + use.hk * g.blocks + use.block) & 63);
      } else heads_of.end(
          cols, d,
          [&](int h, float top, float sum) {
            if (g.whole) {
              s_ml[warp * 16 + h] = make_float2(top, sum);
            } else if (!whole) {
              reinterpret_cast<float2*>(g.part_ml)[part * g.block + h] = make_float2(top, sum);
            } else if (g.stats) {
              const int64_t r = use.b * (int64_t)(kv.kv_heads * g.group) + q0 + h;
              reinterpret_cast<float2*>(g.stats)[r] =
                  make_float2(top == -INFINITY ? 0.f : top, sum == 0.f ? 0.f : 1.f / sum);
            }
          },
          [&](int h, int col, float x, float inv) {
            if (whole) out[h * g.o_head + col] = T(x * inv);
            else po[h * d + col] = x;
          });
    }
    use.next(g);
  }
  // a wait ran out, or the lengths changed under the kernel
  if (kTma && t < count) give_up(2 * t + keys_taken);
  if constexpr (Heads::kPieces) {
    __syncwarp();
    if (s_odd[warp])
      walk_again<T, kTile>(g, s_first[warp], t, w, s_odd[warp], s_ml + warp * 16,
                           reinterpret_cast<float*>(ring));
  }
  if (!g.whole) return;
  if (count == 0 && lane < 16) s_ml[warp * 16 + lane] = make_float2(-INFINITY, 0.f);
  __syncthreads();
  if (whole_len == 0) {
    zero_heads<T>(g, blockIdx.x / (int)kv.kv_heads,
                  (blockIdx.x % (int)kv.kv_heads) * g.group,
                  (blockIdx.x % (int)kv.kv_heads + 1) * g.group);
    return;
  }
  join_whole<T>(g, blockIdx.x / (int)kv.kv_heads, blockIdx.x % (int)kv.kv_heads, whole_len, s_ml,
                reinterpret_cast<const float*>(smem), kPart);
}

// Launches attend_kernel for g.a.kv's head_dim and g.block; one definition per
// element type.
template <typename T>
void launch_attend(const AttendArgs& g, cudaStream_t st);
template <>
void launch_attend<float>(const AttendArgs& g, cudaStream_t st);
template <>
void launch_attend<__half>(const AttendArgs& g, cudaStream_t st);
template <>
void launch_attend<__nv_bfloat16>(const AttendArgs& g, cudaStream_t st);

// The cache as [pages, kv_heads, page, head_dim] for boxes of 16 rows of 128
// bytes; false when TMA cannot take it (a tile might leave its page, or a
// stride is none of a tensor map's).
template <typename T>
bool make_map(const InfercPagedKv& kv, bool values, CUtensorMap* map) {
  if (kv.page_size % kBox != 0 || kv.num_pages == 0) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page_size,
                              (cuuint64_t)kv.kv_heads, (cuuint64_t)kv.num_pages};
  const int64_t s[3] = {values ? kv.v_token_stride : kv.k_token_stride,
                        values ? kv.v_head_stride : kv.k_head_stride,
                        values ? kv.v_page_stride : kv.k_page_stride};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    if (s[i] <= 0) return false;
    strides[i] = (cuuint64_t)s[i] * sizeof(T);
  }
  const cuuint32_t box[4] = {128 / sizeof(T), kBox, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = std::is_same_v<T, float>    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return tc::encode_fn()(map, type, 4, values ? kv.v : kv.k, dims, strides, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename H>
struct Named {
  using type = H;
};

template <typename T, int kDim>
void launch_attend_dim(const AttendArgs& g, cudaStream_t st) {
  using L = Layout<T, kDim>;
  static_assert(L::kSlots >= 3, "the ring needs three slots");
  const unsigned grid = (unsigned)((g.warps + kWarps - 1) / kWarps);
  CUtensorMap k_map{}, v_map{};
  const bool tma = make_map<T>(g.a.kv, false, &k_map) && make_map<T>(g.a.kv, true, &v_map);
  // one head per key head in fp32, up to 8, or up to 16
  const int kind = std::is_same_v<T, float> && kDim <= 128 && g.group == 1 ? 0 : g.block <= 8 ? 1 : 2;
  using One = std::conditional_t<std::is_same_v<T, float> && (kDim == 64 || kDim == 128),
                                 OneHead<kDim == 64 ? 64 : 128>, TensorHeads<T, kDim, 1>>;
  using Eight = TensorHeads<T, kDim, 1>;
  using Sixteen = TensorHeads<T, kDim, 2>;
  const Fetch fetch = !tma ? kCopy : g.scores ? kTmaOnce : kTmaKeep;
  auto kernel_of = [&](auto heads) {
    using Heads = typename decltype(heads)::type;
    return fetch == kCopy      ? attend_kernel<T, kDim, Heads, kCopy>
           : fetch == kTmaKeep ? attend_kernel<T, kDim, Heads, kTmaKeep>
                               : attend_kernel<T, kDim, Heads, kTmaOnce>;
  };
  auto* kernel = kind == 0   ? kernel_of(Named<One>{})
                 : kind == 1 ? kernel_of(Named<Eight>{})
                             : kernel_of(Named<Sixteen>{});
  // one request per kernel and device
  constexpr int kMost = 64;
  static std::atomic<bool> ready[kMost][9];
  int dev = 0;
  IDEV_CUDA(cudaGetDevice(&dev));
  std::atomic<bool>* known = dev < kMost ? &ready[dev][3 * fetch + kind] : nullptr;
  if (!known || !known->load(std::memory_order_relaxed)) {
    IDEV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem));
    if (known) known->store(true, std::memory_order_relaxed);
  }
  launch_pdl(kernel, dim3(grid), dim3(kWarps * 32), L::kSmem, st, g, k_map, v_map);
}

// One fp32 head per key head runs on the CUDA cores, in rows of 64 or 128.
template <typename T>
constexpr bool one_head(int64_t group) {
  return std::is_same_v<T, float> && group == 1;
}

template <typename T>
void launch_attend_any(const AttendArgs& g, cudaStream_t st) {
  const int d = g.a.kv.head_dim;
  if (d <= 64) launch_attend_dim<T, 64>(g, st);
  else if (d <= 96 && !one_head<T>(g.group)) launch_attend_dim<T, 96>(g, st);
  else if (d <= 128) launch_attend_dim<T, 128>(g, st);
  else if (d <= 192) launch_attend_dim<T, 192>(g, st);
  else launch_attend_dim<T, 256>(g, st);
}

// Positions per tile and resident blocks per SM of the kernel for a head_dim.
struct Shape {
  int tile, blocks;
};
template <typename T>
Shape shape_of(int d, int64_t group) {
  auto of = [](auto l) { return Shape{decltype(l)::kTile, decltype(l)::kBlocks}; };
  return d <= 64    ? of(Layout<T, 64>())
         : d <= 96 && !one_head<T>(group) ? of(Layout<T, 96>())
         : d <= 128 ? of(Layout<T, 128>())
         : d <= 192 ? of(Layout<T, 192>())
                    : of(Layout<T, 256>());
}

}  // namespace paged
}  // namespace inferc_dev
