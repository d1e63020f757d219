// Attention of one new token per sequence over the paged cache: the kernel
// that reads the cache. paged_attention.cu has the entry point, the join of
// cut sequences and the running sums; one file per element type instantiates
// this one.
//
// Mathematics. For a key head and the query heads that share it (a block of 8
// or 16), every warp walks its tiles of 16 positions with the running maximum
// m and sum l of the softmax:
//   S^T = K Q^T   (16 positions x heads),   m' = max(m, S),  P = 2^(S - m')
//   O^T = 2^(m - m') O^T + V^T P            (head_dim x heads)
// with scores in the log2 domain. The positions are the matrix instruction's
// rows and the heads its 8 columns, so the whole width is used from 8 heads
// per key head on, and one head per key head still costs only 1 / 2 of what
// 16 rows of queries would.
//
// What bounds it: every byte of K and V is read once and used for 2 flops per
// query head, so HBM. mma.sync is enough (at 8 heads, 0.1 PFLOP/s of it at
// full bandwidth); tcgen05 tiles would need 64 rows and a trip through tensor
// memory for each 16 positions.
//
// Layout. Each warp owns a ring of kSlots shared-memory slots, each 16 rows of
// K or V, filled by 16-byte cp.async some tiles ahead across the boundaries
// of heads and sequences, so that warps never wait for each other and the
// loads never drain. Rows are padded to an odd number of 16-byte pieces (fp32:
// by 16 words), which keeps ldmatrix (fp32: 16-byte loads) free of bank
// conflicts. Rows past a sequence's end, or on a page that does not exist,
// are filled with zeros and their scores set to -inf, so what the page holds
// there is never used.
//
// Numbers. 16-bit products are exact in fp32. P goes into the second product
// as two 16-bit pieces, P = hi + lo, so that rounding it adds less than the
// result's own rounding; fp16 P carries a factor 2^10 (in m), which keeps
// weights down to 2^-34 of the largest. fp32 operands are taken as two tf32
// pieces each, three products (big big, big small, small big): 2^-22 relative.
#pragma once

#include "paged.cuh"

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
  int64_t warps;    // in the grid
  int least;        // tiles per warp, see warps_used
  int64_t* before;  // [batch + 1] tiles before each sequence
  int32_t* jobs;    // [warps, 2] (sequence, head block) whose first part this warp left; -1
  float* part_ml;   // [2 warps, block, 2] maximum and sum of a part
  float* part_o;    // [2 warps, block, head_dim]
  float* scores;    // [batch, q_heads, capacity] or nullptr
  float* stats;     // [batch, q_heads, 2] maximum and 1 / sum (with scores)
  int64_t capacity;
  float* w;
  int64_t w_batch, w_head;
};

constexpr int kWarps = 4;  // per block

template <typename T, int kDim>
struct Layout {
  static constexpr bool kWide = sizeof(T) == 4;
  // row stride in bytes; both operands of fp32 share the larger one's slot
  static constexpr int kRowK = kWide ? (kDim + 16) * 4 : kDim * 2 + 16;
  static constexpr int kRowV = kWide ? (kDim + 8) * 4 : kDim * 2 + 16;
  static constexpr int kSlot = kTile * kRowK;
  // Two blocks (8 warps) per SM with as many slots as their shares of the
  // 227 KB allow, one block where that would leave fewer than three.
  static constexpr int kTwo = 112 * 1024 / (kWarps * kSlot + 64);
  static constexpr int kBlocks = kTwo >= 3 ? 2 : 1;
  static constexpr int kFit = kBlocks == 2 ? kTwo : 220 * 1024 / (kWarps * kSlot + 64);
  static constexpr int kSlots = kFit > 8 ? 8 : kFit;
  static constexpr int kSmem = kWarps * kSlots * (kSlot + 16);
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
struct Cursor {
  int b, head, tile, tiles, len;  // head: key head x head block

  // Goes to sequence b or the first one after it that holds something.
  __device__ __forceinline__ void open(const AttendArgs& g, int first) {
    b = first;
    head = tile = tiles = 0;
    for (; b < (int)g.a.kv.batch; ++b) {
      len = seq_len(g.a, b);
      tiles = (len + kTile - 1) / kTile;
      if (tiles) return;
    }
  }
  __device__ __forceinline__ void next(const AttendArgs& g, int heads) {
    if (++tile < tiles) return;
    tile = 0;
    if (++head < heads) return;
    open(g, b + 1);
  }
};

template <typename T, int kDim, int kCols>
__global__ void __launch_bounds__(kWarps * 32, Layout<T, kDim>::kBlocks)
    attend_kernel(const __grid_constant__ AttendArgs g) {
  using L = Layout<T, kDim>;
  constexpr bool kWide = L::kWide;
  constexpr int kElem = sizeof(T), kThreads = kWarps * 32;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int64_t s_before[kThreads + 1];
  __shared__ int64_t s_warp[kWarps];
  const InfercPagedKv& kv = g.a.kv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  const int heads = (int)kv.kv_heads * g.blocks;
  const int batch = (int)kv.batch;
  const int d = kv.head_dim;
  pdl_launch_dependents();

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
  int64_t total = 0, ahead = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) ahead += s_warp[i];
    total += s_warp[i];
  }
  s_before[tid] = ahead + scan - mine;
  if (tid == 0) s_before[kThreads] = total;
  if (blockIdx.x == 0 && g.before) {
    int64_t at = ahead + scan - mine;
    for (int b = run0; b < run1; ++b) {
      g.before[b] = at;
      at += (int64_t)((seq_len(g.a, b) + kTile - 1) / kTile) * heads;
    }
    if (tid == 0) g.before[batch] = total;
  }
  // A sequence of length 0 gives zeros.
  for (int64_t b = blockIdx.x; b < batch; b += gridDim.x) {
    if (seq_len(g.a, b) > 0) continue;
    const int pieces = d / 8;
    const int q_heads = (int)kv.kv_heads * g.group;
    const float zero[8] = {};
    for (int i = tid; i < q_heads * pieces; i += kThreads)
      store8(reinterpret_cast<T*>(g.out) + b * g.o_batch + (int64_t)(i / pieces) * g.o_head +
                 (i % pieces) * 8,
             zero);
  }
  __syncthreads();

  const int64_t w = (int64_t)blockIdx.x * kWarps + warp;
  if (g.jobs && lane == 0 && w < g.warps) g.jobs[2 * w] = -1;
  const int64_t used = warps_used(total, g.warps, g.least);
  if (w >= used) return;
  const int64_t t0 = first_tile(w, total, used);
  const int count = (int)(first_tile(w + 1, total, used) - t0);

  // The tile t0: the thread whose run holds it, then the sequence, then the head.
  Cursor load;
  {
    int lo = 0, hi = kThreads;  // s_before[lo] <= t0 < s_before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (s_before[mid] <= t0) lo = mid;
      else hi = mid;
    }
    int64_t left = t0 - s_before[lo];
    load.open(g, min(lo * run, batch));
    while (load.b < batch && left >= (int64_t)load.tiles * heads) {
      left -= (int64_t)load.tiles * heads;
      load.open(g, load.b + 1);
    }
    if (load.b >= batch) return;  // only if the lengths change under the kernel
    load.head = (int)(left / load.tiles);
    load.tile = (int)(left % load.tiles);
  }
  Cursor use = load;

  unsigned char* ring = smem + warp * L::kSlots * (L::kSlot + 16);
  uint32_t* masks = reinterpret_cast<uint32_t*>(ring + L::kSlots * L::kSlot);
  const uint32_t ring_addr = smem_addr(ring);
  if (d < kDim)  // columns that no copy fills
    for (int i = lane * 16; i < L::kSlots * L::kSlot; i += 32 * 16)
      *reinterpret_cast<uint4*>(ring + i) = make_uint4(0, 0, 0, 0);
  __syncwarp();

  // ---- loads: one slot at a time, the keys of a tile, then its values
  constexpr int kPieces = kDim * kElem / 16;  // 16-byte pieces of a full row
  constexpr int kLanes = kPieces <= 8 ? 8 : kPieces <= 16 ? 16 : 32;
  constexpr int kRowsAt = 32 / kLanes, kSteps = kTile / kRowsAt;
  constexpr int kTurns = (kPieces + 31) / 32;
  const int pieces = d * kElem / 16, piece = lane % kLanes;
  int loaded = 0, slot_in = 0;
  bool values = false;
  int64_t off_v = 0;
  bool row_ok = false;
  const char* k_base = reinterpret_cast<const char*>(kv.k) + piece * 16;
  const char* v_base = reinterpret_cast<const char*>(kv.v) + piece * 16;
  auto fill = [&]() {
    if (loaded < count && load.b < batch) {
      int64_t off;
      if (!values) {
        const int j = load.tile * kTile + (lane & 15);
        row_ok = j < load.len;
        int page = 0;
        uint32_t slot = 0;
        if (row_ok) {
          const uint32_t index = g.a.page.div(j);
          slot = j - index * g.a.page.d;
          page = page_of(g.a, kv.page_table + load.b * kv.table_stride, index);
          row_ok = page >= 0;
        }
        const int hk = load.head / g.blocks;
        off = row_ok ? (page * kv.k_page_stride + slot * kv.k_token_stride +
                        hk * kv.k_head_stride) * kElem
                     : 0;
        off_v = row_ok ? (page * kv.v_page_stride + slot * kv.v_token_stride +
                          hk * kv.v_head_stride) * kElem
                       : 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, row_ok);
        if (lane == 0) masks[slot_in] = mask;
      } else {
        off = off_v;
      }
      const char* base = values ? v_base : k_base;
      const uint32_t dst = ring_addr + slot_in * L::kSlot + piece * 16;
      const int stride = values ? L::kRowV : L::kRowK;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int row = i * kRowsAt + lane / kLanes;
        const int64_t from = __shfl_sync(0xffffffffu, off, row);
        const bool ok = __shfl_sync(0xffffffffu, (int)row_ok, row);
#pragma unroll
        for (int t = 0; t < kTurns; ++t)
          if (piece + 32 * t < pieces)
            copy16(dst + row * stride + 512 * t, base + from + 512 * t, ok);
      }
      if (values) {
        ++loaded;
        load.next(g, heads);
      }
      values = !values;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    slot_in = slot_in + 1 == L::kSlots ? 0 : slot_in + 1;
  };
#pragma unroll 1
  for (int i = 0; i < L::kSlots; ++i) fill();

  // ---- the state of one (sequence, head block)
  constexpr int kKSteps = kWide ? kDim / 8 : kDim / 16;  // steps along head_dim
  constexpr int kMTiles = kDim / 16;                     // blocks of 16 columns of V
  constexpr float kLift = std::is_same_v<T, __half> ? 10.f : 0.f;
  uint32_t qf[kCols][kKSteps][2];
  float o[kCols][kMTiles][4];
  float m[kCols][2], l[kCols][2];
  bool begins = false;
  int slot_out = 0;

#pragma unroll 1
  for (int t = 0; t < count && use.b < batch; ++t) {
    const int hk = use.head / g.blocks, q0 = hk * g.group + (use.head % g.blocks) * g.block;
    const int cols = min(g.block, hk * g.group + g.group - q0);
    if (t == 0 || use.tile == 0) {
      begins = use.tile == 0;
      const T* q = reinterpret_cast<const T*>(g.q) + use.b * g.q_batch + q0 * g.q_head;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int h = c * 8 + gid;
        const T* row = q + (int64_t)h * g.q_head;
#pragma unroll
        for (int s = 0; s < kKSteps; ++s) {
          if constexpr (kWide) {
            // columns are taken in the order the 16-byte loads of K give them
            const int at = (s >> 1) * 16 + tig * 4 + (s & 1) * 2;
            const bool in = h < cols && at < d;
            qf[c][s][0] = in ? __float_as_uint(row[at]) : 0u;
            qf[c][s][1] = in ? __float_as_uint(row[at + 1]) : 0u;
          } else {
            const int at = s * 16 + tig * 2;
            qf[c][s][0] = h < cols && at < d ? *reinterpret_cast<const uint32_t*>(row + at) : 0u;
            qf[c][s][1] =
                h < cols && at + 8 < d ? *reinterpret_cast<const uint32_t*>(row + at + 8) : 0u;
          }
        }
        m[c][0] = m[c][1] = -INFINITY;
        l[c][0] = l[c][1] = 0.f;
#pragma unroll
        for (int i = 0; i < kMTiles; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
      }
    }

    // ---- scores
    asm volatile("cp.async.wait_group %0;" ::"n"(L::kSlots - 1) : "memory");
    __syncwarp();
    const uint32_t k_addr = ring_addr + slot_out * L::kSlot;
    const unsigned char* k_ptr = ring + slot_out * L::kSlot;
    const uint32_t mask = masks[slot_out];
    float sc[kCols][4];
    if constexpr (!kWide) {
      float acc[kCols][2][4] = {};
      const uint32_t addr =
          k_addr + ((lane & 7) + ((lane >> 3) & 1) * 8) * L::kRowK + (lane >> 4) * 16;
#pragma unroll
      for (int s = 0; s < kKSteps; ++s) {
        uint32_t a[4];
        ldmatrix4(addr + s * 32, a);
#pragma unroll
        for (int c = 0; c < kCols; ++c) mma16<T>(acc[c][s & 1], a, qf[c][s][0], qf[c][s][1]);
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[c][i] = acc[c][0][i] + acc[c][1][i];
    } else {
      // two chains, so that a product need not wait for the one before
      float acc[kCols][2][4] = {};
      const unsigned char* r0 = k_ptr + gid * L::kRowK + tig * 16;
      const unsigned char* r1 = r0 + 8 * L::kRowK;
#pragma unroll
      for (int s = 0; s < kKSteps; s += 2) {
        const float4 x = *reinterpret_cast<const float4*>(r0 + s * 32);
        const float4 y = *reinterpret_cast<const float4*>(r1 + s * 32);
        uint32_t big[2][4], small[2][4];
        split_tf32(x.x, big[0][0], small[0][0]);
        split_tf32(y.x, big[0][1], small[0][1]);
        split_tf32(x.y, big[0][2], small[0][2]);
        split_tf32(y.y, big[0][3], small[0][3]);
        split_tf32(x.z, big[1][0], small[1][0]);
        split_tf32(y.z, big[1][1], small[1][1]);
        split_tf32(x.w, big[1][2], small[1][2]);
        split_tf32(y.w, big[1][3], small[1][3]);
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t b0, b1, s0, s1;
            split_tf32(__uint_as_float(qf[c][s + u][0]), b0, s0);
            split_tf32(__uint_as_float(qf[c][s + u][1]), b1, s1);
            mma_tf32(acc[c][1], small[u], b0, b1);
            mma_tf32(acc[c][1], big[u], s0, s1);
            mma_tf32(acc[c][0], big[u], b0, b1);
          }
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[c][i] = acc[c][0][i] + acc[c][1][i];
    }
    __syncwarp();
    fill();

    // ---- softmax: positions gid and gid + 8, heads 2 tig and 2 tig + 1 of each column block
    const bool ok0 = mask >> gid & 1, ok1 = mask >> (gid + 8) & 1;
    float top[kCols][2];
    bool grew = false;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      sc[c][0] = ok0 ? sc[c][0] * g.scale : -INFINITY;
      sc[c][1] = ok0 ? sc[c][1] * g.scale : -INFINITY;
      sc[c][2] = ok1 ? sc[c][2] * g.scale : -INFINITY;
      sc[c][3] = ok1 ? sc[c][3] * g.scale : -INFINITY;
      if (g.scores) {
        float* to = g.scores + (use.b * (int64_t)(kv.kv_heads * g.group) + q0 + c * 8 + tig * 2) *
                                   g.capacity + use.tile * kTile + gid;
        const int left = use.len - use.tile * kTile - gid;  // positions from this lane's on
        const int h = c * 8 + tig * 2;
        if (h < cols) {
          if (left > 0) to[0] = sc[c][0];
          if (left > 8) to[8] = sc[c][2];
        }
        if (h + 1 < cols) {
          if (left > 0) to[g.capacity] = sc[c][1];
          if (left > 8) to[g.capacity + 8] = sc[c][3];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(sc[c][i], sc[c][i + 2]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        top[c][i] = x - kLift;
        grew |= top[c][i] > m[c][i];
      }
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
        sc[c][i] = ex2(sc[c][i] - base);
        sc[c][i + 2] = ex2(sc[c][i + 2] - base);
        l[c][i] += sc[c][i] + sc[c][i + 2];
      }

    // ---- values
    slot_out = slot_out + 1 == L::kSlots ? 0 : slot_out + 1;
    asm volatile("cp.async.wait_group %0;" ::"n"(L::kSlots - 1) : "memory");
    __syncwarp();
    const uint32_t v_addr = ring_addr + slot_out * L::kSlot;
    const unsigned char* v_ptr = ring + slot_out * L::kSlot;
    if constexpr (!kWide) {
      uint32_t hi[kCols][2], lo[kCols][2];
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          split_pair16<T>(sc[c][2 * i], sc[c][2 * i + 1], hi[c][i], lo[c][i]);
          hi[c][i] = transpose8x8(hi[c][i]);
          lo[c][i] = transpose8x8(lo[c][i]);
        }
      const uint32_t addr =
          v_addr + ((lane & 7) + (lane >> 4) * 8) * L::kRowV + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int i = 0; i < kMTiles; ++i) {
        uint32_t a[4];
        ldmatrix4_trans(addr + i * 32, a);
#pragma unroll
        for (int c = 0; c < kCols; ++c) mma16<T>(o[c][i], a, lo[c][0], lo[c][1]);
#pragma unroll
        for (int c = 0; c < kCols; ++c) mma16<T>(o[c][i], a, hi[c][0], hi[c][1]);
      }
    } else {
      // P of positions (tig, tig + 4) of each half, head gid: from the lanes that hold them
      uint32_t b_big[kCols][2][2], b_small[kCols][2][2];
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int src = (tig + 4 * i) * 4 + (gid >> 1);
            const float x = __shfl_sync(0xffffffffu, sc[c][2 * half], src);
            const float y = __shfl_sync(0xffffffffu, sc[c][2 * half + 1], src);
            split_tf32(gid & 1 ? y : x, b_big[c][half][i], b_small[c][half][i]);
          }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const unsigned char* r0 = v_ptr + (half * 8 + tig) * L::kRowV + gid * 16;
        const unsigned char* r1 = r0 + 4 * L::kRowV;
#pragma unroll
        for (int i = 0; i < kMTiles; i += 2) {
          const float4 x = *reinterpret_cast<const float4*>(r0 + i * 64);
          const float4 y = *reinterpret_cast<const float4*>(r1 + i * 64);
          uint32_t big[2][4], small[2][4];
          split_tf32(x.x, big[0][0], small[0][0]);
          split_tf32(x.y, big[0][1], small[0][1]);
          split_tf32(y.x, big[0][2], small[0][2]);
          split_tf32(y.y, big[0][3], small[0][3]);
          split_tf32(x.z, big[1][0], small[1][0]);
          split_tf32(x.w, big[1][1], small[1][1]);
          split_tf32(y.z, big[1][2], small[1][2]);
          split_tf32(y.w, big[1][3], small[1][3]);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              mma_tf32(o[c][i + u], small[u], b_big[c][half][0], b_big[c][half][1]);
              mma_tf32(o[c][i + u], big[u], b_small[c][half][0], b_small[c][half][1]);
              mma_tf32(o[c][i + u], big[u], b_big[c][half][0], b_big[c][half][1]);
            }
        }
      }
    }
    __syncwarp();
    fill();
    slot_out = slot_out + 1 == L::kSlots ? 0 : slot_out + 1;

    // ---- the end of the sequence's head block, or of this warp's share
    const bool ends = use.tile + 1 == use.tiles;
    if (ends || t + 1 == count) {
      const bool whole = begins && ends;
      const int64_t part = 2 * w + (begins ? 1 : 0);
      if (begins && !ends && g.jobs && lane == 0) {
        g.jobs[2 * w] = use.b;
        g.jobs[2 * w + 1] = use.head;
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = l[c][i];
          x += __shfl_xor_sync(0xffffffffu, x, 4);
          x += __shfl_xor_sync(0xffffffffu, x, 8);
          x += __shfl_xor_sync(0xffffffffu, x, 16);
          const int h = c * 8 + tig * 2 + i;
          const float inv = x == 0.f ? 0.f : 1.f / x;  // 0: every page was bad
          if (h < cols) {
            if (gid == 0) {
              const float base = m[c][i] == -INFINITY ? 0.f : m[c][i];
              if (!whole) {
                g.part_ml[(part * g.block + h) * 2] = m[c][i];
                g.part_ml[(part * g.block + h) * 2 + 1] = x;
              } else if (g.stats) {
                const int64_t r = use.b * (int64_t)(kv.kv_heads * g.group) + q0 + h;
                g.stats[2 * r] = base;
                g.stats[2 * r + 1] = inv;
              }
            }
            T* out = reinterpret_cast<T*>(g.out) + use.b * g.o_batch + (q0 + h) * g.o_head;
            float* po = g.part_o + (part * g.block + h) * d;
#pragma unroll
            for (int j = 0; j < kMTiles; ++j)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int col = kWide ? (j >> 1) * 32 + gid * 4 + (j & 1) * 2 + half
                                      : j * 16 + half * 8 + gid;
                if (col < d) {
                  if (whole) out[col] = T(o[c][j][2 * half + i] * inv);
                  else po[col] = o[c][j][2 * half + i];
                }
              }
          }
        }
      }
    }
    use.next(g, heads);
  }
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

template <typename T, int kDim>
void launch_attend_dim(const AttendArgs& g, cudaStream_t st) {
  using L = Layout<T, kDim>;
  static_assert(L::kSlots >= 3, "the ring needs three slots");
  const unsigned grid = (unsigned)((g.warps + kWarps - 1) / kWarps);
  auto* kernel = g.block <= 8 ? attend_kernel<T, kDim, 1> : attend_kernel<T, kDim, 2>;
  IDEV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem));
  kernel<<<grid, kWarps * 32, L::kSmem, st>>>(g);
  IDEV_LAUNCHED();
}


template <typename T>
void launch_attend_any(const AttendArgs& g, cudaStream_t st) {
  const int d = g.a.kv.head_dim;
  if (d <= 64) launch_attend_dim<T, 64>(g, st);
  else if (d <= 96) launch_attend_dim<T, 96>(g, st);
  else if (d <= 128) launch_attend_dim<T, 128>(g, st);
  else if (d <= 192) launch_attend_dim<T, 192>(g, st);
  else launch_attend_dim<T, 256>(g, st);
}

template <typename T>
int blocks_per_sm(int d) {
  return d <= 64    ? Layout<T, 64>::kBlocks
         : d <= 96  ? Layout<T, 96>::kBlocks
         : d <= 128 ? Layout<T, 128>::kBlocks
         : d <= 192 ? Layout<T, 192>::kBlocks
                    : Layout<T, 256>::kBlocks;
}

}  // namespace paged
}  // namespace inferc_dev
