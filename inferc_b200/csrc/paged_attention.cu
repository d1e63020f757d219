// Attention of one new token per sequence over the paged cache: entry points,
// and what follows the reading of the cache: the join of sequences that several
// warps read and the running sums of attention weights. paged_attention.cuh reads the cache.
#include <algorithm>
#include <string>

#include "paged_attention.cuh"

namespace inferc_dev {
namespace paged {
namespace {

constexpr int kSMs = 148;  // B200; elsewhere the grid runs in waves
constexpr int kWholeTiles = 16;
constexpr int kJoinThreads = 128;

// Tiles of one head block: of all sequences, and (*ahead) of those before b. By
// the whole block; the lengths may be read while attend_kernel still runs.
__device__ __forceinline__ int64_t all_tiles(const AttendArgs& g, int64_t b, int64_t* ahead_out,
                                             int64_t* s_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t all = 0, ahead = 0;
  for (int i = threadIdx.x; i < (int)g.a.kv.batch; i += kJoinThreads) {
    const int64_t n = (seq_len(g.a, i) + g.tile - 1) / g.tile;
    all += n;
    if (i < b) ahead += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
  }
  if (lane == 0) s_sum[warp] = all, s_sum[kJoinThreads / 32 + warp] = ahead;
  __syncthreads();
  all = ahead = 0;
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) {
    all += s_sum[i];
    ahead += s_sum[kJoinThreads / 32 + i];
  }
  *ahead_out = ahead;
  return all;
}

// Joins what several warps left of a (sequence, head block):
//   M = max m_i,  out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
// Several blocks per head block (`of`), each for some of its columns. Where
// those are fewer than the warps, the jobs are all (sequence, head block)s and
// the parts follow from the lengths, which are read while attend_kernel still
// runs; else a job is a warp that left a first part, and what it wrote. Bound by
// latency: each thread takes four columns of a head and every `shares`-th part
// and fetches four parts at once, so that up to 32 to 128 parts (by the columns)
// cost one round trip, and the shares meet in shared memory.
template <typename T>
__device__ __forceinline__ void join(const AttendArgs& g, int job, bool by_warp, int part, int of,
                                     float4* s_o, float2* s_ml, int64_t* s_sum) {
  constexpr int kAtOnce = 4;
  const InfercPagedKv& kv = g.a.kv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = (int)kv.kv_heads * g.blocks, d = kv.head_dim;
  int64_t b;
  int head;
  Parts parts;
  if (by_warp) {
    pdl_wait();
    const int4 left = g.jobs[job];
    if (left.x < 0) return;
    b = left.x;
    head = left.y;
    parts = parts_within(job, left.z, g.warps);
  } else {
    b = job / heads;
    head = job - (int)b * heads;
    int64_t ahead;
    const int64_t all = all_tiles(g, b, &ahead, s_sum);
    const int64_t tiles = (seq_len(g.a, b) + g.tile - 1) / g.tile;
    if (tiles > 0)
      parts = parts_of(ahead * heads + head * tiles, tiles, all * heads,
                       warps_used(all * heads, g.warps));
    pdl_wait();
    if (tiles == 0 || parts.count == 1) return;
  }

  const int hk = head / g.blocks, q0 = hk * g.group + (head - hk * g.blocks) * g.block;
  const int cols = min(g.block, hk * g.group + g.group - q0);
  const int quads = d / 4, items = cols * quads;  // float4s of the result
  const int item1 = items * (part + 1) / of;
  for (int base = items * part / of; base < item1; base += kJoinThreads) {
    const int n = min(item1 - base, kJoinThreads);
    const int shares = min(kJoinThreads / n, 32);
    const int share = tid / n, item = base + tid - share * n;
    const int h = item / quads, quad = item - h * quads;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (share < shares) {
      for (int i0 = share; i0 < parts.count; i0 += kAtOnce * shares) {
        float2 ml[kAtOnce];
        float4 x[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int i = i0 + u * shares;
          ml[u] = make_float2(-INFINITY, 0.f);
          x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < parts.count) {
            const int64_t row = parts.slot(i) * g.block + h;
            ml[u] = reinterpret_cast<const float2*>(g.part_ml)[row];
            x[u] = reinterpret_cast<const float4*>(g.part_o + row * d)[quad];
          }
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) top = fmaxf(top, ml[u].x);
        const float to = top == -INFINITY ? 0.f : top;
        const float keep = ex2(m - to);
        m = top;
        l *= keep;
        o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const float f = ex2(ml[u].x - to);
          l += f * ml[u].y;
          o.x += f * x[u].x;
          o.y += f * x[u].y;
          o.z += f * x[u].z;
          o.w += f * x[u].w;
        }
      }
    }
    s_ml[tid] = make_float2(m, l);
    s_o[tid] = o;
    __syncthreads();
    auto finish = [&](int h, int quad, float l, float4 o) {
      const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: every page was bad
      T* out = reinterpret_cast<T*>(g.out) + b * g.o_batch + (q0 + h) * g.o_head + quad * 4;
      out[0] = T(o.x * inv);
      out[1] = T(o.y * inv);
      out[2] = T(o.z * inv);
      out[3] = T(o.w * inv);
    };
    if (shares > 8) {  // a warp per item, a lane per share
      for (int i = warp; i < n; i += kJoinThreads / 32) {
        float2 ml = make_float2(-INFINITY, 0.f);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (lane < shares) ml = s_ml[lane * n + i], x = s_o[lane * n + i];
        const float top = warp_max(ml.x), f = ex2(ml.x - (top == -INFINITY ? 0.f : top));
        const float sum = warp_sum(f * ml.y);
        x.x = warp_sum(f * x.x);
        x.y = warp_sum(f * x.y);
        x.z = warp_sum(f * x.z);
        x.w = warp_sum(f * x.w);
        const int h = (base + i) / quads;
        if (lane == 0) finish(h, base + i - h * quads, sum, x);
      }
    } else if (share == 0) {
      float top = m;
      for (int s = 1; s < shares; ++s) top = fmaxf(top, s_ml[s * n + tid].x);
      const float to = top == -INFINITY ? 0.f : top;
      const float keep = ex2(m - to);
      l *= keep;
      o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
      for (int s = 1; s < shares; ++s) {
        const float2 ml = s_ml[s * n + tid];
        const float4 x = s_o[s * n + tid];
        const float f = ex2(ml.x - to);
        l += f * ml.y;
        o.x += f * x.x;
        o.y += f * x.y;
        o.z += f * x.z;
        o.w += f * x.w;
      }
      finish(h, quad, l, o);
    }
    __syncthreads();
  }
}

// (M, 1 / L) of `cols` heads from row `r` on, to stats, by one warp.
__device__ __forceinline__ void head_stats(const AttendArgs& g, const Parts& parts, int cols,
                                           int64_t r, float2* stats) {
  const int lane = threadIdx.x & 31;
  // lanes h and h + 16 take head h, every second part each
  const int mine = lane & 15;
  float2 st = make_float2(0.f, 0.f);
  if (parts.count == 1) {
    if (mine < cols) st = reinterpret_cast<const float2*>(g.stats)[r + mine];
  } else {
    float m = -INFINITY, l = 0.f;
    if (mine < cols)
#pragma unroll 4
      for (int p = lane >> 4; p < parts.count; p += 2) {
        const float2 ml =
            reinterpret_cast<const float2*>(g.part_ml)[parts.slot(p) * g.block + mine];
        const float top = fmaxf(m, ml.x), to = top == -INFINITY ? 0.f : top;
        l = l * ex2(m - to) + ml.y * ex2(ml.x - to);
        m = top;
      }
    const float top = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    const float to = top == -INFINITY ? 0.f : top;
    l *= ex2(m - to);
    // both lanes add in the same order
    const float other = __shfl_xor_sync(0xffffffffu, l, 16);
    l = lane < 16 ? l + other : other + l;
    st = make_float2(to, l == 0.f ? 0.f : 1.f / l);
  }
  __syncwarp();
  if (lane < cols) stats[lane] = st;
  __syncwarp();
}

// Positions [j0, n) of one key head: sum[j] += the weights of `cols` heads, whose
// scores are `stride` floats apart; 32 consecutive positions a load, four loads
// of a head at once.
__device__ __forceinline__ void add_positions(const float* s, int64_t stride, int cols, float* sum,
                                              int j0, int n, const float2* stats) {
  s += j0 + (threadIdx.x & 31);
  sum += j0 + (threadIdx.x & 31);
  int left = n - j0 - (int)(threadIdx.x & 31);  // positions from this lane's on
  for (; __any_sync(0xffffffffu, left > 0); left -= 128, s += 128, sum += 128) {
    float p[4] = {0.f, 0.f, 0.f, 0.f};
    const float* row = s;
#pragma unroll 4
    for (int c = 0; c < cols; ++c, row += stride) {
      const float2 st = stats[c];
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = left > 32 * u ? row[32 * u] : -INFINITY;
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] += ex2(x[u] - st.x) * st.y;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (left > 32 * u) sum[32 * u] += p[u];
  }
}

// Adds each position's softmax weight, 2^(s - M) / L summed over the query
// heads of its key head in their order, to the running sum. The tiles are cut
// among `warps` warps as they were among attend_kernel's, four tiles (128
// positions) at least; where one of those began is in g.starts, so that nothing
// is searched for. A head's M and L come from its parts where it was cut (each
// lane takes some of them), else from what its warp left.
__device__ __forceinline__ void add_weights(const AttendArgs& g, int64_t i, int64_t warps,
                                            float2* stats, int64_t* s_sum) {
  const InfercPagedKv& kv = g.a.kv;
  const int heads = (int)kv.kv_heads * g.blocks;
  const int64_t q_heads = kv.kv_heads * g.group;
  int64_t ahead;
  const int64_t total = all_tiles(g, 0, &ahead, s_sum) * heads;
  const int64_t n = min(warps, (total + 3) / 4);
  int64_t used = 1, t = 0, t1 = 0, w = 0, w0 = 0, w1 = 0;
  if (i < n) {
    used = warps_used(total, g.warps);
    t = first_tile(i, total, n);
    t1 = first_tile(i + 1, total, n);
    w = owner_of(t, total, used);
    w0 = first_tile(w, total, used);
    w1 = first_tile(w + 1, total, used);
  }
  pdl_wait();
  if (t == t1) return;
  const int4 start = g.starts[w];
  if (start.x >= (int)kv.batch) return;  // that warp found no tile: the lengths changed
  // the head block that holds tile t, its place there
  int b = start.x, head = start.y;
  int64_t from = start.z + (t - w0);
  int len = seq_len(g.a, b), tiles = (len + g.tile - 1) / g.tile;
  auto next = [&]() {
    if (++head < heads) return;
    head = 0;
    tiles = 0;
    while (tiles == 0 && ++b < (int)kv.batch) {
      len = seq_len(g.a, b);
      tiles = (len + g.tile - 1) / g.tile;
    }
  };
  while (b < (int)kv.batch && from >= tiles) {
    from -= tiles;
    next();
  }
  // (b stays below batch unless the lengths change under the kernel)
  for (; t < t1 && b < (int)kv.batch; next(), from = 0) {
    const int64_t upto = min((int64_t)tiles, from + (t1 - t));
    const int64_t head0 = t - from;  // tile 0 of this head block
    t += upto - from;
    if (head % g.blocks) continue;  // summed with the first block of its key head
    const int h = head / g.blocks;
    const int n = (int)min((int64_t)len, upto * g.tile);
    const int64_t r = b * q_heads + (int64_t)h * g.group;
    const float* s = g.scores + r * g.capacity;
    float* sum = g.w + b * g.w_batch + h * g.w_head;
    for (int i0 = 0; i0 < g.group; i0 += g.block) {
      const int cols = min(g.block, g.group - i0);
      const int64_t t0 = head0 + i0 / g.block * tiles;
      Parts parts{0, 1};
      if (g.part_ml && (t0 < w0 || t0 + tiles > w1)) parts = parts_of(t0, tiles, total, used);
      head_stats(g, parts, cols, r + i0, stats);
      add_positions(s + i0 * g.capacity, g.capacity, cols, sum, (int)from * g.tile, n, stats);
    }
  }
}

// Behind attend_kernel: the first jobs * of blocks join, the others add weights.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads, 6) finish_kernel(
    const __grid_constant__ AttendArgs g, int jobs, bool by_warp, int of, int64_t sum_warps) {
  __shared__ float4 s_o[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads];
  __shared__ int64_t s_sum[kJoinThreads / 16];
  pdl_launch_dependents();
  if ((int)blockIdx.x < jobs * of) {
    const int job = blockIdx.x / of;
    join<T>(g, job, by_warp, blockIdx.x - job * of, of, s_o, s_ml, s_sum);
  } else {
    const int warp = threadIdx.x >> 5;
    add_weights(g, (int64_t)(blockIdx.x - jobs * of) * (kJoinThreads / 32) + warp, sum_warps,
                s_ml + warp * 16, s_sum);
  }
}

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

int block_of(int64_t group) {
  const int64_t blocks = (group + 15) / 16;
  return (int)((group + blocks - 1) / blocks);
}

// Sizes of the work and of its scratch; those parts of AttendArgs that the
// sizes decide.
struct Plan {
  AttendArgs g{};
  bool cut;  // a sequence may be read by several warps
  int64_t bytes = 0;
};

Plan plan_of(const InfercPagedKv& kv, int64_t q_heads, bool weights, char* ws) {
  Plan p;
  AttendArgs& g = p.g;
  g.group = (int)(q_heads / kv.kv_heads);
  g.block = block_of(g.group);
  g.blocks = (g.group + g.block - 1) / g.block;
  g.capacity = (kv.max_pages * kv.page_size + 3) / 4 * 4;
  const Shape shape = kv.dtype == F32   ? shape_of<float>(kv.head_dim, g.group)
                      : kv.dtype == F16 ? shape_of<__half>(kv.head_dim, g.group)
                                        : shape_of<__nv_bfloat16>(kv.head_dim, g.group);
  g.tile = shape.tile;
  const int64_t tiles = (g.capacity + g.tile - 1) / g.tile;
  const int64_t most = kv.batch * kv.kv_heads * g.blocks * tiles;
  g.warps = std::max<int64_t>(1, std::min<int64_t>((int64_t)kSMs * shape.blocks * kWarps, most));
  // Short sequences of few heads: a block each (see attend_kernel). At most one wave of blocks,
  // whose warps take four tiles each at most; one request of 160 positions and 12 fp32 heads:
  // 5.1 us against 6.9 us. (Longer ones would gain where all lengths are alike: 32 x 8 bf16
  // key heads of 2000 positions 45.7 against 52.4 us; one long sequence among short ones, or few
  // of them, loses: 1 x 8 of 1000 15.6 against 9.3 us.)
  const int64_t pairs = kv.batch * kv.kv_heads;
  g.whole = g.blocks == 1 && tiles <= kWholeTiles && pairs <= kSMs * shape.blocks;
  if (g.whole) g.warps = pairs * kWarps;
  p.cut = tiles > 1 && !g.whole;
  auto take = [&](int64_t bytes) {
    char* at = ws + p.bytes;
    p.bytes += align16(bytes);
    return at;
  };
  if (p.cut) {
    g.jobs = reinterpret_cast<int4*>(take(g.warps * 16));
    g.part_ml = reinterpret_cast<float*>(take(2 * g.warps * g.block * 8));
    g.part_o = reinterpret_cast<float*>(take(2 * g.warps * g.block * kv.head_dim * 4));
  }
  if (weights && !g.whole) {
    g.starts = reinterpret_cast<int4*>(take(g.warps * 16));
    g.stats = reinterpret_cast<float*>(take(kv.batch * q_heads * 8));
  }
  if (weights) {
    g.scores = reinterpret_cast<float*>(take(kv.batch * q_heads * g.capacity * 4));
  }
  return p;
}

void check(const InfercPagedKv* kv, int64_t q_heads, bool weights) {
  check_kv(kv, "PagedDecodeAttention");
  IDEV_CHECK_ARG(q_heads >= 1 && q_heads <= 65535 && q_heads % kv->kv_heads == 0,
                 "PagedDecodeAttention: q_heads must be a multiple of kv_heads");
  IDEV_CHECK_ARG(kv->batch * q_heads <= INT32_MAX,
                 "PagedDecodeAttention: too many heads in one call");
  // the scratch for weights: no more bytes than a device has, let alone than 64 bits count
  IDEV_CHECK_ARG(!weights || kv->batch * q_heads * (kv->max_pages * kv->page_size >> 10) < 1 << 30,
                 "PagedDecodeAttention: too many positions in one call to keep weights");
}

template <typename T>
void run(const Plan& p, cudaStream_t st) {
  const AttendArgs& g = p.g;
  const InfercPagedKv& kv = g.a.kv;
  launch_attend<T>(g, st);
  if (g.whole || (!p.cut && !g.w)) return;
  int64_t jobs = 0;
  int of = 1;
  bool by_warp = false;
  if (p.cut) {
    const int64_t pairs = kv.batch * kv.kv_heads * g.blocks;
    by_warp = pairs > g.warps;
    jobs = by_warp ? g.warps : pairs;
    // few jobs: several blocks each, of four float4s of the result at least
    of = (int)std::min<int64_t>(g.block * (kv.head_dim / 4) / 4,
                                std::max<int64_t>(1, 4 * kSMs / jobs));
    of = std::max(of, 1);
  }
  // sums: what the SMs hold
  const int64_t sum_blocks = g.w ? 6 * kSMs : 0;
  const int64_t grid = jobs * of + sum_blocks;
  launch_pdl(finish_kernel<T>, dim3((unsigned)grid), dim3(kJoinThreads), 0, st, g, (int)jobs, by_warp,
             of, sum_blocks * (kJoinThreads / 32));
}

}  // namespace
}  // namespace paged
}  // namespace inferc_dev

using namespace inferc_dev;
using namespace inferc_dev::paged;

extern "C" {

int64_t inferc_dev_paged_decode_attention_workspace(const InfercPagedKv* kv, int64_t q_heads,
                                                    int with_weights) {
  int64_t bytes = -1;
  guard([&] {
    check(kv, q_heads, with_weights != 0);
    bytes = plan_of(*kv, q_heads, with_weights != 0, nullptr).bytes;
  });
  return bytes;
}

int inferc_dev_paged_decode_attention(const InfercPagedKv* kv, const void* q,
                                      int64_t q_batch_stride, int64_t q_head_stride,
                                      int64_t q_heads, float scale, void* out,
                                      int64_t out_batch_stride, int64_t out_head_stride,
                                      float* weights, int64_t weights_batch_stride,
                                      int64_t weights_head_stride, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  return guard([&] {
    const char* op = "PagedDecodeAttention";
    check(kv, q_heads, weights != nullptr);
    if (kv->batch == 0) return;
    check_rows(op, "query", q, q_batch_stride, q_head_stride, kv->dtype);
    check_rows(op, "output", out, out_batch_stride, out_head_stride, kv->dtype);
    check_apart(op, "output", kv->head_dim, {kv->batch, out_batch_stride},
                {q_heads, out_head_stride});
    if (weights)
      check_apart(op, "weights", kv->max_pages * kv->page_size, {kv->batch, weights_batch_stride},
                  {kv->kv_heads, weights_head_stride});
    Plan p = plan_of(*kv, q_heads, weights != nullptr, static_cast<char*>(workspace));
    IDEV_CHECK_ARG(workspace_bytes >= p.bytes && (p.bytes == 0 || (workspace && aligned16(workspace))),
                   "PagedDecodeAttention: the workspace is too small or not 16-byte aligned");
    AttendArgs& g = p.g;
    g.a.kv = *kv;
    g.a.page = FastDiv((uint32_t)kv->page_size);
    g.a.flag = range_flag_ptr();
    g.q = q;
    g.q_batch = q_batch_stride;
    g.q_head = q_head_stride;
    g.out = out;
    g.o_batch = out_batch_stride;
    g.o_head = out_head_stride;
    g.scale = scale * 1.4426950408889634f;
    g.w = weights;
    g.w_batch = weights_batch_stride;
    g.w_head = weights_head_stride;
    cudaStream_t st = as_stream(stream);
    if (kv->dtype == F32) run<float>(p, st);
    else if (kv->dtype == F16) run<__half>(p, st);
    else run<__nv_bfloat16>(p, st);
  });
}

}  // extern "C"
