// The paged cache's writers: per-head RMS norm with rotary positions, append
// of new tokens, and eviction by accumulated attention weight
// (inferc_dev_qk_norm_rotary, inferc_dev_paged_kv_append,
// inferc_dev_paged_kv_evict). All three move rows of head_dim values and do
// a few operations per value, so they are bound by HBM, and by launch latency
// when few tokens are in flight.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <string>

#include "paged.cuh"

namespace inferc_dev {

namespace paged {

// [0]: an index pointed outside its buffer; [1]: a wait for a copy gave up
__device__ int g_flags[2];

int* range_flag_ptr() {
  constexpr int kMost = 64;
  static std::atomic<int*> known[kMost];  // one lookup per device
  int dev = 0;
  IDEV_CUDA(cudaGetDevice(&dev));
  int* p = dev < kMost ? known[dev].load(std::memory_order_relaxed) : nullptr;
  if (!p) {
    IDEV_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_flags));
    if (dev < kMost) known[dev].store(p, std::memory_order_relaxed);
  }
  return p;
}

int elem_bytes(int dtype) { return dtype == F32 ? 4 : 2; }

void check_rows(const char* op, const char* what, const void* p, int64_t stride_a,
                int64_t stride_b, int dtype) {
  const int64_t unit = 16 / elem_bytes(dtype);
  IDEV_CHECK_ARG(p != nullptr, std::string(op) + ": null " + what);
  IDEV_CHECK_ARG(aligned16(p) && stride_a % unit == 0 && stride_b % unit == 0,
                 std::string(op) + ": " + what + " must be 16-byte aligned, its strides too");
}

static void check_dtype_dim(const char* op, int dtype, int64_t head_dim) {
  IDEV_CHECK_ARG(dtype == F32 || dtype == F16 || dtype == BF16,
                 std::string(op) + ": dtype must be float, float16 or bfloat16");
  IDEV_CHECK_ARG(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0,
                 std::string(op) + ": head_dim must be a multiple of 8 in [8, 256]");
}

void check_kv(const InfercPagedKv* kv, const char* op) {
  const std::string o = std::string(op) + ": ";
  IDEV_CHECK_ARG(kv != nullptr, o + "null cache descriptor");
  check_dtype_dim(op, kv->dtype, kv->head_dim);
  IDEV_CHECK_ARG(kv->num_pages >= 0 && kv->num_pages <= INT32_MAX && kv->kv_heads >= 1 &&
                     kv->kv_heads <= 65535 && kv->page_size >= 1 && kv->batch >= 0 &&
                     kv->batch <= (1 << 20) && kv->max_pages >= 0,
                 o + "bad cache shape");
  IDEV_CHECK_ARG(kv->page_size <= INT32_MAX && kv->max_pages <= INT32_MAX &&
                     kv->page_size * kv->max_pages <= INT32_MAX,
                 o + "page_size * max_pages must stay below 2^31");
  IDEV_CHECK_ARG(kv->table_stride >= kv->max_pages, o + "page table rows overlap");
  if (kv->batch == 0) return;
  IDEV_CHECK_ARG(kv->lens != nullptr && (kv->max_pages == 0 || kv->page_table != nullptr),
                 o + "null page table or lengths");
  if (kv->num_pages == 0) return;
  check_rows(op, "key cache", kv->k, kv->k_page_stride, kv->k_head_stride, kv->dtype);
  check_rows(op, "value cache", kv->v, kv->v_page_stride, kv->v_head_stride, kv->dtype);
  check_rows(op, "key cache", kv->k, kv->k_token_stride, 0, kv->dtype);
  check_rows(op, "value cache", kv->v, kv->v_token_stride, 0, kv->dtype);
}

}  // namespace paged

int read_and_clear_paged() {
  int v[2] = {0, 0};
  IDEV_CUDA(cudaMemcpyFromSymbol(v, paged::g_flags, sizeof v));
  if (v[0] | v[1]) {
    const int z[2] = {0, 0};
    IDEV_CUDA(cudaMemcpyToSymbol(paged::g_flags, z, sizeof z));
  }
  return v[0] | v[1] << 1;
}

namespace paged {
namespace {

// --------------------------------------------------- norm, rotation, append

struct Heads {
  const void* src;
  void* dst;
  int64_t src_token, src_head, dst_token, dst_head;
  int heads;
};

struct RowArgs {
  Args a;  // a.kv.batch == 0: no cache, keys go to k.dst
  InfercHeadRotary rot;
  Heads q, k, v;
  const int32_t* cu;
  int64_t tokens;
  int d;
  bool norm_q, norm_k, turn;
};

// Largest b in [0, n) with cu[b] <= t, one warp, 32 probes a step; -1 if none.
__device__ __forceinline__ int64_t find_seq(const int32_t* cu, int64_t n, int64_t t, int lane) {
  int64_t lo = 0, size = n;
  while (size > 1) {
    const int64_t step = (size + 31) / 32;
    const int64_t at = lo + lane * step;
    const bool below = lane * step < size && cu[at] <= t;
    const int below_n = __popc(__ballot_sync(0xffffffffu, below));
    if (below_n == 0) return -1;
    const int64_t skip = (below_n - 1) * step;
    lo += skip;
    size = min(step, size - skip);
  }
  return n > 0 && cu[lo] <= t ? lo : -1;
}

// One warp per (token, block of heads). A head's row is spread over G lanes,
// 8 values (16 bytes of a 16-bit type) each, so the mean of squares is a
// log2(G)-step shuffle and a row is read and written once, in whole sectors.
template <typename T, int G>
__global__ void rows_kernel(const __grid_constant__ RowArgs r, int head_blocks, int64_t warps) {
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (w >= warps) return;
  const int lane = threadIdx.x & 31, c = lane % G, sub = lane / G;
  const int64_t t = w / head_blocks;
  const int head = (int)(w % head_blocks) * (32 / G) + sub;
  int64_t pos = t, b = t;
  const bool paged = r.a.kv.batch > 0;
  int page = 0;
  uint32_t slot = 0;
  if (paged) {
    int64_t first = t, count = 1;
    if (r.cu) {
      if (t >= r.cu[r.a.kv.batch]) return;  // behind the last sequence
      b = find_seq(r.cu, r.a.kv.batch, t, lane);
      if (b < 0) { *r.a.flag = 1; return; }
      first = r.cu[b];
      count = r.cu[b + 1] - first;
    }
    const int64_t len = r.a.kv.lens[b];
    pos = len - count + (t - first);
    if (pos < 0 || pos >= len || len > r.a.kv.max_pages * r.a.kv.page_size) {
      *r.a.flag = 1;
      return;
    }
    const uint32_t index = r.a.page.div((uint32_t)pos);
    slot = (uint32_t)pos - index * r.a.page.d;
    page = page_of(r.a, r.a.kv.page_table + b * r.a.kv.table_stride, index);
    if (page < 0) return;
  }
  if (r.rot.positions) pos = r.rot.positions[t];
  if (r.turn && (pos < 0 || pos >= r.rot.table_len)) { *r.a.flag = 1; return; }

  const int total = r.q.heads + r.k.heads + r.v.heads;
  const bool live = head < total && c * 8 < r.d;
  const bool is_q = head < r.q.heads, is_k = !is_q && head < r.q.heads + r.k.heads;
  const int h = is_q ? head : is_k ? head - r.q.heads : head - r.q.heads - r.k.heads;
  const Heads& s = is_q ? r.q : is_k ? r.k : r.v;
  T* dst = reinterpret_cast<T*>(s.dst) + t * s.dst_token + h * s.dst_head;
  if (paged && !is_q) {
    const InfercPagedKv& kv = r.a.kv;
    dst = is_k ? reinterpret_cast<T*>(kv.k) + page * kv.k_page_stride + h * kv.k_head_stride +
                     (int64_t)slot * kv.k_token_stride
               : reinterpret_cast<T*>(kv.v) + page * kv.v_page_stride + h * kv.v_head_stride +
                     (int64_t)slot * kv.v_token_stride;
  }
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live) load8(reinterpret_cast<const T*>(s.src) + t * s.src_token + h * s.src_head + c * 8, x);

  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (live && ((is_q && r.norm_q) || (is_k && r.norm_k))) {
    const float inv = 1.0f / sqrtf(sum / (float)r.d + r.rot.eps);
    const float* gamma = (is_q ? r.rot.q_gamma : r.rot.k_gamma) + c * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * gamma[i];
  }
  if (r.turn) {
    const int half = r.rot.rotary_dim / 2;
    const float* cs = r.rot.cos + pos * r.rot.table_stride;
    const float* sn = r.rot.sin + pos * r.rot.table_stride;
    const bool turns = live && (is_q || is_k);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = c * 8 + i;
      const bool in = col < 2 * half;
      const bool second = r.rot.interleaved ? (i & 1) : col >= half;
      const int pair = r.rot.interleaved ? col >> 1 : second ? col - half : col;
      float other;
      if (r.rot.interleaved) {
        other = x[i ^ 1];
      } else if (half % 8 == 0) {
        const int src = second ? c - half / 8 : c + half / 8;
        other = __shfl_sync(0xffffffffu, x[i], (lane - c) + (src & (G - 1)));
      } else {
        // pairs that straddle lanes at an odd offset: each value of the partner lanes in turn
        const int pc = second ? col - half : col + half;
        other = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float z = __shfl_sync(0xffffffffu, x[j], (lane - c) + ((pc >> 3) & (G - 1)));
          if ((pc & 7) == j) other = z;
        }
      }
      y[i] = x[i];
      if (turns && in) {
        const float co = cs[pair], si = sn[pair];
        y[i] = second ? x[i] * co + other * si : x[i] * co - other * si;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
  }
  if (live) store8(dst + c * 8, x);
}

template <typename T>
void launch_rows(const RowArgs& r, cudaStream_t st) {
  const int heads = r.q.heads + r.k.heads + r.v.heads;
  if (r.tokens == 0 || heads == 0) return;
  const int g = r.d <= 64 ? 8 : r.d <= 128 ? 16 : 32;
  const int blocks = (heads + 32 / g - 1) / (32 / g);
  const int64_t warps = r.tokens * blocks;
  const int64_t grid = (warps + 7) / 8;
  IDEV_CHECK_ARG(grid <= INT32_MAX, "too many tokens in one call");
  if (g == 8) rows_kernel<T, 8><<<(unsigned)grid, 256, 0, st>>>(r, blocks, warps);
  else if (g == 16) rows_kernel<T, 16><<<(unsigned)grid, 256, 0, st>>>(r, blocks, warps);
  else rows_kernel<T, 32><<<(unsigned)grid, 256, 0, st>>>(r, blocks, warps);
  IDEV_LAUNCHED();
}

void dispatch_rows(int dtype, const RowArgs& r, cudaStream_t st) {
  if (dtype == F32) launch_rows<float>(r, st);
  else if (dtype == F16) launch_rows<__half>(r, st);
  else launch_rows<__nv_bfloat16>(r, st);
}

void set_rotary(RowArgs& r, const InfercHeadRotary* rot, const char* op) {
  std::memset(&r.rot, 0, sizeof r.rot);
  if (!rot) return;
  const std::string o = std::string(op) + ": ";
  IDEV_CHECK_ARG(rot->rotary_dim >= 0 && rot->rotary_dim % 2 == 0 && rot->rotary_dim <= r.d,
                 o + "rotary_dim must be even and at most head_dim");
  IDEV_CHECK_ARG(!(rot->q_gamma || rot->k_gamma) || rot->eps >= 0.f, o + "eps must not be negative");
  if (rot->rotary_dim > 0)
    IDEV_CHECK_ARG(rot->cos && rot->sin && rot->table_len >= 1 &&
                       rot->table_stride >= rot->rotary_dim / 2,
                   o + "rotation needs cos and sin tables [table_len, rotary_dim / 2]");
  r.rot = *rot;
  r.norm_q = rot->q_gamma != nullptr;
  r.norm_k = rot->k_gamma != nullptr;
  r.turn = rot->rotary_dim > 0;
}

// ------------------------------------------------------------------ evict

struct EvictArgs {
  Args a;
  const int32_t* dst_table;  // nullptr: in place
  int64_t dst_stride, dst_pages;
  float* w;
  int64_t w_batch, w_head;
  float* w_out;
  int64_t wo_batch, wo_head;
  int keep, recent;
  int32_t* lens_out;
  int32_t* kept;
};

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;

// Order of weights as unsigned numbers: -0 equals 0, every NaN is the largest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the block of `v` before this thread; *total: over all of it.
__device__ __forceinline__ uint64_t block_exclusive(uint64_t v, uint64_t* warp_sums,
                                                    uint64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t n = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += n;
  }
  __syncthreads();  // warp_sums of the previous call are read
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    uint64_t x = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t n = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += n;
    }
    warp_sums[lane] = x;
  }
  __syncthreads();
  *total = warp_sums[31];
  return s - v + (warp ? warp_sums[warp - 1] : 0);
}

// One block per (sequence, key head): finds the weight of rank keep - recent
// by three histograms of 11, 11 and 10 bits of its key, then walks the
// positions in order, packing what stays. A position's new place is the
// number of larger weights before it plus the equal ones before it that stay,
// so ties go to the lowest index whatever the threads' order.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const __grid_constant__ EvictArgs e) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint64_t sums[32];
  __shared__ uint32_t s_prefix, s_need;
  const int hk = (int)e.a.kv.kv_heads;
  const int64_t b = blockIdx.x / hk;
  const int h = blockIdx.x % hk, tid = threadIdx.x;
  const int n = seq_len(e.a, b);
  const int m = min(n, e.keep);
  float* w = e.w + b * e.w_batch + h * e.w_head;
  float* wo = e.w_out + b * e.wo_batch + h * e.wo_head;
  int32_t* kept = e.kept + ((int64_t)b * hk + h) * e.keep;
  if (h == 0 && tid == 0) e.lens_out[b] = m;
  for (int i = m + tid; i < e.keep; i += kSelThreads) kept[i] = -1;
  if (n <= e.keep) {
    for (int i = tid; i < n; i += kSelThreads) {
      kept[i] = i;
      if (wo != w) wo[i] = w[i];
    }
    return;
  }
  const int limit = n - e.recent, need = e.keep - e.recent;
  uint32_t prefix = 0, mask = 0, left = need;
  if (need > 0) {
    const int shifts[3] = {21, 10, 0};
    const uint32_t widths[3] = {2047u, 2047u, 1023u};
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int j = tid; j < limit; j += kSelThreads) {
        const uint32_t k = weight_key(w[j]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shifts[pass]) & widths[pass]], 1u);
      }
      __syncthreads();
      // bins from the largest down; this thread's two are 2 tid and 2 tid + 1
      const uint32_t hi = hist[kBins - 1 - 2 * tid], lo = hist[kBins - 2 - 2 * tid];
      uint64_t total;
      const uint32_t before = (uint32_t)block_exclusive((uint64_t)hi + lo, sums, &total);
      if (before < left && left <= before + hi + lo) {
        const bool first = left <= before + hi;
        s_prefix = (uint32_t)(kBins - 1 - 2 * tid - (first ? 0 : 1));
        s_need = left - before - (first ? 0 : hi);
      }
      __syncthreads();
      prefix |= s_prefix << shifts[pass];
      mask |= widths[pass] << shifts[pass];
      left = s_need;
    }
  }
  // `prefix` is the key of that weight; `left` positions with this very key stay
  uint64_t done = 0;  // larger ones so far (high half), equal ones (low half)
  for (int j0 = 0; j0 < n; j0 += kSelThreads) {
    const int j = j0 + tid;
    float v = 0.f;
    bool gt = false, eq = false;
    if (j < n) v = w[j];
    if (j < limit && need > 0) {
      const uint32_t k = weight_key(v);
      gt = k > prefix;
      eq = k == prefix;
    }
    uint64_t total;
    const uint64_t at =
        done + block_exclusive(((uint64_t)gt << 32) | (uint64_t)eq, sums, &total);
    const uint32_t eq_before = (uint32_t)at, gt_before = (uint32_t)(at >> 32);
    // (the scan's barriers also separate this chunk's reads from the writes below)
    if (gt || (eq && eq_before < left)) {
      const uint32_t to = gt_before + min(eq_before, left);
      kept[to] = j;
      wo[to] = v;
    } else if (j >= limit && j < n) {
      kept[need + j - limit] = j;
      wo[need + j - limit] = v;
    }
    done += total;
  }
  __syncthreads();
  for (int j = e.keep + tid; j < n; j += kSelThreads) wo[j] = 0.f;
}

constexpr int kMoveThreads = 256, kMoveItems = 4, kMoveCluster = 8;

// Moves the kept rows of one (sequence, key head) of the keys or the values
// to the front. In place, a row's source lies at or behind its destination
// (kept[i] >= i), so of a stretch of rows all loads come before any store
// (a barrier over the cluster that shares the sequence), and later stretches'
// sources lie behind what earlier ones wrote.
template <bool kInPlace>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictArgs e,
                                                                  int lanes, FastDiv by_lanes) {
  const int part = blockIdx.x % kMoveCluster;
  int64_t job = blockIdx.x / kMoveCluster;
  const bool is_v = job & 1;
  job >>= 1;
  const int hk = (int)e.a.kv.kv_heads;
  const int64_t b = job / hk;
  const int h = (int)(job % hk);
  const InfercPagedKv& kv = e.a.kv;
  const int es = kv.dtype == F32 ? 4 : 2;
  char* base = reinterpret_cast<char*>(is_v ? kv.v : kv.k) +
               h * (is_v ? kv.v_head_stride : kv.k_head_stride) * es;
  const int64_t page_bytes = (is_v ? kv.v_page_stride : kv.k_page_stride) * es;
  const int64_t slot_bytes = (is_v ? kv.v_token_stride : kv.k_token_stride) * es;
  const int32_t* src_row = kv.page_table + b * kv.table_stride;
  const int32_t* dst_row = kInPlace ? src_row : e.dst_table + b * e.dst_stride;
  pdl_wait();
  const int m = min(e.lens_out[b], e.keep);
  const int32_t* kept = e.kept + ((int64_t)b * hk + h) * e.keep;
  const int per_block = kMoveThreads * kMoveItems;
  // items (row, 16-byte piece), counted in 32 bits: m * lanes < 2^31 is checked by the host
  const uint32_t items = (uint32_t)m * lanes;
  for (uint32_t i0 = 0; i0 < items; i0 += per_block * kMoveCluster) {
    uint4 val[kMoveItems];
    char* to[kMoveItems];
#pragma unroll
    for (int u = 0; u < kMoveItems; ++u) {
      const uint32_t i = i0 + part * per_block + u * kMoveThreads + threadIdx.x;
      to[u] = nullptr;
      if (i >= items) continue;
      const uint32_t row = by_lanes.div(i), piece = i - row * lanes;
      const uint32_t from = (uint32_t)kept[row];
      if (kInPlace && from == row) continue;
      const uint32_t sp = e.a.page.div(from), dp = e.a.page.div(row);
      const int src = page_of(e.a, src_row, sp), dst = page_of(e.a, dst_row, dp);
      if (src < 0 || dst < 0) continue;
      val[u] = *reinterpret_cast<const uint4*>(base + src * page_bytes +
                                               (from - sp * e.a.page.d) * slot_bytes + piece * 16);
      to[u] = base + dst * page_bytes + (row - dp * e.a.page.d) * slot_bytes + piece * 16;
    }
    if (kInPlace) {
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
#pragma unroll
    for (int u = 0; u < kMoveItems; ++u)
      if (to[u]) *reinterpret_cast<uint4*>(to[u]) = val[u];
  }
}

void launch_evict(const EvictArgs& e, cudaStream_t st) {
  const InfercPagedKv& kv = e.a.kv;
  const int64_t jobs = kv.batch * kv.kv_heads;
  evict_select_kernel<<<(unsigned)jobs, kSelThreads, 0, st>>>(e);
  IDEV_LAUNCHED();
  const int lanes = kv.head_dim * elem_bytes(kv.dtype) / 16;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(jobs * 2 * kMoveCluster));
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kMoveCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = e.dst_table ? 1 : 2;
  const FastDiv by((uint32_t)lanes);
  if (e.dst_table) IDEV_CUDA(cudaLaunchKernelEx(&cfg, evict_move_kernel<false>, e, lanes, by));
  else IDEV_CUDA(cudaLaunchKernelEx(&cfg, evict_move_kernel<true>, e, lanes, by));
}

}  // namespace
}  // namespace paged
}  // namespace inferc_dev

using namespace inferc_dev;
using namespace inferc_dev::paged;

extern "C" {

int inferc_dev_qk_norm_rotary(const InfercHeadRotary* rot, int dtype, const void* q,
                              int64_t q_token_stride, int64_t q_head_stride, const void* k,
                              int64_t k_token_stride, int64_t k_head_stride, void* q_out,
                              int64_t q_out_token_stride, int64_t q_out_head_stride, void* k_out,
                              int64_t k_out_token_stride, int64_t k_out_head_stride,
                              int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                              void* stream) {
  return guard([&] {
    const char* op = "QKNormRotary";
    IDEV_CHECK_ARG(rot != nullptr, "QKNormRotary: null rotary descriptor");
    check_dtype_dim(op, dtype, head_dim);
    IDEV_CHECK_ARG(tokens >= 0 && tokens <= INT32_MAX && q_heads >= 0 && q_heads <= 65535 &&
                       kv_heads >= 0 && kv_heads <= 65535,
                   "QKNormRotary: bad shape");
    RowArgs r{};
    r.d = (int)head_dim;
    r.tokens = tokens;
    set_rotary(r, rot, op);
    if (tokens == 0) return;
    if (q_heads > 0) {
      check_rows(op, "query", q, q_token_stride, q_head_stride, dtype);
      check_rows(op, "query output", q_out, q_out_token_stride, q_out_head_stride, dtype);
    }
    if (kv_heads > 0) {
      check_rows(op, "key", k, k_token_stride, k_head_stride, dtype);
      check_rows(op, "key output", k_out, k_out_token_stride, k_out_head_stride, dtype);
    }
    r.q = {q, q_out, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride,
           (int)q_heads};
    r.k = {k, k_out, k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride,
           (int)kv_heads};
    r.a.flag = range_flag_ptr();
    dispatch_rows(dtype, r, as_stream(stream));
  });
}

int inferc_dev_paged_kv_append(const InfercPagedKv* kv, const InfercHeadRotary* rot, const void* q,
                               int64_t q_token_stride, int64_t q_head_stride, const void* k,
                               int64_t k_token_stride, int64_t k_head_stride, const void* v,
                               int64_t v_token_stride, int64_t v_head_stride, void* q_out,
                               int64_t q_out_token_stride, int64_t q_out_head_stride,
                               int64_t q_heads, const int32_t* cu_tokens, int64_t tokens,
                               void* stream) {
  return guard([&] {
    const char* op = "PagedKVAppend";
    check_kv(kv, op);
    IDEV_CHECK_ARG(tokens >= 0 && tokens <= INT32_MAX && q_heads >= 0 && q_heads <= 65535,
                   "PagedKVAppend: bad shape");
    IDEV_CHECK_ARG(cu_tokens != nullptr || tokens == kv->batch,
                   "PagedKVAppend: without cu_tokens there is one token per sequence");
    IDEV_CHECK_ARG(rot != nullptr || q_heads == 0,
                   "PagedKVAppend: queries come with a norm or a rotation");
    RowArgs r{};
    r.d = kv->head_dim;
    r.tokens = tokens;
    set_rotary(r, rot, op);
    if (tokens == 0 || kv->batch == 0) return;
    check_rows(op, "key", k, k_token_stride, k_head_stride, kv->dtype);
    check_rows(op, "value", v, v_token_stride, v_head_stride, kv->dtype);
    if (q_heads > 0) {
      check_rows(op, "query", q, q_token_stride, q_head_stride, kv->dtype);
      check_rows(op, "query output", q_out, q_out_token_stride, q_out_head_stride, kv->dtype);
    }
    r.a.kv = *kv;
    r.a.page = FastDiv((uint32_t)kv->page_size);
    r.a.flag = range_flag_ptr();
    r.q = {q, q_out, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride,
           (int)q_heads};
    r.k = {k, nullptr, k_token_stride, k_head_stride, 0, 0, (int)kv->kv_heads};
    r.v = {v, nullptr, v_token_stride, v_head_stride, 0, 0, (int)kv->kv_heads};
    r.cu = cu_tokens;
    dispatch_rows(kv->dtype, r, as_stream(stream));
  });
}

int inferc_dev_paged_kv_evict(const InfercPagedKv* kv, const int32_t* dst_table,
                              int64_t dst_max_pages, int64_t dst_table_stride, float* weights,
                              int64_t weights_batch_stride, int64_t weights_head_stride,
                              float* weights_out, int64_t weights_out_batch_stride,
                              int64_t weights_out_head_stride, int64_t keep, int64_t recent,
                              int32_t* lens_out, int32_t* kept, void* stream) {
  return guard([&] {
    const char* op = "PagedKVEvict";
    check_kv(kv, op);
    IDEV_CHECK_ARG(keep >= 1 && keep <= INT32_MAX && recent >= 0 && recent <= keep,
                   "PagedKVEvict: keep must be at least 1 and recent in [0, keep]");
    const int64_t most = std::min<int64_t>(keep, kv->max_pages * kv->page_size);
    IDEV_CHECK_ARG(most * 64 <= INT32_MAX, "PagedKVEvict: too many positions to keep");
    if (dst_table == kv->page_table) dst_table = nullptr;
    if (dst_table)
      IDEV_CHECK_ARG(dst_max_pages >= 0 && dst_max_pages <= INT32_MAX &&
                         dst_table_stride >= dst_max_pages &&
                         dst_max_pages * kv->page_size >= most,
                     "PagedKVEvict: the destination's page table is too small");
    if (kv->batch == 0) return;
    IDEV_CHECK_ARG(kv->batch * kv->kv_heads <= INT32_MAX / (2 * kMoveCluster),
                   "PagedKVEvict: too many heads in one call");
    IDEV_CHECK_ARG(weights && lens_out && kept, "PagedKVEvict: null weights, lens_out or kept");
    IDEV_CHECK_ARG(lens_out + kv->batch <= kv->lens || kv->lens + kv->batch <= lens_out,
                   "PagedKVEvict: lens_out must not overlap lens");
    EvictArgs e{};
    e.a.kv = *kv;
    e.a.page = FastDiv((uint32_t)kv->page_size);
    e.a.flag = range_flag_ptr();
    e.dst_table = dst_table;
    e.dst_stride = dst_table_stride;
    e.dst_pages = dst_max_pages;
    e.w = weights;
    e.w_batch = weights_batch_stride;
    e.w_head = weights_head_stride;
    e.w_out = weights_out ? weights_out : weights;
    e.wo_batch = weights_out ? weights_out_batch_stride : weights_batch_stride;
    e.wo_head = weights_out ? weights_out_head_stride : weights_head_stride;
    e.keep = (int)keep;
    e.recent = (int)recent;
    e.lens_out = lens_out;
    e.kept = kept;
    launch_evict(e, as_stream(stream));
  });
}

}  // extern "C"
