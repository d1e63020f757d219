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

#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace inferc_dev {

namespace paged {

// [0]: an index pointed outside its buffer; [1]: a wait for a copy gave up
__device__ int g_flags[2];

// Where they are on each device; nullptr until an operator was called there.
constexpr int kMostDevices = 64;
static std::atomic<int*> g_known[kMostDevices];

int* range_flag_ptr() {
  int dev = 0;
  IDEV_CUDA(cudaGetDevice(&dev));
  int* p = dev < kMostDevices ? g_known[dev].load() : nullptr;
  if (!p) {
    IDEV_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_flags));
    if (dev < kMostDevices) g_known[dev].store(p);
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

void check_apart(const char* op, const char* what, int64_t d, Steps a, Steps b, Steps c) {
  Steps steps[3] = {a, b, c};
  auto size = [](int64_t stride) { return stride < 0 ? -(__int128)stride : (__int128)stride; };
  std::sort(steps, steps + 3, [&](const Steps& x, const Steps& y) {
    return size(x.stride) < size(y.stride);
  });
  __int128 extent = d;  // of what the smaller steps reach
  for (const Steps& s : steps) {
    if (s.count == 0) return;
    if (s.count == 1) continue;
    IDEV_CHECK_ARG(size(s.stride) >= extent,
                   std::string(op) + ": rows of the " + what + " overlap");
    extent += size(s.stride) * (s.count - 1);
  }
}

// The caches, where they are written.
static void check_caches_apart(const char* op, const InfercPagedKv& kv) {
  check_apart(op, "key cache", kv.head_dim, {kv.num_pages, kv.k_page_stride},
              {kv.kv_heads, kv.k_head_stride}, {kv.page_size, kv.k_token_stride});
  check_apart(op, "value cache", kv.head_dim, {kv.num_pages, kv.v_page_stride},
              {kv.kv_heads, kv.v_head_stride}, {kv.page_size, kv.v_token_stride});
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
  // (positions are counted in 32 bits, with room for a grid's strides)
  IDEV_CHECK_ARG(kv->page_size <= kMostPositions && kv->max_pages <= kMostPositions &&
                     kv->page_size * kv->max_pages <= kMostPositions,
                 o + "page_size * max_pages must be at most 2^30");
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
  int dev = 0;
  IDEV_CUDA(cudaGetDevice(&dev));
  // callers without a paged cache do not wait for a copy of its flags
  if (dev < paged::kMostDevices && !paged::g_known[dev].load()) return 0;
  int v[2] = {0, 0};
  IDEV_CUDA(cudaMemcpyFromSymbol(v, paged::g_flags, sizeof v));
  // only what was seen: the other may be raised meanwhile, by work on another stream
  for (int i = 0; i < 2; ++i) {
    const int z = 0;
    if (v[i]) IDEV_CUDA(cudaMemcpyToSymbol(paged::g_flags, &z, sizeof z, i * sizeof z));
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
  int d, turn;  // turn: how the pairs lie (Turn)
};

// The sequence that token t belongs to, where its tokens begin and how many
// they are, by one warp: 32 boundaries a step, so that up to 31 sequences cost
// one load. b: -1 behind the last sequence, -2 when cu is no list of boundaries.
struct Owner {
  int64_t b, begin, count;
};
__device__ __forceinline__ Owner owner_of_token(const int32_t* cu, int64_t n, int64_t t, int lane) {
  int64_t lo = 0, size = n + 1;  // the last boundary at t or below is in [lo, lo + size)
  for (;;) {
    const int64_t step = (size + 31) / 32, at = lane * step;
    const int64_t mine = at < size ? cu[lo + at] : INT64_MAX;
    const int below = __popc(__ballot_sync(0xffffffffu, mine <= t));
    if (below == 0) return {-2, 0, 0};
    if (step == 1) {
      const int64_t b = lo + below - 1;
      if (b == n) return {-1, 0, 0};
      const int64_t begin = __shfl_sync(0xffffffffu, mine, below - 1);
      int64_t end = __shfl_sync(0xffffffffu, mine, below & 31);
      if (below == size || below == 32) end = cu[b + 1];
      return {b, begin, end - begin};
    }
    lo += (below - 1) * step;
    size = min(step, size - (below - 1) * step);
  }
}

// How a row's pairs lie in its lanes.
enum Turn : int {
  kNone = 0,     // no rotation
  kHalves = 1,   // (i, i + half), half a multiple of 4: a lane holds four columns and their partners
  kWithin = 2,   // (2 i, 2 i + 1): in the lane itself
  kAcross = 3    // (i, i + half) at an odd offset: through shared memory
};

// Rows a group of lanes fetches before it uses the first: 64 bytes a lane.
template <typename T>
constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;

// The eight columns of lane c: first .. first + 3 and first + second .. + 3.
struct Columns {
  int first, second;
};
template <int kTurn>
__device__ __forceinline__ Columns columns_of(int c, int half) {
  if (kTurn == kHalves && c * 4 < half) return {c * 4, half};
  return {c * 8, 4};  // (behind the rotated columns too: half / 4 lanes hold 2 half columns)
}

// Rows [hb, h1) as far as they go. Lanes without columns keep zeros, and those
// without a row what they had (its results are not stored).
template <typename T, int G>
__device__ __forceinline__ void fetch_rows(const T* src, int64_t src_head, int hb, int h1,
                                           bool column, const Columns& col,
                                           Raw8<T> (&raw)[kAhead<T>]) {
  const int sub = (threadIdx.x & 31) / G;
  src += (hb + sub) * src_head + col.first;
#pragma unroll
  for (int u = 0; u < kAhead<T>; ++u) {
    if (column && hb + u * (32 / G) + sub < h1) raw[u].load(src, col.second);
    src += 32 / G * src_head;
  }
}

// Norm and rotation of the heads [h0, h1) of the queries or the keys of one
// token by one warp: G lanes share a row, 8 values each. With gamma, c and s folded,
//   y_i = inv * (x_i * own_i + x_partner * other_i),
// own_i = gamma_i c_i, other_i = -+ gamma_partner s_i (once per token). Lanes hold
// the columns so that partners meet in one lane, and a row costs three
// operations per value beside its mean.
template <typename T, int G, int kTurn>
__device__ __forceinline__ void rows_of(const T* src, int64_t src_head, T* dst, int64_t dst_head,
                                        int h0, int h1, const float* gamma,
                                        const InfercHeadRotary& rot, int64_t pos, int d,
                                        float* stage, Raw8<T> (&raw)[kAhead<T>], bool fetched) {
  constexpr int kAtOnce = 32 / G;
  const int lane = threadIdx.x & 31, c = lane % G, sub = lane / G;
  const bool column = c * 8 < d;
  const float inv_d = 1.0f / (float)d;
  const int half = rot.rotary_dim / 2;
  const Columns col = columns_of<kTurn>(c, half);
  dst += (h0 + sub) * dst_head + col.first;
  const int64_t dst_step = kAtOnce * dst_head;

  float own[8], other[8];
  uint32_t in = 0;  // columns that are rotated
  bool ready = false;
  // One row: what `r` holds, to `to` where `live`.
  auto row = [&](const Raw8<T>& r, T* to, bool live) {
    float x[8], y[8], inv = 1.f;
    r.widen(x);
    if (gamma) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      inv = rsqrtf(sum * inv_d + rot.eps);
    }
    if constexpr (kTurn == kAcross) {
      __syncwarp();
      store8(stage + lane * 8, x);
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kTurn == kWithin) {
        y[i] = x[i ^ 1];
      } else if constexpr (kTurn == kHalves) {
        y[i] = x[i ^ 4];
      } else if constexpr (kTurn == kAcross) {
        const int at = c * 8 + i;
        y[i] = in >> i & 1 ? stage[(lane - c) * 8 + (at < half ? at + half : at - half)] : 0.f;
      }
    }
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = x[i] * own[i];
    if constexpr (kTurn == kHalves) {  // a lane's columns are rotated all or none
      if (in)
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] += y[i] * other[i];
    } else if constexpr (kTurn != kNone) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in >> i & 1) z[i] += y[i] * other[i];
    }
    if (gamma)
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] *= inv;
    if (live) {
      store4(to, z);
      store4(to + col.second, z + 4);
    }
  };
  for (int hb = h0; hb < h1; hb += kAtOnce * kAhead<T>) {
    if (!fetched) fetch_rows<T, G>(src, src_head, hb, h1, column, col, raw);
    fetched = false;
    if (!ready) {  // behind the first rows' loads
      ready = true;
#pragma unroll
      for (int i = 0; i < 8; ++i) own[i] = 1.f, other[i] = 0.f;
      if (gamma && column) {
        const float4 a = *reinterpret_cast<const float4*>(gamma + col.first);
        const float4 b = *reinterpret_cast<const float4*>(gamma + col.first + col.second);
        own[0] = a.x; own[1] = a.y; own[2] = a.z; own[3] = a.w;
        own[4] = b.x; own[5] = b.y; own[6] = b.z; own[7] = b.w;
      }
      if (kTurn != kNone && column && col.first < 2 * half) {
        const float* cs = rot.cos + pos * rot.table_stride;
        const float* sn = rot.sin + pos * rot.table_stride;
        if constexpr (kTurn == kHalves) {
          if (c * 4 < half) {
            in = 0xff;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float co = cs[c * 4 + i], si = sn[c * 4 + i];
              other[i] = -si * own[i + 4];
              other[i + 4] = si * own[i];
              own[i] *= co;
              own[i + 4] *= co;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = c * 8 + i;
            const bool second = kTurn == kWithin ? i & 1 : at >= half;
            const int pair = kTurn == kWithin ? at >> 1 : second ? at - half : at;
            const int to = kTurn == kWithin ? at ^ 1 : second ? at - half : at + half;
            if (at < 2 * half) {
              in |= 1u << i;
              own[i] *= cs[pair];
              other[i] = (second ? sn[pair] : -sn[pair]) * (gamma ? gamma[to] : 1.f);
            }
          }
        }
      }
    }
    if (hb + kAtOnce * kAhead<T> <= h1) {  // all live: their chains run side by side
#pragma unroll
      for (int u = 0; u < kAhead<T>; ++u, dst += dst_step) row(raw[u], dst, column);
    } else {
#pragma unroll
      for (int u = 0; u < kAhead<T>; ++u, dst += dst_step)
        if (hb + u * kAtOnce < h1)  // the same for the whole warp
          row(raw[u], dst, column && hb + u * kAtOnce + sub < h1);
    }
  }
}

// One warp per (token, block of `per_warp` heads), the heads numbered queries,
// keys, values. What a token's position and the gammas give stays in registers
// for all its heads: read for each head again, the cosines and sines were twice
// the bytes of a 16-bit row (8190 tokens of 40 bf16 heads of 128: 110 us; so
// 39 us, 0.67 of the measured copy rate).
template <typename T, int G, int kTurn>
__global__ void __launch_bounds__(256, 3)
    rows_kernel(const __grid_constant__ RowArgs r, int per_warp, int head_blocks, int64_t warps) {
  __shared__ __align__(16) float stage[kTurn == kAcross ? 8 : 1][32 * 8];
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  pdl_wait();
  if (w >= warps) return;
  const int lane = threadIdx.x & 31, c = lane % G, sub = lane / G;
  const int64_t t = divide(w, head_blocks);
  const int first = (int)(w - t * head_blocks) * per_warp;
  const int total = r.q.heads + r.k.heads + r.v.heads;
  const int last = min(first + per_warp, total);
  const bool paged = r.a.kv.batch > 0;
  const InfercPagedKv& kv = r.a.kv;
  // The first rows are on their way while the token's place is looked up.
  Raw8<T> raw[kAhead<T>];
  const int begin_kind = first < r.q.heads ? 0 : 1;
  {
    const Heads& s = begin_kind ? r.k : r.q;
    const int before = begin_kind ? r.q.heads : 0;
    fetch_rows<T, G>(reinterpret_cast<const T*>(s.src) + t * s.src_token, s.src_head,
                     first - before, min(last - before, s.heads), c * 8 < r.d,
                     columns_of<kTurn>(c, r.rot.rotary_dim / 2), raw);
  }
  int64_t pos = t, b = t;
  int page = 0;
  uint32_t slot = 0;
  if (r.rot.positions) pos = r.rot.positions[t];
  if (paged) {
    int64_t begin = t, count = 1;
    if (r.cu) {
      const Owner o = owner_of_token(r.cu, kv.batch, t, lane);
      if (o.b == -1) return;  // behind the last sequence
      if (o.b < 0) { *r.a.flag = 1; return; }
      b = o.b;
      begin = o.begin;
      count = o.count;
      // tokens that belong to a sequence and are not among the rows
      if (w == 0 && lane == 0 && (r.cu[0] != 0 || r.cu[kv.batch] > r.tokens)) *r.a.flag = 1;
    }
    const int64_t len = kv.lens[b], at = len - count + (t - begin);
    if (at < 0 || at >= len || len > kv.max_pages * kv.page_size) {
      *r.a.flag = 1;
      return;
    }
    const uint32_t index = r.a.page.div((uint32_t)at);
    slot = (uint32_t)at - index * r.a.page.d;
    page = page_of(r.a, kv.page_table + b * kv.table_stride, index);
    if (page < 0) return;
    if (!r.rot.positions) pos = at;
  }
  if (kTurn != kNone && (pos < 0 || pos >= r.rot.table_len)) { *r.a.flag = 1; return; }

#pragma unroll 1
  for (int kind = begin_kind; kind < 2; ++kind) {
    const Heads& s = kind ? r.k : r.q;
    const int before = kind ? r.q.heads : 0;
    const int h0 = max(first - before, 0), h1 = min(last - before, s.heads);
    if (h0 >= h1) continue;
    T* dst = reinterpret_cast<T*>(s.dst) + t * s.dst_token;
    int64_t dst_head = s.dst_head;
    if (paged && kind) {
      dst = reinterpret_cast<T*>(kv.k) + page * kv.k_page_stride +
            (int64_t)slot * kv.k_token_stride;
      dst_head = kv.k_head_stride;
    }
    rows_of<T, G, kTurn>(reinterpret_cast<const T*>(s.src) + t * s.src_token, s.src_head, dst,
                         dst_head, h0, h1, kind ? r.rot.k_gamma : r.rot.q_gamma, r.rot, pos, r.d,
                         stage[kTurn == kAcross ? threadIdx.x >> 5 : 0], raw, kind == begin_kind);
  }
  // values: as they are
  const int before = r.q.heads + r.k.heads;
  const T* src = reinterpret_cast<const T*>(r.v.src) + t * r.v.src_token + c * 8;
  T* dst = reinterpret_cast<T*>(kv.v) + page * kv.v_page_stride +
           (int64_t)slot * kv.v_token_stride + c * 8;
  if (c * 8 < r.d)
#pragma unroll 4
    for (int h = max(first - before, 0) + sub; h < min(last - before, r.v.heads); h += 32 / G) {
      const uint4* from = reinterpret_cast<const uint4*>(src + h * r.v.src_head);
      uint4* to = reinterpret_cast<uint4*>(dst + h * kv.v_head_stride);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) to[i] = from[i];
    }
}

template <typename T, int G>
void launch_rows_of(const RowArgs& r, cudaStream_t st) {
  const int heads = r.q.heads + r.k.heads + r.v.heads;
  // Heads of a token per warp: what spreads the rows over the warps that the SMs
  // hold (24 each), so that a decode step's few tokens do not wait for one
  // another and what a token costs is paid once where there are many.
  const int unit = 32 / G;  // heads that a warp takes at once
  int per_warp = (int)std::min<int64_t>((r.tokens * heads + 148 * 24 - 1) / (148 * 24), heads);
  per_warp = std::min((per_warp + unit - 1) / unit * unit, (heads + unit - 1) / unit * unit);
  const int blocks = (heads + per_warp - 1) / per_warp;
  per_warp = ((heads + blocks - 1) / blocks + unit - 1) / unit * unit;  // alike
  const int64_t warps = r.tokens * blocks;
  const int64_t grid = (warps + 7) / 8;
  IDEV_CHECK_ARG(grid <= INT32_MAX, "too many tokens in one call");
  auto* kernel = r.turn == kNone    ? rows_kernel<T, G, kNone>
                 : r.turn == kHalves ? rows_kernel<T, G, kHalves>
                 : r.turn == kWithin ? rows_kernel<T, G, kWithin>
                                     : rows_kernel<T, G, kAcross>;
  launch_pdl(kernel, dim3((unsigned)grid), dim3(256), 0, st, r, per_warp, blocks, warps);
}

template <typename T>
void launch_rows(const RowArgs& r, cudaStream_t st) {
  if (r.tokens == 0 || r.q.heads + r.k.heads + r.v.heads == 0) return;
  if (r.d <= 64) launch_rows_of<T, 8>(r, st);
  else if (r.d <= 128) launch_rows_of<T, 16>(r, st);
  else launch_rows_of<T, 32>(r, st);
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
  IDEV_CHECK_ARG(!(rot->q_gamma || rot->k_gamma) ||
                     (rot->eps >= 0.f && aligned16(rot->q_gamma) && aligned16(rot->k_gamma)),
                 o + "eps must not be negative, gammas 16-byte aligned");
  if (rot->rotary_dim > 0)
    IDEV_CHECK_ARG(rot->cos && rot->sin && rot->table_len >= 1 &&
                       rot->table_stride >= rot->rotary_dim / 2,
                   o + "rotation needs cos and sin tables [table_len, rotary_dim / 2]");
  r.rot = *rot;
  r.turn = rot->rotary_dim == 0       ? kNone
           : rot->interleaved         ? kWithin
           : rot->rotary_dim % 8 == 0  ? kHalves
                                       : kAcross;
}

// ------------------------------------------------------------------ evict

constexpr int kMoveCluster = 8;  // blocks at most that share a (sequence, key head)

struct EvictArgs {
  Args a;
  const int32_t* dst_table;  // nullptr: in place
  int64_t dst_stride;
  float* w;
  int64_t w_batch, w_head;
  float* w_out;
  int64_t wo_batch, wo_head;
  int keep, recent;
  int32_t* lens_out;
  int32_t* kept;
};

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32;
constexpr int kBins = 2048;
constexpr int kDeep = 4;              // 16-byte loads a lane has in flight, of K and of V
constexpr int kKeysHeld = 16 * 1024;  // weights a block keeps in shared memory
constexpr int kChooseAlone = 8 * 1024;  // positions up to which every block chooses by itself

// Order of weights as unsigned numbers: -0 equals 0, every NaN is the largest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the block of `v` before this thread; *total: over all of it. One
// barrier: calls take turns between two rows of `sums`, so that a row is read by
// all before it is written again.
template <typename V>
__device__ __forceinline__ V block_exclusive(V v, V (*sums)[kEvictWarps], int& turn, V* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V n = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += n;
  }
  if (lane == 31) sums[turn][warp] = s;
  __syncthreads();
  V w = lane < kEvictWarps ? sums[turn][lane] : 0;
#pragma unroll
  for (int o = 1; o < kEvictWarps; o <<= 1) {
    const V n = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += n;
  }
  turn ^= 1;
  *total = __shfl_sync(0xffffffffu, w, kEvictWarps - 1);
  const V before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return s - v + (warp ? before : 0);
}

// One cluster per (sequence, key head).
//
// Choice: the weight of rank keep - recent by histograms of 11, 11 and 10 bits
// of its key, ending early when a bin stays whole. Up to kChooseAlone positions
// every block of the cluster counts all of them, which costs less than the
// cluster barriers it saves (1024 positions: 10 against 14 us); beyond, each
// counts its slice and the blocks add up each other's counts through
// distributed shared memory. A position's new place is the number of larger weights
// before it plus the equal ones before it that stay, so ties go to the lowest
// position whatever the threads' order.
//
// Move: rows go to the front in steps of the whole cluster. In place, a row's
// source lies at or behind its destination (kept[i] >= i), so of a step's rows
// all loads come before any store (a cluster barrier), and the sources of later
// steps lie behind what earlier ones wrote. A warp looks up the pages of its
// rows one row per lane and passes the addresses on by shuffles: the kLanes
// lanes of a row fetch 16 bytes each. (One thread per 16 bytes, each finding
// its own page, took 98 instructions per piece and 131 us for 543 MB; so 99 us,
// 0.84 of the measured copy rate.)
template <int kLanes, int kTurns, bool kInPlace>
__global__ void __launch_bounds__(kEvictThreads, 2)
    evict_kernel(const __grid_constant__ EvictArgs e, int keys_held) {
  __shared__ __align__(16) uint32_t hist[3][kBins];
  __shared__ uint32_t sums[2][kEvictWarps];
  __shared__ uint64_t sums2[2][kEvictWarps];
  __shared__ uint64_t s_count;  // larger (high half) and equal weights in this block's slice
  __shared__ uint32_t s_bin, s_left, s_whole;
  extern __shared__ uint32_t keys[];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const InfercPagedKv& kv = e.a.kv;
  const int hk = (int)kv.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t job = blockIdx.x / blocks;
  const int64_t b = job / hk;
  const int h = (int)(job - b * hk);
  pdl_wait();
  const int n = seq_len(e.a, b);
  const int m = min(n, e.keep);
  const float* w = e.w + b * e.w_batch + h * e.w_head;
  float* wo = e.w_out + b * e.wo_batch + h * e.wo_head;
  int32_t* kept = e.kept + job * e.keep;
  const int all_threads = blocks * kEvictThreads, all_tid = rank * kEvictThreads + tid;
  // rows per warp and step of the move, and whether this block moves row r
  constexpr int kAtOnce = 32 / kLanes, kRows = kDeep / kTurns * kAtOnce;
  constexpr int kBlockRows = kEvictWarps * kRows;
  const bool alone = n <= kChooseAlone && n <= keys_held;  // the same for the whole cluster
  const int slices = alone ? 1 : blocks, at_slice = alone ? 0 : rank;
  auto sync = [&]() {
    if (alone) __syncthreads();
    else cluster.sync();
  };
  auto keep_row = [&](int r, int from) {
    if (!alone || (r / kBlockRows) % blocks == rank) kept[r] = from;
  };
  if (h == 0 && all_tid == 0) e.lens_out[b] = m;
  for (int i = m + all_tid; i < e.keep; i += all_threads) kept[i] = -1;

  // ---- choice
  if (n <= e.keep) {
    if (alone)
      for (int i = tid; i < n; i += kEvictThreads) keep_row(i, i);
    else
      for (int i = all_tid; i < n; i += all_threads) kept[i] = i;
    if (kInPlace && !e.dst_table && wo == w) return;  // the whole cluster
  } else {
    const int limit = n - e.recent, need = e.keep - e.recent;
    const int slice = ((n + slices - 1) / slices + 3) & ~3;
    const int s0 = min(at_slice * slice, n), s1 = min(s0 + slice, n);
    const int c1 = min(s1, limit);  // candidates: [s0, c1)
    const bool held = slice <= keys_held;
    auto key_at = [&](int j) { return held ? keys[j - s0] : weight_key(w[j]); };
    for (int i = tid * 4; i < 3 * kBins; i += kEvictThreads * 4)
      *reinterpret_cast<uint4*>(&hist[0][0] + i) = make_uint4(0, 0, 0, 0);
    if (held)
      for (int j = s0 + tid; j < c1; j += kEvictThreads) keys[j - s0] = weight_key(w[j]);
    __syncthreads();
    uint32_t prefix = 0, mask = 0, left = need;
    int turn = 0;
    if (need > 0) {
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t width = pass == 2 ? 1023u : 2047u;
        for (int j = s0 + tid; j < c1; j += kEvictThreads) {
          const uint32_t k = key_at(j);
          if ((k & mask) == prefix) atomicAdd(&hist[pass][(k >> shift) & width], 1u);
        }
        sync();
        // bins from the largest down, four a thread
        const int low = kBins - 4 - 4 * tid;
        uint4 c = make_uint4(0, 0, 0, 0);
        if (alone) {
          c = *reinterpret_cast<const uint4*>(&hist[pass][low]);
        } else {
          uint4 x[kMoveCluster];  // all on their way before the first is used
#pragma unroll
          for (int r = 0; r < kMoveCluster; ++r) {
            x[r] = make_uint4(0, 0, 0, 0);
            if (r < blocks)
              x[r] = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&hist[pass][low], r));
          }
#pragma unroll
          for (int r = 0; r < kMoveCluster; ++r) {
            c.x += x[r].x; c.y += x[r].y; c.z += x[r].z; c.w += x[r].w;
          }
        }
        uint32_t all;
        const uint32_t before = block_exclusive(c.x + c.y + c.z + c.w, sums, turn, &all);
        const uint32_t count[4] = {c.w, c.z, c.y, c.x};
        uint32_t run = before;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (run < left && left <= run + count[i]) {
            s_bin = low + 3 - i;
            s_left = left - run;
            s_whole = left - run == count[i];
          }
          run += count[i];
        }
        __syncthreads();
        prefix |= s_bin << shift;
        mask |= width << shift;
        left = s_left;
        if (s_whole) break;  // the same in every block
      }
    }
    // (k & mask) > prefix stays, and of those equal to it the first `left`
    // A thread takes a run of consecutive positions (an odd number of them, so that the keys
    // it reads lie in another bank than its neighbours'): counts what stays, adds up what
    // stays before it, and walks the run again.
    const int run = (max(c1 - s0, 0) + kEvictThreads - 1) / kEvictThreads | 1;
    const int j0 = (int)min((int64_t)s0 + (int64_t)tid * run, (int64_t)c1);
    const int j1 = need > 0 ? min(j0 + run, c1) : j0;
    uint64_t mine = 0;  // larger ones (high half) and equal ones
    for (int j = j0; j < j1; ++j) {
      const uint32_t k = key_at(j) & mask;
      mine += ((uint64_t)(k > prefix) << 32) | (uint64_t)(k == prefix);
    }
    uint64_t total, done = 0;
    uint64_t at = block_exclusive(mine, sums2, turn, &total);
    if (!alone) {
      if (tid == 0) s_count = total;
      cluster.sync();
      uint64_t x = lane < rank ? *cluster.map_shared_rank(&s_count, lane) : 0;
#pragma unroll
      for (int o = 1; o < kMoveCluster; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      done = __shfl_sync(0xffffffffu, x, 0);  // in the slices before this one
    }
    at += done;
    for (int j = j0; j < j1; ++j) {
      const uint32_t k = key_at(j) & mask;
      const uint32_t eq_before = (uint32_t)at, gt_before = (uint32_t)(at >> 32);
      const uint32_t to = gt_before + min(eq_before, left);
      if ((k > prefix || (k == prefix && eq_before < left)) && to < (uint32_t)need) keep_row(to, j);
      at += ((uint64_t)(k > prefix) << 32) | (uint64_t)(k == prefix);
    }
    for (int j = max(s0, limit) + tid; j < s1; j += kEvictThreads) keep_row(need + j - limit, j);
  }
  sync();  // `kept` is whole (and no block leaves while another reads its counts)

  // ---- move
  const int es = kv.dtype == F32 ? 4 : 2;
  const int pieces = kv.head_dim * es / 16;
  const int32_t* src_row = kv.page_table + b * kv.table_stride;
  const int32_t* dst_row = e.dst_table ? e.dst_table + b * e.dst_stride : src_row;
  const char* k_head = static_cast<const char*>(kv.k) + h * kv.k_head_stride * es;
  const char* v_head = static_cast<const char*>(kv.v) + h * kv.v_head_stride * es;
  // A warp's 32 lanes look up the rows of 32 / kRows steps at once, so that the chain of kept
  // position, page and address is waited for once in as many steps.
  const int step = blocks * kBlockRows;
  for (int base = 0; base < m; base += 32 / kRows * step) {
    const int row = base + lane / kRows * step + rank * kBlockRows + warp * kRows + lane % kRows;
    bool ok = false;
    int64_t sk = 0, sv = 0, dk = 0, dv = 0;
    uint32_t from = 0;
    if (row < m) {
      // (below n unless the weights change under the kernel)
      from = min((uint32_t)kept[row], (uint32_t)(n - 1));
      if (e.dst_table || from != (uint32_t)row) {
        const uint32_t sp = e.a.page.div(from), dp = e.a.page.div(row);
        const int src = page_of(e.a, src_row, sp), dst = page_of(e.a, dst_row, dp);
        const int64_t ss = from - sp * e.a.page.d, ds = row - dp * e.a.page.d;
        ok = src >= 0 && dst >= 0;
        if (ok) {
          sk = (src * kv.k_page_stride + ss * kv.k_token_stride) * es;
          sv = (src * kv.v_page_stride + ss * kv.v_token_stride) * es;
          dk = (dst * kv.k_page_stride + ds * kv.k_token_stride) * es;
          dv = (dst * kv.v_page_stride + ds * kv.v_token_stride) * es;
        }
      }
    }
    for (int s = 0; s < 32 / kRows && base + s * step < m; ++s) {
      uint4 k_val[kDeep], v_val[kDeep];
      auto row_at = [&](int u) { return s * kRows + u / kTurns * kAtOnce + lane / kLanes; };
      auto piece_at = [&](int u) { return lane % kLanes + u % kTurns * 32; };
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int r = row_at(u), piece = piece_at(u);
        const int64_t from_k = __shfl_sync(0xffffffffu, sk, r);
        const int64_t from_v = __shfl_sync(0xffffffffu, sv, r);
        const bool live = __shfl_sync(0xffffffffu, (int)ok, r) && piece < pieces;
        if (live) {
          k_val[u] = *reinterpret_cast<const uint4*>(k_head + from_k + piece * 16);
          v_val[u] = *reinterpret_cast<const uint4*>(v_head + from_v + piece * 16);
        }
      }
      const bool weighs = lane / kRows == s && row < m;
      float weight = 0.f;
      if (weighs) weight = w[from];
      if (kInPlace) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      }
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int r = row_at(u), piece = piece_at(u);
        const int64_t to_k = __shfl_sync(0xffffffffu, dk, r);
        const int64_t to_v = __shfl_sync(0xffffffffu, dv, r);
        const bool live = __shfl_sync(0xffffffffu, (int)ok, r) && piece < pieces;
        if (live) {
          *reinterpret_cast<uint4*>(const_cast<char*>(k_head) + to_k + piece * 16) = k_val[u];
          *reinterpret_cast<uint4*>(const_cast<char*>(v_head) + to_v + piece * 16) = v_val[u];
        }
      }
      if (weighs) wo[row] = weight;
    }
  }
  // every load of w is done: in place, before the last step's barrier
  for (int j = m + all_tid; j < n; j += all_threads) wo[j] = 0.f;
}

void launch_evict(const EvictArgs& e, cudaStream_t st) {
  const InfercPagedKv& kv = e.a.kv;
  const int64_t jobs = kv.batch * kv.kv_heads;
  const int64_t capacity = kv.max_pages * kv.page_size;
  // Blocks per (sequence, key head), a power of two so that clusters fill the
  // SMs (of 6, two of three SMs stood idle). Where each chooses by itself, one
  // per SM (two took 111 us for 16 x 8 heads of 4352 positions, one 99 us),
  // else two; none with fewer positions than threads.
  const bool alone = capacity <= kChooseAlone;
  int blocks = 1;
  while (blocks < kMoveCluster && jobs * blocks * 2 <= (alone ? 1 : 2) * 148 &&
         capacity > blocks * kEvictThreads)
    blocks *= 2;
  const int slices = alone ? 1 : blocks;
  const int64_t slice = ((capacity + slices - 1) / slices + 3) / 4 * 4;
  const int held = (int)std::min<int64_t>(slice, kKeysHeld);
  const int pieces = kv.head_dim * elem_bytes(kv.dtype) / 16;
  const bool in_place = !e.dst_table || e.w_out == e.w;
  using Kernel = void (*)(EvictArgs, int);
  Kernel kernel = pieces <= 8    ? (in_place ? evict_kernel<8, 1, true> : evict_kernel<8, 1, false>)
                  : pieces <= 16 ? (in_place ? evict_kernel<16, 1, true> : evict_kernel<16, 1, false>)
                  : pieces <= 32 ? (in_place ? evict_kernel<32, 1, true> : evict_kernel<32, 1, false>)
                                 : (in_place ? evict_kernel<32, 2, true> : evict_kernel<32, 2, false>);
  const size_t smem = (size_t)held * 4;
  if (smem > 16 * 1024)  // with the histograms, past the 48 KB every kernel may have
    IDEV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   kKeysHeld * 4));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(jobs * blocks));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  IDEV_CUDA(cudaLaunchKernelEx(&cfg, kernel, e, held));
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
      check_apart(op, "query output", head_dim, {tokens, q_out_token_stride},
                  {q_heads, q_out_head_stride});
    }
    if (kv_heads > 0) {
      check_rows(op, "key", k, k_token_stride, k_head_stride, dtype);
      check_rows(op, "key output", k_out, k_out_token_stride, k_out_head_stride, dtype);
      check_apart(op, "key output", head_dim, {tokens, k_out_token_stride},
                  {kv_heads, k_out_head_stride});
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
      check_apart(op, "query output", kv->head_dim, {tokens, q_out_token_stride},
                  {q_heads, q_out_head_stride});
    }
    check_caches_apart(op, *kv);
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
    IDEV_CHECK_ARG(keep >= 1 && keep <= kMostPositions && recent >= 0 && recent <= keep,
                   "PagedKVEvict: keep must be in [1, 2^30] and recent in [0, keep]");
    const int64_t most = std::min<int64_t>(keep, kv->max_pages * kv->page_size);
    if (dst_table == kv->page_table && (kv->batch <= 1 || dst_table_stride == kv->table_stride))
      dst_table = nullptr;
    IDEV_CHECK_ARG(!dst_table || dst_table != kv->page_table,
                   "PagedKVEvict: dst_table starts as page_table does, but has another stride");
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
    check_caches_apart(op, *kv);
    if (!weights_out) {
      weights_out = weights;
      weights_out_batch_stride = weights_batch_stride;
      weights_out_head_stride = weights_head_stride;
    }
    check_apart(op, "weights", kv->max_pages * kv->page_size,
                {kv->batch, weights_out_batch_stride}, {kv->kv_heads, weights_out_head_stride});
    IDEV_CHECK_ARG(weights_out != weights || kv->batch * kv->kv_heads == 1 ||
                       ((weights_out_batch_stride == weights_batch_stride || kv->batch == 1) &&
                        (weights_out_head_stride == weights_head_stride || kv->kv_heads == 1)),
                   "PagedKVEvict: weights_out starts as weights do, but has other strides");
    const Rows2 read{reinterpret_cast<intptr_t>(weights) / 4, kv->max_pages * kv->page_size,
                     {{kv->batch, weights_batch_stride}, {kv->kv_heads, weights_head_stride}}};
    const Rows2 written{reinterpret_cast<intptr_t>(weights_out) / 4, read.length,
                        {{kv->batch, weights_out_batch_stride},
                         {kv->kv_heads, weights_out_head_stride}}};
    IDEV_CHECK_ARG(weights_out == weights || !rows_meet(read, written),
                   "PagedKVEvict: weights_out must be weights or share nothing with them");
    EvictArgs e{};
    e.a.kv = *kv;
    e.a.page = FastDiv((uint32_t)kv->page_size);
    e.a.flag = range_flag_ptr();
    e.dst_table = dst_table;
    e.dst_stride = dst_table_stride;
    e.w = weights;
    e.w_batch = weights_batch_stride;
    e.w_head = weights_head_stride;
    e.w_out = weights_out;
    e.wo_batch = weights_out_batch_stride;
    e.wo_head = weights_out_head_stride;
    e.keep = (int)keep;
    e.recent = (int)recent;
    e.lens_out = lens_out;
    e.kept = kept;
    launch_evict(e, as_stream(stream));
  });
}

}  // extern "C"
