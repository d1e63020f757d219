// Attention of one new token per sequence over the paged cache
// (inferc_dev_paged_decode_attention).
#include <algorithm>
#include <string>

#include "paged.cuh"

namespace inferc_dev {
namespace paged {
namespace {

struct AttendArgs {
  Args a;
  const void* q;
  int64_t q_batch, q_head;
  void* out;
  int64_t o_batch, o_head;
  float scale;  // times log2(e)
  int group;    // query heads per key head
  float* scores;  // [batch, q_heads, capacity] scaled scores in the log2 domain, or nullptr
  float* stats;   // [batch, q_heads, 2] maximum and 1 / sum
  int64_t capacity;
  float* w;
  int64_t w_batch, w_head;
};

constexpr int kThreads = 256;

// One block per (query head, sequence); G lanes share a key.
template <typename T, int G>
__global__ void attend_kernel(const __grid_constant__ AttendArgs g) {
  constexpr int kSubs = kThreads / G;
  __shared__ float sm_m[kSubs], sm_l[kSubs];
  extern __shared__ float sm_o[];  // [kSubs][d]
  const InfercPagedKv& kv = g.a.kv;
  const int h = blockIdx.x, d = kv.head_dim, tid = threadIdx.x;
  const int64_t b = blockIdx.y;
  const int c = tid % G, sub = tid / G, hk = h / g.group;
  const int n = seq_len(g.a, b);
  const bool live = c * 8 < d;
  T* out = reinterpret_cast<T*>(g.out) + b * g.o_batch + h * g.o_head;
  float q[8] = {}, o[8] = {}, m = -INFINITY, l = 0.f;
  if (live) load8(reinterpret_cast<const T*>(g.q) + b * g.q_batch + h * g.q_head + c * 8, q);
  const int32_t* row = kv.page_table + b * kv.table_stride;
  const T* kc = reinterpret_cast<const T*>(kv.k) + hk * kv.k_head_stride + c * 8;
  const T* vc = reinterpret_cast<const T*>(kv.v) + hk * kv.v_head_stride + c * 8;
  float* scores = g.scores ? g.scores + (b * gridDim.x + h) * g.capacity : nullptr;
  for (int j0 = 0; j0 < n; j0 += kSubs) {
    const int j = j0 + sub;
    int page = -1;
    uint32_t slot = 0;
    if (j < n) {
      const uint32_t index = g.a.page.div(j);
      slot = j - index * g.a.page.d;
      page = page_of(g.a, row, index);
    }
    float x[8] = {}, s = 0.f;
    if (page >= 0 && live) load8(kc + page * kv.k_page_stride + slot * kv.k_token_stride, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += q[i] * x[i];
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= g.scale;
    if (j >= n) continue;
    if (page < 0) s = -INFINITY;
    if (scores && c == 0) scores[j] = s;
    if (page < 0) continue;
    const float m2 = fmaxf(m, s);
    const float base = m2 == -INFINITY ? 0.f : m2;
    const float keep = exp2f(m - base), p = exp2f(s - base);
    m = m2;
    l = l * keep + p;
    if (live) load8(vc + page * kv.v_page_stride + slot * kv.v_token_stride, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * keep + p * x[i];
  }
  if (c == 0) sm_m[sub] = m, sm_l[sub] = l;
  if (live)
    for (int i = 0; i < 8; ++i) sm_o[sub * d + c * 8 + i] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int s = 0; s < kSubs; ++s) top = fmaxf(top, sm_m[s]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int s = 0; s < kSubs; ++s) sum += sm_l[s] * exp2f(sm_m[s] - base);
  const float inv = n == 0 ? 0.f : 1.0f / sum;
  if (tid == 0 && g.stats) {
    g.stats[2 * (b * gridDim.x + h)] = base;
    g.stats[2 * (b * gridDim.x + h) + 1] = inv;
  }
  if (tid < d / 8) {
    float r[8] = {};
    for (int s = 0; s < kSubs; ++s) {
      const float f = exp2f(sm_m[s] - base);
      for (int i = 0; i < 8; ++i) r[i] += f * sm_o[s * d + tid * 8 + i];
    }
    for (int i = 0; i < 8; ++i) r[i] = n == 0 ? 0.f : r[i] * inv;
    store8(out + tid * 8, r);
  }
}

// Adds each position's softmax weight, summed over the group's query heads.
__global__ void weights_kernel(const __grid_constant__ AttendArgs g) {
  const InfercPagedKv& kv = g.a.kv;
  const int64_t b = blockIdx.y / kv.kv_heads;
  const int h = blockIdx.y % kv.kv_heads;
  const int64_t q_heads = kv.kv_heads * g.group;
  const int n = seq_len(g.a, b);
  float* w = g.w + b * g.w_batch + h * g.w_head;
  for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < n; j += gridDim.x * blockDim.x) {
    float sum = 0.f;
    for (int i = 0; i < g.group; ++i) {
      const int64_t r = b * q_heads + h * g.group + i;
      sum += exp2f(g.scores[r * g.capacity + j] - g.stats[2 * r]) * g.stats[2 * r + 1];
    }
    w[j] += sum;
  }
}

template <typename T>
void launch(const AttendArgs& g, cudaStream_t st) {
  const InfercPagedKv& kv = g.a.kv;
  const int d = kv.head_dim;
  const dim3 grid((unsigned)(kv.kv_heads * g.group), (unsigned)kv.batch);
  if (d <= 64) attend_kernel<T, 8><<<grid, kThreads, kThreads / 8 * d * 4, st>>>(g);
  else if (d <= 128) attend_kernel<T, 16><<<grid, kThreads, kThreads / 16 * d * 4, st>>>(g);
  else attend_kernel<T, 32><<<grid, kThreads, kThreads / 32 * d * 4, st>>>(g);
  IDEV_LAUNCHED();
  if (g.w) {
    weights_kernel<<<dim3(32, (unsigned)(kv.batch * kv.kv_heads)), 256, 0, st>>>(g);
    IDEV_LAUNCHED();
  }
}

int64_t workspace_bytes(const InfercPagedKv& kv, int64_t q_heads, bool weights) {
  const int64_t rows = kv.batch * q_heads;
  return weights ? rows * (kv.max_pages * kv.page_size + 2) * 4 : 0;
}

void check(const InfercPagedKv* kv, int64_t q_heads) {
  check_kv(kv, "PagedDecodeAttention");
  IDEV_CHECK_ARG(q_heads >= 1 && q_heads <= 65535 && q_heads % kv->kv_heads == 0,
                 "PagedDecodeAttention: q_heads must be a multiple of kv_heads");
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
    check(kv, q_heads);
    bytes = workspace_bytes(*kv, q_heads, with_weights != 0);
  });
  return bytes;
}

int inferc_dev_paged_decode_attention(const InfercPagedKv* kv, const void* q,
                                      int64_t q_batch_stride, int64_t q_head_stride,
                                      int64_t q_heads, float scale, void* out,
                                      int64_t out_batch_stride, int64_t out_head_stride,
                                      float* weights, int64_t weights_batch_stride,
                                      int64_t weights_head_stride, void* workspace,
                                      int64_t workspace_bytes_given, void* stream) {
  return guard([&] {
    const char* op = "PagedDecodeAttention";
    check(kv, q_heads);
    if (kv->batch == 0) return;
    check_rows(op, "query", q, q_batch_stride, q_head_stride, kv->dtype);
    check_rows(op, "output", out, out_batch_stride, out_head_stride, kv->dtype);
    const int64_t need = workspace_bytes(*kv, q_heads, weights != nullptr);
    IDEV_CHECK_ARG(workspace_bytes_given >= need && (need == 0 || (workspace && aligned16(workspace))),
                   "PagedDecodeAttention: the workspace is too small or not 16-byte aligned");
    AttendArgs g{};
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
    g.group = (int)(q_heads / kv->kv_heads);
    g.capacity = kv->max_pages * kv->page_size;
    if (weights) {
      g.scores = static_cast<float*>(workspace);
      g.stats = g.scores + kv->batch * q_heads * g.capacity;
      g.w = weights;
      g.w_batch = weights_batch_stride;
      g.w_head = weights_head_stride;
    }
    cudaStream_t st = as_stream(stream);
    if (kv->dtype == F32) launch<float>(g, st);
    else if (kv->dtype == F16) launch<__half>(g, st);
    else launch<__nv_bfloat16>(g, st);
  });
}

}  // extern "C"
