// The paged cache's device view: element types, row access, page lookup and
// the flag for indexes that point outside their buffers. Shared by
// paged_kv.cu (norm, rotation, append, evict) and paged_attention.cu.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "paged_plan.h"

namespace inferc_dev {
namespace paged {

constexpr int64_t kMostPositions = 1 << 30;  // of a sequence

enum DType : int { F32 = 1, F16 = 10, BF16 = 16 };  // ONNX TensorProto codes

// Eight values of a row as they lie in memory, four from each of two places
// (which may adjoin), to be widened when they are used.
template <typename T>
struct Raw8 {
  using Four = std::conditional_t<sizeof(T) == 4, uint4, uint2>;
  Four part[2] = {};
  __device__ __forceinline__ void load(const T* p, int second = 4) {
    part[0] = *reinterpret_cast<const Four*>(p);
    part[1] = *reinterpret_cast<const Four*>(p + second);
  }
  __device__ __forceinline__ void widen(float* x) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (std::is_same_v<T, float>) {
        x[4 * i] = __uint_as_float(part[i].x);
        x[4 * i + 1] = __uint_as_float(part[i].y);
        x[4 * i + 2] = __uint_as_float(part[i].z);
        x[4 * i + 3] = __uint_as_float(part[i].w);
      } else {
        const uint32_t w[2] = {part[i].x, part[i].y};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float2 f;
          if constexpr (std::is_same_v<T, __half>)
            f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          else
            f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
          x[4 * i + 2 * j] = f.x;
          x[4 * i + 2 * j + 1] = f.y;
        }
      }
    }
  }
};

// Four values rounded to T, to a place of 4 * sizeof(T) alignment.
template <typename T>
__device__ __forceinline__ void store4(T* p, const float* x) {
  if constexpr (std::is_same_v<T, float>) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  Raw8<T> raw;
  raw.load(p);
  raw.widen(x);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (std::is_same_v<T, float>) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Device arguments of every paged kernel: the caller's descriptor, the
// division by the page size, and two flags: flag[0] is raised by an index that
// points outside its buffer, flag[1] by a wait that gave up.
struct Args {
  InfercPagedKv kv;
  FastDiv page;
  int* flag;
};

// Positions of sequence b, clamped into what its page table can name.
__device__ __forceinline__ int seq_len(const Args& a, int64_t b) {
  const int n = a.kv.lens[b];
  const int cap = (int)(a.kv.max_pages * a.kv.page_size);
  if (n >= 0 && n <= cap) return n;
  *a.flag = 1;
  return n < 0 ? 0 : cap;
}

// Page of position p of a sequence whose table row is `row`; -1 (and the
// flag) when the id is no page.
__device__ __forceinline__ int page_of(const Args& a, const int32_t* row, uint32_t index) {
  const int id = row[index];
  if (id >= 0 && id < a.kv.num_pages) return id;
  *a.flag = 1;
  return -1;
}

// Address of the flags on the current device; inferc_dev_stream_synchronize
// reports them.
int* range_flag_ptr();
// Throws INFERC_ERR_INVALID when the descriptor is not one the kernels take.
void check_kv(const InfercPagedKv* kv, const char* op);
void check_rows(const char* op, const char* what, const void* p, int64_t stride_a,
                int64_t stride_b, int dtype);
// Throws it when rows of `d` elements that a kernel writes, at i * a.stride +
// j * b.stride + k * c.stride, may share elements.
struct Steps {
  int64_t count, stride;
};
void check_apart(const char* op, const char* what, int64_t d, Steps a, Steps b,
                 Steps c = {1, 0});
int elem_bytes(int dtype);

}  // namespace paged

// Bit 0: an index was out of range; bit 1: a wait gave up.
int read_and_clear_paged();

}  // namespace inferc_dev
