// kv8_device.h -- device helpers of the 8-bit paged cache's kernels.
#pragma once

#include "kv8.h"
#include "step_common.h"

namespace dsdk {
namespace {

typedef _Float16 F16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 F16x8 __attribute__((ext_vector_type(8)));
typedef float F32x2 __attribute__((ext_vector_type(2)));
typedef float F32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 Bf16x2 __attribute__((ext_vector_type(2)));

constexpr float kKv8Tiny = 0x1p-126f;  // the least scale

// One request of a batch, checked: false (reported) where what the device
// data says does not fit the batch's sizes.  No index outside the caller's
// arrays is formed from a request that passed.
struct Kv8Request {
  int row0 = 0;   // its first row of q, k, v, out
  int n = 0;      // its new (query) tokens
  int past = 0;
  int list = 0;   // its first entry of page_ids
  int pages = 0;  // entries
};

__device__ __forceinline__ bool Kv8ReadList(const dsd_kv8_batch& b, int r, Kv8Request* q) {
  if (b.list_stride > 0) {
    q->list = r * b.list_stride;
    q->pages = b.page_counts[r];
    return q->pages >= 0 && q->pages <= b.list_stride && q->pages <= b.total_pages - q->list;
  }
  q->list = b.page_offsets[r];
  const int end = b.page_offsets[r + 1];
  q->pages = end - q->list;
  return q->list >= 0 && end >= q->list && end <= b.total_pages;
}

// With new tokens: rows, past and a list that holds them all.
__device__ __forceinline__ bool Kv8ReadTokens(const dsd_kv8_batch& b, int r, int page,
                                              Kv8Request* q) {
  q->row0 = b.token_offsets[r];
  const int end = b.token_offsets[r + 1];
  q->past = b.past_tokens[r];
  const bool list_ok = Kv8ReadList(b, r, q);
  if (q->row0 < 0 || end < q->row0 || end > b.tokens) return false;
  q->n = end - q->row0;
  if (q->n == 0) return true;
  return list_ok && q->n <= b.max_tokens && q->past >= 0 &&
         static_cast<int64_t>(q->past) + q->n <= static_cast<int64_t>(q->pages) * page &&
         q->past <= 0x7fffffff - q->n;
}

// Orders one wave's LDS writes before its reads of what other lanes wrote.
__device__ __forceinline__ void WaveLdsFence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Eight consecutive elements as floats; vec: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void Load8(const T* p, bool vec, float* x) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const F32x4 a = *reinterpret_cast<const F32x4*>(p);
    const F32x4 b = *reinterpret_cast<const F32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 a = *reinterpret_cast<const T8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
  }
}

template <typename T>
__device__ __forceinline__ void Store8(T* p, bool vec, const float* x) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = static_cast<T>(x[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<F32x4*>(p) = F32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<F32x4*>(p + 4) = F32x4{x[4], x[5], x[6], x[7]};
  } else {
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = static_cast<T>(x[i]);
    *reinterpret_cast<T8*>(p) = a;
  }
}

}  // namespace
}  // namespace dsdk
