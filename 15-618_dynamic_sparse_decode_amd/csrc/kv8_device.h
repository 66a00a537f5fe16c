// kv8_device.h -- device helpers of the 8-bit paged cache's kernels.
#pragma once

#include <type_traits>

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

// N consecutive elements as they lie in memory (16-bit ones two a word).
template <typename T, int N>
struct Packed {
  unsigned w[N * sizeof(T) / 4];

  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (std::is_same<T, float>::value) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __bf16>::value) {
      return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    } else {
      return static_cast<float>(
          __builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)))));
    }
  }
  // Elements i (even) and i + 1.
  __device__ __forceinline__ void Set2(int i, float x, float y) {
    if constexpr (std::is_same<T, float>::value) {
      w[i] = __float_as_uint(x);
      w[i + 1] = __float_as_uint(y);
    } else {
      typedef T T2 __attribute__((ext_vector_type(2)));
      const F32x2 v = {x, y};
      w[i >> 1] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, T2));
    }
  }
  // Elements [at, at + 8) from p; vec: p is 16-byte aligned.
  __device__ __forceinline__ void Load8(int at, const T* p, bool vec) {
    unsigned* to = w + at * static_cast<int>(sizeof(T)) / 4;
    if (vec) {
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T)) * 2; k += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned*>(p) + k);
        to[k] = v.x;
        to[k + 1] = v.y;
        to[k + 2] = v.z;
        to[k + 3] = v.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 8; ++k) to[k] = __float_as_uint(p[k]);
    } else {
      const uint16_t* from = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        to[k] = from[2 * k] | static_cast<unsigned>(from[2 * k + 1]) << 16;
      }
    }
  }
  __device__ __forceinline__ void Store8(int at, T* p, bool vec) const {
    const unsigned* from = w + at * static_cast<int>(sizeof(T)) / 4;
    if (vec) {
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T)) * 2; k += 4) {
        *reinterpret_cast<uint4*>(reinterpret_cast<unsigned*>(p) + k) =
            make_uint4(from[k], from[k + 1], from[k + 2], from[k + 3]);
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = __uint_as_float(from[k]);
    } else {
      uint16_t* to = reinterpret_cast<uint16_t*>(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        to[2 * k] = static_cast<uint16_t>(from[k]);
        to[2 * k + 1] = static_cast<uint16_t>(from[k] >> 16);
      }
    }
  }
};

// Eight consecutive elements as floats.
template <typename T>
__device__ __forceinline__ void Load8(const T* p, bool vec, float* x) {
  Packed<T, 8> raw;
  raw.Load8(0, p, vec);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = raw[i];
}

}  // namespace
}  // namespace dsdk
