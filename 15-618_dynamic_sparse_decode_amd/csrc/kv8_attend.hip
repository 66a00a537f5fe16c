// kv8_attend.hip -- dsd_kv8_attend, and dsd_kv8_attend_prompt and _cross of few rows
// (gfx950):
// softmax attention over the pages of an 8-bit cache.
//
// Mathematics.  Codes are exact in half precision, so q K^T is a product of
// half-precision matrices: q scaled by a power of two so that its row's
// largest element lies in [2^13, 2^14) -- one term for 16-bit queries (what
// falls below half precision's range is 2^-38 of that element), two for
// float32 ones -- times the codes; the page's scale and the power of two go on
// the logits afterwards, in float32.  Weights p = 2^(s - m) (s in the log2
// domain, m the running maximum) meet the value codes the same way, as p * v *
// 2^(m - n + 15) with v the page's value scale and n the running maximum of s +
// log2 v, so at most 2^15 whatever the scales and logits: half precision rounds them to
// 2^-11, or 2^-22 as two terms where the output is finer than bf16 (bf16 outputs,
// whose own rounding is 2^-8, are off by 0.0017 of their size either way; two terms
// took 12.2 us in place of 11.5 for one request of 1000 tokens, 38.9 in place of
// 37.6 for drafted tokens).  All sums are float32.
//
// Bound by HBM for long lists: a token's codes and scales are read once for all
// query heads of its key head.  Measured (kernel times): 32 requests of 32768
// tokens, 8 key heads of 128, pages of 16: 366 us for 2.15 GB, 5.9 TB/s, what
// reads alone reach here; 64 requests of 32 pages of 64: 44 us, 6.2 TB/s; 16
// requests of 512-2048 tokens, 32 key heads, float32: 36 us, 5.2 TB/s; 4 of
// 65536-131072, int8, heads of 64: 42 us, 5.3 TB/s, and 5 for the merge; one of
// 1000 tokens: 11.6 us, a chain of ids -> scales and codes -> products.
#include "kv8_attend_block.h"

#include <algorithm>

namespace dsdk {
namespace {

// Grid (key heads * row tiles, batch, pieces).
template <typename T, int FMT, int NU, int kDim, int W>
__global__ __launch_bounds__(W* kWave, NU <= 2 ? 2 : 1) void Kv8AttendKernel(Kv8AttendArgs a,
                                                                            Plan p) {
  extern __shared__ __align__(16) float lds[];
  AttendBlock<T, FMT, NU, kDim, W, false>(a, p, blockIdx.x, blockIdx.y, blockIdx.z, lds);
}

// Grid (256 numbers of a row each, batch).
template <typename T>
__global__ __launch_bounds__(256) void Kv8GroupQueriesKernel(const T* q, int64_t q_stride,
                                                             int group, int dim, int elements,
                                                             float* sums) {
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= elements) return;
  const int head = e / dim, d = e - head * dim;
  const T* p = q + blockIdx.y * q_stride + static_cast<int64_t>(head) * group * dim + d;
  float sum = static_cast<float>(p[0]);
  for (int g = 1; g < group; ++g) sum += static_cast<float>(p[g * dim]);
  sums[static_cast<int64_t>(blockIdx.y) * elements + e] = sum;
}

constexpr int kWaves = kAttendWaves;

// Whether a call has rows enough for kv8_prompt.hip and kv8_cross.hip.  Both sides (us, this
// file's form and that one's): 16 requests with 128 rows behind 8000 tokens 175
// and 134; with 64 rows behind 1000 tokens 21 and 40; one with 64 rows behind
// 60000 tokens 101 and 157.
bool ManyRows(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  return static_cast<int64_t>(b.max_tokens) * (q_heads / c.heads) > 64;
}

// Calls f with the kernel of a head size.
template <typename T, int FMT, typename F>
void WithKernel(int dim, F&& f) {
  if (dim == 64) return f(Kv8AttendKernel<T, FMT, 1, 64, kWaves>);
  if (dim < 64) return f(Kv8AttendKernel<T, FMT, 1, 0, kWaves>);
  if (dim == 128) return f(Kv8AttendKernel<T, FMT, 2, 128, kWaves>);
  if (dim < 128) return f(Kv8AttendKernel<T, FMT, 2, 0, kWaves>);
  return f(Kv8AttendKernel<T, FMT, 4, 0, kWaves>);
}

template <typename T, int FMT>
void Launch(const Kv8AttendArgs& a, const Plan& p, hipStream_t stream) {
  const dim3 grid(a.c.heads * p.blocks, a.b.batch, p.pieces);
  WithKernel<T, FMT>(a.c.dim, [&](auto kernel) {
    kernel<<<grid, kWaves * kWave, AttendLdsBytes(a.c.dim), stream>>>(a, p);
  });
  DSD_HIP_CHECK(hipGetLastError());
  Merge<T>(a, p, stream);
}

template <typename T>
void LaunchType(const Kv8AttendArgs& a, const Plan& p, hipStream_t stream) {
  a.c.format == DSD_KV8_INT8 ? Launch<T, DSD_KV8_INT8>(a, p, stream)
                             : Launch<T, DSD_KV8_E4M3>(a, p, stream);
}

template <typename T, int FMT>
void PreloadDim(const Kv8View& c) {
  WithKernel<T, FMT>(c.dim, [&](auto kernel) {
    PreloadKernel(kernel);
    DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(AttendLdsBytes(c.dim))));
  });
}

template <typename T>
void PreloadType(const Kv8View& c) {
  c.format == DSD_KV8_INT8 ? PreloadDim<T, DSD_KV8_INT8>(c) : PreloadDim<T, DSD_KV8_E4M3>(c);
  PreloadKernel(Kv8MergeKernel<T>);
  PreloadKernel(Kv8MergeRowsKernel<T>);
  PreloadKernel(Kv8GroupQueriesKernel<T>);
}

}  // namespace

size_t Kv8WorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  if (b.batch == 0) return 0;
  dsd_kv8_batch one = b;
  one.max_tokens = 1;
  size_t bytes = MostPartBytes(c, AttendPlan(c, one, q_heads, false), kAttendTarget);
  if (b.max_tokens > 1) {
    bytes = std::max(bytes, MostPartBytes(c, AttendPlan(c, b, q_heads, true), kAttendTarget));
  }
  // (of one token a request too, where query heads enough share a key head)
  if (ManyRows(c, b, q_heads)) bytes = std::max(bytes, Kv8PromptWorkspaceBytes(c, b, q_heads));
  return bytes;
}

void LaunchKv8GroupQueries(const Kv8View& c, int batch, int type, int q_heads, const void* q,
                           int64_t q_stride, float* sums, hipStream_t stream) {
  const int elements = c.heads * c.dim;
  const dim3 grid((elements + 255) / 256, batch);
  auto launch = [&](auto* rows) {
    using T = std::remove_cv_t<std::remove_pointer_t<decltype(rows)>>;
    Kv8GroupQueriesKernel<T><<<grid, 256, 0, stream>>>(rows, q_stride, q_heads / c.heads, c.dim,
                                                       elements, sums);
  };
  switch (type) {
    case DSD_TYPE_F32: launch(static_cast<const float*>(q)); break;
    case DSD_TYPE_BF16: launch(static_cast<const __bf16*>(q)); break;
    default: launch(static_cast<const _Float16*>(q));
  }
  DSD_HIP_CHECK(hipGetLastError());
}

void PreloadKv8Attend(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
}

void LaunchKv8Attend(const Kv8AttendArgs& a, hipStream_t stream) {
  if (a.b.batch == 0 || (a.many && a.b.tokens == 0)) return;
  if (a.many && ManyRows(a.c, a.b, a.q_heads)) {
    return a.causal ? LaunchKv8Prompt(a, stream) : LaunchKv8Cross(a, stream);
  }
  Plan p = AttendPlan(a.c, a.b, a.q_heads, a.many);
  PlaceParts(&p, a);
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(a, p, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(a, p, stream);
    default: return LaunchType<_Float16>(a, p, stream);
  }
}

}  // namespace dsdk
