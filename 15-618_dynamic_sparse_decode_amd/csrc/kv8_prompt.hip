// kv8_prompt.hip -- dsd_kv8_attend_prompt for prompts and chunks of them
// (gfx950): the mathematics of kv8_attend.hip, for many rows.
//
// Bound by the matrix and vector units together: a block of 64 tokens and 32
// rows is 1024 cycles of matrix products and, its exponentials a quarter rate,
// about as many of vector work.  A workgroup's 128 rows share the tokens' codes:
// its four waves turn a group of 64 tokens into half-precision numbers once,
// in LDS, while they work on the group before, two workgroups a CU, so that one
// wave's products run beside another's exponentials.
//
// Measured (kernel times): one prompt of 8192 tokens, 32 bf16 query heads of 128
// over 8 key heads, 620 us for 550 GFLOP on one card and 665 on another (830-890
// TFLOP/s; a large bf16 matrix product alone reaches 1356 here), the matrix units
// busy 42 % of the time and the vector units 56 %; 16 prompts of 1-700 tokens 84 us
// (27 GFLOP: the longest prompts' last rows end it); f16 rows 925 us, float32 1459.  On the way there (the long prompt):
// shared groups in LDS in place of 16 rows a workgroup 1230 -> 695 us, operands
// asked for four products ahead -> 658, products and exponentials in turn and
// maxima that lag (kSlack) -> 631, the value scale in the exponent -> 621.
#include "kv8_prompt_block.h"

namespace dsdk {
namespace {

// Grid (key heads * blocks of 128 rows, batch, pieces).
template <typename T, int FMT, int NU, int kDim>
__global__ __launch_bounds__(kThreads, NU <= 2 && sizeof(T) == 2 ? 2 : 1) void
Kv8PromptKernel(Kv8AttendArgs a, Plan plan) {
  extern __shared__ __align__(16) _Float16 smem[];
  PromptBlock<T, FMT, NU, kDim, true, false>(a, plan, blockIdx.x, blockIdx.y, blockIdx.z, smem);
}

// Calls f with the kernel of a head size.
template <typename T, int FMT, typename F>
void WithKernel(int dim, F&& f) {
  if (dim == 64) return f(Kv8PromptKernel<T, FMT, 1, 64>);
  if (dim < 64) return f(Kv8PromptKernel<T, FMT, 1, 0>);
  if (dim == 128) return f(Kv8PromptKernel<T, FMT, 2, 128>);
  if (dim < 128) return f(Kv8PromptKernel<T, FMT, 2, 0>);
  return f(Kv8PromptKernel<T, FMT, 4, 0>);
}

template <typename T, int FMT>
void Launch(const Kv8AttendArgs& a, hipStream_t stream) {
  Plan p = PromptPlan(a.c, a.b, a.q_heads);
  PlaceParts(&p, a);
  const dim3 grid(a.c.heads * p.blocks, a.b.batch, p.pieces);
  WithKernel<T, FMT>(a.c.dim, [&](auto kernel) {
    kernel<<<grid, kThreads, PromptLdsBytes(a.c.dim), stream>>>(a, p);
  });
  DSD_HIP_CHECK(hipGetLastError());
  Merge<T>(a, p, stream);
}

template <typename T>
void LaunchType(const Kv8AttendArgs& a, hipStream_t stream) {
  a.c.format == DSD_KV8_INT8 ? Launch<T, DSD_KV8_INT8>(a, stream)
                             : Launch<T, DSD_KV8_E4M3>(a, stream);
}

template <typename T, int FMT>
void PreloadDim(const Kv8View& c) {
  WithKernel<T, FMT>(c.dim, [&](auto kernel) {
    PreloadKernel(kernel);
    DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(PromptLdsBytes(c.dim))));
  });
}

template <typename T>
void PreloadType(const Kv8View& c) {
  c.format == DSD_KV8_INT8 ? PreloadDim<T, DSD_KV8_INT8>(c) : PreloadDim<T, DSD_KV8_E4M3>(c);
}

}  // namespace

void PreloadKv8Prompt(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
}

size_t Kv8PromptWorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  return MostPartBytes(c, PromptPlan(c, b, q_heads), kPromptTarget);
}

void LaunchKv8Prompt(const Kv8AttendArgs& a, hipStream_t stream) {
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(a, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(a, stream);
    default: return LaunchType<_Float16>(a, stream);
  }
}

}  // namespace dsdk
