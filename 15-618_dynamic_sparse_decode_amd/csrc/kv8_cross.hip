// kv8_cross.hip -- dsd_kv8_attend_cross for many rows (gfx950): query tokens that see
// all tokens of their request's list (an encoder's states, a document), the mathematics
// and the tiles of kv8_prompt.hip without its diagonal.
//
// A list's pages may hold fewer tokens than they have places, any of them: a group of
// 64 tokens is masked where one of its chunks is not full, which the wave votes on.
#include "kv8_prompt_block.h"

namespace dsdk {
namespace {

// The request whose list is the i-th longest, so that long ones are not begun last (up to
// 64 requests, a lane each; more are taken as they come).  All lanes of a wave.
__device__ __forceinline__ int ByLength(const dsd_kv8_batch& b, int i) {
  if (b.batch == 1 || b.batch > kWave) return i;
  const int lane = threadIdx.x & (kWave - 1);
  Kv8Request q;
  int pages = -1;
  if (lane < b.batch) pages = Kv8ReadList(b, lane, &q) ? q.pages : 0;
  int before = 0;
  for (int k = 0; k < b.batch; ++k) {
    const int other = __builtin_amdgcn_readlane(pages, k);
    before += other > pages || (other == pages && k < lane) ? 1 : 0;
  }
  return __ffsll(__ballot(lane < b.batch && before == i)) - 1;
}

// Grid (key heads * blocks of 128 rows, batch, pieces).
template <typename T, int FMT, int NU, int kDim>
__global__ __launch_bounds__(kThreads, NU <= 2 && sizeof(T) == 2 ? 2 : 1) void
Kv8CrossKernel(Kv8AttendArgs a, Plan plan) {
  extern __shared__ __align__(16) _Float16 smem[];
  PromptBlock<T, FMT, NU, kDim, false, false>(a, plan, blockIdx.x, ByLength(a.b, blockIdx.y),
                                              blockIdx.z, smem);
}

// Calls f with the kernel of a head size.
template <typename T, int FMT, typename F>
void WithKernel(int dim, F&& f) {
  if (dim == 64) return f(Kv8CrossKernel<T, FMT, 1, 64>);
  if (dim < 64) return f(Kv8CrossKernel<T, FMT, 1, 0>);
  if (dim == 128) return f(Kv8CrossKernel<T, FMT, 2, 128>);
  if (dim < 128) return f(Kv8CrossKernel<T, FMT, 2, 0>);
  return f(Kv8CrossKernel<T, FMT, 4, 0>);
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
  PreloadKernel(Kv8MergeKernel<T>);
  PreloadKernel(Kv8MergeRowsKernel<T>);
}

}  // namespace

void PreloadKv8Cross(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
}

void LaunchKv8Cross(const Kv8AttendArgs& a, hipStream_t stream) {
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(a, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(a, stream);
    default: return LaunchType<_Float16>(a, stream);
  }
}

}  // namespace dsdk
