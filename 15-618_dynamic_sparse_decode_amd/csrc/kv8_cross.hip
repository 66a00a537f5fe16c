// kv8_cross.hip -- dsd_kv8_attend_cross for many rows (gfx950): query tokens that see
// all tokens of their request's list (an encoder's states, a document), the mathematics
// and the tiles of kv8_prompt.hip without its diagonal.
//
// A list's pages may hold fewer tokens than they have places, any of them: a group of
// 64 tokens is masked where one of its chunks is not full, which the wave votes on.
//
// What bounds it: a group's turning into halves and its exponentials (vector units), LDS,
// and the products (matrix units), in turn.  bf16, 32 query heads on 8 of 128: 4096
// queries over 8192 tokens 546 us, 1007 TFLOP/s (557 on another card; a large bf16 matrix
// product reaches 1356 here), f16 rows, whose weights take two terms, 725, float32 ones,
// whose queries do too, 1255; 16 requests of 1 to 300 queries over 200 to 3000 tokens, int8,
// 131 us a call (139 under a profiler), where the longest lists' 47 groups in turn end the
// launch.  Heads of 144 to 256 spill: a wave has 32 rows of all dims in registers, 103 to
// 173 of them in scratch, and 4096 over 8192 of 16 heads on 8 of 256 takes 2713 us, 203
// TFLOP/s.
#include "kv8_prompt_block.h"

namespace dsdk {
namespace {

constexpr int kWideWaves = 8;
constexpr int kWideRows = 32 * kWideWaves;

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

// Eight waves to a workgroup where a request has more than 128 rows: the halves of a group
// of 64 tokens then go to LDS, whose writes are a quarter of its reads' rate (31 bytes a
// cycle measured), once for 256 rows.  4096 tokens over 8192: 543 us, four waves 604; 1024
// over 8192: 240 and 217 (a workgroup a CU either way), 512: 237 and 135.  16-bit rows of
// heads of up to 128 (others' registers hold one workgroup of four waves a CU).
template <typename T>
bool Wide(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  const int group = q_heads / c.heads;
  const int64_t rows = static_cast<int64_t>(b.max_tokens) * group;
  const int64_t blocks = (rows + kWideRows - 1) / kWideRows * c.heads * b.batch;
  return sizeof(T) == 2 && c.dim <= 128 && rows > kRows && blocks >= 256;
}

// Grid (key heads * blocks of 32 W rows, batch, pieces).
template <typename T, int FMT, int NU, int kDim, int W>
__global__ __launch_bounds__(W* kWave, NU <= 2 && sizeof(T) == 2 ? 2 : 1) void
Kv8CrossKernel(Kv8AttendArgs a, Plan plan) {
  extern __shared__ __align__(16) _Float16 smem[];
  PromptBlock<T, FMT, NU, kDim, false, false, W>(a, plan, blockIdx.x, ByLength(a.b, blockIdx.y),
                                                 blockIdx.z, smem);
}

// Calls f with the kernel of a head size, and its threads.
template <typename T, int FMT, typename F>
void WithKernel(int dim, bool wide, F&& f) {
  if constexpr (sizeof(T) == 2) {
    if (wide) {
      if (dim == 64) return f(Kv8CrossKernel<T, FMT, 1, 64, kWideWaves>, kWideWaves * kWave);
      if (dim < 64) return f(Kv8CrossKernel<T, FMT, 1, 0, kWideWaves>, kWideWaves * kWave);
      if (dim == 128) return f(Kv8CrossKernel<T, FMT, 2, 128, kWideWaves>, kWideWaves * kWave);
      return f(Kv8CrossKernel<T, FMT, 2, 0, kWideWaves>, kWideWaves * kWave);
    }
  }
  if (dim == 64) return f(Kv8CrossKernel<T, FMT, 1, 64, kPromptWaves>, kThreads);
  if (dim < 64) return f(Kv8CrossKernel<T, FMT, 1, 0, kPromptWaves>, kThreads);
  if (dim == 128) return f(Kv8CrossKernel<T, FMT, 2, 128, kPromptWaves>, kThreads);
  if (dim < 128) return f(Kv8CrossKernel<T, FMT, 2, 0, kPromptWaves>, kThreads);
  return f(Kv8CrossKernel<T, FMT, 4, 0, kPromptWaves>, kThreads);
}

template <typename T, int FMT>
void Launch(const Kv8AttendArgs& a, hipStream_t stream) {
  const bool wide = Wide<T>(a.c, a.b, a.q_heads);
  Plan p = PromptPlan(a.c, a.b, a.q_heads, wide ? kWideRows : kRows);
  PlaceParts(&p, a);
  const dim3 grid(a.c.heads * p.blocks, a.b.batch, p.pieces);
  WithKernel<T, FMT>(a.c.dim, wide, [&](auto kernel, int threads) {
    kernel<<<grid, threads, PromptLdsBytes(a.c.dim), stream>>>(a, p);
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
  for (const bool wide : {false, true}) {
    if (wide && c.dim > 128) continue;
    WithKernel<T, FMT>(c.dim, wide, [&](auto kernel, int) {
      PreloadKernel(kernel);
      DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(PromptLdsBytes(c.dim))));
    });
  }
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
