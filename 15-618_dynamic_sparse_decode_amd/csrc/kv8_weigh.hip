// kv8_weigh.hip -- dsd_kv8_attend_weigh (gfx950): dsd_kv8_attend, and each token's softmax
// weight, summed over the query heads of its key head, added to the caller's array.
//
// Mathematics.  A weight is 2^(s - m) / l with s the logit in the log2 domain and m, l
// its row's maximum and sum, which are known once the whole list has been read.  Reading
// the keys a second time would be half of the bytes again; the logits are 4 bytes a token
// and query head beside 2 dim / group of codes (a sixteenth at 4 heads of 128), so the
// attention writes them to the workspace and a second launch turns them into weights.
// Sums over a group's heads are float32, in order; a token's own sum takes one atomic
// addition (a page that several requests list gets all of theirs, in any order).
// Logits lie by their list's place in page_ids.  Where page_offsets falls, a list behind
// may name entries of one before: its logits are formed a second time instead.
//
// What bounds it: HBM.  32 requests of 32768 tokens, 32 query heads on 8 of 128, bf16:
// attention 460 us for 2.15 GB of codes and 134 MB of logits, where reads alone reach
// 6.3 TB/s and sixteen parts read to one written 5.0 to 5.35 (430 to 456 us); the weights
// 60 us for 134 MB of logits read and 67 MB read and written; the whole call 538 us.
#include "kv8_attend_block.h"

namespace dsdk {
namespace {

// Grid (key heads * row tiles, batch, pieces).
template <typename T, int FMT, int NU, int kDim>
__global__ __launch_bounds__(kAttendWaves* kWave, NU <= 2 ? 2 : 1) void Kv8AttendLogitsKernel(
    Kv8AttendArgs a, Plan p, float* logits) {
  extern __shared__ __align__(16) float lds[];
  AttendBlock<T, FMT, NU, kDim, kAttendWaves, false, true>(
      a, p, blockIdx.x, blockIdx.y, blockIdx.z, lds, logits, LaterList(a.b, blockIdx.y));
}

// A logit (times log2 e) from the query and the codes, in 64 bits: of lists that the
// attention kept none of.  Element i of the queries, byte c of the codes.
__device__ __forceinline__ double QueryNumber(const Kv8AttendArgs& a, int64_t i) {
  switch (a.type) {
    case DSD_TYPE_F32: return static_cast<double>(static_cast<const float*>(a.q)[i]);
    case DSD_TYPE_BF16: return static_cast<double>(static_cast<float>(static_cast<const __bf16*>(a.q)[i]));
    default: return static_cast<double>(static_cast<float>(static_cast<const _Float16*>(a.q)[i]));
  }
}
__device__ __forceinline__ float LogitOf(const Kv8AttendArgs& a, int64_t query, int64_t key, float scale) {
  double sum = 0.0;
#pragma unroll 1
  for (int d = 0; d < a.c.dim; ++d) {
    const uint8_t c = a.c.keys[key + d];
    const double k = a.c.format == DSD_KV8_INT8
                         ? static_cast<double>(static_cast<int8_t>(c))
                         : static_cast<double>(__builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 0));
    sum = fma(QueryNumber(a, query + d), k, sum);
  }
  return static_cast<float>(sum * static_cast<double>(scale) * (static_cast<double>(a.scale) * kLog2e));
}

constexpr int kRowTile = 64;

// Maxima and reciprocal sums of rows [row0, row0 + rows) of a key head.
__device__ __forceinline__ void RowSums(const Kv8AttendArgs& a, const Plan& p, int r, int head, int row0,
                                        int rows, int pieces, float* row_base, float* row_inv) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  for (int i = wave; i < rows; i += 4) {
    PieceStats st = {-INFINITY, -1.0f, 0.0f};
    if (lane < pieces) st = p.stats[PartSlot(p, a.c.heads, r, head, row0 + i) + lane];
    const bool some = !(st.l < 0.0f);
    float peak = some ? st.m : -INFINITY;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) peak = fmaxf(peak, __shfl_xor(peak, o, kWave));
    const float base = peak == -INFINITY ? 0.0f : peak;
    float sum = some ? st.l * Exp2(st.m - base) : 0.0f;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) sum += __shfl_xor(sum, o, kWave);
    if (lane == 0) {
      row_base[i] = base;
      row_inv[i] = 1.0f / sum;
    }
  }
}

// All of a list's weights by one workgroup of 256, the logits formed again.
__device__ __forceinline__ void WeighAgain(const Kv8AttendArgs& a, const Plan& p, const Span& s, int r,
                                           int head, float* row_base, float* row_inv, float* weights) {
  const Kv8View& c = a.c;
  for (int row0 = 0; row0 < p.group; row0 += kRowTile) {
    const int rows = min(kRowTile, p.group - row0);
    __syncthreads();
    RowSums(a, p, r, head, row0, rows, Pieces(p, s), row_base, row_inv);
    __syncthreads();
#pragma unroll 1
    for (int slot = 0; slot < s.q.pages; ++slot) {
      const int page = a.b.page_ids[s.q.list + slot];
      const int count = InPool(page, c.capacity) ? min(c.token_counts[page], c.page) : 0;
      const int64_t pair = static_cast<int64_t>(page) * c.heads + head;
      for (int at = threadIdx.x; at < count; at += 256) {
        float w = 0.0f;
#pragma unroll 1
        for (int i = 0; i < rows; ++i) {
          const int64_t query = r * a.q_stride + static_cast<int64_t>(head * p.group + row0 + i) * c.dim;
          const float x = LogitOf(a, query, (pair * c.page + at) * c.dim, c.key_scales[pair]);
          w = fmaf(Exp2(x - row_base[i]), row_inv[i], w);
        }
        unsafeAtomicAdd(weights + pair * c.page + at, w);
      }
    }
  }
}

// Grid (shares of a list and one more, key heads, batch): a wave has kBlocks blocks of 64
// tokens at a time on their way, lane l their place l; the first ones' logits and pages are
// asked for before the rows' sums are formed.  The last share has the lists without logits.
constexpr int kBlocks = 4;
constexpr int kFirstRows = 4;
__global__ __launch_bounds__(256) void Kv8WeighKernel(Kv8AttendArgs a, Plan p, const float* logits,
                                                      float* weights) {
  __shared__ float row_base[kRowTile], row_inv[kRowTile];
  const Kv8View& c = a.c;
  const int r = blockIdx.z, head = blockIdx.y;
  const int shares = static_cast<int>(gridDim.x) - 1;
  const int later = LaterList(a.b, r);
  Span s;
  if (!FindSpan(a, p.group, r, 0, p.group, &s)) return;
  if (static_cast<int>(blockIdx.x) == shares) {
    if (__ballot(later != 0) != 0) WeighAgain(a, p, s, r, head, row_base, row_inv, weights);
    return;
  }
  const int blocks = (s.chunks + 3) / 4;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int first = static_cast<int>(blockIdx.x) * 4 * kBlocks;
  if (first >= blocks) return;
  const int pieces = Pieces(p, s);
  const unsigned inverse = 0xffffffffu / static_cast<unsigned>(c.chunks) + 1u;
  const float* from = logits + LogitBlock(a, p, head, r, s.q.list, 0) +
                      ((lane >> 2 & 3) * 4 + (lane >> 4)) * p.group * 4 + (lane & 3);
  const int block_floats = 64 * p.group;
  for (int row0 = 0; row0 < p.group; row0 += kRowTile) {
    const int rows = min(kRowTile, p.group - row0);
    float y[kFirstRows][kBlocks];
    int page[kBlocks], off[kBlocks];
    auto logit = [&](int b0, int k, int i) {  // (of a block behind the last: the last one's)
      return from[static_cast<int64_t>(min(b0 + k, blocks - 1)) * block_floats +
                  4 * (row0 + min(i, rows - 1))];
    };
    auto fetch = [&](int b0) {
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const int at = min((b0 + k) * 64 + lane, s.q.pages * c.page - 1);
        const int slot = c.chunks == 1 ? at >> 4 : static_cast<int>(__umulhi(at >> 4, inverse));
        off[k] = at - slot * c.page;
        page[k] = a.b.page_ids[s.q.list + slot];
#pragma unroll
        for (int i = 0; i < kFirstRows; ++i) y[i][k] = logit(b0, k, i);
      }
    };
    int b0 = first + wave * kBlocks;
    fetch(min(b0, blocks - 1));
    __syncthreads();
    RowSums(a, p, r, head, row0, rows, pieces, row_base, row_inv);
    __syncthreads();
    if (__ballot(later != 0) != 0) return;
    for (; b0 < blocks; b0 += shares * 4 * kBlocks) {
      if (b0 != first + wave * kBlocks) fetch(b0);
      int count[kBlocks];
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        count[k] = InPool(page[k], c.capacity) ? c.token_counts[page[k]] : 0;
      }
      float w[kBlocks] = {};
#pragma unroll
      for (int i = 0; i < kFirstRows; ++i) {
        if (i >= rows) break;
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
          w[k] = fmaf(Exp2(y[i][k] - row_base[i]), row_inv[i], w[k]);
        }
      }
#pragma unroll 4
      for (int i = kFirstRows; i < rows; ++i) {
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
          w[k] = fmaf(Exp2(logit(b0, k, i) - row_base[i]), row_inv[i], w[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        if ((b0 + k) * 64 + lane < s.q.pages * c.page && off[k] < count[k]) {
          unsafeAtomicAdd(weights + (static_cast<int64_t>(page[k]) * c.heads + head) * c.page + off[k],
                          w[k]);
        }
      }
    }
  }
}

// Calls f with the kernel of a head size.
template <typename T, int FMT, typename F>
void WithKernel(int dim, F&& f) {
  if (dim == 64) return f(Kv8AttendLogitsKernel<T, FMT, 1, 64>);
  if (dim < 64) return f(Kv8AttendLogitsKernel<T, FMT, 1, 0>);
  if (dim == 128) return f(Kv8AttendLogitsKernel<T, FMT, 2, 128>);
  if (dim < 128) return f(Kv8AttendLogitsKernel<T, FMT, 2, 0>);
  return f(Kv8AttendLogitsKernel<T, FMT, 4, 0>);
}

// The workspace: parts (of lists in pieces), stats, logits.
size_t PartBytes(const Kv8View& c, const dsd_kv8_batch& b, const Plan& p) {
  return p.pieces == 1 ? 0 : PlanSlots(c, b, p) * sizeof(float) * c.dim;
}
size_t StatsBytes(const Kv8View& c, const dsd_kv8_batch& b, const Plan& p) {
  return (PlanSlots(c, b, p) * sizeof(PieceStats) + 15) / 16 * 16;
}
size_t LogitBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  Kv8AttendArgs a;
  a.c = c;
  a.b = b;
  return static_cast<size_t>(q_heads) * LogitBlocks(a) * 64 * sizeof(float);
}

template <typename T, int FMT>
void Launch(const Kv8AttendArgs& a, float* weights, hipStream_t stream) {
  Plan p = AttendPlan(a.c, a.b, a.q_heads, false);
  unsigned char* space = static_cast<unsigned char*>(a.workspace);
  p.part = reinterpret_cast<float*>(space);
  space += PartBytes(a.c, a.b, p);
  p.stats = reinterpret_cast<PieceStats*>(space);
  space += StatsBytes(a.c, a.b, p);
  float* logits = reinterpret_cast<float*>(space);
  const dim3 grid(a.c.heads * p.blocks, a.b.batch, p.pieces);
  WithKernel<T, FMT>(a.c.dim, [&](auto kernel) {
    kernel<<<grid, kAttendWaves * kWave, AttendLdsBytes(a.c.dim, true), stream>>>(a, p, logits);
  });
  DSD_HIP_CHECK(hipGetLastError());
  Merge<T>(a, p, stream);
  const int64_t shares = (ListGroups(a.c, a.b) + 4 * kBlocks - 1) / (4 * kBlocks);
  const dim3 over(static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(shares, 1), 65536)) + 1,
                  a.c.heads, a.b.batch);
  Kv8WeighKernel<<<over, 256, 0, stream>>>(a, p, logits, weights);
  DSD_HIP_CHECK(hipGetLastError());
}

template <typename T>
void LaunchType(const Kv8AttendArgs& a, float* weights, hipStream_t stream) {
  a.c.format == DSD_KV8_INT8 ? Launch<T, DSD_KV8_INT8>(a, weights, stream)
                             : Launch<T, DSD_KV8_E4M3>(a, weights, stream);
}

template <typename T, int FMT>
void PreloadDim(const Kv8View& c) {
  WithKernel<T, FMT>(c.dim, [&](auto kernel) {
    PreloadKernel(kernel);
    DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(AttendLdsBytes(c.dim, true))));
  });
}

template <typename T>
void PreloadType(const Kv8View& c) {
  c.format == DSD_KV8_INT8 ? PreloadDim<T, DSD_KV8_INT8>(c) : PreloadDim<T, DSD_KV8_E4M3>(c);
  PreloadKernel(Kv8MergeKernel<T>);
  PreloadKernel(Kv8MergeRowsKernel<T>);
}

}  // namespace

size_t Kv8WeighBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  if (b.batch == 0) return 0;
  const Plan p = AttendPlan(c, b, q_heads, false);
  return PartBytes(c, b, p) + StatsBytes(c, b, p) + LogitBytes(c, b, q_heads);
}

// Of any batch of at most these sizes: pieces where a launch would have few workgroups,
// a row's sums where it has many.
size_t Kv8WeighWorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  if (b.batch == 0) return 0;
  Plan p = AttendPlan(c, b, q_heads, false);
  const size_t parts = MostPartBytes(c, p, kAttendTarget);
  p.pieces = 1;
  return (parts + 15) / 16 * 16 + StatsBytes(c, b, p) + LogitBytes(c, b, q_heads);
}

void PreloadKv8Weigh(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
  PreloadKernel(Kv8WeighKernel);
}

void LaunchKv8Weigh(const Kv8AttendArgs& a, float* weights, hipStream_t stream) {
  if (a.b.batch == 0) return;
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(a, weights, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(a, weights, stream);
    default: return LaunchType<_Float16>(a, weights, stream);
  }
}

}  // namespace dsdk
