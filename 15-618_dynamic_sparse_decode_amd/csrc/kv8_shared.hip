// kv8_shared.hip -- dsd_kv8_attend_shared (gfx950): one query token a request over a
// prefix that its group shares, then over its own list.
//
// Mathematics.  Softmax over two lists is that of each, joined: with a list's maximum m,
// sum l of 2^(s - m) and sum o of those times values, the whole is sum(2^(m - M) o) /
// sum(2^(m - M) l), M the greatest m.  So the requests of a group are rows of one
// attention over the group's list (as many rows a key head as requests times query heads
// of it), each request's own list is another, and a last launch joins the rows' pieces.
//
// What bounds it: for few rows a prefix HBM, for many the matrix and vector units.  bf16,
// 32 query heads on 8 of 128: 8 requests behind 2000 tokens 10 us and 4.5 for the joining;
// 64 behind 32768, own lists of 200 to 2000, 81 and 10 (36 us of bytes, 26 of products, and
// as much again of turning codes into halves, twice for 256 rows); float32, 32 / 32 heads,
// 16 requests in 4 groups behind 4096 to 16384, 111 and 5.5, 5.3 TB/s.  Heads of 144
// to 256 of many rows spill as kv8_cross.hip's do: the 64 behind 32768 of 16 heads on 8 of
// 256 take 360 us a call.
#include "kv8_attend_block.h"
#include "kv8_prompt_block.h"

#include <algorithm>

namespace dsdk {
namespace {

// The prefixes' pieces, then the own lists'.
struct SharedArgs {
  Kv8AttendArgs pre, own;
  Plan pre_plan, own_plan;
  int pre_items = 0;  // workgroups over prefixes, first in the grid
};

// A launch's index over units (key heads * row blocks) of lists of pieces.
struct Item {
  int unit, list, piece;
};
__device__ __forceinline__ Item ItemOf(int i, int units, int lists) {
  const int rest = i / units;
  return {i - rest * units, rest % lists, rest / lists};
}

// Both, 16 rows a workgroup.
template <typename T, int FMT, int NU, int kDim>
__global__ __launch_bounds__(kAttendWaves* kWave, NU <= 2 ? 2 : 1) void Kv8SharedKernel(
    SharedArgs s) {
  extern __shared__ __align__(16) float lds[];
  const int i = blockIdx.x;
  const bool pre = i < s.pre_items;
  const Kv8AttendArgs& a = pre ? s.pre : s.own;
  const Plan& p = pre ? s.pre_plan : s.own_plan;
  const Item at = ItemOf(pre ? i : i - s.pre_items, a.c.heads * p.blocks, a.b.batch);
  AttendBlock<T, FMT, NU, kDim, kAttendWaves, true>(a, p, at.unit, at.list, at.piece, lds);
}

// The same for prefixes of many rows, 128 a workgroup: their workgroups are bound by the
// matrix and vector units, the own lists' by HBM, so one launch runs them side by side.
template <typename T, int FMT, int NU, int kDim>
__global__ __launch_bounds__(kThreads, NU <= 2 && sizeof(T) == 2 ? 2 : 1) void
Kv8SharedRowsKernel(SharedArgs s) {
  extern __shared__ __align__(16) float lds[];
  const int i = blockIdx.x;
  if (i < s.pre_items) {
    const Item at = ItemOf(i, s.pre.c.heads * s.pre_plan.blocks, s.pre.b.batch);
    PromptBlock<T, FMT, NU, kDim, false, true>(s.pre, s.pre_plan, at.unit, at.list, at.piece,
                                               reinterpret_cast<_Float16*>(lds));
  } else {
    const Item at = ItemOf(i - s.pre_items, s.own.c.heads * s.own_plan.blocks, s.own.b.batch);
    AttendBlock<T, FMT, NU, kDim, kAttendWaves, true>(s.own, s.own_plan, at.unit, at.list, at.piece,
                                                      lds);
  }
}

// The group of request r, -1: none (two: reported).  All lanes of a wave.
__device__ __forceinline__ int GroupOf(const Kv8AttendArgs& pre, int r) {
  const int lane = threadIdx.x & (kWave - 1);
  int group = -1, claims = 0;
  for (int g0 = 0; g0 < pre.b.batch; g0 += kWave) {
    const int g = g0 + lane;
    Kv8Request q;
    const bool mine = g < pre.b.batch && Kv8ReadRows(pre.b, g, &q) && q.row0 <= r && r < q.row0 + q.n;
    const unsigned long long ours = __ballot(mine);
    claims += static_cast<int>(__popcll(ours));
    if (ours != 0) group = g0 + __ffsll(ours) - 1;
  }
  if (claims > 1 && lane == 0) ReportFailure(pre.fail, kFailShape);
  return claims == 1 ? group : -1;
}

// A row's pieces joined, a workgroup a row.  Grid (query heads, batch).  All of the row's
// slots are asked for before it is known which of them have pieces.
template <typename T>
__global__ __launch_bounds__(256) void Kv8JoinKernel(SharedArgs s) {
  __shared__ float factor[kMostPieces];
  __shared__ Power last;
  __shared__ int counts[2];
  __shared__ F32x4 part_sum[256];
  const int D = s.own.c.dim, quads = D / 4;
  const int r = blockIdx.y, q_head = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1);
  const int stride = s.own_plan.stride, base = s.own_plan.base;
  const int64_t slot0 =
      (static_cast<int64_t>(r) * s.own.c.heads * s.own_plan.group + q_head) * stride;
  const int shares = 256 / quads;  // threads per quad
  const int share = threadIdx.x / quads, d = 4 * (threadIdx.x - share * quads);
  const float* part = s.own_plan.part + slot0 * D + d;
  constexpr int kAhead = 4;
  F32x4 x[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int z = share + i * shares;
    if (share < shares && z < stride) x[i] = *reinterpret_cast<const F32x4*>(part + z * D);
  }
  if (threadIdx.x < kWave) {
    PieceStats st = {-INFINITY, -1.0f, 0.0f};
    if (lane < stride) st = s.own_plan.stats[slot0 + lane];
    Span span;
    int n_pre = 0, n_own = 0;
    const int group = GroupOf(s.pre, r);
    if (group >= 0 && FindSpan(s.pre, s.pre_plan.group, group, 0, 1, &span)) {
      n_pre = Pieces(s.pre_plan, span);
    }
    if (FindSpan(s.own, s.own_plan.group, r, 0, 1, &span)) n_own = Pieces(s.own_plan, span);
    const bool has = lane < n_pre || (lane >= base && lane < base + n_own);
    if (!has) st = {-INFINITY, -1.0f, 0.0f};
    Power to_out;
    factor[lane] = JoinFactor<kWave>(st, !(st.l < 0.0f), &to_out);
    if (lane == 0) {
      last = to_out;
      counts[0] = n_pre;
      counts[1] = base + n_own;
    }
  }
  __syncthreads();
  const int n_pre = counts[0], end = counts[1];
  F32x4 o = {0, 0, 0, 0};
  if (share < shares) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int z = share + i * shares;
      if (z < n_pre || (z >= base && z < end)) o += x[i] * factor[z];
    }
#pragma unroll 4
    for (int z = share + kAhead * shares; z < end; z += shares) {
      if (z < n_pre || z >= base) o += *reinterpret_cast<const F32x4*>(part + z * D) * factor[z];
    }
  }
  part_sum[threadIdx.x] = o;
  __syncthreads();
  if (share > 0) return;
  for (int i = 1; i < shares; ++i) o += part_sum[i * quads + threadIdx.x];
  o = o * last.most * last.rest;
  T* out = static_cast<T*>(s.own.out) + r * s.own.out_stride + static_cast<int64_t>(q_head) * D + d;
  StoreRow4(out, reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0, o);
}

// ---- plans ------------------------------------------------------------------------

// The rows' slots: at most kMostSlots where a row has more than a prefix piece and an own.
constexpr int64_t kMostSlots = 65536;

struct SharedPlan {
  SharedArgs s;
  bool many = false;  // prefixes by blocks of 128 rows
};

SharedPlan MakePlan(const Kv8AttendArgs& own, const dsd_kv8_prefix& prefix) {
  SharedPlan m;
  const int most_requests = std::max(std::min(prefix.max_requests, own.b.batch), 1);
  SharedArgs& s = m.s;
  s.own = own;
  s.pre = own;
  s.pre.many = true;
  s.pre.b = dsd_kv8_batch{};
  s.pre.b.batch = prefix.groups;
  s.pre.b.tokens = own.b.batch;
  s.pre.b.max_tokens = most_requests;
  s.pre.b.max_pages = prefix.max_pages;
  s.pre.b.total_pages = prefix.total_pages;
  s.pre.b.page_offsets = prefix.page_offsets;
  s.pre.b.page_ids = prefix.page_ids;
  s.pre.b.token_offsets = prefix.request_offsets;
  const Kv8View& c = own.c;
  const int group = own.q_heads / c.heads;
  m.many = static_cast<int64_t>(most_requests) * group > 64;
  auto shape = [&](Plan* p, int64_t requests, int block) {
    p->group = group;
    p->rows = requests * group;
    p->block = block;
    p->blocks = static_cast<int>((p->rows + block - 1) / block);
  };
  shape(&s.pre_plan, most_requests, m.many ? kRows : 16);
  shape(&s.own_plan, 1, 16);
  // Pieces of the same length for both, so many that the workgroups fill the chip once.
  const int64_t pre_units = static_cast<int64_t>(c.heads) * s.pre_plan.blocks * prefix.groups;
  const int64_t own_units = static_cast<int64_t>(c.heads) * s.own_plan.blocks * own.b.batch;
  const int64_t pre_groups = ListGroups(c, s.pre.b), own_groups = ListGroups(c, own.b);
  const int64_t rows = static_cast<int64_t>(own.b.batch) * own.q_heads;
  const int64_t most = std::max<int64_t>(std::min<int64_t>(kMostPieces, kMostSlots / rows), 2);
  auto cut = [&](Plan* p, int64_t groups, int64_t length, int64_t at_most) {
    CutLists(p, groups, std::min((groups + length - 1) / length, at_most), 1);
  };
  const int64_t pre = pre_units * pre_groups, own_all = own_units * own_groups;
  const int64_t all = own_all + (m.many ? 0 : pre);
  const int64_t length = std::max<int64_t>((all + kAttendTarget - 1) / kAttendTarget, kAttendWaves);
  cut(&s.own_plan, own_groups, length, most / 2);
  int64_t pre_length = length;
  if (m.many) {
    // Blocks of 128 rows: one workgroup a CU beside the own lists' (a group of 64 tokens
    // 2.3 us) or two that the own lists' follow (2.45 us, which at 3.8 TB/s take what is
    // left).  64 requests behind 32768 tokens, own lists of 200-2000: 82 and 93 us.  (Measured
    // at bf16 heads of 128; other types' and sizes' groups take longer, which shifts where the
    // two meet, not the results.)
    const double step = static_cast<double>(pre) / kPromptTarget;
    const double own_us = static_cast<double>(own_all) * 128 * c.dim / 3.8e6;
    const int64_t target = own_us > (2 * 2.3 - 2.45) * step ? kPromptTarget / 2 : kPromptTarget;
    pre_length = std::max<int64_t>((pre + target - 1) / target, 1);
  }
  cut(&s.pre_plan, pre_groups, pre_length, most - s.own_plan.pieces);
  s.pre_plan.stride = s.own_plan.stride = s.pre_plan.pieces + s.own_plan.pieces;
  s.own_plan.base = s.pre_plan.pieces;
  return m;
}

// Workgroups of a launch, one direction (its threads are counted in 32 bits).
int64_t Items(const Kv8View& c, const Plan& p, const dsd_kv8_batch& b) {
  return static_cast<int64_t>(c.heads) * p.blocks * b.batch * p.pieces;
}
constexpr int64_t kMostItems = 0xffffff;

size_t SlotBytes(const Kv8View& c) { return sizeof(float) * c.dim + sizeof(PieceStats); }

size_t RowsLdsBytes(int dim) { return std::max(PromptLdsBytes(dim), AttendLdsBytes(dim)); }

// ---- launches -----------------------------------------------------------------------

#define DSD_WITH_DIM(KERNEL)                            \
  if (dim == 64) return f(KERNEL<T, FMT, 1, 64>);       \
  if (dim < 64) return f(KERNEL<T, FMT, 1, 0>);         \
  if (dim == 128) return f(KERNEL<T, FMT, 2, 128>);     \
  if (dim < 128) return f(KERNEL<T, FMT, 2, 0>);        \
  return f(KERNEL<T, FMT, 4, 0>)

// Calls f with the kernel of a head size.
template <typename T, int FMT, typename F>
void WithShared(int dim, F&& f) {
  DSD_WITH_DIM(Kv8SharedKernel);
}
template <typename T, int FMT, typename F>
void WithSharedRows(int dim, F&& f) {
  DSD_WITH_DIM(Kv8SharedRowsKernel);
}
#undef DSD_WITH_DIM

template <typename T, int FMT>
void Launch(SharedPlan m, hipStream_t stream) {
  SharedArgs& s = m.s;
  const int dim = s.own.c.dim;
  s.pre_items = static_cast<int>(Items(s.pre.c, s.pre_plan, s.pre.b));
  const int items = s.pre_items + static_cast<int>(Items(s.own.c, s.own_plan, s.own.b));
  if (m.many) {
    WithSharedRows<T, FMT>(dim, [&](auto kernel) {
      kernel<<<items, kThreads, RowsLdsBytes(dim), stream>>>(s);
    });
  } else {
    WithShared<T, FMT>(dim, [&](auto kernel) {
      kernel<<<items, kAttendWaves * kWave, AttendLdsBytes(dim), stream>>>(s);
    });
  }
  DSD_HIP_CHECK(hipGetLastError());
  Kv8JoinKernel<T><<<dim3(s.own.q_heads, s.own.b.batch), 256, 0, stream>>>(s);
  DSD_HIP_CHECK(hipGetLastError());
}

template <typename T>
void LaunchType(const SharedPlan& m, hipStream_t stream) {
  m.s.own.c.format == DSD_KV8_INT8 ? Launch<T, DSD_KV8_INT8>(m, stream)
                                   : Launch<T, DSD_KV8_E4M3>(m, stream);
}

template <typename T, int FMT>
void PreloadDim(const Kv8View& c) {
  auto load = [](auto kernel, size_t lds) {
    PreloadKernel(kernel);
    DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(lds)));
  };
  WithShared<T, FMT>(c.dim, [&](auto kernel) { load(kernel, AttendLdsBytes(c.dim)); });
  WithSharedRows<T, FMT>(c.dim, [&](auto kernel) { load(kernel, RowsLdsBytes(c.dim)); });
}

template <typename T>
void PreloadType(const Kv8View& c) {
  c.format == DSD_KV8_INT8 ? PreloadDim<T, DSD_KV8_INT8>(c) : PreloadDim<T, DSD_KV8_E4M3>(c);
  PreloadKernel(Kv8JoinKernel<T>);
}

}  // namespace

bool Kv8SharedFits(const Kv8AttendArgs& a, const dsd_kv8_prefix& prefix) {
  const SharedPlan m = MakePlan(a, prefix);
  return Items(a.c, m.s.pre_plan, m.s.pre.b) + Items(a.c, m.s.own_plan, a.b) <= kMostItems;
}

size_t Kv8SharedBytes(const Kv8View& c, const dsd_kv8_batch& b, const dsd_kv8_prefix& prefix,
                      int q_heads) {
  if (b.batch == 0) return 0;
  Kv8AttendArgs a;
  a.c = c;
  a.b = b;
  a.q_heads = q_heads;
  const SharedPlan m = MakePlan(a, prefix);
  return static_cast<size_t>(b.batch) * q_heads * m.s.own_plan.stride * SlotBytes(c);
}

size_t Kv8SharedWorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  const size_t rows = static_cast<size_t>(b.batch) * q_heads;
  return std::min<size_t>(rows * kMostPieces, kMostSlots + 2 * rows) * SlotBytes(c);
}

void PreloadKv8Shared(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
}

void LaunchKv8Shared(const Kv8AttendArgs& a, const dsd_kv8_prefix& prefix, hipStream_t stream) {
  if (a.b.batch == 0) return;
  if (prefix.groups == 0) return LaunchKv8Attend(a, stream);
  SharedPlan m = MakePlan(a, prefix);
  const size_t slots = static_cast<size_t>(a.b.batch) * a.q_heads * m.s.own_plan.stride;
  m.s.pre_plan.part = m.s.own_plan.part = static_cast<float*>(a.workspace);
  m.s.pre_plan.stats = m.s.own_plan.stats =
      reinterpret_cast<PieceStats*>(static_cast<float*>(a.workspace) + slots * a.c.dim);
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(m, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(m, stream);
    default: return LaunchType<_Float16>(m, stream);
  }
}

}  // namespace dsdk
