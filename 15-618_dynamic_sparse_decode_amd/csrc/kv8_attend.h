// kv8_attend.h -- what the attention kernels of the 8-bit paged cache share.
#pragma once

#include <type_traits>

#include "kv8_device.h"

namespace dsdk {
namespace {

// Maxima beyond which a logit's products are rounded before the maximum is taken off:
// one is off by half its last place, 2^-7 here and whole powers of two further out,
// and the exponential of what a fused product keeps of it would grow by as much.
constexpr float kFar = 0x1p18f;
constexpr float kWeightBits = 15.0f;  // weights reach 2^15 (half precision ends at 2^16)

// The larger (sum) of the four lanes that share lane % 16.
__device__ __forceinline__ float Max4(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float Sum4(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// 2^x as a product of two: Exp2 gives nothing below 2^-126, and a row whose values
// have scales near that has factors below it.  Of x >= -64 the second is one.
struct Power {
  float most, rest;
};
__device__ __forceinline__ Power PowerOf(float x) {
  const bool low = x < -64.0f;
  return {Exp2(low ? x + 64.0f : x), low ? 0x1p-64f : 1.0f};
}

// Eight codes (two words) as half-precision numbers.
template <int FMT>
__device__ __forceinline__ F16x8 Numbers8(unsigned w0, unsigned w1) {
  F16x2 x[4];
  if constexpr (FMT == DSD_KV8_INT8) {
    // 1024 + (code + 128) in the last bits of a half's fraction, less 1152
    const F16x2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    x[0] = __builtin_bit_cast(F16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) - bias;
    x[1] = __builtin_bit_cast(F16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) - bias;
    x[2] = __builtin_bit_cast(F16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) - bias;
    x[3] = __builtin_bit_cast(F16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) - bias;
  } else {
    x[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
    x[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
    x[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
    x[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
  }
  F16x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = x[i][0];
    r[2 * i + 1] = x[i][1];
  }
  return r;
}

// The high bit of each byte that is an e4m3 NaN.
__device__ __forceinline__ unsigned NanBytes(unsigned w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// What a workgroup attends: rows [first, first + some) of request r (row i:
// token i / group, query head i % group of the key head), chunks of 16 tokens.
struct Span {
  Kv8Request q;
  int rows = 0;    // of the request
  int chunks = 0;  // that the workgroup's rows look at
};

__device__ __forceinline__ bool FindSpan(const Kv8AttendArgs& a, int group, int r, int first,
                                         int some, Span* s) {
  bool ok;
  if (a.causal) {
    ok = Kv8ReadTokens(a.b, r, a.c.page, &s->q);
  } else {
    ok = Kv8ReadList(a.b, r, &s->q);
    s->q.row0 = r;
    s->q.n = 1;
  }
  if (!ok || s->q.pages > 0x7fffff00 / a.c.page) {
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailShape);
    // (a decode request still gets its zeros)
    if (a.causal) return false;
    s->q.pages = 0;
  }
  s->rows = s->q.n * group;
  if (first >= s->rows) return false;
  if (a.causal) {
    const int last = (min(first + some, s->rows) - 1) / group;
    s->chunks = (s->q.past + last) / 16 + 1;
  } else {
    s->chunks = s->q.pages * a.c.chunks;
  }
  return true;
}

// One page of a request's list, staged in LDS.
struct PageInfo {
  int page;     // (0 for one that holds no token)
  int tokens;   // in the cache
  float key_scale;
  float value_scale;
};
constexpr int kStage = 512;  // pages staged at a time

__device__ __forceinline__ PageInfo ReadPage(const Kv8AttendArgs& a, const Span& s, int head,
                                             int slot) {
  const Kv8View& c = a.c;
  PageInfo k;
  k.page = a.b.page_ids[s.q.list + slot];
  const bool ok = InPool(k.page, c.capacity);
  if (!ok) ReportFailure(a.fail, kFailPageId);
  k.page = ok ? k.page : 0;
  k.tokens = 0;
  if (ok) k.tokens = a.causal ? s.q.past + s.q.n - slot * c.page : c.token_counts[k.page];
  k.tokens = min(max(k.tokens, 0), c.page);
  const int at = k.page * c.heads + head;
  k.key_scale = k.tokens > 0 ? c.key_scales[at] : 1.0f;
  k.value_scale = k.tokens > 0 ? fmaxf(c.value_scales[at], kKv8Tiny) : 1.0f;
  return k;
}

template <typename T>
constexpr int kQueryTerms = sizeof(T) == 4 ? 2 : 1;
template <typename T>
constexpr int kWeightTerms = std::is_same<T, __bf16>::value ? 1 : 2;

// A query row's scale: `up` brings its largest element to [2^13, 2^14) (with the
// sign of the call's scale), `back` is what its products with codes lack.
struct QueryScale {
  float up = 1.0f;
  float back = 0.0f;
};
__device__ __forceinline__ QueryScale ScaleQuery(float most, float scale) {
  int e = 0;
  (void)frexpf(most, &e);
  e = most > 0.0f ? max(min(14 - e, 126), -126) : 0;
  QueryScale s;
  s.up = copysignf(__uint_as_float(static_cast<unsigned>(e + 127) << 23), scale);
  s.back = fabsf(scale) * kLog2e * __uint_as_float(static_cast<unsigned>(127 - e) << 23);
  return s;
}

// y into element i of a query operand's terms.
template <int NQ>
__device__ __forceinline__ void SplitQuery(float y, F16x8 (&q)[NQ], int i) {
  const _Float16 hi = static_cast<_Float16>(y);
  q[0][i] = hi;
  if constexpr (NQ == 2) {
    const float rest = y - static_cast<float>(hi);
    q[1][i] = static_cast<_Float16>(fabsf(y) < INFINITY ? rest : 0.0f);
  }
}

// y0, y1 into elements i, i + 1 of a weight operand's terms.
template <int NP>
__device__ __forceinline__ void SplitWeights(float y0, float y1, F16x8 (&w)[NP], int i) {
  const F32x2 y = {y0, y1};
  const F16x2 hi = __builtin_convertvector(y, F16x2);
  w[0][i] = hi[0];
  w[0][i + 1] = hi[1];
  if constexpr (NP == 2) {
    const F32x2 rest = {y0 - static_cast<float>(hi[0]), y1 - static_cast<float>(hi[1])};
    const F16x2 lo = __builtin_convertvector(rest, F16x2);
    w[1][i] = lo[0];
    w[1][i + 1] = lo[1];
  }
}

// Four numbers of an output row; vec: they lie on four elements' bytes.
template <typename T>
__device__ __forceinline__ void StoreRow4(T* p, bool vec, F32x4 o) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const T4 x = __builtin_convertvector(o, T4);
  if (vec) {
    *reinterpret_cast<T4*>(p) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = x[e];
  }
}

// ---- lists cut into pieces ------------------------------------------------------
// Where a launch has fewer workgroups than the chip runs at once, each row
// block's list is cut into pieces of equal numbers of 64-token groups, by the
// batch's sizes alone (the lengths themselves are on the device); a second launch
// joins them.
constexpr int kMostPieces = 64;
// A row's piece: its sum of weights is l * 2^m, of weights times values its part *
// 2^(m + top).  (The parts are relative to a maximum of their own: a page whose
// tokens weigh 2^-150 of another's may have values 2^150 times as large.)
struct PieceStats {
  float m, l;  // l < 0: no token
  float top;
};
struct Plan {
  int group = 1;     // query heads per key head
  int64_t rows = 1;  // of a request and key head, at most
  int block = 16;    // rows of a workgroup
  int blocks = 1;    // of a request and key head, at most
  int pieces = 1;    // a list is cut into at most this many
  int piece = 1;     // groups of 64 tokens in a piece
  float* part = nullptr;    // [batch][key heads][rows][pieces][dim]
  PieceStats* stats = nullptr;  // [batch][key heads][rows][pieces]
};
__device__ __forceinline__ int64_t PartSlot(const Plan& p, int heads, int r, int head, int row) {
  return ((static_cast<int64_t>(r) * heads + head) * p.rows + row) * p.pieces;
}
// The pieces that a span's list is cut into.
__device__ __forceinline__ int Pieces(const Plan& p, const Span& s) {
  const int groups = (s.chunks + 3) / 4;
  return min(p.pieces, max(1, (groups + p.piece - 1) / p.piece));
}

// The factors that join a row's pieces (`some`: this lane's has a token): its own of
// each lane's piece, then `last` of their sum.  The first kLanes lanes have pieces.
template <int kLanes>
__device__ __forceinline__ float JoinFactor(const PieceStats& st, bool some, Power* last) {
  float peak = some ? st.m : -INFINITY;
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) peak = fmaxf(peak, __shfl_xor(peak, o, kWave));
  const float base = peak == -INFINITY ? 0.0f : peak;
  float sum = some ? st.l * Exp2(st.m - base) : 0.0f;
  const float x = some ? st.m - base + st.top : -INFINITY;
  float top = x;
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    sum += __shfl_xor(sum, o, kWave);
    top = fmaxf(top, __shfl_xor(top, o, kWave));
  }
  top = top == -INFINITY ? 0.0f : top;
  Power to_out = PowerOf(top);
  if (__ballot(some) != 0) to_out.most /= sum;
  *last = {__shfl(to_out.most, 0, kWave), __shfl(to_out.rest, 0, kWave)};
  return Exp2(x - top);
}

// One row's pieces.  Grid (key heads * rows, batch): the pieces' factors first, in
// LDS, while the first parts are on their way; the threads beyond a row's quads
// take every 256 / quads-th piece, and their sums are added in that order.
template <typename T>
__global__ __launch_bounds__(256) void Kv8MergeKernel(Kv8AttendArgs a, Plan p) {
  __shared__ float factor[kMostPieces];
  __shared__ Power last;
  __shared__ F32x4 part_sum[256];
  const Kv8View& c = a.c;
  const int D = c.dim, quads = D / 4;
  const int r = blockIdx.y, head = blockIdx.x % c.heads;
  const int at = blockIdx.x / c.heads, first = at / p.block * p.block;
  Span s;
  if (!FindSpan(a, p.group, r, first, p.block, &s)) return;
  const int pieces = Pieces(p, s);
  if (pieces == 1 || at >= s.rows) return;
  const int64_t slot0 = PartSlot(p, c.heads, r, head, at);
  const int lane = threadIdx.x & (kWave - 1);
  const int shares = 256 / quads;  // threads per quad
  const int share = threadIdx.x / quads, d = 4 * (threadIdx.x - share * quads);
  if (threadIdx.x < kWave) {
    PieceStats st = {-INFINITY, -1.0f, 0.0f};
    if (lane < pieces) st = p.stats[slot0 + lane];
    Power to_out;
    factor[lane] = JoinFactor<kWave>(st, !(st.l < 0.0f), &to_out);
    if (lane == 0) last = to_out;
  }
  // (loads that do not need the factors are on their way meanwhile)
  constexpr int kAhead = 4;
  const float* part = p.part + slot0 * D + d;
  F32x4 x[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int z = share + i * shares;
    x[i] = F32x4{0, 0, 0, 0};
    if (share < shares && z < pieces) {
      x[i] = *reinterpret_cast<const F32x4*>(part + z * D);
    }
  }
  __syncthreads();
  F32x4 o = {0, 0, 0, 0};
  if (share < shares) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int z = share + i * shares;
      if (z < pieces) o += x[i] * factor[z];
    }
#pragma unroll 4
    for (int z = share + kAhead * shares; z < pieces; z += shares) {
      o += *reinterpret_cast<const F32x4*>(part + z * D) * factor[z];
    }
  }
  part_sum[threadIdx.x] = o;
  __syncthreads();
  if (share > 0) return;
  for (int i = 1; i < shares; ++i) o += part_sum[i * quads + threadIdx.x];
  o = o * last.most * last.rest;
  const int tok = at / p.group;
  T* out = static_cast<T*>(a.out) + (s.q.row0 + tok) * a.out_stride +
           static_cast<int64_t>(head * p.group + at - tok * p.group) * D + d;
  StoreRow4(out, reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0, o);
}

// The same for few pieces and many rows: a wave a row, four a workgroup.  Grid
// (key heads * rows / 4, batch).  1024 rows are a quarter of the waves that the
// chip holds; 2048 rows of 4 pieces took 6.5 us, with a workgroup a row 7.8.
constexpr int kFewPieces = 8;
template <typename T>
__global__ __launch_bounds__(256) void Kv8MergeRowsKernel(Kv8AttendArgs a, Plan p) {
  const Kv8View& c = a.c;
  const int D = c.dim, quads = D / 4;
  const int lane = threadIdx.x & (kWave - 1);
  const int r = blockIdx.y;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (index >= c.heads * p.rows) return;
  const int head = static_cast<int>(index / p.rows);
  const int at = static_cast<int>(index - head * p.rows), first = at / p.block * p.block;
  Span s;
  if (!FindSpan(a, p.group, r, first, p.block, &s)) return;
  const int pieces = Pieces(p, s);
  if (pieces == 1 || at >= s.rows) return;
  const int64_t slot0 = PartSlot(p, c.heads, r, head, at);
  PieceStats st = {-INFINITY, -1.0f, 0.0f};
  if (lane < pieces) st = p.stats[slot0 + lane];
  const float* part = p.part + slot0 * D + 4 * lane;
  F32x4 x[kFewPieces];
#pragma unroll
  for (int z = 0; z < kFewPieces; ++z) {
    x[z] = F32x4{0, 0, 0, 0};
    if (lane < quads && z < pieces) x[z] = *reinterpret_cast<const F32x4*>(part + z * D);
  }
  Power last;
  const float factor = JoinFactor<kFewPieces>(st, !(st.l < 0.0f), &last);
  F32x4 o = {0, 0, 0, 0};
#pragma unroll
  for (int z = 0; z < kFewPieces; ++z) {
    const float f = __shfl(factor, z, kWave);
    if (z < pieces) o += x[z] * f;
  }
  if (lane >= quads) return;
  o = o * last.most * last.rest;
  const int tok = at / p.group, d = 4 * lane;
  T* out = static_cast<T*>(a.out) + (s.q.row0 + tok) * a.out_stride +
           static_cast<int64_t>(head * p.group + at - tok * p.group) * D + d;
  StoreRow4(out, reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0, o);
}

// Into `want` pieces, at most kMostPieces, of at least `least` groups.
inline int64_t ListGroups(const Kv8View& c, const dsd_kv8_batch& b) {
  return (static_cast<int64_t>(b.max_pages) * c.page + 63) / 64;
}
inline void CutLists(Plan* p, int64_t groups, int64_t want, int64_t least) {
  if (want > (groups + least - 1) / least) want = (groups + least - 1) / least;
  if (want > kMostPieces) want = kMostPieces;
  p->pieces = static_cast<int>(want > 1 ? want : 1);
  const int64_t piece = (groups + p->pieces - 1) / p->pieces;
  p->piece = static_cast<int>(piece > 1 ? piece : 1);
}

inline size_t PlanSlots(const Kv8View& c, const dsd_kv8_batch& b, const Plan& p) {
  return static_cast<size_t>(b.batch) * c.heads * p.rows * p.pieces;
}
inline size_t PlanBytes(const Kv8View& c, const dsd_kv8_batch& b, const Plan& p) {
  return p.pieces == 1 ? 0 : PlanSlots(c, b, p) * (sizeof(float) * c.dim + sizeof(PieceStats));
}
// What any batch needs at most whose rows per request are no more: lists are cut
// into as many pieces as keep the workgroups within `target`.
inline size_t MostPartBytes(const Kv8View& c, const Plan& p, int target) {
  const size_t rows = static_cast<size_t>(p.rows < p.block ? p.rows : p.block);
  return target * rows * (sizeof(float) * c.dim + sizeof(PieceStats));
}
// The pieces' places in the call's workspace; without one lists stay whole.
inline void PlaceParts(Plan* p, const Kv8AttendArgs& a) {
  if (p->pieces > 1 && (a.workspace == nullptr || a.workspace_bytes < PlanBytes(a.c, a.b, *p))) {
    p->pieces = 1;
    p->piece = 1;
  }
  if (p->pieces == 1) return;
  p->part = static_cast<float*>(a.workspace);
  p->stats = reinterpret_cast<PieceStats*>(p->part + PlanSlots(a.c, a.b, *p) * a.c.dim);
}

template <typename T>
void Merge(const Kv8AttendArgs& a, const Plan& p, hipStream_t stream) {
  if (p.pieces == 1) return;
  const int64_t rows = a.c.heads * p.rows;
  if (p.pieces <= kFewPieces && rows * a.b.batch >= 1024) {
    const dim3 grid(static_cast<unsigned>((rows + 3) / 4), a.b.batch);
    Kv8MergeRowsKernel<T><<<grid, 256, 0, stream>>>(a, p);
  } else {
    Kv8MergeKernel<T><<<dim3(static_cast<unsigned>(rows), a.b.batch), 256, 0, stream>>>(a, p);
  }
  DSD_HIP_CHECK(hipGetLastError());
}

}  // namespace
}  // namespace dsdk
