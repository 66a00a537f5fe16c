// kv8_attend.h -- what the attention kernels of the 8-bit paged cache share.
#pragma once

#include <type_traits>

#include "kv8_device.h"

namespace dsdk {
namespace {

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

}  // namespace
}  // namespace dsdk
