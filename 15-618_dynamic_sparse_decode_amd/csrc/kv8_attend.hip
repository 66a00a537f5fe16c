// kv8_attend.hip -- dsd_kv8_attend and dsd_kv8_attend_prompt (gfx950):
// softmax attention over the pages of an 8-bit cache.
//
// Mathematics.  Codes are exact in half precision, so q K^T is a product of
// half-precision matrices: q scaled by a power of two so that its row's
// largest element lies in [2^13, 2^14) -- one term for 16-bit queries (what
// falls below half precision's range is 2^-39 of that element), two for
// float32 ones -- times the codes; the page's scale and the power of two go on
// the logits afterwards, in float32.  Weights p = 2^(s - m) (s in the log2
// domain, m the running maximum) meet the value codes the same way, as p * v *
// 2^(m - n + 15) with v the page's value scale and n the running maximum of s +
// log2 v, so at most 2^15 whatever the scales: half precision rounds them to
// 2^-11, or 2^-22 as two terms where the output is finer than bf16.  All sums
// are float32.
#include "kv8_device.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

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

// A launch as its kernels see it.
struct Plan {
  int group = 1;   // query heads per key head
  int tiles = 1;   // row tiles of a request and key head, at most
  int pieces = 1;  // a list is cut into at most this many
  int piece = 1;   // groups of 64 tokens in a piece
  int rows = 16;   // rows of a tile held in the workspace
  float* part = nullptr;    // [batch][heads * tiles][pieces][rows][dim]
  float2* stats = nullptr;  // [batch][heads * tiles][pieces][rows]: (m, l), l < 0: no token
};

// What a workgroup attends: rows [first, first + 16) of request r (row i:
// token i / group, query head i % group of the key head), chunks of 16 tokens.
struct Span {
  Kv8Request q;
  int rows = 0;    // of the request
  int chunks = 0;  // that the tile's rows look at
  int pieces = 1;  // that these are cut into
};

__device__ __forceinline__ bool FindSpan(const Kv8AttendArgs& a, const Plan& p, int r, int first,
                                         Span* s) {
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
  s->rows = s->q.n * p.group;
  if (first >= s->rows) return false;
  if (a.causal) {
    const int last = (min(first + 16, s->rows) - 1) / p.group;
    s->chunks = (s->q.past + last) / 16 + 1;
  } else {
    s->chunks = s->q.pages * a.c.chunks;
  }
  const int groups = (s->chunks + 3) / 4;
  s->pieces = min(p.pieces, max(1, (groups + p.piece - 1) / p.piece));
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

// Grid (key heads * row tiles, batch, pieces); W waves, each of which takes
// every W-th group of 64 tokens of the piece for all of the tile's 16 rows.
// Lane (n, g) = (lane % 16, lane / 16).  Logits come out transposed, S^T = K
// Q^T in four tiles of 16 tokens whose rows are dealt so that lane (n, g) gets
// all 16 tokens of the group's chunk g for row n; they are then the second
// operand of O^T = V^T P^T as they stand (the order of a product's inner index
// is free), whose first operand, 16 tokens of one dim, is one load of the
// values' layout.  No number crosses lanes but for the maxima.
// kDim: head_dim where it is 64 * NU (no bounds tests), else 0.
template <typename T, int FMT, int NU, int kDim, int W>
__global__ __launch_bounds__(W* kWave, NU <= 2 ? 2 : 1) void Kv8AttendKernel(Kv8AttendArgs a, Plan p) {
  constexpr int NQ = kQueryTerms<T>, NP = kWeightTerms<T>, NT = 4 * NU;
  extern __shared__ __align__(16) float lds[];
  const Kv8View& c = a.c;
  const int D = kDim > 0 ? kDim : c.dim, tiles = kDim > 0 ? NT : D / 16;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int n = lane & 15, g = lane >> 4;
  const int r = blockIdx.y, head = blockIdx.x % c.heads;
  const int first = blockIdx.x / c.heads * 16;
  Span s;
  if (!FindSpan(a, p, r, first, &s)) return;
  if (static_cast<int>(blockIdx.z) >= s.pieces) return;
  const int groups = (s.chunks + 3) / 4;
  const int begin = blockIdx.z * p.piece;
  const int end = static_cast<int>(blockIdx.z) == s.pieces - 1 ? groups : begin + p.piece;

  // Row n's query: units g + 4 u of 16 dims, eight at a time.
  const int row = first + n;
  const bool there = row < s.rows;
  const int token = there ? row / p.group : 0;
  F16x8 q[NU][2][NQ];
  float to_logit = 0.0f;  // what a product with codes lacks but the page's scale; >= 0
  auto load_query = [&] {
    const int q_head = head * p.group + (there ? row - token * p.group : 0);
    const T* qp = static_cast<const T*>(a.q) + (s.q.row0 + token) * a.q_stride +
                  static_cast<int64_t>(q_head) * D;
    float x[NU][16];
    float most = 0.0f;
    const bool even = reinterpret_cast<uintptr_t>(qp) % 16 == 0;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int d = (g + 4 * u) * 16;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[u][e] = 0.0f;
      if (there && d < D) {
        Load8(qp + d, even, x[u]);
        Load8(qp + d + 8, even, x[u] + 8);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float size = fabsf(x[u][e]);
        most = fmaxf(most, size < INFINITY ? size : 0.0f);
      }
    }
    most = Max4(most);
    int e = 0;
    (void)frexpf(most, &e);
    e = most > 0.0f ? max(min(14 - e, 126), -126) : 0;
    const float up = copysignf(__uint_as_float(static_cast<unsigned>(e + 127) << 23), a.scale);
    to_logit =
        fabsf(a.scale) * kLog2e * __uint_as_float(static_cast<unsigned>(127 - e) << 23);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = x[u][i] * up;
        const _Float16 hi = static_cast<_Float16>(y);
        q[u][i >> 3][0][i & 7] = hi;
        if constexpr (NQ == 2) {
          const float rest = y - static_cast<float>(hi);
          q[u][i >> 3][1][i & 7] = static_cast<_Float16>(fabsf(y) < INFINITY ? rest : 0.0f);
        }
      }
    }
  };
  const int sees = a.causal ? s.q.past + token + 1 : 0x7fffffff;  // row n's tokens

  F32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = F32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  float mv = -INFINITY;  // of s + log2(value scale): acc is relative to it
  bool seen = false;

  // The list's pages are staged in LDS, so that a group's addresses are known
  // before its turn: its keys are asked for as soon as the logits of the group
  // before have taken their registers' contents, its values after the products.
  PageInfo* info = reinterpret_cast<PageInfo*>(lds);
  const int per_stage = max((kStage - 2) * c.chunks / 4, 1);  // groups
  const unsigned inverse = 0xffffffffu / static_cast<unsigned>(c.chunks) + 1u;
  const int page_bytes = c.page * D;
  uint4 kw[4][NU], vw[NT];
  for (int g0 = begin; g0 < end; g0 += per_stage) {
    const int g1 = min(end, g0 + per_stage);
    const int slot0 = 4 * g0 / c.chunks;
    const int slots = (min(4 * g1, s.chunks) - 1) / c.chunks + 1 - slot0;
    if (g0 > begin) __syncthreads();
    for (int i = threadIdx.x; i < slots; i += W * kWave) {
      info[i] = ReadPage(a, s, head, slot0 + i);
    }
    __syncthreads();
    // Chunk i of the list: its place among the staged ones, its part of the page.
    auto place = [&](int i, int* sub) {
      const int slot = c.chunks == 1 ? i : static_cast<int>(__umulhi(i, inverse));
      *sub = i - slot * c.chunks;
      return min(slot - slot0, slots - 1);
    };
    auto load_keys = [&](int grp) {
      int sub;
      const int page = info[place(4 * grp + (n >> 2), &sub)].page;
      const uint8_t* kp = c.keys + static_cast<int64_t>(page * c.heads + head) * page_bytes +
                          (sub * 16 + (n & 3)) * D + g * 16;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          if (kDim > 0 || (g + 4 * u) * 16 < D) {
            kw[t][u] = *reinterpret_cast<const uint4*>(kp + 4 * t * D + 64 * u);
          } else {
            kw[t][u] = make_uint4(0, 0, 0, 0);
          }
        }
      }
    };
    PageInfo now;   // the values' page, and its tokens from the chunk's first on
    auto load_values = [&](int grp) {
      int sub;
      now = info[place(4 * grp + g, &sub)];
      now.tokens = 4 * grp + g < s.chunks ? now.tokens - sub * 16 : 0;
      const uint8_t* vp = c.values +
                          static_cast<int64_t>(now.page * c.heads + head) * page_bytes +
                          (sub * D + n) * 16;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t < tiles) vw[t] = *reinterpret_cast<const uint4*>(vp + 256 * t);
      }
    };
    int grp = g0 + wave;
    if (grp < g1) {
      load_keys(grp);
      load_values(grp);
    }
    if (g0 == begin) load_query();  // (its latency beside the first group's)
    for (; grp < g1; grp += W) {
      const bool more = grp + W < g1;
      F32x4 x[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x[t] = F32x4{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const F16x8 k0 = Numbers8<FMT>(kw[t][u].x, kw[t][u].y);
          const F16x8 k1 = Numbers8<FMT>(kw[t][u].z, kw[t][u].w);
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[u][0][i], x[t], 0, 0, 0);
            x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[u][1][i], x[t], 0, 0, 0);
          }
        }
      }
      if (more) load_keys(grp + W);

      // Row n's tokens of the chunk: those in the cache that it sees.
      const int count = min(now.tokens, sees - (4 * grp + g) * 16);
      const bool whole = __ballot(count < 16) == 0;
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (4 * t + i >= count) x[t][i] = -INFINITY;
          }
        }
      }
      const float f = fmaxf(to_logit * now.key_scale, kKv8Tiny);
      float most = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        most = fmaxf(most, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
      }
      most *= f;
      seen = seen || count > 0;
      const float m_new = fmaxf(m, Max4(most));
      const float mv_new = fmaxf(mv, Max4(most + __builtin_amdgcn_logf(now.value_scale)));
      const float base = m_new == -INFINITY ? 0.0f : m_new;
      const float base_v = mv_new == -INFINITY ? 0.0f : mv_new;
      if (__ballot(m_new > m || mv_new > mv) != 0) {
        l *= Exp2(m - base);
        const float shrink = Exp2(mv - base_v);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] *= shrink;
        m = m_new;
        mv = mv_new;
      }
      const float to_half = now.value_scale * Exp2(base - base_v + kWeightBits);
      F16x8 w[2][NP];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = Exp2(fmaf(x[t][i], f, -base));
          l += e;
          y[i] = e * to_half;
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const F32x2 pair = {y[i], y[i + 1]};
          const F16x2 hi = __builtin_convertvector(pair, F16x2);
          w[t >> 1][0][4 * (t & 1) + i] = hi[0];
          w[t >> 1][0][4 * (t & 1) + i + 1] = hi[1];
          if constexpr (NP == 2) {
            const F32x2 rest = {y[i] - static_cast<float>(hi[0]),
                                y[i + 1] - static_cast<float>(hi[1])};
            const F16x2 lo = __builtin_convertvector(rest, F16x2);
            w[t >> 1][1][4 * (t & 1) + i] = lo[0];
            w[t >> 1][1][4 * (t & 1) + i + 1] = lo[1];
          }
        }
      }
      if (!whole) {
        // Codes behind a request's tokens may be anything, and 0 * NaN is not 0.
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          unsigned* word = reinterpret_cast<unsigned*>(&vw[t]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int have = min(max(now.tokens - 4 * i, 0), 4);
            word[i] &= have == 4 ? 0xffffffffu : (1u << (8 * have)) - 1u;
          }
        }
        // Nor may NaN codes of tokens that only later rows see reach the others:
        // they are taken out, and the rows that see one get NaN.
        if (FMT == DSD_KV8_E4M3 && a.causal) {
          bool nan = false;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (t < tiles) {
              nan = nan || ((NanBytes(vw[t].x) | NanBytes(vw[t].y)) |
                            (NanBytes(vw[t].z) | NanBytes(vw[t].w))) != 0u;
            }
          }
          if (__ballot(nan) != 0) {
            F16x8 visible[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              visible[i >> 3][i & 7] = static_cast<_Float16>(i < count ? 1.0f : 0.0f);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if (t < tiles) {
                unsigned* word = reinterpret_cast<unsigned*>(&vw[t]);
                unsigned ones[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const unsigned bytes = (NanBytes(word[i]) >> 7) * 0xffu;
                  ones[i] = bytes & 0x38383838u;  // 1.0
                  word[i] &= ~bytes;
                }
                F32x4 hits = {0, 0, 0, 0};
                hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(Numbers8<FMT>(ones[0], ones[1]),
                                                              visible[0], hits, 0, 0, 0);
                hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(Numbers8<FMT>(ones[2], ones[3]),
                                                              visible[1], hits, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if (hits[i] > 0.0f) acc[t][i] = __builtin_nanf("");
                }
              }
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t < tiles) {
          const F16x8 v0 = Numbers8<FMT>(vw[t].x, vw[t].y);
          const F16x8 v1 = Numbers8<FMT>(vw[t].z, vw[t].w);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w[0][i], acc[t], 0, 0, 0);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w[1][i], acc[t], 0, 0, 0);
          }
        }
      }
      if (more) load_values(grp + W);
    }
  }

  // The waves' streams, through LDS: [W][16] m, l and mv, [W][16][D + 4] acc.
  __syncthreads();
  float* s_m = lds;
  float* s_l = lds + 16 * W;
  float* s_mv = lds + 32 * W;
  float* s_acc = lds + 48 * W;
  l = Sum4(l);
  const bool any = Max4(seen ? 1.0f : 0.0f) > 0.0f;
  if (g == 0) {
    s_m[wave * 16 + n] = m;
    s_l[wave * 16 + n] = any ? l : -1.0f;
    s_mv[wave * 16 + n] = mv;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t < tiles) {
      *reinterpret_cast<F32x4*>(s_acc + (wave * 16 + n) * (D + 4) + 16 * t + 4 * g) = acc[t];
    }
  }
  __syncthreads();
  const int quads = D / 4;
  for (int i = threadIdx.x; i < 16 * quads; i += W * kWave) {
    const int k = i / quads, d = 4 * (i - k * quads);
    const int at = first + k;
    if (at >= s.rows) break;
    float peak = -INFINITY;
    bool some = false;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (!(s_l[w * 16 + k] < 0.0f)) {
        peak = fmaxf(peak, s_m[w * 16 + k]);
        some = true;
      }
    }
    const float base = peak == -INFINITY ? 0.0f : peak;
    float sum = 0.0f;
    F32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (!(s_l[w * 16 + k] < 0.0f)) {
        sum += s_l[w * 16 + k] * Exp2(s_m[w * 16 + k] - base);
        o += *reinterpret_cast<const F32x4*>(s_acc + (w * 16 + k) * (D + 4) + d) *
             Exp2(s_mv[w * 16 + k] - base - kWeightBits);
      }
    }
    if (s.pieces == 1) {
      const int tok = at / p.group;
      T* out = static_cast<T*>(a.out) + (s.q.row0 + tok) * a.out_stride +
               static_cast<int64_t>(head * p.group + at - tok * p.group) * D + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(some ? o[e] / sum : 0.0f);
    } else {
      const int64_t slot =
          ((static_cast<int64_t>(r) * gridDim.x + blockIdx.x) * p.pieces + blockIdx.z) * p.rows + k;
      *reinterpret_cast<F32x4*>(p.part + slot * D + d) = o;
      if (d == 0) p.stats[slot] = make_float2(peak, some ? sum : -1.0f);
    }
  }
}

// One row's pieces.  Grid (key heads * row tiles, batch, rows of a tile): the
// pieces' factors first, in LDS, so that the sums' loads wait for nothing; the
// threads beyond a row's quads take every 256 / quads-th piece, and their sums
// are added in that order.
constexpr int kMostPieces = 64;
template <typename T>
__global__ __launch_bounds__(256) void Kv8MergeKernel(Kv8AttendArgs a, Plan p) {
  __shared__ float factor[kMostPieces];
  __shared__ F32x4 part_sum[256];
  const Kv8View& c = a.c;
  const int D = c.dim, quads = D / 4;
  const int r = blockIdx.y, head = blockIdx.x % c.heads, first = blockIdx.x / c.heads * 16;
  const int k = blockIdx.z, at = first + k;
  Span s;
  if (!FindSpan(a, p, r, first, &s) || s.pieces == 1 || at >= s.rows) return;
  const int64_t slot0 =
      (static_cast<int64_t>(r) * gridDim.x + blockIdx.x) * p.pieces * p.rows + k;
  const int lane = threadIdx.x & (kWave - 1);
  const int shares = 256 / quads;  // threads per quad
  const int share = threadIdx.x / quads, d = 4 * (threadIdx.x - share * quads);
  if (threadIdx.x < kWave) {
    float2 st = make_float2(-INFINITY, -1.0f);
    if (lane < s.pieces) st = p.stats[slot0 + static_cast<int64_t>(lane) * p.rows];
    const bool some = !(st.y < 0.0f);
    float peak = some ? st.x : -INFINITY;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) peak = fmaxf(peak, __shfl_xor(peak, o, kWave));
    const float e = some ? Exp2(st.x - (peak == -INFINITY ? 0.0f : peak)) : 0.0f;
    float sum = some ? st.y * e : 0.0f;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) sum += __shfl_xor(sum, o, kWave);
    factor[lane] = (__ballot(some) != 0 ? 1.0f / sum : 1.0f) * e;
  }
  // (loads that do not need the factors are on their way meanwhile)
  constexpr int kAhead = 4;
  const float* part = p.part + slot0 * D + d;
  const int64_t step = static_cast<int64_t>(p.rows) * D;
  F32x4 x[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int z = share + i * shares;
    x[i] = F32x4{0, 0, 0, 0};
    if (share < shares && z < s.pieces) {
      x[i] = *reinterpret_cast<const F32x4*>(part + z * step);
    }
  }
  __syncthreads();
  F32x4 o = {0, 0, 0, 0};
  if (share < shares) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int z = share + i * shares;
      if (z < s.pieces) o += x[i] * factor[z];
    }
#pragma unroll 4
    for (int z = share + kAhead * shares; z < s.pieces; z += shares) {
      o += *reinterpret_cast<const F32x4*>(part + z * step) * factor[z];
    }
  }
  part_sum[threadIdx.x] = o;
  __syncthreads();
  if (share > 0) return;
  for (int i = 1; i < shares; ++i) o += part_sum[i * quads + threadIdx.x];
  const int tok = at / p.group;
  T* out = static_cast<T*>(a.out) + (s.q.row0 + tok) * a.out_stride +
           static_cast<int64_t>(head * p.group + at - tok * p.group) * D + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(o[e]);
}

constexpr int kWaves = 4;
constexpr int kTarget = 768;  // workgroups worth spreading lists for

// How a batch's lists are cut, by its sizes alone (the lengths themselves are
// on the device).
Plan MakePlan(const Kv8View& c, const dsd_kv8_batch& b, int q_heads, bool causal) {
  Plan p;
  p.group = q_heads / c.heads;
  const int64_t rows = static_cast<int64_t>(causal ? b.max_tokens : 1) * p.group;
  p.tiles = static_cast<int>((rows + 15) / 16);
  p.rows = static_cast<int>(std::min<int64_t>(rows, 16));
  const int64_t groups = (static_cast<int64_t>(b.max_pages) * c.page + 63) / 64;
  const int64_t units = static_cast<int64_t>(c.heads) * p.tiles * b.batch;
  int64_t want = (kTarget + units - 1) / std::max<int64_t>(units, 1);
  want = std::min<int64_t>({want, (groups + kWaves - 1) / kWaves, kMostPieces});
  p.pieces = static_cast<int>(std::max<int64_t>(want, 1));
  p.piece = static_cast<int>(std::max<int64_t>((groups + p.pieces - 1) / p.pieces, 1));
  return p;
}

size_t PlanBytes(const Kv8View& c, const dsd_kv8_batch& b, const Plan& p) {
  if (p.pieces == 1) return 0;
  return static_cast<size_t>(b.batch) * c.heads * p.tiles * p.pieces * p.rows *
         (sizeof(float) * c.dim + sizeof(float2));
}

size_t LdsBytes(int dim) {
  return std::max(sizeof(float) * (48 * kWaves + kWaves * 16 * (dim + 4)),
                  sizeof(PageInfo) * kStage);
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
  const dim3 grid(a.c.heads * p.tiles, a.b.batch, p.pieces);
  WithKernel<T, FMT>(a.c.dim, [&](auto kernel) {
    kernel<<<grid, kWaves * kWave, LdsBytes(a.c.dim), stream>>>(a, p);
  });
  DSD_HIP_CHECK(hipGetLastError());
  if (p.pieces > 1) {
    Kv8MergeKernel<T><<<dim3(grid.x, grid.y, p.rows), 256, 0, stream>>>(a, p);
    DSD_HIP_CHECK(hipGetLastError());
  }
}

template <typename T>
void LaunchType(const Kv8AttendArgs& a, const Plan& p, hipStream_t stream) {
  a.c.format == DSD_KV8_INT8 ? Launch<T, DSD_KV8_INT8>(a, p, stream)
                             : Launch<T, DSD_KV8_E4M3>(a, p, stream);
}

template <typename T, int FMT>
void PreloadDim(const Kv8View& c) {
  WithKernel<T, FMT>(c.dim, [](auto kernel) { PreloadKernel(kernel); });
}

template <typename T>
void PreloadType(const Kv8View& c) {
  c.format == DSD_KV8_INT8 ? PreloadDim<T, DSD_KV8_INT8>(c) : PreloadDim<T, DSD_KV8_E4M3>(c);
  PreloadKernel(Kv8MergeKernel<T>);
}

}  // namespace

size_t Kv8WorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  if (b.batch == 0) return 0;
  return std::max(PlanBytes(c, b, MakePlan(c, b, q_heads, false)),
                  PlanBytes(c, b, MakePlan(c, b, q_heads, true)));
}

void PreloadKv8Attend(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
}

void LaunchKv8Attend(const Kv8AttendArgs& a, hipStream_t stream) {
  if (a.b.batch == 0 || (a.causal && a.b.tokens == 0)) return;
  Plan p = MakePlan(a.c, a.b, a.q_heads, a.causal);
  if (p.pieces > 1) {
    if (a.workspace == nullptr || a.workspace_bytes < PlanBytes(a.c, a.b, p)) {
      p.pieces = 1;
      p.piece = 1;
    } else {
      const size_t slots = static_cast<size_t>(a.b.batch) * a.c.heads * p.tiles * p.pieces * p.rows;
      p.part = static_cast<float*>(a.workspace);
      p.stats = reinterpret_cast<float2*>(p.part + slots * a.c.dim);
    }
  }
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(a, p, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(a, p, stream);
    default: return LaunchType<_Float16>(a, p, stream);
  }
}

}  // namespace dsdk
