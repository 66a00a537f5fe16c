// kv8_prompt_block.h -- attention of 128 rows over a piece of a page list, what one
// workgroup of the 8-bit cache's attention kernels for many rows does.
#pragma once

#include <algorithm>

#include "kv8_attend.h"

namespace dsdk {
namespace {

typedef float F32x16 __attribute__((ext_vector_type(16)));

constexpr int kPromptWaves = 4;
constexpr int kThreads = kPromptWaves * kWave;
constexpr int kRows = 32 * kPromptWaves;  // of a workgroup of so many waves
constexpr int kGroup = 64;             // tokens
// The running maxima follow a row's once it is 2^4 ahead of them (following it at
// once, 64 products an update, cost 6%): weights reach 2^(11 + 4).
constexpr float kSlack = 4.0f;
constexpr float kPromptBits = 11.0f;
constexpr int kValueStride = kGroup + 8;  // halves of a dim's row in LDS (16 bytes off the banks)

// The larger (sum) of the two lanes that share lane % 32.
__device__ __forceinline__ float Max2(float x) {
  const auto a =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float Sum2(float x) {
  const auto a =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// What a group's products need of its four chunks of 16 tokens.
struct ChunkInfo {
  float key_scale;
  float value_scale;
  float log_value_scale;
  int tokens;  // in the cache
};

__host__ __device__ inline int KeyHalves(int dim) { return kGroup * (dim + 8); }
__host__ __device__ inline int ValueHalves(int dim) { return (dim + 31) / 32 * 32 * kValueStride; }

// LDS: two buffers of a group's keys [64][dim + 8] and values [dim][72] in half
// precision (rows 16 bytes off each other's banks), then the staged pages, two
// groups' chunks and each dim's first token whose value is NaN.
inline size_t PromptLdsBytes(int dim) {
  return 2 * sizeof(_Float16) * (KeyHalves(dim) + ValueHalves(dim)) + sizeof(PageInfo) * kStage +
         2 * 4 * sizeof(ChunkInfo) + sizeof(int) * dim;
}

// One piece of request r's list for a block of 32 W rows (unit: key heads * blocks, the
// key head fastest, the last rows first).  kCausal: a row sees its request's tokens up
// to its own; else all of the list's, each page's count of them.  kJoin: a later
// launch joins the piece with others.  Wave w
// has rows [32 w, 32 w + 32) of the block, lane (n, h) = (lane % 32, lane / 32)
// row n.  Logits come out transposed, S^T = K Q^T in two tiles of 32 tokens
// dealt so that lane (n, h) holds all 16 tokens of chunk 2 t + h for row n, and
// go into O^T = V^T P^T as they stand.
template <typename T, int FMT, int NU, int kDim, bool kCausal, bool kJoin, int W = kPromptWaves>
__device__ __forceinline__ void PromptBlock(const Kv8AttendArgs& a, const Plan& plan, int unit,
                                            int r, int piece, _Float16* smem) {
  constexpr int NQ = kQueryTerms<T>, NP = kWeightTerms<T>;
  constexpr int kBlockThreads = W * kWave, kBlockRows = 32 * W;
  // 16-byte units of a group's keys (values) that a thread turns
  constexpr int NJ = NU * kThreads > kBlockThreads ? NU * kThreads / kBlockThreads : 1;
  constexpr bool kAllUnits = kDim > 0 && 4 * kDim == NJ * kBlockThreads;
  constexpr int KS = 4 * NU, NT = 2 * NU;
  constexpr int kMfma = 0x008, kDsRead = 0x100;  // (the scheduler's groups)
  constexpr int kAhead = 4;
  const Kv8View& c = a.c;
  const int D = kDim > 0 ? kDim : c.dim, units = D / 16;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int n = lane & 31, h = lane >> 5;
  const int head = unit % c.heads;
  const int first = (plan.blocks - 1 - unit / c.heads) * kBlockRows;
  const int group = plan.group;
  Span s;
  if (!FindSpan(a, group, r, first, kBlockRows, &s)) return;
  const int pieces = Pieces(plan, s);
  const bool parts = kJoin || pieces > 1;
  if (piece >= pieces) return;
  const int begin = piece * plan.piece;
  const int groups = piece == pieces - 1 ? (s.chunks + 3) / 4 : begin + plan.piece;

  _Float16* key_tiles = smem;
  _Float16* value_tiles = smem + 2 * KeyHalves(D);
  PageInfo* info = reinterpret_cast<PageInfo*>(value_tiles + 2 * ValueHalves(D));
  ChunkInfo* chunk_info = reinterpret_cast<ChunkInfo*>(info + kStage);
  int* nan_from = reinterpret_cast<int*>(chunk_info + 8);

  if (!kCausal && s.chunks == 0) {  // no token: zeros
    const int quads = D / 4;
    for (int i = threadIdx.x; i < kBlockRows * quads; i += kBlockThreads) {
      const int row = first + i / quads, d = 4 * (i % quads);
      if (row >= s.rows) break;
      const int token = row / group;
      if (kJoin) {
        const int64_t slot = JoinSlot(plan, c.heads, s.q.row0, head, row) + piece;
        *reinterpret_cast<F32x4*>(plan.part + slot * D + d) = F32x4{0, 0, 0, 0};
        if (d == 0) plan.stats[slot] = {-INFINITY, -1.0f, 0.0f};
        continue;
      }
      T* out = static_cast<T*>(a.out) + (s.q.row0 + token) * a.out_stride +
               static_cast<int64_t>(head * group + row - token * group) * D + d;
      StoreRow4(out, reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0, F32x4{0, 0, 0, 0});
    }
    return;
  }

  // Pages staged ahead of their groups.
  const int per_stage = max((kStage - 2) * c.chunks / 4, 1);
  const unsigned inverse = 0xffffffffu / static_cast<unsigned>(c.chunks) + 1u;
  const int page_bytes = c.page * D;
  int slot0 = 0, slots = 0, stage_end = 0;
  // Whether a page so far was outside the cache: it holds no token, in the middle
  // of a list, and what it stands for (page 0) is masked.  (A vote on the chunks'
  // tokens in every group in place of this cost 1% more.)  Not causal: whether a
  // staged page lacks tokens, as any page of a list may, and groups do vote.
  bool bad = false;
  auto stage = [&](int g0) {
    stage_end = min(groups, g0 + per_stage);
    slot0 = 4 * g0 / c.chunks;
    slots = (min(4 * stage_end, s.chunks) - 1) / c.chunks + 1 - slot0;
    bool mine = false;
    for (int i = threadIdx.x; i < slots; i += kBlockThreads) {
      info[i] = ReadPage(a, s, head, slot0 + i);
      mine = mine || (kCausal ? info[i].tokens == 0 : info[i].tokens < c.page);
    }
    return mine;
  };
  // Chunk i of the list: its page and its part of it; tokens from its first on.
  auto place = [&](int i, int* sub) {
    const int slot = c.chunks == 1 ? i : static_cast<int>(__umulhi(i, inverse));
    *sub = i - slot * c.chunks;
    PageInfo k = info[min(slot - slot0, slots - 1)];
    k.tokens = i < s.chunks ? k.tokens - *sub * 16 : 0;
    return k;
  };

  // A group's codes on their way to LDS: a chunk's keys and its values are dim
  // units of 16 bytes each, at the same offset of both arrays, and thread i has every
  // kBlockThreads-th unit of the group's four chunks.
  uint4 kw[NJ], vw[NJ];
  auto fetch = [&](int grp) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int i = threadIdx.x + kBlockThreads * j;
      if (kAllUnits || i < 4 * D) {
        const int k = i / D;
        int sub;
        const int page = place(4 * grp + k, &sub).page;
        const int64_t at = static_cast<int64_t>(page * c.heads + head) * page_bytes +
                           (sub * D + i - k * D) * 16;
        kw[j] = *reinterpret_cast<const uint4*>(c.keys + at);
        vw[j] = *reinterpret_cast<const uint4*>(c.values + at);
      }
    }
  };
  auto put = [&](int grp, int buf) {
    _Float16* keys = key_tiles + buf * KeyHalves(D);
    _Float16* values = value_tiles + buf * ValueHalves(D);
    if (threadIdx.x < 4) {
      int sub;
      const PageInfo k = place(4 * grp + threadIdx.x, &sub);
      chunk_info[4 * buf + threadIdx.x] = {k.key_scale, k.value_scale,
                                           __builtin_amdgcn_logf(k.value_scale), k.tokens};
    }
    const bool tail = bad || (kCausal && (grp + 1) * kGroup > s.q.past + s.q.n);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int i = threadIdx.x + kBlockThreads * j;
      if (kAllUnits || i < 4 * D) {
        // as keys: 16 dims of token t; as values: 16 tokens of dim d
        const int t = i / units, u = i - t * units;
        const int k = i / D, d = i - k * D;
        _Float16* to = keys + t * (D + 8) + u * 16;
        *reinterpret_cast<F16x8*>(to) = Numbers8<FMT>(kw[j].x, kw[j].y);
        *reinterpret_cast<F16x8*>(to + 8) = Numbers8<FMT>(kw[j].z, kw[j].w);
        unsigned w[4] = {vw[j].x, vw[j].y, vw[j].z, vw[j].w};
        if (tail) {
          // Codes behind the request's tokens may be anything, and 0 * NaN is not 0.
          int tokens = kCausal ? s.q.past + s.q.n - grp * kGroup - 16 * k : 16;
          if (bad) {
            int sub;
            tokens = min(tokens, place(4 * grp + k, &sub).tokens);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int have = min(max(tokens - 4 * e, 0), 4);
            w[e] &= have == 4 ? 0xffffffffu : (1u << (8 * have)) - 1u;
          }
        }
        if constexpr (FMT == DSD_KV8_E4M3) {
          // A NaN must not reach the rows that do not see its token: it is taken
          // out, and the first of a dim remembered.
          if (((NanBytes(w[0]) | NanBytes(w[1])) | (NanBytes(w[2]) | NanBytes(w[3]))) != 0u) {
#pragma unroll
            for (int e = 3; e >= 0; --e) {
              const unsigned is = NanBytes(w[e]);
              if (is != 0u) {
                atomicMin(&nan_from[d], grp * kGroup + 16 * k + 4 * e + (__ffs(is) >> 3) - 1);
              }
              w[e] &= ~((is >> 7) * 0xffu);
            }
          }
        }
        to = values + d * kValueStride + 16 * k;
        *reinterpret_cast<F16x8*>(to) = Numbers8<FMT>(w[0], w[1]);
        *reinterpret_cast<F16x8*>(to + 8) = Numbers8<FMT>(w[2], w[3]);
      }
    }
  };

  // Row n's query, 8 dims of each 16 (16 k + 8 h on).
  const int row0 = first + 32 * wave;
  const int row = row0 + n;
  const bool there = row < s.rows;
  const int token = (there ? row : s.rows - 1) / group;
  const int q_head = head * group + (there ? row - token * group : 0);
  F16x8 q[KS][NQ];
  float to_logit;  // what a product with codes lacks but the page's scale; >= 0
  for (int i = threadIdx.x; i < D; i += kBlockThreads) nan_from[i] = 0x7fffffff;
  const bool bad_here = stage(begin);
  {
    const T* qp = static_cast<const T*>(a.q) + (s.q.row0 + token) * a.q_stride +
                  static_cast<int64_t>(q_head) * D;
    const bool even = reinterpret_cast<uintptr_t>(qp) % 16 == 0;
    float x[KS][8];
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = 0.0f;
      if (there && (kDim > 0 || k < units)) Load8(qp + 16 * k + 8 * h, even, x[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float size = fabsf(x[k][e]);
        most = fmaxf(most, size < INFINITY ? size : 0.0f);
      }
    }
    const QueryScale scale = ScaleQuery(Max2(most), a.scale);
    to_logit = scale.back;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) SplitQuery(x[k][e] * scale.up, q[k], e);
    }
  }
  // Row n's tokens, the most that one of the wave's rows sees, what all of them see.
  const int sees = kCausal ? s.q.past + token + 1 : 0x7fffffff;
  const int wave_sees =
      row0 >= s.rows ? 0
                     : (kCausal ? s.q.past + (min(row0 + 31, s.rows - 1)) / group + 1 : 0x7fffffff);
  const int all_see = kCausal ? s.q.past + row0 / group + 1 : 0x7fffffff;

  F32x16 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  float top = -INFINITY;  // of s + log2(value scale), less m: acc is relative to it
  // (m and top follow within kSlack)
  bool seen = false;  // not causal: a token

  bad = __syncthreads_or(bad_here) != 0;
  fetch(begin);
  put(begin, begin & 1);
  for (int grp = begin; grp < groups; ++grp) {
    const int buf = grp & 1;
    __syncthreads();
    if (grp + 1 < groups) {
      if (grp + 1 == stage_end) {
        const bool more_bad = stage(grp + 1);
        bad = __syncthreads_or((kCausal && bad) || more_bad) != 0;
      }
      fetch(grp + 1);
    }
    if (grp * kGroup < wave_sees) {
      const _Float16* keys = key_tiles + buf * KeyHalves(D) +
                             (16 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3)) * (D + 8) + 8 * h;
      const _Float16* values =
          value_tiles + buf * ValueHalves(D) + n * kValueStride + 16 * h;
      F32x16 x[2];
      float to_half[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[t][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if (kDim > 0 || k < units) {
            const F16x8 w = *reinterpret_cast<const F16x8*>(keys + 32 * t * (D + 8) + 16 * k);
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
              x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, q[k][i], x[t], 0, 0, 0);
            }
          }
        }
      }
      if constexpr (kDim > 0) {
        // kAhead operands on their way before the first product, then one a product.
        __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
        for (int i = 0; i < 2 * KS - kAhead; ++i) {
          __builtin_amdgcn_sched_group_barrier(kMfma, NQ, 0);
          __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, kAhead * NQ, 0);
      }
      ChunkInfo ci[2];
      float f[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ci[t] = chunk_info[4 * buf + 2 * t + h];
        f[t] = fmaxf(to_logit * ci[t].key_scale, kKv8Tiny);
      }
      const bool whole = kCausal ? (grp + 1) * kGroup <= all_see && !bad
                                 : __ballot(min(ci[0].tokens, ci[1].tokens) < 16) == 0;
      if (!kCausal) seen = seen || max(ci[0].tokens, ci[1].tokens) > 0;
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          int count = kCausal ? sees - (grp * kGroup + 32 * t + 16 * h) : ci[t].tokens;
          if (kCausal && bad) count = min(count, ci[t].tokens);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (i >= count) x[t][i] = -INFINITY;
          }
        }
      }
      float most[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        most[t] = x[t][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most[t] = fmaxf(most[t], x[t][i]);
        most[t] *= f[t];
      }
      const float m_new = fmaxf(m, Max2(fmaxf(most[0], most[1])));
      const float base_was = m == -INFINITY ? 0.0f : m;
      const float top_new = Max2(fmaxf(most[0] - base_was + ci[0].log_value_scale,
                                       most[1] - base_was + ci[1].log_value_scale));
      if (__ballot(m_new - m > kSlack || top_new - top > kSlack) != 0) {
        const float from = m_new == -INFINITY ? 0.0f : m_new;
        const float was = top + (m - from);
        top = fmaxf(was, Max2(fmaxf(most[0] - from + ci[0].log_value_scale,
                                    most[1] - from + ci[1].log_value_scale)));
        l *= Exp2(m - from);
        const float shrink = Exp2(was - (top == -INFINITY ? 0.0f : top));
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] *= shrink;
        m = m_new;
      }
      const float base = m == -INFINITY ? 0.0f : m;
      const float base_top = top == -INFINITY ? 0.0f : top;
      // A weight is 2^(s - base + lift), lift = log2 of the value scale - base_top + 11,
      // of which the row's sum wants 2^(s - base): the chunk's own sum times 2^-lift
      // (what lift - base loses to its rounding is then an error of s, in both sums).
      // (Where lift < -60 the weights are no half-precision number either way.)
      float sum[2] = {0.0f, 0.0f}, lift[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        lift[t] = fmaxf(ci[t].log_value_scale - base_top + kPromptBits, -60.0f);
        to_half[t] = lift[t] - base;
      }
      if (__ballot(fabsf(base) > kFar) != 0) {  // seldom
        if (fabsf(base) > kFar) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[t][i] = x[t][i] * f[t] - base;
            f[t] = 1.0f;
            to_half[t] = lift[t];
          }
        }
      }
      // The weights of the first 32 tokens; then their products with the weights
      // of the others in between, as the two units take turns; then the others'.
      // Operands are asked for kAhead products before theirs.
      F16x8 w[2][2][NP];
      auto weights = [&](int t, int i) {  // elements i, i + 1
        const float y0 = Exp2(fmaf(x[t][i], f[t], to_half[t]));
        const float y1 = Exp2(fmaf(x[t][i + 1], f[t], to_half[t]));
        sum[t] += y0 + y1;
        SplitWeights(y0, y1, w[t][i >> 3], i & 7);
      };
      constexpr int kSteps = 2 * NT;
      F16x8 v[2 * kSteps];
      auto operand = [&](int step) {
        const int t = step / kSteps, d = step % kSteps / 2, k = step % 2;
        if (kDim > 0 || 32 * d < D) {
          v[step] = *reinterpret_cast<const F16x8*>(values + 32 * d * kValueStride + 32 * t + 8 * k);
        }
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) operand(i);
#pragma unroll
      for (int i = 0; i < 16; i += 2) weights(0, i);
      if (kDim > 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int step = 0; step < 2 * kSteps; ++step) {
        const int t = step / kSteps, d = step % kSteps / 2, k = step % 2;
        if (step + kAhead < 2 * kSteps) operand(step + kAhead);
        if (kDim > 0 || 32 * d < D) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[step], w[t][k][i], acc[d], 0, 0, 0);
          }
        }
        if (t == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i * kSteps / 8 == step) weights(1, 2 * i);
          }
          if (kDim > 0) __builtin_amdgcn_sched_barrier(0);
        }
      }
      l += sum[0] * Exp2(-lift[0]);
      l += sum[1] * Exp2(-lift[1]);
    }
    if (grp + 1 < groups) put(grp + 1, buf ^ 1);
  }

  l = Sum2(l);
  const bool any = kCausal || Max2(seen ? 1.0f : 0.0f) > 0.0f;
  if (!there) return;
  const float lacks = (top == -INFINITY ? 0.0f : top) - kPromptBits;  // acc: 2^lacks
  Power to_out = PowerOf(lacks);
  const bool none = kCausal ? (bad && m == -INFINITY) || sees <= begin * kGroup : !any;  // no token here
  float* part = nullptr;
  if (parts) {
    const int64_t slot = (kJoin ? JoinSlot(plan, c.heads, s.q.row0, head, row)
                                : PartSlot(plan, c.heads, r, head, row)) + piece;
    part = plan.part + slot * D;
    if (h == 0) plan.stats[slot] = {m, none ? -1.0f : l, lacks};
    to_out = {1.0f, 1.0f};
  } else {
    to_out.most /= none ? 1.0f : l;
  }
  if (__ballot(to_out.rest != 1.0f) != 0) {  // seldom
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] *= to_out.rest;
  }
  T* out = static_cast<T*>(a.out) + (s.q.row0 + token) * a.out_stride +
           static_cast<int64_t>(q_head) * D;
  const bool even = reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * t + 2 * i + 4 * h;
      if (kDim > 0 || d < D) {
        F32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = acc[t][i + e] * to_out.most;
        if constexpr (FMT == DSD_KV8_E4M3) {
          const int4 nan = *reinterpret_cast<const int4*>(nan_from + d);
          const int least = min(min(nan.x, nan.y), min(nan.z, nan.w));
          if (least < sees) {
            if (nan.x < sees) o[0] = __builtin_nanf("");
            if (nan.y < sees) o[1] = __builtin_nanf("");
            if (nan.z < sees) o[2] = __builtin_nanf("");
            if (nan.w < sees) o[3] = __builtin_nanf("");
          }
        }
        if (parts) {
          *reinterpret_cast<F32x4*>(part + d) = o;
        } else {
          StoreRow4(out + d, even, o);
        }
      }
    }
  }
}

constexpr int kPromptTarget = 512;  // workgroups the chip runs at once
inline Plan PromptPlan(const Kv8View& c, const dsd_kv8_batch& b, int q_heads, int block = kRows) {
  Plan p;
  p.group = q_heads / c.heads;
  p.rows = static_cast<int64_t>(b.max_tokens) * p.group;
  p.block = block;
  p.blocks = static_cast<int>((p.rows + block - 1) / block);
  const int64_t units = static_cast<int64_t>(c.heads) * p.blocks * b.batch;
  const int64_t most = kPromptTarget * kRows / block / std::max<int64_t>(units, 1);
  // A group takes a workgroup about 1.5 us (a causal one of bf16 heads of 128, for all
  // forms alike: others' take longer); pieces cost the second launch, 5 us,
  // and a write and a read of their sums at about 3 TB/s.
  const int64_t groups = ListGroups(c, b);
  const double rows = static_cast<double>(b.batch) * c.heads * static_cast<double>(p.rows);
  const double piece_us = rows * c.dim * 8 / 3e6;
  int64_t best = 1;
  double best_us = 1.5 * static_cast<double>(groups);
  for (int64_t n = 2; n <= std::min<int64_t>(most, kMostPieces); ++n) {
    const double us = 1.5 * static_cast<double>((groups + n - 1) / n) + 5.0 + piece_us * n;
    if (us < best_us) {
      best_us = us;
      best = n;
    }
  }
  CutLists(&p, groups, best, 1);
  return p;
}

}  // namespace
}  // namespace dsdk
