// kv8_attend_block.h -- attention of 16 rows over a piece of a page list, what one
// workgroup of the 8-bit cache's attention kernels for few rows does.
#pragma once

#include <algorithm>

#include "kv8_attend.h"

namespace dsdk {
namespace {

constexpr float kMostFactor = 100.0f;  // powers of two beyond which weights are formed in steps

// 16 bytes of codes; once: they are not wanted again.
template <bool kOnce>
__device__ __forceinline__ uint4 LoadCodes(const uint8_t* p) {
  if constexpr (kOnce) {
    typedef unsigned U4 __attribute__((ext_vector_type(4)));
    const U4 x = __builtin_nontemporal_load(reinterpret_cast<const U4*>(p));
    return make_uint4(x[0], x[1], x[2], x[3]);
  } else {
    return *reinterpret_cast<const uint4*>(p);
  }
}

// kWeigh: a wave's logits that are held in LDS, 16 blocks of 4 rows (its LDS behind the
// staged pages: two workgroups of 72 KB a CU).
constexpr int kSlotFloats = 4096;

// Where the logits of a key head and 64 tokens of request r's list begin: [4 tokens of
// four][4 chunks of 16][rows of the key head][4], so that a wave's store of one of its
// four tiles is 64 bytes and more a chunk side by side, whole lines (rows of a head's
// tokens each in a line of its own took 497 us in place of the figure in kv8_weigh.hip).
// A list's first block is a whole one of its own.  Lists that begin no earlier than those
// before them end have blocks that no other writes; one behind a fall of page_offsets may
// name entries of an earlier one and keeps no logits (LaterList).
__host__ __device__ inline int64_t LogitBlocks(const Kv8AttendArgs& a) {
  return static_cast<int64_t>(a.b.total_pages) * a.c.page / 64 + a.b.batch + 1;
}
__device__ __forceinline__ int64_t LogitBlock(const Kv8AttendArgs& a, const Plan& p, int head, int r,
                                              int list, int block) {
  const int64_t first = static_cast<int64_t>(list) * a.c.page / 64 + r;
  return (head * LogitBlocks(a) + first + block) * 64 * p.group;
}
// Not 0 in some lane of the wave: page_offsets falls before request r's entry.
__device__ __forceinline__ int LaterList(const dsd_kv8_batch& b, int r) {
  if (b.list_stride > 0 || r == 0) return 0;
  const int lane = threadIdx.x & (kWave - 1), i = min(lane, r - 1);
  int fell = b.page_offsets[i + 1] < b.page_offsets[i] ? 1 : 0;
#pragma unroll 8
  for (int j = kWave + lane; j < r; j += kWave) {
    fell |= b.page_offsets[j + 1] < b.page_offsets[j] ? 1 : 0;
  }
  return fell;
}

// One piece of request r's list for one tile of 16 rows (unit: key heads * row tiles,
// the key head fastest); W waves, each of which takes
// every W-th group of 64 tokens of the piece for all of the tile's 16 rows.
// Lane (n, g) = (lane % 16, lane / 16).  Logits come out transposed, S^T = K
// Q^T in four tiles of 16 tokens whose rows are dealt so that lane (n, g) gets
// all 16 tokens of the group's chunk g for row n; they are then the second
// operand of O^T = V^T P^T as they stand (the order of a product's inner index
// is free), whose first operand, 16 tokens of one dim, is one load of the
// values' layout.  No number crosses lanes but for the maxima.
// kJoin: a later launch joins the piece with others.  kWeigh: logits (times log2 e) go
// to `logits` as well, unless a lane's `later` says that the list has no place there,
// and the rows' sums to p.stats.
// kDim: head_dim where it is 64 * NU (no bounds tests), else 0.
template <typename T, int FMT, int NU, int kDim, int W, bool kJoin, bool kWeigh = false>
__device__ __forceinline__ void AttendBlock(const Kv8AttendArgs& a, const Plan& p, int unit, int r,
                                            int piece, float* lds, float* logits = nullptr,
                                            int later = 0) {
  constexpr int NQ = kQueryTerms<T>, NP = kWeightTerms<T>, NT = 4 * NU;
  // The loads of a wave's last group are issued too (its own once more): a wait for the
  // values then counts the next keys and the stores, whichever path led there, and does
  // not wait for them.
  constexpr bool kSteady = kWeigh || kJoin;
  const Kv8View& c = a.c;
  const int D = kDim > 0 ? kDim : c.dim, tiles = kDim > 0 ? NT : D / 16;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int n = lane & 15, g = lane >> 4;
  const int head = unit % c.heads;
  const int first = unit / c.heads * 16;
  Span s;
  if (!FindSpan(a, p.group, r, first, 16, &s)) return;
  const int pieces = Pieces(p, s);
  if (piece >= pieces) return;
  const int groups = (s.chunks + 3) / 4;
  const int begin = piece * p.piece;
  const int end = piece == pieces - 1 ? groups : begin + p.piece;

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
    const QueryScale scale = ScaleQuery(Max4(most), a.scale);
    to_logit = scale.back;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) SplitQuery(x[u][i] * scale.up, q[u][i >> 3], i & 7);
    }
  };
  const int sees = a.causal ? s.q.past + token + 1 : 0x7fffffff;  // row n's tokens

  F32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = F32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  float top = -INFINITY;  // of s + log2(value scale), less m: acc is relative to it
  bool seen = false;

  // The list's pages are staged in LDS, so that a group's addresses are known
  // before its turn: its keys are asked for as soon as the logits of the group
  // before have taken their registers' contents, its values after the products.
  PageInfo* info = reinterpret_cast<PageInfo*>(lds);
  const int per_stage = max((kStage - 2) * c.chunks / 4, 1);  // groups
  const unsigned inverse = 0xffffffffu / static_cast<unsigned>(c.chunks) + 1u;
  const int page_bytes = c.page * D;
  uint4 kw[4][NU], vw[NT];
  // kWeigh: a wave's logits are kept in LDS and written many blocks at a time: a write
  // here and there among the reads costs HBM a fifth of its rate, bursts of them a
  // twentieth (16 bytes read a byte written, alone: 459 us for 2 GiB and 413 of 341
  // without writes; 355 where the reads leave the caches alone besides).
  const int tile_rows = kWeigh ? min(p.group - first, 16) : 16;
  const int most_held = kSlotFloats / (64 * tile_rows);
  float* kept = lds + (sizeof(PageInfo) * kStage / sizeof(float)) + wave * kSlotFloats;
  int held = 0;
  auto flush = [&](int last) {  // blocks last, last - W, ...
    const int quads = 16 * tile_rows;
    const int some = __ballot(later != 0) == 0 ? held : 0;
    for (int i = 0; i < some; ++i) {
      float* to = logits + LogitBlock(a, p, head, r, s.q.list, last - (held - 1 - i) * W) + first * 4;
      const float* from = kept + i * 64 * tile_rows;
      for (int e = lane; e < quads; e += kWave) {
        const int tg = e / tile_rows;  // (a compile-time 16 rows are no rule)
        *reinterpret_cast<F32x4*>(to + (tg * (p.group - tile_rows) + e) * 4) =
            *reinterpret_cast<const F32x4*>(from + 4 * e);
      }
    }
    held = 0;
  };
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
            kw[t][u] = LoadCodes<kWeigh>(kp + 4 * t * D + 64 * u);
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
        if (t < tiles) vw[t] = LoadCodes<kWeigh>(vp + 256 * t);
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
      const int next = more ? grp + W : grp;
      if (kSteady || more) load_keys(next);

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
      if constexpr (kWeigh) {
        // (the block's rows of this tile, [4 t][4 g][tile rows][4], in a slot of the wave)
        if (there) {
          float* to = kept + held * 64 * tile_rows + (g * tile_rows + n) * 4;
#pragma unroll
          for (int t = 0; t < 4; ++t) *reinterpret_cast<F32x4*>(to + 16 * t * tile_rows) = x[t] * f;
        }
        if (++held == most_held || !more) {
          WaveLdsFence();
          flush(grp);
          WaveLdsFence();
        }
      }
      float most = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        most = fmaxf(most, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
      }
      most *= f;
      seen = seen || count > 0;
      const float m_new = fmaxf(m, Max4(most));
      const float base = m_new == -INFINITY ? 0.0f : m_new;
      const float log_v = __builtin_amdgcn_logf(now.value_scale);
      const float was = top + (m - base);
      const float top_new = fmaxf(was, Max4(most - base + log_v));
      const float base_top = top_new == -INFINITY ? 0.0f : top_new;
      if (__ballot(m_new > m || top_new > was) != 0) {
        l *= Exp2(m - base);
        const float shrink = Exp2(was - base_top);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] *= shrink;
        m = m_new;
        top = top_new;
      }
      // A weight is p * to_half, p = 2^(s - base).  Where the largest p's values are
      // next to nothing (a page of zeros has the scale 2^-126) the two factors reach
      // 2^141 and more, the product 2^15 all the same: such a lane's 2^rise goes
      // from to_half to p, and to_half is formed in two steps.
      const float up = kWeightBits - base_top;
      float to_half = now.value_scale * Exp2(up);
      float slope = f, start = -base, to_sum = 1.0f;
      if (__ballot(up > kMostFactor || log_v + up > kMostFactor || fabsf(base) > kFar) != 0) {  // seldom
        const float rise = fmaxf(ceilf(log_v + up - kMostFactor), 0.0f);
        const float lift = up - rise > 0.5f * kMostFactor ? 0.5f * kMostFactor : 0.0f;
        to_half = now.value_scale * Exp2(lift) * Exp2(up - rise - lift);
        start = rise - base;
        to_sum = Exp2(-rise);
        if (fabsf(base) > kFar) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t][i] = x[t][i] * f - base;
          }
          slope = 1.0f;
          start = rise;
        }
      }
      F16x8 w[2][NP];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float e0 = Exp2(fmaf(x[t][i], slope, start));
          const float e1 = Exp2(fmaf(x[t][i + 1], slope, start));
          l = fmaf(e0 + e1, to_sum, l);
          SplitWeights(e0 * to_half, e1 * to_half, w[t >> 1], 4 * (t & 1) + i);
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
      if (kSteady || more) load_values(next);
    }
  }

  // The waves' streams, through LDS: [W][16] m, l and top, [W][16][D + 4] acc.
  __syncthreads();
  float* s_m = lds;
  float* s_l = lds + 16 * W;
  float* s_top = lds + 32 * W;
  float* s_acc = lds + 48 * W;
  l = Sum4(l);
  const bool any = Max4(seen ? 1.0f : 0.0f) > 0.0f;
  if (g == 0) {
    s_m[wave * 16 + n] = m;
    s_l[wave * 16 + n] = any ? l : -1.0f;
    s_top[wave * 16 + n] = top;
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
    float most = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (!(s_l[w * 16 + k] < 0.0f)) {
        most = fmaxf(most, s_m[w * 16 + k] - base + s_top[w * 16 + k]);
      }
    }
    most = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f;
    F32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (!(s_l[w * 16 + k] < 0.0f)) {
        const float e = s_m[w * 16 + k] - base;
        sum += s_l[w * 16 + k] * Exp2(e);
        o += *reinterpret_cast<const F32x4*>(s_acc + (w * 16 + k) * (D + 4) + d) *
             Exp2(e + s_top[w * 16 + k] - most);
      }
    }
    const float x = most - kWeightBits;  // o lacks 2^x
    if (kWeigh && pieces == 1 && d == 0) {
      p.stats[PartSlot(p, c.heads, r, head, at)] = {peak, some ? sum : -1.0f, x};
    }
    if (!kJoin && pieces == 1) {
      const int tok = at / p.group;
      T* out = static_cast<T*>(a.out) + (s.q.row0 + tok) * a.out_stride +
               static_cast<int64_t>(head * p.group + at - tok * p.group) * D + d;
      const F32x4 zero = {0, 0, 0, 0};
      const Power to_out = PowerOf(x);
      StoreRow4(out, reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0,
                some ? o * (to_out.most / sum) * to_out.rest : zero);
    } else {
      const int64_t slot = (kJoin ? JoinSlot(p, c.heads, s.q.row0, head, at)
                                  : PartSlot(p, c.heads, r, head, at)) + piece;
      *reinterpret_cast<F32x4*>(p.part + slot * D + d) = o;
      if (d == 0) p.stats[slot] = {peak, some ? sum : -1.0f, x};
    }
  }
}

constexpr int kAttendWaves = 4;

inline size_t AttendLdsBytes(int dim, bool weigh = false) {
  const size_t joined = sizeof(float) * (48 * kAttendWaves + kAttendWaves * 16 * (dim + 4));
  const size_t staged =
      sizeof(PageInfo) * kStage + (weigh ? sizeof(float) * kSlotFloats * kAttendWaves : 0);
  return joined > staged ? joined : staged;
}

// Two workgroups fit a CU (registers), 512 the chip.
constexpr int kAttendTarget = 512;

// Pieces that lists of so many groups are cut into, `units` workgroups to a piece.
// In us: a launch about 5.5; a step, a group for each of the four waves, 1.15 and
// more where workgroups share the memory's rate, up to 5.9 TB/s; the merge, with
// its launch, 3.5 to 5.9.  Heads of 128 (32 / 8), bf16, us whole and in pieces:
// one of 512 tokens 8.2 and 10.3, of 2000 15.0 and 10.4, of 32000 158 and 22; 16
// of 1000 12.9 and 16.8, of 2000 17.7 and 19.9, of 8000 64 and 56; 32 of 500 11.7
// and 17.1.  Lists are seldom equally long, and pieces end more evenly: of choices
// within 3% the one with most pieces.
inline int64_t PiecesWanted(int64_t groups, int64_t most, int64_t units, int dim) {
  const int64_t steps = (groups + kAttendWaves - 1) / kAttendWaves;
  const double share = 8.7e-5 * dim;  // us of a step's bytes of one workgroup
  auto cost = [&](int64_t n) {
    const double workgroups = static_cast<double>(units * n);
    const double step = std::max(1.15 + 0.6 * share * workgroups, share * workgroups);
    const double merge = n > 1 ? 3.5 + 2.4 * std::min(1.0, workgroups / 256) : 0.0;
    return 5.5 + static_cast<double>((steps + n - 1) / n) * step + merge;
  };
  most = std::min(most, steps);
  double best = cost(1);
  for (int64_t n = 2; n <= most; ++n) best = std::min(best, cost(n));
  int64_t n = most;
  while (n > 1 && cost(n) > 1.03 * best) --n;
  return n;
}

inline Plan AttendPlan(const Kv8View& c, const dsd_kv8_batch& b, int q_heads, bool many) {
  Plan p;
  p.group = q_heads / c.heads;
  p.rows = static_cast<int64_t>(many ? b.max_tokens : 1) * p.group;
  p.block = 16;
  p.blocks = static_cast<int>((p.rows + p.block - 1) / p.block);
  const int64_t units = static_cast<int64_t>(c.heads) * p.blocks * b.batch;
  const int64_t groups = ListGroups(c, b);
  const int64_t most = std::min<int64_t>(kAttendTarget / std::max<int64_t>(units, 1), kMostPieces);
  CutLists(&p, groups, PiecesWanted(groups, std::max<int64_t>(most, 1), units, c.dim), kAttendWaves);
  return p;
}

}  // namespace
}  // namespace dsdk
