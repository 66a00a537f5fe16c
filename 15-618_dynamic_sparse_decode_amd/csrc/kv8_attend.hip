// kv8_attend.hip -- dsd_kv8_attend and dsd_kv8_attend_prompt (gfx950):
// softmax attention over the pages of an 8-bit cache.
//
// Mathematics.  Codes are exact in half precision, so q K^T is a product of
// half-precision matrices: q scaled by a power of two so that its row's
// largest element lies in [2^13, 2^14) -- one term for 16-bit queries (what
// falls below half precision's range is 2^-38 of that element), two for
// float32 ones -- times the codes; the page's scale and the power of two go on
// the logits afterwards, in float32.  Weights p = 2^(s - m) (s in the log2
// domain, m the running maximum) meet the value codes the same way, as p * v *
// 2^(m - n + 15) with v the page's value scale and n the running maximum of s +
// log2 v, so at most 2^15 whatever the scales and logits: half precision rounds them to
// 2^-11, or 2^-22 as two terms where the output is finer than bf16 (bf16 outputs,
// whose own rounding is 2^-8, are off by 0.0017 of their size either way; two terms
// took 12.2 us in place of 11.5 for one request of 1000 tokens, 38.9 in place of
// 37.6 for drafted tokens).  All sums are float32.
//
// Bound by HBM for long lists: a token's codes and scales are read once for all
// query heads of its key head.  Measured (kernel times): 32 requests of 32768
// tokens, 8 key heads of 128, pages of 16: 366 us for 2.15 GB, 5.9 TB/s, what
// reads alone reach here; 64 requests of 32 pages of 64: 44 us, 6.2 TB/s; 16
// requests of 512-2048 tokens, 32 key heads, float32: 36 us, 5.2 TB/s; 4 of
// 65536-131072, int8, heads of 64: 42 us, 5.3 TB/s, and 5 for the merge; one of
// 1000 tokens: 11.6 us, a chain of ids -> scales and codes -> products.
#include "kv8_attend.h"

#include <algorithm>
#include <cmath>

namespace dsdk {
namespace {

constexpr float kMostFactor = 100.0f;  // powers of two beyond which weights are formed in steps

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
__global__ __launch_bounds__(W* kWave, NU <= 2 ? 2 : 1) void Kv8AttendKernel(Kv8AttendArgs a,
                                                                            Plan p) {
  constexpr int NQ = kQueryTerms<T>, NP = kWeightTerms<T>, NT = 4 * NU;
  extern __shared__ __align__(16) float lds[];
  const Kv8View& c = a.c;
  const int D = kDim > 0 ? kDim : c.dim, tiles = kDim > 0 ? NT : D / 16;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int n = lane & 15, g = lane >> 4;
  const int r = blockIdx.y, head = blockIdx.x % c.heads;
  const int first = blockIdx.x / c.heads * 16;
  Span s;
  if (!FindSpan(a, p.group, r, first, 16, &s)) return;
  const int pieces = Pieces(p, s);
  if (static_cast<int>(blockIdx.z) >= pieces) return;
  const int groups = (s.chunks + 3) / 4;
  const int begin = blockIdx.z * p.piece;
  const int end = static_cast<int>(blockIdx.z) == pieces - 1 ? groups : begin + p.piece;

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
      if (more) load_values(grp + W);
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
    if (pieces == 1) {
      const int tok = at / p.group;
      T* out = static_cast<T*>(a.out) + (s.q.row0 + tok) * a.out_stride +
               static_cast<int64_t>(head * p.group + at - tok * p.group) * D + d;
      const F32x4 zero = {0, 0, 0, 0};
      const Power to_out = PowerOf(x);
      StoreRow4(out, reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0,
                some ? o * (to_out.most / sum) * to_out.rest : zero);
    } else {
      const int64_t slot = PartSlot(p, c.heads, r, head, at) + blockIdx.z;
      *reinterpret_cast<F32x4*>(p.part + slot * D + d) = o;
      if (d == 0) p.stats[slot] = {peak, some ? sum : -1.0f, x};
    }
  }
}

// Grid (256 numbers of a row each, batch).
template <typename T>
__global__ __launch_bounds__(256) void Kv8GroupQueriesKernel(const T* q, int64_t q_stride,
                                                             int group, int dim, int elements,
                                                             float* sums) {
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= elements) return;
  const int head = e / dim, d = e - head * dim;
  const T* p = q + blockIdx.y * q_stride + static_cast<int64_t>(head) * group * dim + d;
  float sum = static_cast<float>(p[0]);
  for (int g = 1; g < group; ++g) sum += static_cast<float>(p[g * dim]);
  sums[static_cast<int64_t>(blockIdx.y) * elements + e] = sum;
}

constexpr int kWaves = 4;

// Two workgroups fit a CU (registers), 512 the chip.
constexpr int kTarget = 512;

// Pieces that lists of so many groups are cut into, `units` workgroups to a piece.
// In us: a launch about 5.5; a step, a group for each of the four waves, 1.15 and
// more where workgroups share the memory's rate, up to 5.9 TB/s; the merge, with
// its launch, 3.5 to 5.9.  Heads of 128 (32 / 8), bf16, us whole and in pieces:
// one of 512 tokens 8.2 and 10.3, of 2000 15.0 and 10.4, of 32000 158 and 22; 16
// of 1000 12.9 and 16.8, of 2000 17.7 and 19.9, of 8000 64 and 56; 32 of 500 11.7
// and 17.1.  Lists are seldom equally long, and pieces end more evenly: of choices
// within 3% the one with most pieces.
int64_t PiecesWanted(int64_t groups, int64_t most, int64_t units, int dim) {
  const int64_t steps = (groups + kWaves - 1) / kWaves;
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

Plan MakePlan(const Kv8View& c, const dsd_kv8_batch& b, int q_heads, bool causal) {
  Plan p;
  p.group = q_heads / c.heads;
  p.rows = static_cast<int64_t>(causal ? b.max_tokens : 1) * p.group;
  p.block = 16;
  p.blocks = static_cast<int>((p.rows + p.block - 1) / p.block);
  const int64_t units = static_cast<int64_t>(c.heads) * p.blocks * b.batch;
  const int64_t groups = ListGroups(c, b);
  const int64_t most = std::min<int64_t>(kTarget / std::max<int64_t>(units, 1), kMostPieces);
  CutLists(&p, groups, PiecesWanted(groups, std::max<int64_t>(most, 1), units, c.dim), kWaves);
  return p;
}

// Whether a prompt call has rows enough for kv8_prompt.hip.  Both sides (us, this
// file's form and that one's): 16 requests with 128 rows behind 8000 tokens 175
// and 134; with 64 rows behind 1000 tokens 21 and 40; one with 64 rows behind
// 60000 tokens 101 and 157.
bool ManyRows(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  return static_cast<int64_t>(b.max_tokens) * (q_heads / c.heads) > 64;
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
  const dim3 grid(a.c.heads * p.blocks, a.b.batch, p.pieces);
  WithKernel<T, FMT>(a.c.dim, [&](auto kernel) {
    kernel<<<grid, kWaves * kWave, LdsBytes(a.c.dim), stream>>>(a, p);
  });
  DSD_HIP_CHECK(hipGetLastError());
  Merge<T>(a, p, stream);
}

template <typename T>
void LaunchType(const Kv8AttendArgs& a, const Plan& p, hipStream_t stream) {
  a.c.format == DSD_KV8_INT8 ? Launch<T, DSD_KV8_INT8>(a, p, stream)
                             : Launch<T, DSD_KV8_E4M3>(a, p, stream);
}

template <typename T, int FMT>
void PreloadDim(const Kv8View& c) {
  WithKernel<T, FMT>(c.dim, [&](auto kernel) {
    PreloadKernel(kernel);
    DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(LdsBytes(c.dim))));
  });
}

template <typename T>
void PreloadType(const Kv8View& c) {
  c.format == DSD_KV8_INT8 ? PreloadDim<T, DSD_KV8_INT8>(c) : PreloadDim<T, DSD_KV8_E4M3>(c);
  PreloadKernel(Kv8MergeKernel<T>);
  PreloadKernel(Kv8MergeRowsKernel<T>);
  PreloadKernel(Kv8GroupQueriesKernel<T>);
}

}  // namespace

size_t Kv8WorkspaceBytes(const Kv8View& c, const dsd_kv8_batch& b, int q_heads) {
  if (b.batch == 0) return 0;
  dsd_kv8_batch one = b;
  one.max_tokens = 1;
  size_t bytes = MostPartBytes(c, MakePlan(c, one, q_heads, false), kTarget);
  if (b.max_tokens > 1) {
    bytes = std::max(bytes, MostPartBytes(c, MakePlan(c, b, q_heads, true), kTarget));
  }
  // (of one token a request too, where query heads enough share a key head)
  if (ManyRows(c, b, q_heads)) bytes = std::max(bytes, Kv8PromptWorkspaceBytes(c, b, q_heads));
  return bytes;
}

void LaunchKv8GroupQueries(const Kv8View& c, int batch, int type, int q_heads, const void* q,
                           int64_t q_stride, float* sums, hipStream_t stream) {
  const int elements = c.heads * c.dim;
  const dim3 grid((elements + 255) / 256, batch);
  auto launch = [&](auto* rows) {
    using T = std::remove_cv_t<std::remove_pointer_t<decltype(rows)>>;
    Kv8GroupQueriesKernel<T><<<grid, 256, 0, stream>>>(rows, q_stride, q_heads / c.heads, c.dim,
                                                       elements, sums);
  };
  switch (type) {
    case DSD_TYPE_F32: launch(static_cast<const float*>(q)); break;
    case DSD_TYPE_BF16: launch(static_cast<const __bf16*>(q)); break;
    default: launch(static_cast<const _Float16*>(q));
  }
  DSD_HIP_CHECK(hipGetLastError());
}

void PreloadKv8Attend(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
}

void LaunchKv8Attend(const Kv8AttendArgs& a, hipStream_t stream) {
  if (a.b.batch == 0 || (a.causal && a.b.tokens == 0)) return;
  if (a.causal && ManyRows(a.c, a.b, a.q_heads)) return LaunchKv8Prompt(a, stream);
  Plan p = MakePlan(a.c, a.b, a.q_heads, a.causal);
  PlaceParts(&p, a);
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(a, p, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(a, p, stream);
    default: return LaunchType<_Float16>(a, p, stream);
  }
}

}  // namespace dsdk
