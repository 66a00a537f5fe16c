// kv8_append.hip -- dsd_kv8_append (gfx950): a batch's new tokens rotated,
// quantised and written behind what an 8-bit paged cache holds, and their
// queries rotated.
//
// Mathematics.  Pair (x, y) of a head turns by a = position * inv_freq:
// (x cos a - y sin a, y cos a + x sin a).  Angles are taken in half turns
// (position * (inv_freq / pi), exact in 64 bits far beyond a million
// positions, where 32 bits are off by whole hundredths of a radian) and the
// products in 64 bits too: a key's code then falls on the right side of every
// rounding border.  The codes of a page share one scale s >= largest / M (M =
// 448 or 127), so a token that needs a larger one takes the page's earlier
// codes with it: code <- nearest(code * old / s).
//
// Bound by HBM: queries, keys and values are read once, rotated queries and
// codes written once.  A workgroup takes one page's new tokens of some key
// heads and of the query heads that read them, so an angle's sine and cosine
// are formed once for all of these.  Within it a wave takes one side (keys or
// values) of one head at a time.
#include "kv8_device.h"

#include <algorithm>

namespace dsdk {
namespace {

template <int FMT>
constexpr float kLargest = FMT == DSD_KV8_INT8 ? 127.0f : 448.0f;

// The least scale whose largest code reaches `most` (finite, >= 0).
template <int FMT>
__device__ __forceinline__ float ScaleFor(float most) {
  if constexpr (FMT == DSD_KV8_INT8) {
    return fmaxf(static_cast<float>(static_cast<double>(most) / 127.0), kKv8Tiny);
  } else {
    // most = f * 2^e, f in [0.5, 1); 448 = 0.875 * 2^9
    int e;
    const float f = frexpf(most, &e);
    const int power = max(e - 9 + (f > 0.875f ? 1 : 0), -126);
    return most > 0.0f ? __uint_as_float(static_cast<unsigned>(power + 127) << 23) : kKv8Tiny;
  }
}

// x in 32 bits so that a further rounding is that of x itself: towards zero,
// the last bit set where anything was lost.
__device__ __forceinline__ float ToOdd(double x) {
  const float y = static_cast<float>(x);
  const double back = static_cast<double>(y);
  if (back == x || !(fabs(x) < 0x1p127)) return y;
  unsigned bits = __float_as_uint(y);
  if (fabs(back) > fabs(x)) --bits;
  return __uint_as_float(bits | 1u);
}

// A scale with its reciprocals.
struct Scale {
  float s = 0.0f;
  float inv = 0.0f;     // e4m3
  double inv64 = 0.0;   // int8
  template <int FMT>
  __device__ __forceinline__ void Set(float scale) {
    s = scale;
    if constexpr (FMT == DSD_KV8_INT8) {
      inv64 = 1.0 / static_cast<double>(scale);
    } else {
      inv = 1.0f / scale;  // (exact: a power of two)
    }
  }
};

// The nearest integer to x / s within [-127, 127], halves to the even one; 0
// for NaN.  The product with the reciprocal may be off by one where x / s lies
// next to a half; the remainder, exact for x of 32 bits, decides there.
__device__ __forceinline__ int NearestInt8(double x, const Scale& s) {
  const double top = 127.0 * static_cast<double>(s.s);
  if (!(fabs(x) < top)) return x > 0.0 ? 127 : (x < 0.0 ? -127 : 0);
  double n = rint(x * s.inv64);
  const double rest = fma(-n, static_cast<double>(s.s), x);
  const double half = 0.5 * static_cast<double>(s.s);
  const double size = fabs(rest);
  if (size >= half) {
    const bool odd = (static_cast<int>(n) & 1) != 0;
    if (size > half || odd) n += rest > 0.0 ? 1.0 : -1.0;
  }
  return static_cast<int>(n);
}

// Four codes of x / s, one a byte.
template <int FMT, typename X>
__device__ __forceinline__ unsigned Codes4(X x0, X x1, X x2, X x3, const Scale& s) {
  if constexpr (FMT == DSD_KV8_INT8) {
    const unsigned a = static_cast<unsigned>(NearestInt8(x0, s)) & 0xffu;
    const unsigned b = static_cast<unsigned>(NearestInt8(x1, s)) & 0xffu;
    const unsigned c = static_cast<unsigned>(NearestInt8(x2, s)) & 0xffu;
    const unsigned d = static_cast<unsigned>(NearestInt8(x3, s)) & 0xffu;
    return a | (b << 8) | (c << 16) | (d << 24);
  } else {
    float y[4];
    const X x[4] = {x0, x1, x2, x3};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float z;
      if constexpr (sizeof(X) == 8) {
        z = ToOdd(x[i]);
      } else {
        z = x[i];
      }
      z *= s.inv;
      y[i] = z != z ? z : fminf(fmaxf(z, -448.0f), 448.0f);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true));
  }
}

// The four numbers that a word's codes stand for.
template <int FMT>
__device__ __forceinline__ void Numbers4(unsigned w, float* x) {
  if constexpr (FMT == DSD_KV8_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = static_cast<float>(static_cast<int>(w << (24 - 8 * i)) >> 24);
    }
  } else {
    const F32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const F32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = a[0];
    x[1] = a[1];
    x[2] = b[0];
    x[3] = b[1];
  }
}

// Codes brought from scale `old` to the larger s.
template <int FMT>
__device__ __forceinline__ unsigned Rescale4(unsigned w, float old, const Scale& s) {
  float x[4];
  Numbers4<FMT>(w, x);
  double y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = static_cast<double>(x[i]) * static_cast<double>(old);
  return Codes4<FMT>(y[0], y[1], y[2], y[3], s);
}

__device__ __forceinline__ float FiniteSize(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

__device__ __forceinline__ float WaveMax(float x) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) x = fmaxf(x, __shfl_xor(x, o, kWave));
  return x;
}

// Where a head's 16 elements of unit u lie: 8 from a on, 8 from b on, and
// whether they turn with the sines of pairs [8 u, 8 u + 8).
struct Unit {
  int a = 0, b = 0;
  bool turns = false;
};
__device__ __forceinline__ Unit UnitOf(int u, const Kv8Rotation& rot) {
  Unit x;
  x.turns = 8 * u < rot.pairs;
  if (x.turns && !rot.interleaved) {
    x.a = 8 * u;
    x.b = rot.pairs + 8 * u;
  } else {
    x.a = 16 * u;
    x.b = 16 * u + 8;
  }
  return x;
}

// The sines of 16 tokens in LDS: (cos, sin) of token o's pair 8 u + i at
// [o][i][u], so that the lanes of a row, one unit each, read next to each
// other.
__device__ __forceinline__ int SineAt(int o, int i, int u, int turning) {
  return (o * 8 + i) * turning + u;
}

// x[0..8) at a, x[8..16) at b, turned into y; cs: the unit's first pair, the
// others `step` apart.
__device__ __forceinline__ void Turn(const float* x, const double2* cs, int step, const Unit& u,
                                     int interleaved, double* y) {
  if (!u.turns) {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = static_cast<double>(x[i]);
  } else if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double c = cs[i * step].x, s = cs[i * step].y;
      const double p = static_cast<double>(x[2 * i]), q = static_cast<double>(x[2 * i + 1]);
      y[2 * i] = p * c - q * s;
      y[2 * i + 1] = q * c + p * s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double c = cs[i * step].x, s = cs[i * step].y;
      const double p = static_cast<double>(x[i]), q = static_cast<double>(x[8 + i]);
      y[i] = p * c - q * s;
      y[8 + i] = q * c + p * s;
    }
  }
}

// One page's part of a call.
struct Task {
  int page = 0;
  int first = 0;  // new tokens: offsets [first, end) of the page
  int end = 0;
  int row = 0;    // the row of offset 0 (may be negative)
  int index = 0;  // the index in its request of offset 0
};

// The task of workgroup u: request r's pages take workgroups from
// floor(token_offsets[r] / page) + 2 r on, at least as many as its tokens can
// touch (one each where every request has one token).  Every wave computes
// the same.
__device__ __forceinline__ bool FindTask(const Kv8AppendArgs& a, int u, Task* t) {
  const dsd_kv8_batch& b = a.b;
  const int ps = a.c.page;
  int r = u, within = 0;
  if (b.max_tokens > 1) {
    const int lane = threadIdx.x & (kWave - 1);
    int below = 0;
    for (int b0 = 0; b0 < b.batch; b0 += kWave) {
      const int i = b0 + lane;
      bool mine = false;
      if (i < b.batch) mine = b.token_offsets[i] / ps + 2 * i <= u;
      const int got = __popcll(__ballot(mine));
      below += got;
      if (got < kWave) break;
    }
    r = below - 1;
    if (r < 0) return false;
    within = u - (b.token_offsets[r] / ps + 2 * r);
    if (within < 0) return false;
  }
  if (r >= b.batch) return false;
  Kv8Request q;
  if (!Kv8ReadTokens(b, r, ps, &q)) {
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailShape);
    return false;
  }
  if (q.n == 0) return false;
  const int slot0 = q.past / ps, last = (q.past + q.n - 1) / ps;
  const int slot = slot0 + within;
  if (slot > last) return false;
  t->page = b.page_ids[q.list + slot];
  if (!InPool(t->page, a.c.capacity)) {
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailPageId);
    return false;
  }
  t->index = slot * ps;
  t->first = max(q.past - t->index, 0);
  t->end = min(q.past + q.n - t->index, ps);
  t->row = q.row0 + t->index - q.past;
  return true;
}

// The sines and cosines of a chunk's tokens, offsets [lo, hi) of the 16 from
// c0 on, [16][pairs].
__device__ __forceinline__ void FillSines(const Kv8AppendArgs& a, const Task& t, int c0, int lo,
                                          int hi, double2* cs) {
  const int pairs = a.rot.pairs;
  const int n = (hi - lo) * pairs;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int k = i / pairs, p = i - k * pairs;
    const int o = c0 + lo + k;
    const int at = a.b.positions != nullptr ? a.b.positions[t.row + o] : t.index + o;
    double s, c;
    sincospi(static_cast<double>(at) * a.rot.turns[p], &s, &c);
    cs[SineAt(lo + k, p & 7, p >> 3, pairs / 8)] = {c * a.rot.magnitude, s * a.rot.magnitude};
  }
}

// ---- keys ----------------------------------------------------------------------
// Lane l has unit (l + 64 j) % units of token (l + 64 j) / units, j < NU =
// ceil(dim / 64).

template <typename T, int NU>
__device__ __forceinline__ void LoadKeys(const Kv8AppendArgs& a, bool vec, const Task& t, int h,
                                         int c0, int lo, int hi, float (&x)[NU][16]) {
  const int lane = threadIdx.x & (kWave - 1);
  const int units = a.c.dim / 16;
  const T* k = static_cast<const T*>(a.k) + static_cast<int64_t>(h) * a.c.dim;
#pragma unroll
  for (int j = 0; j < NU; ++j) {
    const int i = lane + kWave * j;
    const int o = i / units, u = i - o * units;
    if (o >= lo && o < hi) {
      const Unit w = UnitOf(u, a.rot);
      const T* p = k + (t.row + c0 + o) * a.k_stride;
      Load8(p + w.a, vec, x[j]);
      Load8(p + w.b, vec, x[j] + 8);
    }
  }
}

template <int NU>
__device__ __forceinline__ float LargestKey(const Kv8AppendArgs& a, int lo, int hi,
                                            const double2* cs, const float (&x)[NU][16]) {
  const int lane = threadIdx.x & (kWave - 1);
  const int units = a.c.dim / 16, turning = a.rot.pairs / 8;
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < NU; ++j) {
    const int i = lane + kWave * j;
    const int o = i / units, u = i - o * units;
    if (o >= lo && o < hi) {
      double y[16];
      Turn(x[j], cs + SineAt(o, 0, u, turning), turning, UnitOf(u, a.rot), a.rot.interleaved, y);
#pragma unroll
      for (int e = 0; e < 16; ++e) most = fmaxf(most, FiniteSize(static_cast<float>(y[e])));
    }
  }
  return most;
}

// One chunk's codes: offsets [lo, hi) new (x, turned again), those before them
// as they are or brought from `had` to s.  tile:
// 16 x dim bytes of LDS.  sums: the lane's dims 2 lane, 2 lane + 1 of each 128,
// summed over offsets [0, hi).
template <int FMT, int NU>
__device__ __forceinline__ void StoreKeys(const Kv8AppendArgs& a, uint8_t* block, int lo, int hi,
                                          float had, bool grew, const Scale& s,
                                          const float (&x)[NU][16], const double2* cs,
                                          uint8_t* tile, float (&sums)[(NU + 1) / 2][2]) {
  const int lane = threadIdx.x & (kWave - 1);
  const int D = a.c.dim;
  const int units = D / 16;
  const int turning = a.rot.pairs / 8;
  const int from = grew ? 0 : lo;  // offsets written
  if (lo > 0 && (grew || a.c.summaries != nullptr)) {
    for (int i = lane; i < lo * units; i += kWave) {
      uint4 w = *reinterpret_cast<const uint4*>(block + 16 * i);
      if (grew) {
        w.x = Rescale4<FMT>(w.x, had, s);
        w.y = Rescale4<FMT>(w.y, had, s);
        w.z = Rescale4<FMT>(w.z, had, s);
        w.w = Rescale4<FMT>(w.w, had, s);
      }
      *reinterpret_cast<uint4*>(tile + 16 * i) = w;
    }
  }
#pragma unroll
  for (int j = 0; j < NU; ++j) {
    const int i = lane + kWave * j;
    const int o = i / units, u = i - o * units;
    if (o >= lo && o < hi) {
      const Unit w = UnitOf(u, a.rot);
      double y[16];
      Turn(x[j], cs + SineAt(o, 0, u, turning), turning, w, a.rot.interleaved, y);
      uint2 p, q;
      p.x = Codes4<FMT>(y[0], y[1], y[2], y[3], s);
      p.y = Codes4<FMT>(y[4], y[5], y[6], y[7], s);
      q.x = Codes4<FMT>(y[8], y[9], y[10], y[11], s);
      q.y = Codes4<FMT>(y[12], y[13], y[14], y[15], s);
      *reinterpret_cast<uint2*>(tile + o * D + w.a) = p;
      *reinterpret_cast<uint2*>(tile + o * D + w.b) = q;
    }
  }
  WaveLdsFence();
  for (int i = from * units + lane; i < hi * units; i += kWave) {
    *reinterpret_cast<uint4*>(block + 16 * i) = *reinterpret_cast<const uint4*>(tile + 16 * i);
  }
  if (a.c.summaries != nullptr) {
#pragma unroll
    for (int m = 0; m < (NU + 1) / 2; ++m) {
      const int d = 128 * m + 2 * lane;
      if (d < D) {
        for (int o = 0; o < hi; ++o) {
          float x[4];
          Numbers4<FMT>(*reinterpret_cast<const uint16_t*>(tile + o * D + d), x);
          sums[m][0] += x[0];
          sums[m][1] += x[1];
        }
      }
    }
  }
  WaveLdsFence();
}

// ---- values --------------------------------------------------------------------
// Lane l has dims 2 l, 2 l + 1 of each 128 and the 16 tokens of a chunk.

template <typename T>
__device__ __forceinline__ void LoadValues(const Kv8AppendArgs& a, bool vec, const Task& t, int h,
                                           int c0, int lo, int hi, int d, float (&x)[2][16]) {
  const T* v = static_cast<const T*>(a.v) + static_cast<int64_t>(h) * a.c.dim + d;
  typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int o = 0; o < 16; ++o) {
    x[0][o] = 0.0f;
    x[1][o] = 0.0f;
    if (o >= lo && o < hi && d < a.c.dim) {
      const T* p = v + (t.row + c0 + o) * a.v_stride;
      if (vec) {
        const T2 w = *reinterpret_cast<const T2*>(p);
        x[0][o] = static_cast<float>(w[0]);
        x[1][o] = static_cast<float>(w[1]);
      } else {
        x[0][o] = static_cast<float>(p[0]);
        x[1][o] = static_cast<float>(p[1]);
      }
    }
  }
}

__device__ __forceinline__ float LargestValue(const float (&x)[2][16]) {
  float most = 0.0f;
#pragma unroll
  for (int o = 0; o < 16; ++o) {
    most = fmaxf(most, fmaxf(FiniteSize(x[0][o]), FiniteSize(x[1][o])));
  }
  return most;
}

// The byte mask of tokens [lo, hi) in word i (tokens 4 i ..) of a column.
__device__ __forceinline__ unsigned TokenMask(int i, int lo, int hi) {
  const int l = min(max(lo - 4 * i, 0), 4), h = min(max(hi - 4 * i, 0), 4);
  const unsigned below_h = h == 4 ? 0xffffffffu : (1u << (8 * h)) - 1u;
  const unsigned below_l = l == 4 ? 0xffffffffu : (1u << (8 * l)) - 1u;
  return below_h & ~below_l;
}

// column: the 16 codes of one dim.  Tokens outside [0, hi) stay as they are.
template <int FMT>
__device__ __forceinline__ void StoreValues(uint8_t* column, int lo, int hi, float had, bool grew,
                                            const Scale& s, const float (&x)[16]) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = lo < hi ? Codes4<FMT>(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], s) : 0u;
  }
  if (lo > 0 || hi < 16) {
    const uint4 old = *reinterpret_cast<const uint4*>(column);
    const unsigned was[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned now = TokenMask(i, lo, hi);
      const unsigned before = grew ? TokenMask(i, 0, lo) : 0u;
      unsigned kept = was[i];
      if (before != 0u) kept = (kept & ~before) | (Rescale4<FMT>(kept, had, s) & before);
      w[i] = (w[i] & now) | (kept & ~now);
    }
  }
  *reinterpret_cast<uint4*>(column) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- the kernel ----------------------------------------------------------------
// Grid (pages' workgroups, groups of `per` key heads): 2 * per waves, wave w the
// keys (w even) or values of key head w / 2 of the group; then all of them the
// group's queries.  LDS: the sines of 16 tokens, then a 16 x dim tile per head.
constexpr int kMostPer = 4;

// Rotates the queries of offsets [c0 + lo, c0 + hi), heads [h0, h1).
template <typename T>
__device__ __forceinline__ void Queries(const Kv8AppendArgs& a, bool vec, const Task& t, int h0,
                                        int h1, int c0, int lo, int hi, const double2* cs) {
  const int units = a.c.dim / 16, row_heads = h1 - h0, turning = a.rot.pairs / 8;
  const int per_step = blockDim.x / units;
  const int mine = threadIdx.x / units, u = threadIdx.x - mine * units;
  if (mine >= per_step) return;
  const Unit w = UnitOf(u, a.rot);
  for (int i = mine; i < (hi - lo) * row_heads; i += per_step) {
    const int k = i / row_heads;
    const int o = lo + k;
    const int64_t head = static_cast<int64_t>(h0 + i - k * row_heads) * a.c.dim;
    const int64_t at = t.row + c0 + o;
    const T* p = static_cast<const T*>(a.q) + at * a.q_stride + head;
    T* out = static_cast<T*>(a.q_out) + at * a.out_stride + head;
    float x[16];
    double y[16];
    Load8(p + w.a, vec, x);
    Load8(p + w.b, vec, x + 8);
    Turn(x, cs + SineAt(o, 0, u, turning), turning, w, a.rot.interleaved, y);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = static_cast<float>(y[e]);
    Store8(out + w.a, vec, x);
    Store8(out + w.b, vec, x + 8);
  }
}

// What a wave's side of a page starts from and ends with.
struct Side {
  uint8_t* codes = nullptr;  // the page's, of its head
  float* scale = nullptr;
  float had = 0.0f;
};

// A chunk's new offsets within it.
struct Part {
  int c0 = 0, lo = 0, hi = 0;
};
__device__ __forceinline__ Part PartOf(const Task& t, int c) {
  Part p;
  p.c0 = 16 * c;
  p.lo = min(max(t.first - p.c0, 0), 16);
  p.hi = min(t.end - p.c0, 16);
  return p;
}

// The workgroup's barriers: both sides pass the same ones.  Before pass 1's
// chunk c its sines replace the chunk's before; pass 2 forms them again unless
// the new tokens lie in one chunk.
__device__ __forceinline__ void NextSines(const Kv8AppendArgs& a, const Task& t, const Part& p,
                                          double2* cs) {
  __syncthreads();
  FillSines(a, t, p.c0, p.lo, p.hi, cs);
  __syncthreads();
}

// The largest new number first, then the codes.  New tokens of one chunk stay
// in registers between the two; of several they are read again, from the cache.
template <typename T, int FMT, int NU>
__device__ __forceinline__ void KeySide(const Kv8AppendArgs& a, bool vec, const Task& t, int h0,
                                        int h1, int h, const Side& side, double2* cs,
                                        uint8_t* tile) {
  constexpr int NV = (NU + 1) / 2;
  const int group = a.q_heads / a.c.heads, lane = threadIdx.x & (kWave - 1);
  const int chunk0 = t.first / 16, chunk1 = (t.end - 1) / 16;
  const bool mine = h < h1;
  float x[NU][16];
  float most = 0.0f;
  for (int c = chunk0; c <= chunk1; ++c) {
    const Part p = PartOf(t, c);
    if (mine) LoadKeys<T, NU>(a, vec, t, h, p.c0, p.lo, p.hi, x);
    NextSines(a, t, p, cs);
    if (mine) most = fmaxf(most, LargestKey<NU>(a, p.lo, p.hi, cs, x));
    if (group > 0) Queries<T>(a, vec, t, h0 * group, h1 * group, p.c0, p.lo, p.hi, cs);
  }
  Scale s;
  s.Set<FMT>(fmaxf(side.had, ScaleFor<FMT>(WaveMax(most))));
  const bool grew = t.first > 0 && s.s > side.had;
  const bool means = a.c.summaries != nullptr;
  float sums[NV][2] = {};
  for (int c = 0; c <= chunk1; ++c) {
    const Part p = PartOf(t, c);
    if (chunk0 != chunk1 && p.lo < p.hi) {
      if (mine) LoadKeys<T, NU>(a, vec, t, h, p.c0, p.lo, p.hi, x);
      NextSines(a, t, p, cs);
    }
    if (mine && (p.lo < p.hi || grew || means)) {
      StoreKeys<FMT, NU>(a, side.codes + p.c0 * a.c.dim, p.lo, p.hi, side.had, grew, s, x, cs,
                         tile, sums);
    }
  }
  if (!mine) return;
  if (lane == 0) {
    *side.scale = s.s;
    if (h == 0) a.c.token_counts[t.page] = t.end;
  }
  if (means) {
    const double f = static_cast<double>(s.s);
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int d = 128 * m + 2 * lane;
      if (d < a.c.dim) {
        float* out =
            a.c.summaries + (static_cast<int64_t>(t.page) * a.c.heads + h) * a.c.dim + d;
        out[0] = static_cast<float>(static_cast<double>(sums[m][0]) * f / t.end);
        out[1] = static_cast<float>(static_cast<double>(sums[m][1]) * f / t.end);
      }
    }
  }
}

template <typename T, int FMT, int NU>
__device__ __forceinline__ void ValueSide(const Kv8AppendArgs& a, bool vec, const Task& t, int h0,
                                          int h1, int h, const Side& side, double2* cs) {
  constexpr int NV = (NU + 1) / 2;
  const int group = a.q_heads / a.c.heads, lane = threadIdx.x & (kWave - 1);
  const int chunk0 = t.first / 16, chunk1 = (t.end - 1) / 16;
  const bool mine = h < h1;
  float x[NV][2][16];
  float most = 0.0f;
  for (int c = chunk0; c <= chunk1; ++c) {
    const Part p = PartOf(t, c);
    if (mine) {
#pragma unroll
      for (int m = 0; m < NV; ++m) {
        LoadValues<T>(a, vec, t, h, p.c0, p.lo, p.hi, 128 * m + 2 * lane, x[m]);
      }
    }
    NextSines(a, t, p, cs);
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      if (mine) most = fmaxf(most, LargestValue(x[m]));
    }
    if (group > 0) Queries<T>(a, vec, t, h0 * group, h1 * group, p.c0, p.lo, p.hi, cs);
  }
  Scale s;
  s.Set<FMT>(fmaxf(side.had, ScaleFor<FMT>(WaveMax(most))));
  const bool grew = t.first > 0 && s.s > side.had;
  for (int c = grew ? 0 : chunk0; c <= chunk1; ++c) {
    const Part p = PartOf(t, c);
    if (chunk0 != chunk1 && p.lo < p.hi) NextSines(a, t, p, cs);
    if (!mine) continue;
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int d = 128 * m + 2 * lane;
      if (chunk0 != chunk1 && p.lo < p.hi) {
        LoadValues<T>(a, vec, t, h, p.c0, p.lo, p.hi, d, x[m]);
      }
      if (d < a.c.dim) {
        uint8_t* column = side.codes + p.c0 * a.c.dim + d * 16;
        StoreValues<FMT>(column, p.lo, p.hi, side.had, grew, s, x[m][0]);
        StoreValues<FMT>(column + 16, p.lo, p.hi, side.had, grew, s, x[m][1]);
      }
    }
  }
  if (mine && lane == 0) *side.scale = s.s;
}

template <typename T, int FMT, int NU>
__global__ __launch_bounds__(2 * kMostPer * kWave) void Kv8AppendKernel(Kv8AppendArgs a, int per,
                                                                        bool vec) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int wave = threadIdx.x / kWave;
  if (a.b.max_tokens > 1 && blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && wave == 0) {
    // (a malformed request may have no workgroup that looks at it)
    for (int r = threadIdx.x; r < a.b.batch; r += kWave) {
      Kv8Request q;
      if (!Kv8ReadTokens(a.b, r, a.c.page, &q)) ReportFailure(a.fail, kFailShape);
    }
  }
  Task t;
  if (!FindTask(a, blockIdx.x, &t)) return;
  const int heads = a.c.heads;
  const int h0 = blockIdx.y * per, h1 = min(h0 + per, heads);
  const int h = h0 + wave / 2;
  double2* cs = reinterpret_cast<double2*>(smem);
  const bool keys = (wave & 1) == 0;
  const int64_t page_head = static_cast<int64_t>(t.page) * heads + min(h, heads - 1);
  Side side;
  side.codes = (keys ? a.c.keys : a.c.values) + page_head * a.c.page * a.c.dim;
  side.scale = (keys ? a.c.key_scales : a.c.value_scales) + page_head;
  side.had = t.first > 0 ? *side.scale : 0.0f;
  if (keys) {
    uint8_t* tile = smem + sizeof(double2) * 16 * a.rot.pairs + wave / 2 * 16 * a.c.dim;
    KeySide<T, FMT, NU>(a, vec, t, h0, h1, h, side, cs, tile);
  } else {
    ValueSide<T, FMT, NU>(a, vec, t, h0, h1, h, side, cs);
  }
}

template <typename T, int FMT, int NU>
void Launch(const Kv8AppendArgs& a, bool vec, hipStream_t stream) {
  const int per = std::min(2, a.c.heads);
  const int64_t units = a.b.max_tokens > 1
                            ? a.b.tokens / a.c.page + 2 * static_cast<int64_t>(a.b.batch)
                            : a.b.batch;
  const size_t lds = sizeof(double2) * 16 * a.rot.pairs + per * 16 * a.c.dim;
  const dim3 grid(static_cast<unsigned>(units), (a.c.heads + per - 1) / per);
  Kv8AppendKernel<T, FMT, NU><<<grid, 2 * per * kWave, lds, stream>>>(a, per, vec);
  DSD_HIP_CHECK(hipGetLastError());
}

template <typename T, int FMT>
void LaunchDim(const Kv8AppendArgs& a, bool vec, hipStream_t stream) {
  if (a.c.dim <= 64) return Launch<T, FMT, 1>(a, vec, stream);
  if (a.c.dim <= 128) return Launch<T, FMT, 2>(a, vec, stream);
  return Launch<T, FMT, 4>(a, vec, stream);
}

template <typename T>
void LaunchType(const Kv8AppendArgs& a, hipStream_t stream) {
  // 16-byte accesses where every row starts on 16 bytes (its heads then do, dim
  // being a multiple of 16)
  constexpr int64_t step = 16 / sizeof(T);
  auto even = [&](const void* p, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % step == 0;
  };
  const bool vec = even(a.k, a.k_stride) && even(a.v, a.v_stride) &&
                   (a.q_heads == 0 || (even(a.q, a.q_stride) && even(a.q_out, a.out_stride)));
  a.c.format == DSD_KV8_INT8 ? LaunchDim<T, DSD_KV8_INT8>(a, vec, stream)
                             : LaunchDim<T, DSD_KV8_E4M3>(a, vec, stream);
}

template <typename T, int FMT>
void PreloadDim(const Kv8View& c) {
  if (c.dim <= 64) return PreloadKernel(Kv8AppendKernel<T, FMT, 1>);
  if (c.dim <= 128) return PreloadKernel(Kv8AppendKernel<T, FMT, 2>);
  return PreloadKernel(Kv8AppendKernel<T, FMT, 4>);
}

template <typename T>
void PreloadType(const Kv8View& c) {
  c.format == DSD_KV8_INT8 ? PreloadDim<T, DSD_KV8_INT8>(c) : PreloadDim<T, DSD_KV8_E4M3>(c);
}

}  // namespace

void PreloadKv8Append(const Kv8View& c) {
  PreloadType<float>(c);
  PreloadType<__bf16>(c);
  PreloadType<_Float16>(c);
}

void LaunchKv8Append(const Kv8AppendArgs& a, hipStream_t stream) {
  if (a.b.batch == 0 || a.b.tokens == 0) return;
  switch (a.type) {
    case DSD_TYPE_F32: return LaunchType<float>(a, stream);
    case DSD_TYPE_BF16: return LaunchType<__bf16>(a, stream);
    default: return LaunchType<_Float16>(a, stream);
  }
}

}  // namespace dsdk
