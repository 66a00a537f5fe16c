// kv8_append.hip -- dsd_kv8_append (gfx950): a batch's new tokens rotated,
// quantised and written behind what an 8-bit paged cache holds, and their
// queries rotated.
//
// Mathematics.  Pair (x, y) of a head turns by a = position * inv_freq:
// (x cos a - y sin a, y cos a + x sin a).  A position is its four bytes, so
// (cos a, sin a) is the product of four complex numbers out of a table of 4 x
// 256 a pair, in 64 bits (32-bit angles are off by whole hundredths of a radian
// at a million positions); the turns are 64-bit too: a key's code then falls on
// the right side of every rounding border.  (Forming sines in place cost 25
// registers, a quarter of the waves, and three times the instructions.)  The codes of a page share one scale s >= largest / M (M =
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

// Pair i of a unit whose elements are x[at..at + 8) at a, x[at + 8..at + 16) at
// b: its place from `at` on and its numbers turned.  cs: the unit's first pair, the others `step` apart.
// (The schedule is held to a pair at a time: left to interleave them the
// compiler takes twice the registers, half the waves a CU.)
struct Turned {
  int i0, i1;
  double y0, y1;
};
template <typename X>
__device__ __forceinline__ Turned TurnPair(const X& x, int at, int i, const double2* cs, int step,
                                           const Unit& u, bool interleaved) {
  Turned t;
  t.i0 = interleaved ? 2 * i : i;
  t.i1 = interleaved ? 2 * i + 1 : 8 + i;
  const double p = static_cast<double>(x[at + t.i0]);
  const double q = static_cast<double>(x[at + t.i1]);
  t.y0 = p;
  t.y1 = q;
  if (u.turns) {
    const double2 w = cs[i * step];
    t.y0 = p * w.x - q * w.y;
    t.y1 = q * w.x + p * w.y;
  }
  return t;
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
// c0 on (SineAt).
__device__ __forceinline__ double2 Times(double2 a, double2 b) {
  return {a.x * b.x - a.y * b.y, a.x * b.y + a.y * b.x};
}
__device__ __forceinline__ void FillSines(const Kv8AppendArgs& a, const Task& t, int c0, int lo,
                                          int hi, double2* cs) {
  const int pairs = a.rot.pairs;
  const int n = (hi - lo) * pairs;
  const double2* table = a.rot.table;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int k = i / pairs, p = i - k * pairs;
    const int o = c0 + lo + k;
    const int at = a.b.positions != nullptr ? a.b.positions[t.row + o] : t.index + o;
    const unsigned far = at < 0 ? 0u - static_cast<unsigned>(at) : static_cast<unsigned>(at);
    const double2 w = Times(Times(table[(far & 255u) * pairs + p],
                                  table[(256u + ((far >> 8) & 255u)) * pairs + p]),
                            Times(table[(512u + ((far >> 16) & 255u)) * pairs + p],
                                  table[(768u + (far >> 24)) * pairs + p]));
    const double s = at < 0 ? -w.y : w.y;
    cs[SineAt(lo + k, p & 7, p >> 3, pairs / 8)] = {w.x * a.rot.magnitude,
                                                  s * a.rot.magnitude};
  }
}

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

// A side's new numbers of one chunk in a lane's registers.  Keys: lane l has unit
// (l + 64 j) % units of token (l + 64 j) / units, j < NU = ceil(dim / 64), at
// x[16 j ..].  Values: dims 2 l, 2 l + 1 of the m-th 128, all 16 tokens, at
// x[32 m + 2 token ..].
template <typename T, int NU>
struct Numbers {
  static constexpr int kPlanes = (NU + 1) / 2;
  Packed<T, 32 * kPlanes> x;
};

template <typename T, int NU>
__device__ __forceinline__ void LoadKeys(const Kv8AppendArgs& a, bool vec, const Task& t, int h,
                                         const Part& p, Numbers<T, NU>* x) {
  const int lane = threadIdx.x & (kWave - 1);
  const int units = a.c.dim / 16;
  const T* k = static_cast<const T*>(a.k) + static_cast<int64_t>(h) * a.c.dim;
#pragma unroll
  for (int j = 0; j < NU; ++j) {
    const int i = lane + kWave * j;
    const int o = i / units, u = i - o * units;
    if (o >= p.lo && o < p.hi) {
      const Unit w = UnitOf(u, a.rot);
      const T* from = k + (t.row + p.c0 + o) * a.k_stride;
      x->x.Load8(16 * j, from + w.a, vec);
      x->x.Load8(16 * j + 8, from + w.b, vec);
    }
  }
}

template <typename T, int NU, bool kInterleaved>
__device__ __forceinline__ float LargestKey(const Kv8AppendArgs& a, const Part& p,
                                            const double2* cs, const Numbers<T, NU>& x) {
  const int lane = threadIdx.x & (kWave - 1);
  const int units = a.c.dim / 16, turning = a.rot.pairs / 8;
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < NU; ++j) {
    const int i = lane + kWave * j;
    const int o = i / units, u = i - o * units;
    if (o >= p.lo && o < p.hi) {
      const Unit w = UnitOf(u, a.rot);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Turned y = TurnPair(x.x, 16 * j, e, cs + SineAt(o, 0, u, turning), turning, w,
                                  kInterleaved);
        most = fmaxf(most, fmaxf(FiniteSize(static_cast<float>(y.y0)),
                                 FiniteSize(static_cast<float>(y.y1))));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  return most;
}

// One chunk's codes: offsets [lo, hi) new (x, turned again), those before them
// as they are or brought from `had` to s.  tile: 16 x dim bytes of LDS.  sums:
// the lane's dims 2 lane, 2 lane + 1 of each 128, summed over offsets [0, hi).
template <int FMT, typename T, int NU, bool kInterleaved>
__device__ __forceinline__ void StoreKeys(const Kv8AppendArgs& a, uint8_t* block, const Part& p,
                                          float had, bool grew, const Scale& s,
                                          const Numbers<T, NU>& x, const double2* cs,
                                          uint8_t* tile, float (&sums)[(NU + 1) / 2][2]) {
  const int lane = threadIdx.x & (kWave - 1);
  const int D = a.c.dim;
  const int units = D / 16, turning = a.rot.pairs / 8;
  const int lo = p.lo, hi = p.hi;
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
      // four pairs at a time: two words of codes
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        double y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const Turned z = TurnPair(x.x, 16 * j, e + k, cs + SineAt(o, 0, u, turning), turning, w,
                                    kInterleaved);
          y[kInterleaved ? 2 * k : k] = z.y0;
          y[kInterleaved ? 2 * k + 1 : 4 + k] = z.y1;
        }
        const unsigned c0 = Codes4<FMT>(y[0], y[1], y[2], y[3], s);
        const unsigned c1 = Codes4<FMT>(y[4], y[5], y[6], y[7], s);
        // interleaved: elements 2 e .. 2 e + 8; else e .. e + 4 of both parts
        uint8_t* to = tile + o * D;
        if constexpr (kInterleaved) {
          *reinterpret_cast<uint2*>(to + (e == 0 ? w.a : w.b)) = make_uint2(c0, c1);
        } else {
          *reinterpret_cast<unsigned*>(to + w.a + e) = c0;
          *reinterpret_cast<unsigned*>(to + w.b + e) = c1;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
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
          float v[4];
          Numbers4<FMT>(*reinterpret_cast<const uint16_t*>(tile + o * D + d), v);
          sums[m][0] += v[0];
          sums[m][1] += v[1];
        }
      }
    }
  }
  WaveLdsFence();
}

template <typename T, int NU>
__device__ __forceinline__ void LoadValues(const Kv8AppendArgs& a, bool vec, const Task& t, int h,
                                           const Part& p, Numbers<T, NU>* x) {
  const int lane = threadIdx.x & (kWave - 1);
  constexpr int kWords = sizeof(T) / 2;  // of two elements
#pragma unroll
  for (int m = 0; m < Numbers<T, NU>::kPlanes; ++m) {
    const int d = 128 * m + 2 * lane;
    const T* v = static_cast<const T*>(a.v) + static_cast<int64_t>(h) * a.c.dim + d;
#pragma unroll
    for (int o = 0; o < 16; ++o) {
      unsigned* to = x->x.w + (16 * m + o) * kWords;
#pragma unroll
      for (int k = 0; k < kWords; ++k) to[k] = 0u;
      if (o >= p.lo && o < p.hi && d < a.c.dim) {
        const T* from = v + (t.row + p.c0 + o) * a.v_stride;
        if (vec || sizeof(T) == 4) {
#pragma unroll
          for (int k = 0; k < kWords; ++k) to[k] = reinterpret_cast<const unsigned*>(from)[k];
        } else {
          const uint16_t* half = reinterpret_cast<const uint16_t*>(from);
          to[0] = half[0] | static_cast<unsigned>(half[1]) << 16;
        }
      }
    }
  }
}

template <typename T, int NU>
__device__ __forceinline__ float LargestValue(const Numbers<T, NU>& x) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 32 * Numbers<T, NU>::kPlanes; ++i) {
    most = fmaxf(most, FiniteSize(x.x[i]));
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

// column: the 16 codes of one dim, token t's number x[at + 2 t].  Tokens outside
// [0, hi) stay as they are.
template <int FMT, typename X>
__device__ __forceinline__ void StoreValues(uint8_t* column, int lo, int hi, float had, bool grew,
                                            const Scale& s, const X& x, int at) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = 0u;
    if (lo < hi) {
      w[i] = Codes4<FMT>(x[at + 8 * i], x[at + 8 * i + 2], x[at + 8 * i + 4], x[at + 8 * i + 6], s);
    }
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

// Rotates the queries of a chunk's new tokens, heads [h0, h1).
template <typename T, bool kInterleaved>
__device__ __forceinline__ void Queries(const Kv8AppendArgs& a, bool vec, const Task& t, int h0,
                                        int h1, const Part& p, const double2* cs) {
  const int units = a.c.dim / 16, row_heads = h1 - h0, turning = a.rot.pairs / 8;
  const int per_step = blockDim.x / units;
  const int mine = threadIdx.x / units, u = threadIdx.x - mine * units;
  if (mine >= per_step) return;
  const Unit w = UnitOf(u, a.rot);
  for (int i = mine; i < (p.hi - p.lo) * row_heads; i += per_step) {
    const int k = i / row_heads;
    const int o = p.lo + k;
    const int64_t head = static_cast<int64_t>(h0 + i - k * row_heads) * a.c.dim;
    const int64_t at = t.row + p.c0 + o;
    const T* from = static_cast<const T*>(a.q) + at * a.q_stride + head;
    T* out = static_cast<T*>(a.q_out) + at * a.out_stride + head;
    Packed<T, 16> x;
    x.Load8(0, from + w.a, vec);
    x.Load8(8, from + w.b, vec);
    // two pairs at a time: whole words of results
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const double2* at_cs = cs + SineAt(o, 0, u, turning);
      const Turned y = TurnPair(x, 0, e, at_cs, turning, w, kInterleaved);
      const Turned z = TurnPair(x, 0, e + 1, at_cs, turning, w, kInterleaved);
      if constexpr (kInterleaved) {
        x.Set2(y.i0, static_cast<float>(y.y0), static_cast<float>(y.y1));
        x.Set2(z.i0, static_cast<float>(z.y0), static_cast<float>(z.y1));
      } else {
        x.Set2(y.i0, static_cast<float>(y.y0), static_cast<float>(z.y0));
        x.Set2(y.i1, static_cast<float>(y.y1), static_cast<float>(z.y1));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    x.Store8(0, out + w.a, vec);
    x.Store8(8, out + w.b, vec);
  }
}

template <typename T, int FMT, int NU, bool kInterleaved>
__global__ __launch_bounds__(2 * kMostPer * kWave) void Kv8AppendKernel(Kv8AppendArgs a, int per,
                                                                        bool vec) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  if (a.b.max_tokens > 1 && blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && wave == 0) {
    // (a malformed request may have no workgroup that looks at it)
    for (int r = threadIdx.x; r < a.b.batch; r += kWave) {
      Kv8Request q;
      if (!Kv8ReadTokens(a.b, r, a.c.page, &q)) ReportFailure(a.fail, kFailShape);
    }
  }
  Task t;
  if (!FindTask(a, blockIdx.x, &t)) return;
  constexpr int NV = Numbers<T, NU>::kPlanes;
  const int heads = a.c.heads, D = a.c.dim, group = a.q_heads / heads;
  const int h0 = blockIdx.y * per, h1 = min(h0 + per, heads);
  const int h = h0 + wave / 2;
  const bool mine = h < h1, keys = (wave & 1) == 0;
  double2* cs = reinterpret_cast<double2*>(smem);
  uint8_t* tile = smem + sizeof(double2) * 16 * a.rot.pairs + wave / 2 * 16 * D;
  const int64_t page_head = static_cast<int64_t>(t.page) * heads + min(h, heads - 1);
  uint8_t* codes = (keys ? a.c.keys : a.c.values) + page_head * a.c.page * D;
  float* scale = (keys ? a.c.key_scales : a.c.value_scales) + page_head;
  const float had = t.first > 0 ? *scale : 0.0f;
  const bool means = keys && a.c.summaries != nullptr;
  const int chunk0 = t.first / 16, chunk1 = (t.end - 1) / 16;
  const bool one = chunk0 == chunk1;

  // First the largest new number, then the codes.  New tokens of one chunk stay
  // in registers between the two; of several they are read again, from the
  // cache, and their sines formed again.
  Numbers<T, NU> x;
  float most = 0.0f;
  float sums[NV][2] = {};
  Scale s;
  bool grew = false;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) {
      s.template Set<FMT>(fmaxf(had, ScaleFor<FMT>(WaveMax(most))));
      grew = t.first > 0 && s.s > had;
    }
#pragma unroll 1
    for (int c = pass == 1 && (grew || means) ? 0 : chunk0; c <= chunk1; ++c) {
      const Part p = PartOf(t, c);
      if (p.lo < p.hi && (pass == 0 || !one)) {
        if (mine && keys) {
          LoadKeys<T, NU>(a, vec, t, h, p, &x);
        } else if (mine) {
          LoadValues<T, NU>(a, vec, t, h, p, &x);
        }
        __syncthreads();
        FillSines(a, t, p.c0, p.lo, p.hi, cs);
        __syncthreads();
      }
      if (pass == 0) {
        if (mine) {
          most = fmaxf(most, keys ? LargestKey<T, NU, kInterleaved>(a, p, cs, x)
                                  : LargestValue<T, NU>(x));
        }
        if (group > 0) {
          Queries<T, kInterleaved>(a, vec, t, h0 * group, h1 * group, p, cs);
        }
      } else if (mine && keys) {
        StoreKeys<FMT, T, NU, kInterleaved>(a, codes + p.c0 * D, p, had, grew, s, x, cs, tile,
                                            sums);
      } else if (mine) {
#pragma unroll
        for (int m = 0; m < NV; ++m) {
          const int d = 128 * m + 2 * lane;
          if (d < D) {
            uint8_t* column = codes + p.c0 * D + d * 16;
            StoreValues<FMT>(column, p.lo, p.hi, had, grew, s, x.x, 32 * m);
            StoreValues<FMT>(column + 16, p.lo, p.hi, had, grew, s, x.x, 32 * m + 1);
          }
        }
      }
    }
  }
  if (!mine) return;
  if (lane == 0) {
    *scale = s.s;
    if (h == 0 && keys) a.c.token_counts[t.page] = t.end;
  }
  if (means) {
    const double f = static_cast<double>(s.s);
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int d = 128 * m + 2 * lane;
      if (d < D) {
        float* out = a.c.summaries + page_head * D + d;
        out[0] = static_cast<float>(static_cast<double>(sums[m][0]) * f / t.end);
        out[1] = static_cast<float>(static_cast<double>(sums[m][1]) * f / t.end);
      }
    }
  }
}

// Calls f with the kernel of a head size.
template <typename T, int FMT, bool kInterleaved, typename F>
void WithDim(int dim, F&& f) {
  if (dim <= 64) return f(Kv8AppendKernel<T, FMT, 1, kInterleaved>);
  if (dim <= 128) return f(Kv8AppendKernel<T, FMT, 2, kInterleaved>);
  return f(Kv8AppendKernel<T, FMT, 4, kInterleaved>);
}
template <typename T, typename F>
void WithKernel(int format, int dim, bool interleaved, F&& f) {
  if (format == DSD_KV8_INT8) {
    interleaved ? WithDim<T, DSD_KV8_INT8, true>(dim, f) : WithDim<T, DSD_KV8_INT8, false>(dim, f);
  } else {
    interleaved ? WithDim<T, DSD_KV8_E4M3, true>(dim, f) : WithDim<T, DSD_KV8_E4M3, false>(dim, f);
  }
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
  const int per = std::min(2, a.c.heads);
  const int64_t units = a.b.max_tokens > 1
                            ? a.b.tokens / a.c.page + 2 * static_cast<int64_t>(a.b.batch)
                            : a.b.batch;
  const size_t lds = sizeof(double2) * 16 * a.rot.pairs + per * 16 * a.c.dim;
  const dim3 grid(static_cast<unsigned>(units), (a.c.heads + per - 1) / per);
  WithKernel<T>(a.c.format, a.c.dim, a.rot.interleaved != 0, [&](auto kernel) {
    kernel<<<grid, 2 * per * kWave, lds, stream>>>(a, per, vec);
  });
  DSD_HIP_CHECK(hipGetLastError());
}

template <typename T>
void PreloadType(const Kv8View& c) {
  for (bool interleaved : {false, true}) {
    WithKernel<T>(c.format, c.dim, interleaved, [](auto kernel) { PreloadKernel(kernel); });
  }
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
