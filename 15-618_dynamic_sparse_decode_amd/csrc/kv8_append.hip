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
// registers, a quarter of the waves, and three times the instructions.)  The
// codes of a page share one scale s >= largest / M (M = 448 or 127), so a token
// that needs a larger one takes the page's earlier codes with it: code <-
// nearest(code * old / s).
//
// Bound by HBM: queries, keys and values are read once, rotated queries and
// codes written once.  A workgroup takes one page's new tokens of some key
// heads and of the query heads that read them, so an angle's sine and cosine
// are formed once for all of these.  Within it a wave takes one side (keys or
// values) of one head at a time.
//
// Measured (kernel times): 8192 tokens of 32 bf16 query and 8 key heads of 128,
// pages of 16, 40-41 us for 186 MB, 4.6 TB/s (a large copy reaches 4.7); int8 49.
// Float32, 32 heads of each, 16 prompts of 100-1500 tokens in pages of 64: 310 us
// for 0.98 GB (int8 436, which turns each key twice); the 64-bit turns take a third of the vector units' time, and of the
// waits most are for a page's largest number, with four waves a SIMD (the sines of
// 64 tokens fill LDS).  Pages of 128, the prompt of 8192: 105 us, int8 125.  One
// token: 7.2 us, 64 of them 8.2, a chain of offsets ->
// ids -> scales -> codes after the launch.  Tried on the way: two heads of 16
// waves in place of one of 8 in pages of 64 (374 us against 331), a loop over a
// page's chunks in that kernel (spills), the first queries asked for before the
// codes are written (no gain).
#include "kv8_device.h"

#include <algorithm>
#include <stdexcept>

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
  const unsigned bits = __float_as_uint(y) - (fabs(back) > fabs(x) ? 1u : 0u);
  return __uint_as_float(bits | (back != x && x == x ? 1u : 0u));
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

// The same of finite numbers and a power of two, by the conversion's own scale.
__device__ __forceinline__ unsigned PlainCodes4(float x0, float x1, float x2, float x3, float s) {
  typedef short S2 __attribute__((ext_vector_type(2)));
  S2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x0, x1, s, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x2, x3, s, true);
  return __builtin_bit_cast(unsigned, w);
}
// Of four tokens' words of two 16-bit numbers each, their first or second ones.
template <typename T>
__device__ __forceinline__ unsigned PlainCodes4(unsigned w0, unsigned w1, unsigned w2, unsigned w3,
                                                bool second, float s) {
  typedef short S2 __attribute__((ext_vector_type(2)));
  typedef T T2 __attribute__((ext_vector_type(2)));
  const unsigned take = second ? 0x07060302u : 0x05040100u;
  const T2 a = __builtin_bit_cast(T2, __builtin_amdgcn_perm(w1, w0, take));
  const T2 b = __builtin_bit_cast(T2, __builtin_amdgcn_perm(w3, w2, take));
  S2 w = {0, 0};
  if constexpr (std::is_same<T, __bf16>::value) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, a, s, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, b, s, true);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, a, s, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, b, s, true);
  }
  return __builtin_bit_cast(unsigned, w);
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

// The sines in LDS: (cos, sin) of token o's pair 8 u + i at [o][i ^ o % 4][u], so
// that the lanes of a row, one unit each, read next to each other, and the rows
// beside them other banks.
__device__ __forceinline__ int SineAt(int o, int i, int u, int turning) {
  return (o * 8 + (i ^ (o & 3))) * turning + u;
}

// Pair i of a unit whose elements are x[at..at + 8) at a, x[at + 8..at + 16) at
// b: its place from `at` on and its numbers turned.  cs: token o's pairs of the
// unit, `step` apart.
struct Turned {
  int i0, i1;
  double y0, y1;
};
template <typename X>
__device__ __forceinline__ Turned TurnPair(const X& x, int at, int i, const double2* cs, int step,
                                           int o, bool interleaved) {
  Turned t;
  t.i0 = interleaved ? 2 * i : i;
  t.i1 = interleaved ? 2 * i + 1 : 8 + i;
  const double p = static_cast<double>(x[at + t.i0]);
  const double q = static_cast<double>(x[at + t.i1]);
  const double2 w = cs[(i ^ (o & 3)) * step];
  t.y0 = fma(p, w.x, -(q * w.y));
  t.y1 = fma(q, w.x, p * w.y);
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

// The last request whose workgroups start no later than u, of those whose offsets
// are in order (-1: none).
__device__ __forceinline__ int RequestInOrder(const dsd_kv8_batch& b, int ps, int u) {
  const int lane = threadIdx.x & (kWave - 1);
  int r = -1;
  for (int b0 = 0; b0 < b.batch; b0 += kWave) {
    const int i = b0 + lane;
    bool mine = false;
    if (i < b.batch) {
      const int row = b.token_offsets[i], end = b.token_offsets[i + 1];
      mine = row >= 0 && end >= row && end <= b.tokens && end - row <= b.max_tokens &&
             row / ps + 2 * i <= u;
    }
    const unsigned long long ours = __ballot(mine);
    if (ours != 0) r = b0 + kWave - 1 - __builtin_clzll(ours);
  }
  return r;
}

// The task of workgroup u: request r's pages take workgroups from
// floor(token_offsets[r] / page) + 2 r on, at least as many as its tokens can
// touch (one each where every request has one token).  Every wave computes
// the same.
__device__ __forceinline__ bool FindTask(const Kv8AppendArgs& a, int u, Task* t) {
  const dsd_kv8_batch& b = a.b;
  const int ps = a.c.page;
  int r = u, within = 0;
  Kv8Request q;
  bool ok = false;
  if (b.max_tokens > 1) {
    const int lane = threadIdx.x & (kWave - 1);
    int below = 0;
    bool in_order = true;
    for (int b0 = 0; b0 < b.batch; b0 += kWave) {
      const int i = b0 + lane;
      bool mine = false;
      if (i < b.batch) mine = b.token_offsets[i] / ps + 2 * i <= u;
      const unsigned long long ours = __ballot(mine);
      in_order = in_order && (ours & (ours + 1)) == 0;
      const int got = __popcll(ours);
      below += got;
      if (got < kWave) break;
    }
    r = below - 1;
    if (r >= 0) ok = Kv8ReadTokens(b, r, ps, &q);
    // An offset out of order hides the requests behind it, or those before it: the
    // one it belongs to is skipped, the others are not.
    if (!in_order || (r >= 0 && !ok)) {
      r = RequestInOrder(b, ps, u);
      if (r >= 0) ok = Kv8ReadTokens(b, r, ps, &q);
    }
    if (r < 0) return false;
    within = u - (b.token_offsets[r] / ps + 2 * r);
    if (within < 0) return false;
  } else {
    if (r >= b.batch) return false;
    ok = Kv8ReadTokens(b, r, ps, &q);
  }
  if (!ok) {
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailShape);
    return false;
  }
  if (q.n == 0) return false;
  const int slot0 = q.past / ps, last = (q.past + q.n - 1) / ps;
  const int slot = slot0 + within;
  if (slot > last) return false;
  t->page = b.page_ids[q.list + slot];  // (checked where it is used)
  t->index = slot * ps;
  t->first = max(q.past - t->index, 0);
  t->end = min(q.past + q.n - t->index, ps);
  t->row = q.row0 + t->index - q.past;
  return true;
}

// The sines and cosines of the tokens at offsets [lo, hi) from c0 on (SineAt).
__device__ __forceinline__ double2 Times(double2 a, double2 b) {
  return {fma(a.x, b.x, -(a.y * b.y)), fma(a.x, b.y, a.y * b.x)};
}
__device__ __forceinline__ void FillSines(const Kv8AppendArgs& a, const Task& t, int c0, int lo,
                                          int hi, double2* cs) {
  const int pairs = a.rot.pairs;
  if (pairs == 0) return;
  // A thread has one pair of every `step`-th token.
  const int step = max(static_cast<int>(blockDim.x) / pairs, 1);
  const int k = threadIdx.x / pairs, p = threadIdx.x - k * pairs;
  if (k >= step) return;
  const double2* table = a.rot.table + p;
  double2 high = {1.0, 0.0};
  unsigned known = 0xffffffffu;  // whose upper bytes `high` is of
  // (four tokens' entries on their way at once: the tables are in L2)
  constexpr int kAhead = 4;
  for (int o0 = lo + k; o0 < hi; o0 += kAhead * step) {
    int at[kAhead];
    double2 low[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int o = c0 + min(o0 + i * step, hi - 1);
      at[i] = a.b.positions != nullptr ? a.b.positions[t.row + o] : t.index + o;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const unsigned far = at[i] < 0 ? 0u - static_cast<unsigned>(at[i]) : static_cast<unsigned>(at[i]);
      low[i] = table[(far & 255u) * pairs];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int o = o0 + i * step;
      if (o >= hi) break;
      const unsigned far = at[i] < 0 ? 0u - static_cast<unsigned>(at[i]) : static_cast<unsigned>(at[i]);
      if (far >> 8 != known) {
        known = far >> 8;
        high = Times(Times(table[(256u + ((far >> 8) & 255u)) * pairs],
                           table[(512u + ((far >> 16) & 255u)) * pairs]),
                     table[(768u + (far >> 24)) * pairs]);
        high = {high.x * a.rot.magnitude, high.y * a.rot.magnitude};
      }
      const double2 w = Times(low[i], high);
      cs[SineAt(o, p & 7, p >> 3, pairs / 8)] = {w.x, at[i] < 0 ? -w.y : w.y};
    }
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

constexpr unsigned kInfinity = 0x7f800000u;

// The keys turned; returns the bits of the largest magnitude.  e4m3: into y, to
// which they are rounded so that a code of y is the code of the key itself.
// int8 keeps the numbers it was given and turns them again for their codes (and
// leaves out what is not finite here).
template <int FMT, typename T, int NU, bool kInterleaved>
__device__ __forceinline__ unsigned TurnKeys(const Kv8AppendArgs& a, const Part& p,
                                             const double2* cs, const Numbers<T, NU>& x,
                                             float (&y)[16 * NU]) {
  unsigned top = 0;
  const int lane = threadIdx.x & (kWave - 1);
  const int units = a.c.dim / 16, turning = a.rot.pairs / 8;
#pragma unroll
  for (int j = 0; j < NU; ++j) {
    const int i = lane + kWave * j;
    const int o = i / units, u = i - o * units;
    if (o >= p.lo && o < p.hi) {
      if (u < turning) {
        const double2* at = cs + (o * 8 * turning + u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Turned z = TurnPair(x.x, 16 * j, e, at, turning, o, kInterleaved);
          if constexpr (FMT == DSD_KV8_E4M3) {
            y[16 * j + z.i0] = ToOdd(z.y0);
            y[16 * j + z.i1] = ToOdd(z.y1);
          } else {
            top = max(top, max(__float_as_uint(FiniteSize(static_cast<float>(z.y0))),
                               __float_as_uint(FiniteSize(static_cast<float>(z.y1)))));
          }
          // (two pairs at a time: all of them at once take twice the registers)
          if (e & 1) __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          y[16 * j + e] = x.x[16 * j + e];
          if (FMT != DSD_KV8_E4M3) top = max(top, __float_as_uint(FiniteSize(y[16 * j + e])));
        }
      }
    } else if (FMT == DSD_KV8_E4M3) {
#pragma unroll
      for (int e = 0; e < 16; ++e) y[16 * j + e] = 0.0f;
    }
  }
  if constexpr (FMT == DSD_KV8_E4M3) {
#pragma unroll
    for (int e = 0; e < 16 * NU; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
  }
  return top;
}

// The bits of the largest finite magnitude.
template <int N, typename X>
__device__ __forceinline__ unsigned TopFinite(const X& x) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) most = fmaxf(most, FiniteSize(x[i]));
  return __float_as_uint(most);
}

// One chunk's codes: offsets [lo, hi) new (y, or x turned again), those before
// them as they are or brought from `had` to s.  plain: every new number is finite
// and s a power of two.  tile: 16 x dim bytes of LDS.  sums: the lane's dims 2
// lane, 2 lane + 1 of each 128, summed over offsets [0, hi).
template <int FMT, typename T, int NU, bool kInterleaved>
__device__ __forceinline__ void StoreKeys(const Kv8AppendArgs& a, uint8_t* block, const Part& p,
                                          float had, bool grew, const Scale& s, bool plain,
                                          const Numbers<T, NU>& x, const float (&y)[16 * NU],
                                          const double2* cs, uint8_t* tile,
                                          float (&sums)[(NU + 1) / 2][2]) {
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
      uint8_t* to = tile + o * D;
      unsigned c[4];
      if constexpr (FMT == DSD_KV8_E4M3) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = 16 * j + 4 * e;
          c[e] = plain ? PlainCodes4(y[k], y[k + 1], y[k + 2], y[k + 3], s.s)
                       : Codes4<FMT>(y[k], y[k + 1], y[k + 2], y[k + 3], s);
        }
      } else {
        // four pairs at a time: two words of codes
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          double z[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            Turned t;
            if (u < turning) {
              t = TurnPair(x.x, 16 * j, e + k, cs + (o * 8 * turning + u), turning, o,
                           kInterleaved);
            } else {
              t.y0 = static_cast<double>(x.x[16 * j + (kInterleaved ? 2 * (e + k) : e + k)]);
              t.y1 = static_cast<double>(x.x[16 * j + (kInterleaved ? 2 * (e + k) + 1 : 8 + e + k)]);
            }
            z[kInterleaved ? 2 * k : k] = t.y0;
            z[kInterleaved ? 2 * k + 1 : 4 + k] = t.y1;
          }
          // interleaved: elements 2 e .. 2 e + 8; else e .. e + 4 of both parts
          c[kInterleaved ? e / 2 : e / 4] = Codes4<FMT>(z[0], z[1], z[2], z[3], s);
          c[kInterleaved ? e / 2 + 1 : 2 + e / 4] = Codes4<FMT>(z[4], z[5], z[6], z[7], s);
          __builtin_amdgcn_sched_barrier(0);  // (or all of it is live at once)
        }
      }
      *reinterpret_cast<uint2*>(to + w.a) = make_uint2(c[0], c[1]);
      *reinterpret_cast<uint2*>(to + w.b) = make_uint2(c[2], c[3]);
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
#pragma unroll 4
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

// The bits of the largest magnitude.
template <typename T, int NU>
__device__ __forceinline__ unsigned TopValue(const Numbers<T, NU>& x) {
  constexpr int kWords = 32 * Numbers<T, NU>::kPlanes * sizeof(T) / 4;
  if constexpr (sizeof(T) == 4) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) top = max(top, x.x.w[i] & 0x7fffffffu);
    return top;
  } else {
    typedef uint16_t U2 __attribute__((ext_vector_type(2)));
    U2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      top = __builtin_elementwise_max(top, __builtin_bit_cast(U2, x.x.w[i] & 0x7fff7fffu));
    }
    Packed<T, 2> most;
    most.w[0] = max(top[0], top[1]);
    return __float_as_uint(most[0]);
  }
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
template <int FMT, typename T, typename X>
__device__ __forceinline__ void StoreValues(uint8_t* column, int lo, int hi, float had, bool grew,
                                            const Scale& s, bool plain, const X& x, int at) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = at + 8 * i;
    w[i] = 0u;
    if (lo < hi) {
      if (FMT == DSD_KV8_E4M3 && plain) {
        if constexpr (std::is_same<T, float>::value) {
          w[i] = PlainCodes4(x[k], x[k + 2], x[k + 4], x[k + 6], s.s);
        } else {
          const int b = k >> 1;
          w[i] = PlainCodes4<T>(x.w[b], x.w[b + 1], x.w[b + 2], x.w[b + 3], (at & 1) != 0, s.s);
        }
      } else {
        w[i] = Codes4<FMT>(x[k], x[k + 2], x[k + 4], x[k + 6], s);
      }
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

// ---- the kernels ---------------------------------------------------------------

// Rotates the queries of the new tokens [p.lo, p.hi) from p.c0 on, heads [h0, h1).
template <typename T, bool kInterleaved>
__device__ __forceinline__ void Queries(const Kv8AppendArgs& a, bool vec, const Task& t, int h0,
                                        int h1, const Part& p, const double2* cs) {
  const int units = a.c.dim / 16, row_heads = h1 - h0, turning = a.rot.pairs / 8;
  const int per_step = blockDim.x / units;
  const int mine = threadIdx.x / units, u = threadIdx.x - mine * units;
  if (mine >= per_step) return;
  const Unit w = UnitOf(u, a.rot);
  const unsigned inverse = 0xffffffffu / static_cast<unsigned>(row_heads) + 1u;
  // The next row's numbers are asked for before this one's are turned.
  const int end = (p.hi - p.lo) * row_heads;
  Packed<T, 16> next;
  int next_o = 0;
  T* next_out = nullptr;
  auto load = [&](int i) {
    const int k = row_heads == 1 ? i : static_cast<int>(__umulhi(i, inverse));
    next_o = p.lo + k;
    const int64_t head = static_cast<int64_t>(h0 + i - k * row_heads) * a.c.dim;
    const int64_t at = t.row + p.c0 + next_o;
    const T* from = static_cast<const T*>(a.q) + at * a.q_stride + head;
    next_out = static_cast<T*>(a.q_out) + at * a.out_stride + head;
    next.Load8(0, from + w.a, vec);
    next.Load8(8, from + w.b, vec);
  };
  if (mine < end) load(mine);
  for (int i = mine; i < end; i += per_step) {
    Packed<T, 16> x = next;
    const int o = next_o;
    T* out = next_out;
    if (i + per_step < end) load(i + per_step);
    // two pairs at a time: whole words of results
    if (u < turning) {
      const double2* at_cs = cs + (o * 8 * turning + u);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const Turned y = TurnPair(x, 0, e, at_cs, turning, o, kInterleaved);
        const Turned z = TurnPair(x, 0, e + 1, at_cs, turning, o, kInterleaved);
        if constexpr (kInterleaved) {
          x.Set2(y.i0, static_cast<float>(y.y0), static_cast<float>(y.y1));
          x.Set2(z.i0, static_cast<float>(z.y0), static_cast<float>(z.y1));
        } else {
          x.Set2(y.i0, static_cast<float>(y.y0), static_cast<float>(z.y0));
          x.Set2(y.i1, static_cast<float>(y.y1), static_cast<float>(z.y1));
        }
        if (e & 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
    x.Store8(0, out + w.a, vec);
    x.Store8(8, out + w.b, vec);
  }
}

// A malformed request may have no workgroup that looks at it: the last one does.
__device__ __forceinline__ void CheckRequests(const Kv8AppendArgs& a) {
  if (a.b.max_tokens > 1 && blockIdx.x == gridDim.x - 1 && threadIdx.x < kWave) {
    for (int r = threadIdx.x; r < a.b.batch; r += kWave) {
      Kv8Request q;
      if (!Kv8ReadTokens(a.b, r, a.c.page, &q)) ReportFailure(a.fail, kFailShape);
    }
  }
}

__device__ __forceinline__ unsigned WaveTop(unsigned x) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    x = max(x, static_cast<unsigned>(__shfl_xor(static_cast<int>(x), o, kWave)));
  }
  return x;
}

// What a wave does with its side of a head, a chunk at a time.
template <typename T, int FMT, int NU, bool kInterleaved>
struct Lane {
  static constexpr int NV = Numbers<T, NU>::kPlanes;
  Numbers<T, NU> x;
  float y[16 * NU];      // keys turned (e4m3)
  float sums[NV][2] = {};
  float had = 0.0f;      // the page's scale so far (0: none)
  Scale s;               // and from now on
  bool grew = false;
  bool plain = true;     // PlainCodes4 will do

  __device__ __forceinline__ void Load(const Kv8AppendArgs& a, bool vec, const Task& t, bool keys,
                                       int h, const Part& p) {
    if (keys) {
      LoadKeys<T, NU>(a, vec, t, h, p, &x);
    } else {
      LoadValues<T, NU>(a, vec, t, h, p, &x);
    }
  }
  // The bits of the largest finite magnitude.
  __device__ __forceinline__ unsigned Top(const Kv8AppendArgs& a, bool keys, const Part& p,
                                          const double2* cs) {
    unsigned top = keys ? TurnKeys<FMT, T, NU, kInterleaved>(a, p, cs, x, y) : TopValue<T, NU>(x);
    if (__ballot(top >= kInfinity) != 0) {  // seldom
      plain = false;
      top = keys ? TopFinite<16 * NU>(y) : TopFinite<32 * NV>(x.x);
    }
    return top;
  }
  __device__ __forceinline__ void SetScale(const Task& t, unsigned top) {
    s.template Set<FMT>(fmaxf(had, ScaleFor<FMT>(__uint_as_float(top))));
    grew = t.first > 0 && s.s > had;
    plain = plain && (__float_as_uint(s.s) & 0x007fffffu) == 0u;
  }
  __device__ __forceinline__ void Store(const Kv8AppendArgs& a, bool keys, uint8_t* chunk,
                                        const Part& p, const double2* cs, uint8_t* tile) {
    if (keys) {
      StoreKeys<FMT, T, NU, kInterleaved>(a, chunk, p, had, grew, s, plain, x, y, cs, tile, sums);
      return;
    }
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int d = 128 * m + 2 * static_cast<int>(threadIdx.x & (kWave - 1));
      if (d < a.c.dim) {
        StoreValues<FMT, T>(chunk + d * 16, p.lo, p.hi, had, grew, s, plain, x.x, 32 * m);
        StoreValues<FMT, T>(chunk + d * 16 + 16, p.lo, p.hi, had, grew, s, plain, x.x, 32 * m + 1);
      }
    }
  }
  __device__ __forceinline__ void StoreMeans(const Kv8AppendArgs& a, const Task& t,
                                             int64_t page_head) const {
    const double f = static_cast<double>(s.s);
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int d = 128 * m + 2 * static_cast<int>(threadIdx.x & (kWave - 1));
      if (d < a.c.dim) {
        float* out = a.c.summaries + page_head * a.c.dim + d;
        out[0] = static_cast<float>(static_cast<double>(sums[m][0]) * f / t.end);
        out[1] = static_cast<float>(static_cast<double>(sums[m][1]) * f / t.end);
      }
    }
  }
};

// Pages of at most four chunks.  A workgroup for each page and group of `per` key
// heads, a page's one after the other (their rows lie side by side; head groups in
// the grid's second dimension took 331 us in place of 321 on the longest case
// below): 2 * per * chunks waves, wave w the keys (w even) or values of head
// w / 2 % per of the group, chunk w / (2 * per); then all of them the group's
// queries.  Every number is read once and stays in its lane until its code is
// known.  LDS: the sines of a page's tokens, a 16 x dim tile and the sums of
// each key wave, each wave's largest number.
constexpr int kMostWaves = 8;
template <typename T, int FMT, int NU, bool kInterleaved>
__global__ __launch_bounds__(kMostWaves* kWave) void Kv8AppendKernel(Kv8AppendArgs a, int per,
                                                                     bool vec) {
  extern __shared__ __align__(16) unsigned char smem[];
  CheckRequests(a);
  const int groups = (a.c.heads + per - 1) / per;
  Task t;
  if (!FindTask(a, blockIdx.x / groups, &t)) return;
  using L = Lane<T, FMT, NU, kInterleaved>;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int heads = a.c.heads, D = a.c.dim, chunks = a.c.chunks, group = a.q_heads / heads;
  const int h0 = blockIdx.x % groups * per, h1 = min(h0 + per, heads);
  const bool keys = (wave & 1) == 0;
  const int within = wave / 2 % per, chunk = wave / (2 * per);
  const int h = h0 + within;
  const bool mine = h < h1;
  double2* cs = reinterpret_cast<double2*>(smem);
  const double2* my_cs = cs + 128 * chunk * (a.rot.pairs / 8);
  uint8_t* tiles = smem + sizeof(double2) * 16 * chunks * a.rot.pairs;
  uint8_t* tile = tiles + wave / 2 * 16 * D;
  float* all_sums = reinterpret_cast<float*>(tiles + per * chunks * 16 * D);
  unsigned* all_tops = reinterpret_cast<unsigned*>(all_sums + per * chunks * D);

  const Part p = PartOf(t, chunk);
  const bool fresh = mine && p.lo < p.hi;
  L w;
  if (fresh) w.Load(a, vec, t, keys, h, p);
  if (!InPool(t.page, a.c.capacity)) {  // (every wave's the same)
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailPageId);
    return;
  }
  const int64_t page_head = static_cast<int64_t>(t.page) * heads + min(h, heads - 1);
  float* scale = (keys ? a.c.key_scales : a.c.value_scales) + page_head;
  w.had = t.first > 0 ? *scale : 0.0f;
  FillSines(a, t, 0, t.first, t.end, cs);
  __syncthreads();
  unsigned top = fresh ? WaveTop(w.Top(a, keys, p, my_cs)) : 0u;
  if (chunks > 1) {
    if (lane == 0) all_tops[wave] = top;
    __syncthreads();
    for (int i = 0; i < chunks; ++i) top = max(top, all_tops[(i * per + within) * 2 + (wave & 1)]);
  }
  w.SetScale(t, top);
  const bool means = keys && a.c.summaries != nullptr;
  if (mine && p.c0 < t.end && (fresh || w.grew || means)) {
    uint8_t* codes = (keys ? a.c.keys : a.c.values) + (page_head * a.c.page + p.c0) * D;
    w.Store(a, keys, codes, p, my_cs, tile);
  }
  if (mine && chunk == 0 && lane == 0) {
    *scale = w.s.s;
    if (h == 0 && keys) a.c.token_counts[t.page] = t.end;
  }
  if (a.c.summaries != nullptr) {
    if (chunks > 1) {
      if (mine && keys) {
#pragma unroll
        for (int m = 0; m < L::NV; ++m) {
          const int d = 128 * m + 2 * lane;
          if (d < D) {
            *reinterpret_cast<float2*>(all_sums + wave / 2 * D + d) =
                make_float2(w.sums[m][0], w.sums[m][1]);
          }
        }
      }
      __syncthreads();
    }
    if (mine && keys && chunk == 0) {
      for (int i = 1; i < chunks; ++i) {
#pragma unroll
        for (int m = 0; m < L::NV; ++m) {
          const int d = 128 * m + 2 * lane;
          if (d < D) {
            w.sums[m][0] += all_sums[(i * per + within) * D + d];
            w.sums[m][1] += all_sums[(i * per + within) * D + d + 1];
          }
        }
      }
      w.StoreMeans(a, t, page_head);
    }
  }
  if (group > 0) {
    Part all;
    all.lo = t.first;
    all.hi = t.end;
    Queries<T, kInterleaved>(a, vec, t, h0 * group, h1 * group, all, cs);
  }
}

// Larger pages: 2 * per waves, a wave all chunks of its side in turn, the largest
// number of all of them first, then the codes; the second reading comes from the
// cache, and the sines, of one chunk at a time, are formed again.
template <typename T, int FMT, int NU, bool kInterleaved>
__global__ __launch_bounds__(kMostWaves* kWave) void Kv8AppendPageKernel(Kv8AppendArgs a, int per,
                                                                         bool vec) {
  extern __shared__ __align__(16) unsigned char smem[];
  CheckRequests(a);
  const int groups = (a.c.heads + per - 1) / per;
  Task t;
  if (!FindTask(a, blockIdx.x / groups, &t)) return;
  if (!InPool(t.page, a.c.capacity)) {
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailPageId);
    return;
  }
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int heads = a.c.heads, D = a.c.dim, group = a.q_heads / heads;
  const int h0 = blockIdx.x % groups * per, h1 = min(h0 + per, heads);
  const int h = h0 + wave / 2;
  const bool mine = h < h1, keys = (wave & 1) == 0;
  double2* cs = reinterpret_cast<double2*>(smem);
  uint8_t* tile = smem + sizeof(double2) * 16 * a.rot.pairs + wave / 2 * 16 * D;
  const int64_t page_head = static_cast<int64_t>(t.page) * heads + min(h, heads - 1);
  uint8_t* codes = (keys ? a.c.keys : a.c.values) + page_head * a.c.page * D;
  float* scale = (keys ? a.c.key_scales : a.c.value_scales) + page_head;
  const bool means = keys && a.c.summaries != nullptr;
  const int chunk0 = t.first / 16, chunk1 = (t.end - 1) / 16;
  Lane<T, FMT, NU, kInterleaved> w;
  w.had = t.first > 0 ? *scale : 0.0f;
  unsigned top = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) w.SetScale(t, WaveTop(top));
#pragma unroll 1
    for (int c = pass == 1 && (w.grew || means) ? 0 : chunk0; c <= chunk1; ++c) {
      const Part p = PartOf(t, c);
      const bool fresh = p.lo < p.hi;
      if (fresh) {
        if (mine) w.Load(a, vec, t, keys, h, p);
        __syncthreads();
        FillSines(a, t, p.c0, p.lo, p.hi, cs);
        __syncthreads();
        if (mine) {
          const unsigned now = w.Top(a, keys, p, cs);
          if (pass == 0) top = max(top, now);
        }
      }
      if (pass == 1) {
        if (mine) w.Store(a, keys, codes + p.c0 * D, p, cs, tile);
      } else if (group > 0) {
        Queries<T, kInterleaved>(a, vec, t, h0 * group, h1 * group, p, cs);
      }
    }
  }
  if (!mine) return;
  if (lane == 0) {
    *scale = w.s.s;
    if (h == 0 && keys) a.c.token_counts[t.page] = t.end;
  }
  if (means) w.StoreMeans(a, t, page_head);
}

// Calls f with the kernel of a head size.
constexpr int kMostChunks = 4;
template <typename T, int FMT, bool kInterleaved, typename F>
void WithDim(const Kv8View& c, F&& f) {
  if (c.chunks > kMostChunks) {
    if (c.dim <= 64) return f(Kv8AppendPageKernel<T, FMT, 1, kInterleaved>);
    if (c.dim <= 128) return f(Kv8AppendPageKernel<T, FMT, 2, kInterleaved>);
    return f(Kv8AppendPageKernel<T, FMT, 4, kInterleaved>);
  }
  if (c.dim <= 64) return f(Kv8AppendKernel<T, FMT, 1, kInterleaved>);
  if (c.dim <= 128) return f(Kv8AppendKernel<T, FMT, 2, kInterleaved>);
  return f(Kv8AppendKernel<T, FMT, 4, kInterleaved>);
}
template <typename T, typename F>
void WithKernel(const Kv8View& c, bool interleaved, F&& f) {
  if (c.format == DSD_KV8_INT8) {
    interleaved ? WithDim<T, DSD_KV8_INT8, true>(c, f) : WithDim<T, DSD_KV8_INT8, false>(c, f);
  } else {
    interleaved ? WithDim<T, DSD_KV8_E4M3, true>(c, f) : WithDim<T, DSD_KV8_E4M3, false>(c, f);
  }
}
// Waves of a head, and LDS.
int Across(const Kv8View& c) { return c.chunks > kMostChunks ? 1 : c.chunks; }
int HeadsPerGroup(const Kv8View& c) { return std::min(Across(c) == 1 ? 2 : 1, c.heads); }
size_t LdsBytes(const Kv8View& c, int pairs) {
  const int across = Across(c), per = HeadsPerGroup(c);
  return sizeof(double2) * 16 * across * pairs + per * across * (16 + sizeof(float)) * c.dim +
         sizeof(unsigned) * kMostWaves;
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
  const int per = HeadsPerGroup(a.c);
  const int64_t units = a.b.max_tokens > 1
                            ? a.b.tokens / a.c.page + 2 * static_cast<int64_t>(a.b.batch)
                            : a.b.batch;
  const int64_t workgroups = units * ((a.c.heads + per - 1) / per);
  const int threads = 2 * per * Across(a.c) * kWave;
  // (a launch counts its threads in 32 bits)
  if (workgroups > 0xffffffffll / threads) {
    throw std::invalid_argument("too many tokens and heads for one call");
  }
  const unsigned grid = static_cast<unsigned>(workgroups);
  WithKernel<T>(a.c, a.rot.interleaved != 0, [&](auto kernel) {
    kernel<<<grid, threads, LdsBytes(a.c, a.rot.pairs), stream>>>(a, per, vec);
  });
  DSD_HIP_CHECK(hipGetLastError());
}

template <typename T>
void PreloadType(const Kv8View& c) {
  for (bool interleaved : {false, true}) {
    WithKernel<T>(c, interleaved, [&](auto kernel) {
      PreloadKernel(kernel);
      DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(LdsBytes(c, c.dim / 2))));
    });
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
