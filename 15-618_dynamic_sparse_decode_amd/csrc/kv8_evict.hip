// kv8_evict.hip -- dsd_kv8_evict (gfx950): a list's tokens cut to a budget by what they
// weighed, the kept ones of each key head moved, in order, to new pages.
//
// Mathematics.  Which tokens: per request and key head a selection of the `keep` best of
// n tokens, the better the larger the weight, then the lower the place; the first and the
// last ones are better than all others.  A weight's bits, turned so that they order as
// the numbers do, and behind them the place's are searched from the top in digits of up to
// 11 bits: the digit's counts in LDS, from the best down until `keep` is reached.  Once
// few candidates share the digits so far each counts those that are better.
// Then what they become: the numbers code * scale of a new page's tokens (their old pages
// have scales of their own) share the least scale that their largest fits, and each is
// rounded once to it.
//
// What bounds it: the selection is a chain (weights, counts, a digit, counts again) in one
// workgroup a list and key head: 10.5 us for one list of 4300 tokens, 44 for 32 of 32768 (8
// key heads; 33.5 MB of weights).  The form that holds 32 tiles a wave spills 15 registers
// of a lane (1024 threads have 128 each).  A longer list's ids and weights are read again in
// each pass: a whole call that keeps 4096 of 32768 takes 49 us, of 33000 81, of 60000 119.
// The move is bound by HBM: kept tokens lie apart and a value's load is 16 tokens of one
// dim, so 32 lists cut to 4096 touch 0.84 GB for 0.27 GB that are kept and write 0.27, 280 us.
#include "kv8_codes.h"

#include <algorithm>

namespace dsdk {
namespace {

// ---- which tokens ---------------------------------------------------------------

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;
constexpr int kDigit = 11;
constexpr int kBins = 1 << kDigit;
constexpr int kFew = 64;  // candidates that rank themselves: as many reads of LDS each

// A weight's bits in the numbers' order; NaN above all, -0 as 0.  Below every number's is
// kGone (no token), above every one kAlways (kept whatever it weighs).
constexpr unsigned kGone = 0u, kAlways = 0xffffffffu;
__device__ __forceinline__ unsigned KeyOf(float w) {
  const unsigned u = __float_as_uint(w + 0.0f);
  if (w != w) return kAlways - 1u;
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

// The sum over the workgroup's threads before this one; *total: over all.
__device__ __forceinline__ int BlockBefore(int x, int* wave_sums, int* total) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  int sum = x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(sum, o, kWave);
    if (lane >= o) sum += y;
  }
  __syncthreads();  // (the sums of the call before have been read)
  if (lane == kWave - 1) wave_sums[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    const int y = wave_sums[w];
    before += w < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before + sum - x;
}

struct SelectLds {
  int bins[kBins];
  int wave_sums[kSelectWaves];
  int first_end, recent_begin;  // places before the one, from the other on are kept
  unsigned found_digit;
  int found_above, found_count;
  int few;
  uint2 list[kFew];
};

// What is searched: places before `first_end` and from `recent_begin` on are kept, with
// the best of the others `count` in all.
struct Search {
  Kv8Request q;
  int head, r;
  int places, tiles;  // tiles of 64 places that a wave has
  int first_end, recent_begin;
  int count;
  int held;  // tokens
};

// kPacked: all pages but the last are full, so place i is token i.
template <int kHeld, bool kPacked>
__device__ __forceinline__ void SelectPlaces(const Kv8EvictArgs& a, const Search& f,
                                             const float* weights, SelectLds& lds);

// kBatch tiles are read at a time, without a branch between them (beyond the list: its
// last place again), so that their loads are on their way together.
constexpr int kBatch = 8;
struct Places {
  int page[kBatch], off[kBatch];
};
__device__ __forceinline__ Places ReadPlaces(const Kv8EvictArgs& a, int list, int places, int base,
                                             int j0) {
  const Kv8View& c = a.c;
  const unsigned inverse = 0xffffffffu / static_cast<unsigned>(c.chunks) + 1u;
  Places x;
#pragma unroll
  for (int k = 0; k < kBatch; ++k) {
    const int at = min(base + (j0 + k) * kWave, places - 1);
    const int slot = c.chunks == 1 ? at >> 4 : static_cast<int>(__umulhi(at >> 4, inverse));
    x.off[k] = at - slot * c.page;
    x.page[k] = a.b.page_ids[list + slot];
  }
  return x;
}
__device__ __forceinline__ float ReadWeight(const Kv8EvictArgs& a, int head, int page, int off) {
  const int64_t at = InPool(page, a.c.capacity) ? page : 0;
  return a.weights[(at * a.c.heads + head) * a.c.page + off];
}
// Of all a wave's tiles, the next batch's pages beside a batch's weights.
template <int kHeld>
__device__ __forceinline__ void ReadWeights(const Kv8EvictArgs& a, int list, int head, int places,
                                            int tiles, float* weights) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int base = wave * tiles * kWave + lane;
  Places x = ReadPlaces(a, list, places, base, 0);
#pragma unroll
  for (int j0 = 0; j0 < kHeld; j0 += kBatch) {
    if (j0 >= tiles) break;
    const Places y = x;
    if (j0 + kBatch < kHeld) x = ReadPlaces(a, list, places, base, j0 + kBatch);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) weights[j0 + k] = ReadWeight(a, head, y.page[k], y.off[k]);
  }
}
// The tokens of a list's last page.
__device__ __forceinline__ int LastCount(const Kv8EvictArgs& a, const Kv8Request& q) {
  const int page = a.b.page_ids[q.list + q.pages - 1];
  return InPool(page, a.c.capacity) ? min(max(a.c.token_counts[page], 0), a.c.page) : 0;
}

// Grid (key heads, batch).  kHeld: tiles of 64 places that a wave holds in registers; of
// longer lists the weights are read again for each pass.
template <int kHeld>
__global__ __launch_bounds__(kSelectThreads) void Kv8EvictSelectKernel(Kv8EvictArgs a) {
  __shared__ SelectLds lds;
  const Kv8View& c = a.c;
  const int head = blockIdx.x, r = blockIdx.y;
  Kv8Request q;
  if (!Kv8ReadList(a.b, r, &q) || q.pages > 0x7fff0000 / c.page) {
    if (threadIdx.x == 0) {
      ReportFailure(a.fail, kFailShape);
      if (head == 0) a.new_counts[r] = a.kept_tokens[r] = 0;
    }
    return;
  }
  for (int i = threadIdx.x; i < kBins; i += kSelectThreads) lds.bins[i] = 0;
  const int places = q.pages * c.page;
  const int tiles = ((places + kWave - 1) / kWave + kSelectWaves - 1) / kSelectWaves;
  float weights[kHeld];  // (on their way beside the pages' counts)
  if (places > 0 && tiles <= kHeld) ReadWeights<kHeld>(a, q.list, head, places, tiles, weights);
  // Tokens before each thread's pages, and where the first and the last ones lie.
  auto count_of = [&](int slot) {
    const int page = a.b.page_ids[q.list + slot];
    if (!InPool(page, c.capacity)) {
      ReportFailure(a.fail, kFailPageId);
      return 0;
    }
    return min(max(c.token_counts[page], 0), c.page);
  };
  const int share = (q.pages + kSelectThreads - 1) / kSelectThreads;
  const int s0 = min(q.pages, static_cast<int>(threadIdx.x) * share), s1 = min(q.pages, s0 + share);
  int mine = 0;
  bool full = true;
  for (int s = s0; s < s1; ++s) {
    const int n = count_of(s);
    mine += n;
    full = full && (n == c.page || s == q.pages - 1);
  }
  if (threadIdx.x == 0) {
    lds.first_end = 0;
    lds.recent_begin = 0x7fffffff;
  }
  const int behind = q.pages > 0 ? LastCount(a, q) : 0;
  const bool packed = __syncthreads_and(full) != 0;
  int held = packed ? max(q.pages - 1, 0) * c.page + behind : 0;
  int first_end = 0, recent_begin = 0x7fffffff;
  if (packed) {
    if (held > a.keep) {
      first_end = a.first;
      if (a.recent > 0) recent_begin = held - a.recent;
    }
  } else {
    int rank = BlockBefore(mine, lds.wave_sums, &held);
    const bool all = held <= a.keep;
    const int from = all ? held : held - a.recent;  // the rank of the first of the last
    for (int s = s0; s < s1; ++s) {
      const int n = count_of(s);
      if (!all && rank < a.first && a.first <= rank + n) lds.first_end = s * c.page + a.first - rank;
      if (rank <= from && from < rank + n) lds.recent_begin = s * c.page + from - rank;
      rank += n;
    }
    __syncthreads();
    first_end = lds.first_end;
    recent_begin = lds.recent_begin;
  }
  const int count = min(held, a.keep);
  if (threadIdx.x == 0 && head == 0) {
    a.kept_tokens[r] = count;
    a.new_counts[r] = (count + c.page - 1) / c.page;
  }
  const Search f = {q, head, r, places, tiles, first_end, recent_begin, count, held};
  if (tiles <= kHeld) {
    packed ? SelectPlaces<kHeld, true>(a, f, weights, lds)
           : SelectPlaces<kHeld, false>(a, f, weights, lds);
  } else {
    packed ? SelectPlaces<0, true>(a, f, weights, lds) : SelectPlaces<0, false>(a, f, weights, lds);
  }
}

// Wave w has the w-th `tiles` tiles of 64 places, lane l place l of each.
template <int kHeld, bool kPacked>
__device__ __forceinline__ void SelectPlaces(const Kv8EvictArgs& a, const Search& f,
                                             const float* weights, SelectLds& lds) {
  const Kv8View& c = a.c;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int tiles = f.tiles;
  const int base = wave * tiles * kWave + lane;

  auto key_of = [&](int j, float w, bool counted) {
    const int at = base + j * kWave;
    const bool there = j < tiles && (kPacked ? at < f.held : at < f.places && counted);
    return !there ? kGone : (at < f.first_end || at >= f.recent_begin ? kAlways : KeyOf(w));
  };
  // (the pages' counts where not all are full)
  auto counts = [&](const Places& x, bool* counted) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const bool ok = InPool(x.page[k], c.capacity);
      counted[k] = x.off[k] < (ok ? c.token_counts[x.page[k]] : 0);
    }
  };
  unsigned keys[kHeld > 0 ? kHeld : 1];
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int j0 = 0; j0 < kHeld; j0 += kBatch) {
      if (j0 >= tiles) break;
      bool counted[kBatch] = {};
      if constexpr (!kPacked) counts(ReadPlaces(a, f.q.list, f.places, base, j0), counted);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) keys[j0 + k] = key_of(j0 + k, weights[j0 + k], counted[k]);
    }
  }
  // with(j, key) for the wave's tiles in order.
  auto each = [&](auto&& with) {
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        if (j < tiles) with(j, keys[j]);
      }
    } else {
      for (int j0 = 0; j0 < tiles; j0 += kBatch) {
        const Places x = ReadPlaces(a, f.q.list, f.places, base, j0);
        float w[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) w[k] = ReadWeight(a, f.head, x.page[k], x.off[k]);
        bool counted[kBatch] = {};
        if constexpr (!kPacked) counts(x, counted);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) with(j0 + k, key_of(j0 + k, w[k], counted[k]));
      }
    }
  };

  // The count-th best place: of those whose digits so far are its own the next digit is
  // counted, until few are left.
  unsigned key = f.count > 0 ? kGone : kAlways;  // (all are kept, or none)
  int last = -1;  // of the places with its key the last that is kept
  if (f.count > 0 && f.count < f.held) {
    int left = f.count;
    unsigned known = 0, place_known = 0;  // the key's digits so far, then the turned place's
    int few = 0;
    auto turned_place = [&](int j) { return 0x7fffffffu - static_cast<unsigned>(base + j * kWave); };
    // One digit: with(j, key, &bin) says which are counted.
    auto digit = [&](auto&& with) {
      if (threadIdx.x == 0) lds.few = 0;
      each([&](int j, unsigned p) {
        unsigned bin;
        if (with(j, p, &bin)) atomicAdd(&lds.bins[bin], 1);
      });
      __syncthreads();
      // thread t: bins kBins - 1 - 2 t and the one below it, cleared for the next digit
      const int b0 = kBins - 1 - 2 * static_cast<int>(threadIdx.x);
      const int n0 = lds.bins[b0], n1 = lds.bins[b0 - 1];
      lds.bins[b0] = lds.bins[b0 - 1] = 0;
      int sum;
      const int above = BlockBefore(n0 + n1, lds.wave_sums, &sum);
      if (above < left && left <= above + n0 + n1) {
        const bool second = left > above + n0;
        lds.found_digit = static_cast<unsigned>(second ? b0 - 1 : b0);
        lds.found_above = second ? above + n0 : above;
        lds.found_count = second ? n1 : n0;
      }
      __syncthreads();
      left -= lds.found_above;
      few = lds.found_count;
      return lds.found_digit;
    };
    // Those that are left rank themselves.
    auto finish = [&](auto&& with) {
      each([&](int j, unsigned p) {
        if (with(j, p)) lds.list[atomicAdd(&lds.few, 1)] = make_uint2(p, turned_place(j));
      });
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < few) {
        const uint2 mine = lds.list[threadIdx.x];
        int better = 0;
#pragma unroll 4
        for (int i = 0; i < few; ++i) {
          const uint2 x = lds.list[i];
          better += x.x > mine.x || (x.x == mine.x && x.y > mine.y) ? 1 : 0;
        }
        if (better == left - 1) {
          lds.found_digit = mine.x;
          lds.found_above = static_cast<int>(0x7fffffffu - mine.y);
        }
      }
      __syncthreads();
      key = lds.found_digit;
      last = lds.found_above;
    };
    // Bits 21.., 10.., 0.. of the key (11, 11, 10 of them; kGone alone has a first digit of 0).
    known = digit([&](int, unsigned p, unsigned* bin) {
      *bin = p >> 21;
      return p != kGone;
    });
    int shift = 21;
#pragma unroll 1
    while (few > kFew && shift > 0) {
      const int next = max(shift - kDigit, 0);
      const unsigned found = digit([&](int, unsigned p, unsigned* bin) {
        *bin = (p >> next) & ((1u << (shift - next)) - 1u);
        return p >> shift == known;
      });
      known = known << (shift - next) | found;
      shift = next;
    }
    if (few <= kFew) {
      finish([&](int, unsigned p) { return p >> shift == known; });
    } else {
      // many of one key: bits 20.., 9.., 0.. of the turned place (11, 11, 9); places differ,
      // so the last digit leaves one
      shift = 31;
#pragma unroll 1
      while (few > kFew) {
        const int next = max(shift - kDigit, 0);
        const unsigned found = digit([&](int j, unsigned p, unsigned* bin) {
          const unsigned turned = turned_place(j);
          *bin = (turned >> next) & ((1u << (shift - next)) - 1u);
          return p == known && turned >> shift == place_known;
        });
        place_known = place_known << (shift - next) | found;
        shift = next;
      }
      finish([&](int j, unsigned p) {
        return p == known && turned_place(j) >> shift == place_known;
      });
    }
  }

  // How many each wave keeps, then where its kept places go.
  auto keeps = [&](int j, unsigned p) {
    return p > key || (p == key && base + j * kWave <= last);
  };
  int sure = 0;
  each([&](int j, unsigned p) { sure += static_cast<int>(__popcll(__ballot(keeps(j, p)))); });
  __syncthreads();
  if (lane == 0) lds.wave_sums[wave] = sure;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < wave; ++w) at += lds.wave_sums[w];
  int* kept = a.kept + (static_cast<int64_t>(f.r) * c.heads + f.head) * a.keep;
  const unsigned long long below = (1ull << lane) - 1ull;
  each([&](int j, unsigned p) {
    const bool keep = keeps(j, p);
    const unsigned long long taken = __ballot(keep);
    if (keep) kept[at + __popcll(taken & below)] = base + j * kWave;
    at += static_cast<int>(__popcll(taken));
  });
  for (int i = f.count + threadIdx.x; i < a.keep; i += kSelectThreads) kept[i] = -1;
}

// ---- the move ---------------------------------------------------------------------

typedef uint16_t U16x2 __attribute__((ext_vector_type(2)));
typedef int16_t I16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned Max16(unsigned x, unsigned y) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(U16x2, x),
                                                                __builtin_bit_cast(U16x2, y)));
}

// The magnitudes of bytes 0 and 2 (odd: 1 and 3) of four codes, which order as the numbers
// do (an e4m3 NaN's, 127, above all of them).
template <int FMT>
__device__ __forceinline__ unsigned Sizes2(unsigned w, bool odd) {
  if constexpr (FMT == DSD_KV8_INT8) {
    const unsigned high = odd ? w & 0xff00ff00u : (w << 8) & 0xff00ff00u;
    const I16x2 x = __builtin_bit_cast(I16x2, high) >> 1;  // (-128 has a magnitude too)
    const I16x2 zero = {0, 0};
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(x, zero - x));
  } else {
    return (odd ? w >> 8 : w) & 0x007f007fu;
  }
}
template <int FMT>
__device__ __forceinline__ double NumberOf(unsigned size) {
  if constexpr (FMT == DSD_KV8_INT8) {
    return static_cast<double>(size >> 7);
  } else {
    return static_cast<double>(__builtin_amdgcn_cvt_f32_fp8(static_cast<int>(size), 0));
  }
}
// The codes' magnitudes with 0 in place of NaN.
__device__ __forceinline__ unsigned WithoutNan(unsigned w) {
  return w & ~((NanBytes(w) >> 7) * 0xffu);
}

// The least scale whose largest code reaches `most`.
template <int FMT>
__device__ __forceinline__ float ScaleForNumber(double most) {
  if constexpr (FMT == DSD_KV8_INT8) {
    return fmaxf(static_cast<float>(most / 127.0), kKv8Tiny);
  } else {
    int e;
    const double f = frexp(most, &e);
    const int power = min(max(e - 9 + (f > 0.875 ? 1 : 0), -126), 127);
    return most > 0.0 ? __uint_as_float(static_cast<unsigned>(power + 127) << 23) : kKv8Tiny;
  }
}

__device__ __forceinline__ double WaveMost(double x) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) x = fmax(x, __shfl_xor(x, o, kWave));
  return x;
}

// Codes brought from one scale to another.  Exact in 64 bits (Slow4); the quotient of the
// scales in 32 bits does where it is a power of two (e4m3: a product with a code is exact,
// one rounding), and of int8 codes where the product lies further from a border between
// two codes than its error of 127 * 2^-22 (a quarter of the time in 64 bits).
template <int FMT>
__device__ __forceinline__ float RatioOf(float had, const Scale& s, bool* fast) {
  if constexpr (FMT == DSD_KV8_INT8) {
    *fast = true;
    return static_cast<float>(static_cast<double>(had) * s.inv64);
  } else {
    const unsigned bits = __float_as_uint(had);
    // (0: a place without a token; its codes are 0)
    *fast = (bits & 0x807fffffu) == 0u && bits != 0x7f800000u;
    const int e = static_cast<int>(bits >> 23) - static_cast<int>(__float_as_uint(s.s) >> 23);
    return e < -126 || bits == 0u ? 0.0f
                                  : __uint_as_float(static_cast<unsigned>(min(e, 30) + 127) << 23);
  }
}
template <int FMT>
__device__ __forceinline__ unsigned Slow4(unsigned w, const float (&had)[4], const Scale& s) {
  float n[4];
  Numbers4<FMT>(w, n);
  double y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = static_cast<double>(n[e]) * static_cast<double>(had[e]);
  return Codes4<FMT>(y[0], y[1], y[2], y[3], s);
}
// *sure: the result stands (int8).
template <int FMT>
__device__ __forceinline__ unsigned Quick4(unsigned w, const float (&ratio)[4], bool* sure) {
  float n[4];
  Numbers4<FMT>(w, n);
#pragma unroll
  for (int e = 0; e < 4; ++e) n[e] *= ratio[e];
  if constexpr (FMT == DSD_KV8_INT8) {
    unsigned out = 0;
    *sure = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float near = rintf(n[e]);
      *sure = *sure && fabsf(n[e] - near) < 0.5f - 0x1p-13f;
      out |= (static_cast<unsigned>(static_cast<int>(near)) & 0xffu) << (8 * e);
    }
    return out;
  } else {
    *sure = true;
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(n[0], n[1], 0, false);
    return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(n[2], n[3], low, true));
  }
}

__device__ __forceinline__ float ReadLane(float x, int lane) {
  return __uint_as_float(static_cast<unsigned>(
      __builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(x)), lane)));
}

// Grid (key heads * new pages, batch): one new page of one key head.  Waves 2 i have the
// keys, 2 i + 1 the values of chunks i, i + kWaves / 2, ... of 16 tokens (U of them) in
// registers, as codes: keys lane l unit l + 64 j (16 dims) of the chunk's [16][dim],
// values lane l dims l + 64 j, all 16 tokens; of the chunk's token l % 16 it has the place
// and scale.  NU = ceil(dim / 64); kDim: head_dim where it is 64 * NU, else 0.
template <int FMT, int NU, int kDim, int U>
__global__ __launch_bounds__(512) void Kv8EvictMoveKernel(Kv8EvictArgs a) {
  extern __shared__ __align__(16) uint8_t tile[];  // the new keys (for their mean)
  __shared__ double wave_most[8];
  __shared__ float key_scale;
  const Kv8View& c = a.c;
  const int D = kDim > 0 ? kDim : c.dim, units = D / 16, ps = c.page;
  const int head = blockIdx.x % c.heads, index = blockIdx.x / c.heads, r = blockIdx.y;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int waves = blockDim.x / kWave;
  const bool is_key = (wave & 1) == 0;
  auto chunk_of = [&](int u) { return wave / 2 + waves / 2 * u; };
  // (on their way beside the list's; rows behind the last kept token are in the array too)
  const int* kept = a.kept + (static_cast<int64_t>(r) * c.heads + head) * a.keep + index * ps;
  int place[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = 16 * chunk_of(u) + (lane & 15);
    place[u] = i < ps && index * ps + i < a.keep ? kept[i] : -1;
  }
  Kv8Request q;
  const bool listed = Kv8ReadList(a.b, r, &q);
  const int count = min(a.kept_tokens[r] - index * ps, ps);
  if (count <= 0 || !listed) return;
  // (the caller's array may end behind the last page that is filled)
  const int page = a.new_ids[static_cast<int64_t>(r) * a.new_stride + index];
  if (!InPool(page, c.capacity)) {
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailPageId);
    return;
  }
  if (threadIdx.x == 0 && head == 0) c.token_counts[page] = count;
  const int64_t to = static_cast<int64_t>(page) * c.heads + head;
  const unsigned inverse = 0xffffffffu / static_cast<unsigned>(c.chunks) + 1u;
  const int page_bytes = ps * D;
  unsigned w[U][NU][4];
  float had[U];  // of the lane's token
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int chunk = chunk_of(u);
#pragma unroll
    for (int j = 0; j < NU; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[u][j][i] = 0u;
    }
    had[u] = 0.0f;
    if (chunk >= c.chunks) continue;
    const int here = count - 16 * chunk;  // tokens of the chunk
    const bool mine = (lane & 15) < here;
    const int slot = c.chunks == 1 ? place[u] >> 4 : static_cast<int>(__umulhi(place[u] >> 4, inverse));
    const int off = place[u] - slot * ps;
    const int from = mine ? a.b.page_ids[q.list + slot] : 0;
    const int64_t old = static_cast<int64_t>(from) * c.heads + head;
    const int64_t begin =
        !mine ? 0 : old * page_bytes + (is_key ? off * D : (off >> 4) * (16 * D) + (off & 15));
    const int low = static_cast<int>(begin), high = static_cast<int>(begin >> 32);
    if (here <= 0) {
      // (a chunk behind the last token: zeros)
    } else if (is_key) {
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        const int i = min(lane + kWave * j, D - 1), token = i / units;
        const uint64_t at =
            static_cast<uint64_t>(static_cast<unsigned>(__shfl(high, token, kWave))) << 32 |
            static_cast<unsigned>(__shfl(low, token, kWave));
        if (token < here && (kDim > 0 || lane + kWave * j < D)) {
          const uint4 x = *reinterpret_cast<const uint4*>(c.keys + at + 16 * (i - token * units));
          w[u][j][0] = x.x;
          w[u][j][1] = x.y;
          w[u][j][2] = x.z;
          w[u][j][3] = x.w;
        }
      }
    } else {
      // (all on their way at once: no branch between them, a token beyond the last is the
      // last one's and masked)
      unsigned code[16][NU];
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const int token = min(t, here - 1);
        const uint64_t at =
            static_cast<uint64_t>(static_cast<unsigned>(__builtin_amdgcn_readlane(high, token))) << 32 |
            static_cast<unsigned>(__builtin_amdgcn_readlane(low, token));
        const uint8_t* p = c.values + at;
#pragma unroll
        for (int j = 0; j < NU; ++j) code[t][j] = p[min(lane + kWave * j, D - 1) * 16];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int have = min(max(here - 4 * k, 0), 4);
        const unsigned mask = have == 4 ? 0xffffffffu : (1u << (8 * have)) - 1u;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
          w[u][j][k] = (code[4 * k][j] | code[4 * k + 1][j] << 8 | code[4 * k + 2][j] << 16 |
                        code[4 * k + 3][j] << 24) & mask;
        }
      }
    }
    if (mine) had[u] = (is_key ? c.key_scales : c.value_scales)[old];
    if (is_key && lane < 16) {
      a.weights[to * ps + 16 * chunk + lane] = mine ? a.weights[old * ps + off] : 0.0f;
    }
  }
  // The largest number: of a token's codes by their bytes, then of the tokens'.
  double most = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (chunk_of(u) >= c.chunks) continue;
    auto by_tokens = [&](bool nan) {
      double got = 0.0;
      auto codes = [&](int j, int k) { return nan ? WithoutNan(w[u][j][k]) : w[u][j][k]; };
      if (is_key) {
#pragma unroll
        for (int j = 0; j < NU; ++j) {
          unsigned top = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned x = codes(j, k);
            top = Max16(top, Max16(Sizes2<FMT>(x, false), Sizes2<FMT>(x, true)));
          }
          top = max(top & 0xffffu, top >> 16);
          const int token = min(lane + kWave * j, D - 1) / units;
          got = fmax(got, NumberOf<FMT>(top) * static_cast<double>(__shfl(had[u], token, kWave)));
          if (FMT == DSD_KV8_E4M3 && top == 127u) got = INFINITY;
        }
      } else {
        // tokens 4 k + {0, 2} and 4 k + {1, 3}; then half of them from each lane's partner,
        // until a lane has two tokens' of its 8 lanes, of which the wave has 8 groups
        unsigned top[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          top[2 * k] = top[2 * k + 1] = 0;
#pragma unroll
          for (int j = 0; j < NU; ++j) {
            const unsigned x = codes(j, k);
            top[2 * k] = Max16(top[2 * k], Sizes2<FMT>(x, false));
            top[2 * k + 1] = Max16(top[2 * k + 1], Sizes2<FMT>(x, true));
          }
        }
#pragma unroll
        for (int half = 4; half >= 1; half >>= 1) {
          const bool upper = (lane & half) != 0;  // keeps the upper half
#pragma unroll
          for (int k = 0; k < half; ++k) {
            const unsigned give = upper ? top[k] : top[k + half];
            const unsigned keep = upper ? top[k + half] : top[k];
            top[k] = Max16(keep, static_cast<unsigned>(__shfl_xor(static_cast<int>(give), half, kWave)));
          }
        }
#pragma unroll
        for (int o = 8; o < kWave; o <<= 1) {
          top[0] = Max16(top[0], static_cast<unsigned>(__shfl_xor(static_cast<int>(top[0]), o, kWave)));
        }
        // top[0]: index lane & 7 of the eight
        const int token = 4 * ((lane & 7) >> 1) + (lane & 1);
        const unsigned t0 = top[0] & 0xffffu, t1 = top[0] >> 16;
        got = fmax(NumberOf<FMT>(t0) * static_cast<double>(__shfl(had[u], token, kWave)),
                   NumberOf<FMT>(t1) * static_cast<double>(__shfl(had[u], token + 2, kWave)));
        if (FMT == DSD_KV8_E4M3 && (t0 == 127u || t1 == 127u)) got = INFINITY;
      }
      return got;
    };
    double got = by_tokens(false);
    if (FMT == DSD_KV8_E4M3 && __ballot(got == INFINITY) != 0) got = by_tokens(true);  // seldom
    most = fmax(most, got);
  }
  most = WaveMost(most);
  if (lane == 0) wave_most[wave] = most;
  __syncthreads();
  most = 0.0;
  for (int i = wave & 1; i < waves; i += 2) most = fmax(most, wave_most[i]);
  Scale scale;
  scale.Set<FMT>(ScaleForNumber<FMT>(most));
  if (threadIdx.x == 0) c.key_scales[to] = key_scale = scale.s;
  if (threadIdx.x == kWave) c.value_scales[to] = scale.s;

  // Brought to it.
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int chunk = chunk_of(u);
    if (chunk >= c.chunks) continue;
    bool fast;
    const float ratio = RatioOf<FMT>(had[u], scale, &fast);
    const bool all_fast = __ballot(!fast) == 0;
    const bool same =
        all_fast && __ballot((lane & 15) < count - 16 * chunk && ratio != 1.0f) == 0;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int i = lane + kWave * j;
      if (!same) {
        // of the token that the lane's keys are of
        const int token = min(i, D - 1) / units;
        const float key_ratio = is_key ? __shfl(ratio, token, kWave) : 0.0f;
        const float key_had = is_key ? __shfl(had[u], token, kWave) : 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float by[4];
          bool sure = false;
          unsigned x = 0;
          if (all_fast) {
#pragma unroll
            for (int e = 0; e < 4; ++e) by[e] = is_key ? key_ratio : ReadLane(ratio, 4 * k + e);
            x = Quick4<FMT>(w[u][j][k], by, &sure);
          }
          if (!sure) {
#pragma unroll
            for (int e = 0; e < 4; ++e) by[e] = is_key ? key_had : ReadLane(had[u], 4 * k + e);
            x = Slow4<FMT>(w[u][j][k], by, scale);
          }
          w[u][j][k] = x;
        }
      }
      if (kDim == 0 && i >= D) continue;
      const uint4 out = make_uint4(w[u][j][0], w[u][j][1], w[u][j][2], w[u][j][3]);
      const int64_t at = to * page_bytes + chunk * 16 * D + 16 * i;
      *reinterpret_cast<uint4*>((is_key ? c.keys : c.values) + at) = out;
      if (is_key && c.summaries != nullptr) {
        *reinterpret_cast<uint4*>(tile + chunk * 16 * D + 16 * i) = out;
      }
    }
  }
  if (c.summaries == nullptr) return;
  __syncthreads();
  for (int d = 4 * threadIdx.x; d < D; d += 4 * blockDim.x) {
    float sum[4] = {};
    for (int t = 0; t < count; ++t) {
      float x[4];
      Numbers4<FMT>(*reinterpret_cast<const unsigned*>(tile + t * D + d), x);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += x[e];
    }
    F32x4 mean;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mean[e] =
          static_cast<float>(static_cast<double>(sum[e]) * static_cast<double>(key_scale) / count);
    }
    *reinterpret_cast<F32x4*>(c.summaries + to * D + d) = mean;
  }
}

size_t MoveLdsBytes(const Kv8View& c) {
  return c.summaries != nullptr ? static_cast<size_t>(c.page) * c.dim : 0;
}

// Calls f with the kernel of a head and page size.
template <int FMT, int NU, int kDim, typename F>
void WithMove(int chunks, F&& f) {
  if (chunks <= 4) return f(Kv8EvictMoveKernel<FMT, NU, kDim, 1>);
  if (chunks <= 8) return f(Kv8EvictMoveKernel<FMT, NU, kDim, 2>);
  return f(Kv8EvictMoveKernel<FMT, NU, kDim, 4>);
}
template <int FMT, typename F>
void WithMove(const Kv8View& c, F&& f) {
  if (c.dim == 64) return WithMove<FMT, 1, 64>(c.chunks, f);
  if (c.dim < 64) return WithMove<FMT, 1, 0>(c.chunks, f);
  if (c.dim == 128) return WithMove<FMT, 2, 128>(c.chunks, f);
  if (c.dim < 128) return WithMove<FMT, 2, 0>(c.chunks, f);
  return WithMove<FMT, 4, 0>(c.chunks, f);
}
template <typename F>
void WithMove(const Kv8View& c, F&& f) {
  c.format == DSD_KV8_INT8 ? WithMove<DSD_KV8_INT8>(c, f) : WithMove<DSD_KV8_E4M3>(c, f);
}

}  // namespace

size_t Kv8EvictWorkspaceBytes(const Kv8View&, const dsd_kv8_batch& b, int) {
  return (sizeof(int) * static_cast<size_t>(b.batch) + 15) / 16 * 16;
}

void PreloadKv8Evict(const Kv8View& c) {
  PreloadKernel(Kv8EvictSelectKernel<8>);
  PreloadKernel(Kv8EvictSelectKernel<32>);
  WithMove(c, [&](auto kernel) {
    PreloadKernel(kernel);
    DSD_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(MoveLdsBytes(c))));
  });
}

void LaunchKv8Evict(const Kv8EvictArgs& a, hipStream_t stream) {
  if (a.b.batch == 0) return;
  const dim3 lists(a.c.heads, a.b.batch);
  if (static_cast<int64_t>(a.b.max_pages) * a.c.page <= 8 * kSelectThreads) {
    Kv8EvictSelectKernel<8><<<lists, kSelectThreads, 0, stream>>>(a);
  } else {
    Kv8EvictSelectKernel<32><<<lists, kSelectThreads, 0, stream>>>(a);
  }
  DSD_HIP_CHECK(hipGetLastError());
  const int pages = (a.keep + a.c.page - 1) / a.c.page;
  if (pages == 0) return;
  const dim3 grid(a.c.heads * pages, a.b.batch);
  const int threads = 2 * kWave * std::min(a.c.chunks, 4);
  WithMove(a.c, [&](auto kernel) { kernel<<<grid, threads, MoveLdsBytes(a.c), stream>>>(a); });
  DSD_HIP_CHECK(hipGetLastError());
}

}  // namespace dsdk
