// kv8_evict.hip -- dsd_kv8_evict (gfx950): a list's tokens cut to a budget by what they
// weighed, the kept ones of each key head moved, in order, to new pages.
//
// Mathematics.  Which tokens: per request and key head a selection of the need = keep -
// first - recent largest of n weights.  A weight's bits, turned so that they order as
// the numbers do, are searched from the top in digits of 11, 11 and 10 bits: the digit's
// counts in LDS, from the largest down until `need` is reached.  That leaves the need-th
// largest key T and how many keys equal to it are kept, the ones of the lowest places.
// Then what they become: the numbers code * scale of a new page's tokens (their old pages
// have scales of their own) share the least scale that their largest fits, and each is
// rounded once to it.
#include "kv8_codes.h"

#include <algorithm>

namespace dsdk {
namespace {

// ---- which tokens ---------------------------------------------------------------

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;
constexpr int kDigit = 11;
constexpr int kBins = 1 << kDigit;

// A weight's bits in the numbers' order; NaN above all, -0 as 0.
__device__ __forceinline__ unsigned KeyOf(float w) {
  const unsigned u = __float_as_uint(w + 0.0f);
  if (w != w) return 0xffffffffu;
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
  int wave_sums[kSelectWaves], wave_ties[kSelectWaves];
  int first_end, recent_begin;  // places before the one, from the other on are kept
  unsigned found_digit;
  int found_above;
};

// What is searched: places before `first_end` and from `recent_begin` on are kept, `need`
// of the others, `count` in all.
struct Search {
  Kv8Request q;
  int head, r;
  int places, tiles;  // tiles of 64 places that a wave has
  int first_end, recent_begin;
  int need, count;
};

template <int kHeld>
__device__ __forceinline__ void SelectPlaces(const Kv8EvictArgs& a, const Search& f,
                                             SelectLds& lds);

// Grid (key heads, batch).  kHeld: tiles of 64 places that a wave holds in registers; of
// longer lists the weights are read again for each pass.
template <int kHeld>
__global__ __launch_bounds__(kSelectThreads) void Kv8EvictSelectKernel(Kv8EvictArgs a) {
  __shared__ SelectLds lds;
  const Kv8View& c = a.c;
  const int head = blockIdx.x, r = blockIdx.y;
  Kv8Request q;
  if (!Kv8ReadList(a.b, r, &q) || q.pages > 0x7fffff00 / c.page) {
    if (threadIdx.x == 0) {
      ReportFailure(a.fail, kFailShape);
      if (head == 0) a.new_counts[r] = a.kept_tokens[r] = 0;
    }
    return;
  }
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
  for (int s = s0; s < s1; ++s) mine += count_of(s);
  if (threadIdx.x == 0) {
    lds.first_end = 0;
    lds.recent_begin = 0x7fffffff;
  }
  int held;
  int rank = BlockBefore(mine, lds.wave_sums, &held);
  const bool all = held <= a.keep;
  const int need = all ? 0 : a.keep - a.first - a.recent;
  if (!all) {
    const int from = held - a.recent;  // the rank of the first of the last
    for (int s = s0; s < s1; ++s) {
      const int n = count_of(s);
      if (rank < a.first && a.first <= rank + n) lds.first_end = s * c.page + a.first - rank;
      if (rank <= from && from < rank + n) lds.recent_begin = s * c.page + from - rank;
      rank += n;
    }
  } else if (threadIdx.x == 0) {
    lds.first_end = 0x7fffffff;
  }
  __syncthreads();
  const int count = min(held, a.keep);
  if (threadIdx.x == 0 && head == 0) {
    a.kept_tokens[r] = count;
    a.new_counts[r] = (count + c.page - 1) / c.page;
  }

  const int places = q.pages * c.page;
  const int tiles = ((places + kWave - 1) / kWave + kSelectWaves - 1) / kSelectWaves;
  const Search f = {q,    head,  r, places, tiles, lds.first_end, lds.recent_begin,
                    need, count};
  if (tiles <= kHeld) {
    SelectPlaces<kHeld>(a, f, lds);
  } else {
    SelectPlaces<0>(a, f, lds);
  }
}

// Wave w has the w-th `tiles` tiles of 64 places, lane l place l of each.
template <int kHeld>
__device__ __forceinline__ void SelectPlaces(const Kv8EvictArgs& a, const Search& f,
                                             SelectLds& lds) {
  const Kv8View& c = a.c;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int tiles = f.tiles;
  // Places: kGone (no token), kAlways, or a candidate of some key.
  enum { kGone, kAlways, kCandidate };
  const int base = wave * tiles * kWave + lane;
  struct Place {
    int kind;
    unsigned key;
  };
  auto read = [&](int at) {
    Place p = {kGone, 0u};
    if (at < f.places) {
      const int slot = at / c.page, off = at - slot * c.page;
      const int page = a.b.page_ids[f.q.list + slot];
      if (InPool(page, c.capacity) && off < c.token_counts[page]) {
        p.kind = at < f.first_end || at >= f.recent_begin ? kAlways : kCandidate;
        p.key = KeyOf(a.weights[(static_cast<int64_t>(page) * c.heads + f.head) * c.page + off]);
      }
    }
    return p;
  };
  constexpr int kArray = kHeld > 0 ? kHeld : 1;
  unsigned keys[kArray];
  unsigned long long gone = 0, always = 0;  // of tile j at bit j
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const Place p = j < tiles ? read(base + j * kWave) : Place{kGone, 0u};
      keys[j] = p.key;
      gone |= static_cast<unsigned long long>(p.kind == kGone) << j;
      always |= static_cast<unsigned long long>(p.kind == kAlways) << j;
    }
  }
  // with(j, place) for the wave's tiles in order.
  auto each = [&](auto&& with) {
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        if (j < tiles) {
          with(j, Place{(gone >> j & 1) != 0 ? kGone : ((always >> j & 1) != 0 ? kAlways : kCandidate),
                     keys[j]});
        }
      }
    } else {
      for (int j = 0; j < tiles; ++j) with(j, read(base + j * kWave));
    }
  };

  // The need-th largest key, a digit at a time: candidates whose digits so far are the
  // key's are counted by the next one.
  unsigned key = 0xffffffffu;
  int ties = 0;  // of the key's equals, that many are kept
  if (f.need > 0) {
    int left = f.need;
    unsigned known = 0;  // the digits so far, and which bits they are
    unsigned mask = 0;
#pragma unroll 1
    for (int shift = 32 - kDigit; ; shift = max(shift - kDigit, 0)) {
      const int width = mask == 0 || shift > 0 ? kDigit : 32 - 2 * kDigit;
      for (int i = threadIdx.x; i < kBins; i += kSelectThreads) lds.bins[i] = 0;
      __syncthreads();
      each([&](int, const Place& p) {
        if (p.kind == kCandidate && (p.key & mask) == known) {
          atomicAdd(&lds.bins[(p.key >> shift) & ((1u << width) - 1u)], 1);
        }
      });
      __syncthreads();
      // thread t: bins kBins - 1 - 2 t and the one below it
      const int b0 = kBins - 1 - 2 * static_cast<int>(threadIdx.x);
      const int n0 = lds.bins[b0], n1 = lds.bins[b0 - 1];
      int sum;
      const int above = BlockBefore(n0 + n1, lds.wave_sums, &sum);
      if (above < left && left <= above + n0 + n1) {
        const bool second = left > above + n0;
        lds.found_digit = static_cast<unsigned>(second ? b0 - 1 : b0);
        lds.found_above = second ? above + n0 : above;
      }
      __syncthreads();
      left -= lds.found_above;
      known |= lds.found_digit << shift;
      mask |= ((1u << width) - 1u) << shift;
      if (shift == 0) break;
    }
    key = known;
    ties = left;
  }

  // What each wave keeps, then where its kept places go.
  const bool any = f.need > 0;
  int sure = 0, equal = 0;
  each([&](int, const Place& p) {
    const bool candidate = any && p.kind == kCandidate;
    sure += __popcll(__ballot(p.kind == kAlways || (candidate && p.key > key)));
    equal += __popcll(__ballot(candidate && p.key == key));
  });
  __syncthreads();
  if (lane == 0) {
    lds.wave_sums[wave] = sure;
    lds.wave_ties[wave] = equal;
  }
  __syncthreads();
  int at = 0, ties_before = 0;
  for (int w = 0; w < wave; ++w) {
    at += lds.wave_sums[w] + max(min(ties - ties_before, lds.wave_ties[w]), 0);
    ties_before += lds.wave_ties[w];
  }
  int* kept = a.kept + (static_cast<int64_t>(f.r) * c.heads + f.head) * a.keep;
  const unsigned long long below = (1ull << lane) - 1ull;
  each([&](int j, const Place& p) {
    const bool candidate = any && p.kind == kCandidate;
    const bool tie = candidate && p.key == key;
    const unsigned long long tied = __ballot(tie);
    const bool keep = p.kind == kAlways || (candidate && p.key > key) ||
                      (tie && ties_before + static_cast<int>(__popcll(tied & below)) < ties);
    const unsigned long long taken = __ballot(keep);
    if (keep) kept[at + __popcll(taken & below)] = base + j * kWave;
    at += __popcll(taken);
    ties_before += __popcll(tied);
  });
  for (int i = f.count + threadIdx.x; i < a.keep; i += kSelectThreads) kept[i] = -1;
}

// ---- the move ---------------------------------------------------------------------

// Where a kept token lies.
struct Source {
  int page;  // < 0: none
  int off;
  float key_scale;
  float value_scale;
};

// The largest magnitude of four codes' numbers (finite ones).
template <int FMT>
__device__ __forceinline__ float MostOf4(unsigned w) {
  float x[4];
  Numbers4<FMT>(w, x);
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(x[i]));  // (fmaxf passes over NaN)
  return most;
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

// Grid (key heads * new pages, batch): one new page of one key head.  Waves 2 i have the
// keys, 2 i + 1 the values of chunks i, i + kWaves / 2, ... of 16 tokens (U of them) in
// registers, as codes: keys lane l unit l + 64 j (16 dims) of the chunk's [16][dim],
// values lane l dims l + 64 j, all 16 tokens.  NU = ceil(dim / 64).
template <int FMT, int NU, int U>
__global__ __launch_bounds__(512) void Kv8EvictMoveKernel(Kv8EvictArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ double wave_most[8];
  const Kv8View& c = a.c;
  const int D = c.dim, units = D / 16, ps = c.page;
  const int head = blockIdx.x % c.heads, index = blockIdx.x / c.heads, r = blockIdx.y;
  const int count = min(a.kept_tokens[r] - index * ps, ps);
  if (count <= 0) return;
  const int page = a.new_ids[static_cast<int64_t>(r) * a.new_stride + index];
  if (!InPool(page, c.capacity)) {
    if (threadIdx.x == 0) ReportFailure(a.fail, kFailPageId);
    return;
  }
  Kv8Request q;
  if (!Kv8ReadList(a.b, r, &q)) return;
  Source* source = reinterpret_cast<Source*>(smem);
  uint8_t* tile = smem + sizeof(Source) * ps;  // the new keys (for their mean)
  const int* kept = a.kept + (static_cast<int64_t>(r) * c.heads + head) * a.keep + index * ps;
  const int64_t to = static_cast<int64_t>(page) * c.heads + head;
  for (int i = threadIdx.x; i < ps; i += blockDim.x) {
    Source s = {-1, 0, 0.0f, 0.0f};
    float w = 0.0f;
    if (i < count) {
      const int place = kept[i], slot = place / ps;
      s.off = place - slot * ps;
      s.page = a.b.page_ids[q.list + slot];
      const int64_t at = static_cast<int64_t>(s.page) * c.heads + head;
      s.key_scale = c.key_scales[at];
      s.value_scale = c.value_scales[at];
      w = a.weights[at * ps + s.off];
    }
    source[i] = s;
    a.weights[to * ps + i] = w;
  }
  if (threadIdx.x == 0 && head == 0) c.token_counts[page] = count;
  __syncthreads();

  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int waves = blockDim.x / kWave;
  const bool is_key = (wave & 1) == 0;
  const int page_bytes = ps * D;
  unsigned w[U][NU][4];
  double most = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int chunk = wave / 2 + waves / 2 * u;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[u][j][i] = 0u;
    }
    if (chunk >= c.chunks) continue;
    if (is_key) {
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        const int i = lane + kWave * j;
        if (i < D) {
          const int token = i / units;
          const Source s = source[16 * chunk + token];
          if (s.page >= 0) {
            const uint4 x = *reinterpret_cast<const uint4*>(
                c.keys + (static_cast<int64_t>(s.page) * c.heads + head) * page_bytes + s.off * D +
                16 * (i - token * units));
            w[u][j][0] = x.x;
            w[u][j][1] = x.y;
            w[u][j][2] = x.z;
            w[u][j][3] = x.w;
          }
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const Source s = source[16 * chunk + t];
        if (s.page >= 0) {
          const uint8_t* p = c.values +
                             (static_cast<int64_t>(s.page) * c.heads + head) * page_bytes +
                             (s.off >> 4) * (16 * D) + (s.off & 15);
#pragma unroll
          for (int j = 0; j < NU; ++j) {
            const int d = lane + kWave * j;
            if (d < D) w[u][j][t >> 2] |= static_cast<unsigned>(p[d * 16]) << (8 * (t & 3));
          }
        }
      }
    }
  }
  // The largest number.
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int chunk = wave / 2 + waves / 2 * u;
    if (chunk >= c.chunks) continue;
    if (is_key) {
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        const int i = lane + kWave * j;
        if (i < D) {
          float top = 0.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k) top = fmaxf(top, MostOf4<FMT>(w[u][j][k]));
          most = fmax(most, static_cast<double>(top) *
                                static_cast<double>(source[16 * chunk + i / units].key_scale));
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        double scale[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          scale[e] = static_cast<double>(source[16 * chunk + 4 * k + e].value_scale);
        }
#pragma unroll
        for (int j = 0; j < NU; ++j) {
          float x[4];
          Numbers4<FMT>(w[u][j][k], x);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            most = fmax(most, fabs(static_cast<double>(x[e])) * scale[e]);
          }
        }
      }
    }
  }
  most = WaveMost(most);
  if (lane == 0) wave_most[wave] = most;
  __syncthreads();
  most = 0.0;
  for (int i = wave & 1; i < waves; i += 2) most = fmax(most, wave_most[i]);
  Scale scale;
  scale.Set<FMT>(ScaleForNumber<FMT>(most));
  if (threadIdx.x == 0) c.key_scales[to] = scale.s;
  if (threadIdx.x == kWave) c.value_scales[to] = scale.s;

  // Brought to it.
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int chunk = wave / 2 + waves / 2 * u;
    if (chunk >= c.chunks) continue;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int i = lane + kWave * j;
      if (i >= D) continue;
      unsigned x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float n[4];
        Numbers4<FMT>(w[u][j][k], n);
        double y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float had = is_key ? source[16 * chunk + i / units].key_scale
                                   : source[16 * chunk + 4 * k + e].value_scale;
          y[e] = static_cast<double>(n[e]) * static_cast<double>(had);
        }
        x[k] = Codes4<FMT>(y[0], y[1], y[2], y[3], scale);
      }
      const uint4 out = make_uint4(x[0], x[1], x[2], x[3]);
      const int64_t at = to * page_bytes + chunk * 16 * D + 16 * i;
      *reinterpret_cast<uint4*>((is_key ? c.keys : c.values) + at) = out;
      if (is_key && c.summaries != nullptr) {
        *reinterpret_cast<uint4*>(tile + chunk * 16 * D + 16 * i) = out;
      }
    }
  }
  if (c.summaries == nullptr) return;
  __syncthreads();
  __shared__ float key_scale;
  if (threadIdx.x == 0) key_scale = scale.s;
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float sum = 0.0f;
    for (int t = 0; t < count; ++t) {
      float x[4];
      Numbers4<FMT>(tile[t * D + d], x);
      sum += x[0];
    }
    c.summaries[to * D + d] =
        static_cast<float>(static_cast<double>(sum) * static_cast<double>(key_scale) / count);
  }
}

size_t MoveLdsBytes(const Kv8View& c) {
  return sizeof(Source) * c.page + static_cast<size_t>(c.page) * c.dim;
}

// Calls f with the kernel of a head and page size.
template <int FMT, int NU, typename F>
void WithMove(int chunks, F&& f) {
  if (chunks <= 4) return f(Kv8EvictMoveKernel<FMT, NU, 1>);
  if (chunks <= 8) return f(Kv8EvictMoveKernel<FMT, NU, 2>);
  return f(Kv8EvictMoveKernel<FMT, NU, 4>);
}
template <typename F>
void WithMove(const Kv8View& c, F&& f) {
  const bool int8 = c.format == DSD_KV8_INT8;
  if (c.dim <= 64) {
    return int8 ? WithMove<DSD_KV8_INT8, 1>(c.chunks, f) : WithMove<DSD_KV8_E4M3, 1>(c.chunks, f);
  }
  if (c.dim <= 128) {
    return int8 ? WithMove<DSD_KV8_INT8, 2>(c.chunks, f) : WithMove<DSD_KV8_E4M3, 2>(c.chunks, f);
  }
  return int8 ? WithMove<DSD_KV8_INT8, 4>(c.chunks, f) : WithMove<DSD_KV8_E4M3, 4>(c.chunks, f);
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
