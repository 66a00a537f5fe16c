// kv8_codes.h -- numbers to the 8-bit cache's codes and back.
#pragma once

#include "kv8_device.h"

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

}  // namespace
}  // namespace dsdk
