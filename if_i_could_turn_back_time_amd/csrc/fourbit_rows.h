// Rows of fp16, bf16 or fp32 in 16-byte pieces, at any alignment.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "fourbit.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // rows of odd widths begin anywhere

template <int DT>
struct Of;
template <>
struct Of<FB_DT_F32> {
  using T = float;
  static constexpr int V = 4;
};
template <>
struct Of<FB_DT_F16> {
  using T = _Float16;
  static constexpr int V = 8;
};
template <>
struct Of<FB_DT_BF16> {
  using T = __bf16;
  static constexpr int V = 8;
};

// 16 bytes of values from p[from + at] on (at: a multiple of as many), of a row that begins at p[from]
// and has `n` more there.  The last piece of a row of an odd width is read where it ends with the row,
// and `settled` moves its values to the front (value by value it took three times as long as all the
// others); 0 beyond the row.  Apart, so that a caller can ask for many pieces before it needs one.
// EVEN: rows are whole pieces; the rest of the code, and half the registers, go then.
template <int DT, bool EVEN = false>
__device__ inline u32x4 raw(const void* p, int64_t from, int at, int n) {
  using T = typename Of<DT>::T;
  constexpr int V = Of<DT>::V;
  const T* s = static_cast<const T*>(p) + from + at;
  u32x4 w{0, 0, 0, 0};
  if constexpr (EVEN) {
    if (n > 0) w = *reinterpret_cast<const u32x4_any*>(s);
  } else if (n > 0 && (at || n >= V)) {
    w = *reinterpret_cast<const u32x4_any*>(s + min(n - V, 0));
  } else if (n > 0) {  // a row shorter than a piece
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) {
        if constexpr (DT == FB_DT_F32)
          w[i] = __builtin_bit_cast(unsigned, s[i]);
        else
          w[i / 2] |= (unsigned)__builtin_bit_cast(unsigned short, s[i]) << (16 * (i & 1));
      }
  }
  return w;
}
template <int DT, bool EVEN = false>
__device__ inline u32x4 settled(const u32x4& w, int at, int n) {
  constexpr int V = Of<DT>::V;
  if (EVEN || n >= V || n <= 0 || !at) return w;
  const unsigned bits = (V - n) * (128 / V);
  unsigned long long lo = w[0] | (unsigned long long)w[1] << 32;
  unsigned long long hi = w[2] | (unsigned long long)w[3] << 32;
  if (bits >= 64) {
    lo = hi >> (bits - 64);
    hi = 0;
  } else {
    lo = lo >> bits | hi << (64 - bits);
    hi >>= bits;
  }
  return u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
}
template <int DT>
__device__ inline void unpack(const u32x4& w, float (&o)[Of<DT>::V]) {
#pragma unroll
  for (int i = 0; i < Of<DT>::V; ++i) {
    if constexpr (DT == FB_DT_F32) {
      const unsigned u = w[i];  // a bit cast of a vector's element takes the first one
      o[i] = __builtin_bit_cast(float, u);
    } else {
      const unsigned u = w[i / 2];
      if constexpr (DT == FB_DT_F16)
        o[i] = (float)__builtin_bit_cast(_Float16, (unsigned short)(u >> (16 * (i & 1))));
      else
        o[i] = __builtin_bit_cast(float, i & 1 ? u & 0xFFFF0000u : u << 16);
    }
  }
}
template <int DT, bool EVEN = false>
__device__ inline void load(const void* p, int64_t from, int at, int n, float (&o)[Of<DT>::V]) {
  unpack<DT>(settled<DT, EVEN>(raw<DT, EVEN>(p, from, at, n), at, n), o);
}
template <int DT, bool EVEN = false>
__device__ inline void store(void* p, int64_t at, int n, const float (&v)[Of<DT>::V]) {
  using T = typename Of<DT>::T;
  constexpr int V = Of<DT>::V;
  T* d = static_cast<T*>(p) + at;
  if (EVEN ? n > 0 : n >= V) {
    T o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (T)v[i];
    u32x4 w;
    __builtin_memcpy(&w, o, 16);
    *reinterpret_cast<u32x4_any*>(d) = w;
  } else if constexpr (!EVEN) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) d[i] = (T)v[i];
  }
}

}  // namespace
