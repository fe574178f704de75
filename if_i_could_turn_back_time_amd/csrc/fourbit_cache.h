// What the kernels of the 8-bit key/value cache share: its layout, E4M3 codes and block scales.
#ifndef FOURBIT_CACHE_H
#define FOURBIT_CACHE_H

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fourbit.h"

namespace fbc {

constexpr int kBlock = 32;     // tokens of one scale
constexpr int kSide = 16;      // tokens of one channel side by side in v
constexpr int kMinExp = -100;  // of a block's scale; a block of zeros has it
constexpr int kMaxDim = 256;

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// What a kernel needs of a cache and its sequences, checked on the host.
struct Cache {
  uint8_t *k, *v, *ks, *vs;
  const int32_t* table;
  int64_t table_stride;
  const int32_t *lens, *cu;
  int32_t pages, H, D, P, max_pages, T, B;

  __device__ int capacity() const {
    const int64_t n = (int64_t)max_pages * P;
    return n > 0x7FFFFFE0 ? 0x7FFFFFE0 : (int)n;
  }
  // First row and number of sequence b's new tokens, within [0, T).
  __device__ void rows(int b, int& first, int& n) const {
    if (!cu) {
      first = b;
      n = 1;
      return;
    }
    first = min(max(cu[b], 0), T);
    n = min(max(cu[b + 1], first), T) - first;
  }
  // The page of a sequence's block and the block's place in it; -1: none in the pool.
  __device__ int page_of(int b, int block, int& at) const {
    const unsigned per = (unsigned)P / kBlock;
    const unsigned pg = (unsigned)block / per;
    at = block - (int)(pg * per);
    if (pg >= (unsigned)max_pages) return -1;
    const int id = table[b * table_stride + pg];
    return (unsigned)id < (unsigned)pages ? id : -1;
  }
  // Block `at` of a page and head, counted over the whole pool.
  __device__ int64_t block_index(int page, int h, int at) const {
    return ((int64_t)page * H + h) * (P / kBlock) + at;
  }
};

// Host: checks a cache and its sequences.
inline int check_cache(const fb_cache_t* c, const fb_seqs_t* s, Cache& k) {
  if (!c || !s || !c->k || !c->v || !c->k_scale || !c->v_scale || !s->table || !s->lens)
    return FB_ERR_NULL;
  if (c->pages < 1 || c->pages > INT32_MAX || c->heads < 1 || c->heads > 4096 ||
      c->head_dim < 16 || c->head_dim > kMaxDim || c->head_dim % 16 || c->page < kBlock ||
      c->page > (1 << 24) || c->page % kBlock || s->seqs < 1 || s->seqs > 65535 ||
      s->max_pages < 1 || s->table_stride < s->max_pages || s->tokens < 0 || s->max_new < 0 ||
      s->max_len < 0 || (!s->cu && s->tokens != s->seqs))
    return FB_ERR_SHAPE;
  for (const void* p : {(const void*)c->k, (const void*)c->v})
    if (reinterpret_cast<uintptr_t>(p) & 15u) return FB_ERR_ALIGN;
  for (const void* p : {(const void*)s->table, (const void*)s->lens, (const void*)s->cu})
    if (reinterpret_cast<uintptr_t>(p) & 3u) return FB_ERR_ALIGN;
  k = Cache{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale,
            s->table, s->table_stride, s->lens, s->cu, (int32_t)c->pages, c->heads, c->head_dim,
            c->page, s->max_pages, s->tokens, s->seqs};
  return FB_OK;
}

// Host: whether `groups` workgroups of `threads` can be launched in one direction.  Their threads are
// counted in 32 bits: beyond that some would not run.
inline bool fits_grid(int64_t groups, int threads) { return groups * threads <= UINT32_MAX; }

// 2^e for e in [-126, 127].
__device__ inline float exp2i(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }

// The least e >= kMinExp with amax <= 448 * 2^e; amax finite and >= 0.
__device__ inline int block_exp(float amax) {
  const unsigned b = __builtin_bit_cast(unsigned, amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u);
  return max(e, kMinExp);
}

__device__ inline float finite_abs(float v) {
  const float a = __builtin_fabsf(v);
  return a < __builtin_inff() ? a : 0.f;
}

// Eight finite values, scaled into range already, as E4M3 codes: round to nearest even.
__device__ inline u32x2 encode8_finite(const float (&v)[8]) {
  u32x2 r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int x = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w], v[4 * w + 1], 0, false);
    x = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w + 2], v[4 * w + 3], x, true);
    r[w] = (unsigned)x;
  }
  return r;
}

// The same of any values: what is not finite becomes NaN.
__device__ inline u32x2 encode8(const float (&v)[8]) {
  asm volatile("");  // seldom wanted: not to be worked out beside the other and chosen from
  u32x2 r = encode8_finite(v);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    unsigned u = r[w];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(__builtin_fabsf(v[4 * w + j]) < __builtin_inff()))
        u = (u & ~(0xFFu << (8 * j))) | (0x7Fu << (8 * j));
    r[w] = u;
  }
  return r;
}

__device__ inline void decode8(u32x2 c, float (&v)[8]) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], true);
    v[4 * w] = lo[0];
    v[4 * w + 1] = lo[1];
    v[4 * w + 2] = hi[0];
    v[4 * w + 3] = hi[1];
  }
}

// Sum of v over this lane and those before it.
__device__ inline int sum_to_lane(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31
  return v;
}

}  // namespace fbc

#endif
