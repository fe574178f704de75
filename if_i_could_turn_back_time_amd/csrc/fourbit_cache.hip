// Writing to and evicting from the 8-bit key/value cache (layout: fourbit.h).
#include "fourbit_cache.h"

#include <algorithm>

namespace {

using namespace fbc;

// Largest of the workgroup's 256 values; `lds` holds 4 floats.  Every thread calls it.
__device__ inline float block_max(float v, float* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
  return v;
}

struct NewTokens {
  const void *k, *v;
  int64_t k_token, k_head, v_token, v_head;
  bool k_vec, v_vec;
};

// ---------------------------------------------------------------------------------
// Append.  Workgroup = (sequence, head, keys or values) x (one block of 32 tokens that gets new
// ones): the block's scale needs all of its new values, 32 D at most, which stay in registers
// (8 channels of one token per thread and step) between the maximum and the codes.  A value
// block is turned to its 16-token sides through LDS when it is full; single tokens are written
// byte by byte.  Earlier codes are read only where the scale grows.
// ---------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void cache_append_kernel(Cache c, NewTokens x) {
  __shared__ float red[4];
  __shared__ __align__(16) uint8_t side[kBlock * kMaxDim];
  const int tid = threadIdx.x;
  const int which = blockIdx.x & 1;
  const unsigned bh = blockIdx.x >> 1;
  const int b = bh / c.H, h = bh - b * c.H;
  int row0, n;
  c.rows(b, row0, n);
  const int start = c.lens[b];
  if (start < 0 || n < 1) return;
  const int64_t end64 = (int64_t)start + n;
  const int end = end64 < c.capacity() ? (int)end64 : c.capacity();
  const int64_t blk64 = (int64_t)start / kBlock + blockIdx.y;
  if (blk64 * kBlock >= end) return;
  const int blk = (int)blk64, pos0 = blk * kBlock;
  int at;
  const int page = c.page_of(b, blk, at);
  if (page < 0) return;

  const int64_t bi = c.block_index(page, h, at);
  uint8_t* const scale = (which ? c.vs : c.ks) + bi;
  uint8_t* const codes = (which ? c.v : c.k) + bi * kBlock * c.D;
  const int pieces = c.D / 8, total = kBlock * pieces;
  const int lo = max(start - pos0, 0), hi = min(end - pos0, kBlock);  // the new ones' slots
  float val[4][8];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid + 256 * i, t = e / pieces, d = (e - t * pieces) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) val[i][j] = 0.f;
    if (e < total && t >= lo && t < hi) {
      const int64_t row = row0 + (pos0 + t - start);
      if (which)
        load8<DT>(x.v, row * x.v_token + h * x.v_head + d, x.v_vec, val[i]);
      else
        load8<DT>(x.k, row * x.k_token + h * x.k_head + d, x.k_vec, val[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(val[i][j]));
  }
  amax = block_max(amax, red);
  const int before = (int)*scale - 127;
  int e2 = block_exp(amax);
  if (lo > 0) e2 = max(e2, before);  // earlier tokens keep what they have, or round to more
  __syncthreads();  // every thread has read the scale
  if (tid == 0) *scale = (uint8_t)(e2 + 127);
  const float inv = exp2i(min(max(-e2, -126), 127));

  u32x2 code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) val[i][j] *= inv;
    code[i] = encode8(val[i]);
  }
  const bool full = lo == 0 && hi == kBlock;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid + 256 * i, t = e / pieces, d = (e - t * pieces) * 8;
    if (e >= total || t < lo || t >= hi) continue;
    if (!which) {
      *reinterpret_cast<u32x2*>(codes + t * c.D + d) = code[i];
      continue;
    }
    uint8_t* const to = (full ? side : codes) + (t / kSide) * c.D * kSide + d * kSide + t % kSide;
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j * kSide] = (uint8_t)(code[i][j / 4] >> (8 * (j & 3)));
  }
  if (which && full) {
    __syncthreads();
    for (int e = tid; e < 2 * c.D; e += 256)
      *reinterpret_cast<u32x4*>(codes + e * 16) = *reinterpret_cast<const u32x4*>(side + e * 16);
  }
  if (lo > 0 && e2 > before) {  // the same for the whole workgroup
    const float f = exp2i(max(before - e2, -126));
    for (int e = tid; e < lo * pieces; e += 256) {
      const int t = e / pieces, d = (e - t * pieces) * 8;
      u32x2 old;
      uint8_t* const from = which ? codes + (t / kSide) * c.D * kSide + d * kSide + t % kSide
                                  : codes + t * c.D + d;
      if (which) {
        unsigned u[2] = {0, 0};
        for (int j = 0; j < 8; ++j) u[j / 4] |= (unsigned)from[j * kSide] << (8 * (j & 3));
        old = u32x2{u[0], u[1]};
      } else {
        old = *reinterpret_cast<const u32x2*>(from);
      }
      float v[8];
      decode8(old, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f;
      const u32x2 now = encode8(v);
      if (which)
        for (int j = 0; j < 8; ++j) from[j * kSide] = (uint8_t)(now[j / 4] >> (8 * (j & 3)));
      else
        *reinterpret_cast<u32x2*>(from) = now;
    }
  }
}

// ---------------------------------------------------------------------------------
// Eviction, first half: which tokens of a head stay.  Workgroup = (head, sequence).  A radix
// select over the order-preserving 32-bit keys of the weights, 8 bits a pass, finds the key of
// the last token that stays; a second walk in token order writes down what lies above it, as
// many of its equals as are left, earliest first, and the recent ones.
// ---------------------------------------------------------------------------------
__device__ inline unsigned weight_key(float w) {
  unsigned b = __builtin_bit_cast(unsigned, w);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0;  // NaN: below every number
  if (b == 0x80000000u) b = 0;
  return (b >> 31) ? ~b : (b | 0x80000000u);
}

constexpr int kSelect = 1024;

__global__ __launch_bounds__(kSelect) void evict_select_kernel(
    Cache c, const float* __restrict__ weights, int64_t w_seq, int64_t w_head, int w_tokens,
    int keep, int recent, int32_t* __restrict__ kept, float* __restrict__ new_weights,
    int32_t* __restrict__ new_lens) {
  __shared__ unsigned hist[256];
  __shared__ unsigned chosen[2];  // digit, how many above it
  __shared__ int wave_count[2][kSelect / 64];
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
  const int lane = tid & 63, wave = tid >> 6;
  const int n = min(min(max(c.lens[b], 0), c.capacity()), w_tokens);
  const float* const w = weights + b * w_seq + h * w_head;
  const int64_t out = ((int64_t)b * c.H + h) * keep;
  if (h == 0 && tid == 0) new_lens[b] = min(n, keep);
  const int m = max(n - recent, 0);          // the tokens that compete
  int need = keep - min(recent, n);          // for so many places
  const bool all = n <= keep;
  unsigned last = 0;  // key of the last one that stays
  int above = 0;      // how many have a larger one
  if (!all && need > 0) {
    unsigned prefix = 0, mask = 0;
    int left = need;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelect) hist[i] = 0;
      __syncthreads();
      for (int t = tid; t < m; t += kSelect) {
        const unsigned key = weight_key(w[t]);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        unsigned sum = 0;
        while (d > 0 && sum + hist[d] < (unsigned)left) sum += hist[d--];
        chosen[0] = d;
        chosen[1] = sum;
      }
      __syncthreads();
      prefix |= chosen[0] << shift;
      mask |= 255u << shift;
      left -= (int)chosen[1];
      above += (int)chosen[1];
      __syncthreads();
    }
    last = prefix;
  }
  // tokens in order: larger keys, the first need - above equal ones, and the recent ones
  int written = 0, equal_seen = 0;
  const int equal_most = need - above;
  for (int t0 = 0; t0 < n; t0 += kSelect) {
    const int t = t0 + tid;
    bool more = false, equal = false;
    if (t < n) {
      if (all || t >= m) {
        more = true;
      } else if (need > 0) {
        const unsigned key = weight_key(w[t]);
        more = key > last;
        equal = key == last;
      }
    }
    const unsigned long long eq = __ballot(equal);
    if (lane == 0) wave_count[0][wave] = __popcll(eq);
    __syncthreads();
    int rank = equal_seen + __popcll(eq & ((1ull << lane) - 1)), eq_all = 0;
    for (int i = 0; i < kSelect / 64; ++i) {
      if (i < wave) rank += wave_count[0][i];
      eq_all += wave_count[0][i];
    }
    const bool stays = more || (equal && rank < equal_most);
    const unsigned long long st = __ballot(stays);
    if (lane == 0) wave_count[1][wave] = __popcll(st);
    __syncthreads();
    int place = written + __popcll(st & ((1ull << lane) - 1)), st_all = 0;
    for (int i = 0; i < kSelect / 64; ++i) {
      if (i < wave) place += wave_count[1][i];
      st_all += wave_count[1][i];
    }
    if (stays && place < keep) {
      kept[out + place] = t;
      if (new_weights) new_weights[out + place] = w[t];
    }
    written += st_all;
    equal_seen += eq_all;
    __syncthreads();
  }
  for (int i = written + tid; i < keep; i += kSelect) {
    kept[out + i] = -1;
    if (new_weights) new_weights[out + i] = 0.f;
  }
}

// ---------------------------------------------------------------------------------
// Second half: the kept tokens to their new pages.  Workgroup = (one new block, keys or values)
// x head x sequence, as an append of 32 tokens that are decoded from the cache.
// ---------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void evict_move_kernel(Cache c, Cache to, int keep,
                                                         const int32_t* __restrict__ kept) {
  __shared__ float red[4];
  __shared__ __align__(16) uint8_t side[kBlock * kMaxDim];
  const int tid = threadIdx.x, which = blockIdx.x & 1, blk = blockIdx.x >> 1;
  const int h = blockIdx.y, b = blockIdx.z;
  const int32_t* const ids = kept + ((int64_t)b * c.H + h) * keep;
  if (ids[blk * kBlock] < 0) return;
  int at;
  const int page = to.page_of(b, blk, at);
  if (page < 0) return;
  const int pieces = c.D / 8, total = kBlock * pieces;
  float val[4][8];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid + 256 * i, t = e / pieces, d = (e - t * pieces) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) val[i][j] = 0.f;
    const int place = blk * kBlock + t;
    const int from = e < total && place < keep ? ids[place] : -1;
    int src_at, src = -1;
    if (from >= 0) src = c.page_of(b, from / kBlock, src_at);
    if (src >= 0) {
      const int64_t bi = c.block_index(src, h, src_at);
      const int slot = from % kBlock;
      u32x2 code;
      if (which) {
        const uint8_t* p = c.v + bi * kBlock * c.D + (slot / kSide) * c.D * kSide + d * kSide +
                           slot % kSide;
        unsigned u[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j / 4] |= (unsigned)p[j * kSide] << (8 * (j & 3));
        code = u32x2{u[0], u[1]};
      } else {
        code = *reinterpret_cast<const u32x2*>(c.k + bi * kBlock * c.D + slot * c.D + d);
      }
      const float f = exp2i(min(max((int)(which ? c.vs : c.ks)[bi] - 127, -126), 127));
      decode8(code, val[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        val[i][j] *= f;
        amax = fmaxf(amax, finite_abs(val[i][j]));
      }
    }
  }
  amax = block_max(amax, red);
  const int e2 = block_exp(amax);
  const float inv = exp2i(min(max(-e2, -126), 127));
  const int64_t bi = to.block_index(page, h, at);
  uint8_t* const codes = (which ? to.v : to.k) + bi * kBlock * c.D;
  if (tid == 0) (which ? to.vs : to.ks)[bi] = (uint8_t)(e2 + 127);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid + 256 * i, t = e / pieces, d = (e - t * pieces) * 8;
    if (e >= total) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) val[i][j] *= inv;
    const u32x2 code = encode8(val[i]);
    if (!which) {
      *reinterpret_cast<u32x2*>(codes + t * c.D + d) = code;
      continue;
    }
    uint8_t* const s = side + (t / kSide) * c.D * kSide + d * kSide + t % kSide;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j * kSide] = (uint8_t)(code[j / 4] >> (8 * (j & 3)));
  }
  if (which) {
    __syncthreads();
    for (int e = tid; e < 2 * c.D; e += 256)
      *reinterpret_cast<u32x4*>(codes + e * 16) = *reinterpret_cast<const u32x4*>(side + e * 16);
  }
}

bool vec16(const void* p, int64_t a, int64_t b, int bytes) {
  return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(a * bytes) | (uintptr_t)(b * bytes)) & 15u);
}

}  // namespace

extern "C" {

int fb_cache_append(const fb_cache_t* c, const fb_seqs_t* s, const void* k, int64_t k_token,
                    int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                    int32_t dtype, void* stream) {
  Cache kc;
  const int st = check_cache(c, s, kc);
  if (st != FB_OK) return st;
  if (dtype != FB_DT_F16 && dtype != FB_DT_BF16 && dtype != FB_DT_F32) return FB_ERR_DTYPE;
  if (s->tokens == 0 || s->max_new == 0) return FB_OK;
  if (!k || !v) return FB_ERR_NULL;
  const int bytes = dtype == FB_DT_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & (bytes - 1))
    return FB_ERR_ALIGN;
  // blocks that max_new tokens can touch from any start on
  const int64_t ny = ((int64_t)std::min(s->max_new, s->tokens) + kBlock - 2) / kBlock + 1;
  const int64_t nx = (int64_t)s->seqs * c->heads * 2;
  if (ny > 65535 || nx > INT32_MAX) return FB_ERR_SHAPE;
  const NewTokens x{k,      v,      k_token, k_head, v_token,
                    v_head, vec16(k, k_token, k_head, bytes), vec16(v, v_token, v_head, bytes)};
  const dim3 grid((unsigned)nx, (unsigned)ny);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  if (dtype == FB_DT_F16)
    hipLaunchKernelGGL(cache_append_kernel<FB_DT_F16>, grid, dim3(256), 0, hs, kc, x);
  else if (dtype == FB_DT_BF16)
    hipLaunchKernelGGL(cache_append_kernel<FB_DT_BF16>, grid, dim3(256), 0, hs, kc, x);
  else
    hipLaunchKernelGGL(cache_append_kernel<FB_DT_F32>, grid, dim3(256), 0, hs, kc, x);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

int fb_cache_evict(const fb_cache_t* c, const fb_seqs_t* s, const float* weights, int64_t w_seq,
                   int64_t w_head, int32_t w_tokens, int32_t keep, int32_t recent,
                   const int32_t* new_table, int64_t new_stride, int32_t new_pages,
                   int32_t* kept, float* new_weights, int32_t* new_lens, void* stream) {
  Cache kc;
  const int st = check_cache(c, s, kc);
  if (st != FB_OK) return st;
  if (!weights || !new_table || !kept || !new_lens) return FB_ERR_NULL;
  if (keep < 1 || recent < 0 || recent > keep || w_tokens < 1 || new_pages < 1 ||
      new_stride < new_pages || (int64_t)new_pages * c->page < keep)
    return FB_ERR_SHAPE;
  for (const void* p : {(const void*)weights, (const void*)new_table, (const void*)kept,
                        (const void*)new_weights, (const void*)new_lens})
    if (reinterpret_cast<uintptr_t>(p) & 3u) return FB_ERR_ALIGN;
  Cache to = kc;
  to.table = new_table;
  to.table_stride = new_stride;
  to.max_pages = new_pages;
  const int64_t nx = ((int64_t)keep + kBlock - 1) / kBlock * 2;
  if (nx > INT32_MAX) return FB_ERR_SHAPE;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3(c->heads, s->seqs), dim3(kSelect), 0, hs, kc,
                     weights, w_seq, w_head, w_tokens, keep, recent, kept, new_weights, new_lens);
  if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)nx, c->heads, s->seqs), dim3(256), 0, hs,
                     kc, to, keep, kept);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

}  // extern "C"
