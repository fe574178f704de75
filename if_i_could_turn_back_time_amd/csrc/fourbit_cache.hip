// Writing to and evicting from the 8-bit key/value cache (layout: fourbit.h).
#include "fourbit_cache.h"

#include <algorithm>

namespace {

using namespace fbc;

// Largest of the workgroup's values; `lds` holds 4.  Every thread calls it, once for each `lds`.
__device__ inline unsigned block_max(unsigned v, unsigned* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < (int)blockDim.x / 64; ++w) v = max(v, lds[w]);
  return v;
}

// Eight values of a tensor of dtype DT, as they lie.
template <int DT>
struct Eight {
  static constexpr int kWords = DT == FB_DT_F32 ? 8 : 4;
  unsigned w[kWords];

  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ void load(const void* base, int64_t at, bool vec) {
    const char* const p = static_cast<const char*>(base) + at * (DT == FB_DT_F32 ? 4 : 2);
    if (vec) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4 x = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (DT == FB_DT_F32) {
          w[i] = reinterpret_cast<const unsigned*>(p)[i];
        } else {
          const unsigned short* const u = reinterpret_cast<const unsigned short*>(p) + 2 * i;
          w[i] = (unsigned)u[0] | (unsigned)u[1] << 16;
        }
      }
    }
  }
  __device__ float value(int j) const {
    if constexpr (DT == FB_DT_F32) {
      return __builtin_bit_cast(float, w[j]);
    } else {
      const unsigned short u = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
      return DT == FB_DT_F16 ? (float)__builtin_bit_cast(_Float16, u)
                             : __builtin_bit_cast(float, (unsigned)u << 16);
    }
  }
  // Largest magnitude among these and `m`, as bits: of a type's values they are in order.
  __device__ unsigned max_bits(unsigned m) const {
    if constexpr (DT == FB_DT_F32) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      return m;
    } else {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 x = {(unsigned short)m, 0};
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const unsigned bits = w[i] & 0x7FFF7FFFu;
        x = __builtin_elementwise_max(x, __builtin_bit_cast(u16x2, bits));
      }
      return max((unsigned)x[0], (unsigned)x[1]);
    }
  }
  static constexpr unsigned kInf = DT == FB_DT_F32 ? 0x7F800000u : DT == FB_DT_F16 ? 0x7C00u : 0x7F80u;
  static __device__ float magnitude(unsigned bits) {
    if constexpr (DT == FB_DT_F32) return __builtin_bit_cast(float, bits);
    if constexpr (DT == FB_DT_F16) return (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
    return __builtin_bit_cast(float, bits << 16);
  }
};

struct NewTokens {
  const void *k, *v;
  int64_t k_token, k_head, v_token, v_head;
  bool k_vec, v_vec;
};

// ---------------------------------------------------------------------------------
// Append.  Workgroup = (sequence, head, keys or values) x (one block of 32 tokens that gets new
// ones), D threads rounded up to whole waves: the block's scale needs all of its new values, 32 D
// at most, which stay in registers as they came (4 tokens of 8 channels a thread) between the
// maximum, taken over their bits, and the codes.  Four tokens of a value's channel become one
// word; a full block's words go through LDS to whole 16-token sides.  Earlier codes are read only
// where the scale grows, and only a block that holds something not finite looks for it.
// ---------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void cache_append_kernel(Cache c, NewTokens x) {
  __shared__ unsigned red[2][4];
  __shared__ u32x4 side[2 * kMaxDim];
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

  const int pieces = c.D / 8;
  const int lo = max(start - pos0, 0), hi = min(end - pos0, kBlock);  // the new ones' slots
  const int quad = tid / pieces, piece = tid - quad * pieces;  // quad >= 8: nothing to do
  const int t0 = 4 * quad, d = 8 * piece;
  Eight<DT> raw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    raw[i].clear();
    if (t0 + i >= lo && t0 + i < hi) {
      const int64_t row = row0 + (pos0 + t0 + i - start);
      if (which)
        raw[i].load(x.v, row * x.v_token + h * x.v_head + d, x.v_vec);
      else
        raw[i].load(x.k, row * x.k_token + h * x.k_head + d, x.k_vec);
    }
  }
  const int64_t bi = c.block_index(page, h, at);
  uint8_t* const scale = (which ? c.vs : c.ks) + bi;
  uint8_t* const codes = (which ? c.v : c.k) + bi * kBlock * c.D;
  const int before = lo > 0 ? (int)*scale - 127 : kMinExp;  // read before the barrier below
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits = raw[i].max_bits(bits);
  bits = block_max(bits, red[0]);
  const bool finite = bits < Eight<DT>::kInf;
  float amax = Eight<DT>::magnitude(bits);
  if (!finite) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(raw[i].value(j)));
    amax = __builtin_bit_cast(float, block_max(__builtin_bit_cast(unsigned, amax), red[1]));
  }
  // earlier tokens keep what they have, or round to more
  const int e2 = max(block_exp(amax), before);
  if (tid == 0) *scale = (uint8_t)(e2 + 127);
  const float inv = exp2i(min(max(-e2, -126), 127));

  u32x2 code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float val[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) val[j] = raw[i].value(j) * inv;
    code[i] = finite ? encode8_finite(val) : encode8(val);
  }
  if (which) {
    // word j: this quad's four tokens of channel d + j
    unsigned word[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned pick = 0x0C0C0000u | (unsigned)(4 + (j & 3)) << 8 | (unsigned)(j & 3);
      const unsigned ab = __builtin_amdgcn_perm(code[1][j / 4], code[0][j / 4], pick);
      const unsigned cd = __builtin_amdgcn_perm(code[3][j / 4], code[2][j / 4], pick);
      word[j] = ab | cd << 16;
    }
    if (lo == 0 && hi == kBlock) {
      // 16 bytes a channel, their order turned by the piece so that a wave's words meet no bank
      // twice
      const int turn = (piece >> 1) & 7;
      if (quad < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          reinterpret_cast<unsigned*>(side + (quad >> 2) * c.D + (d + (j ^ turn)))[quad & 3] = word[j];
      }
      __syncthreads();
      for (int e = tid; e < 2 * c.D; e += blockDim.x) {
        const int ch = e < c.D ? e : e - c.D;
        reinterpret_cast<u32x4*>(codes)[e] = side[e - ch + (ch ^ ((ch >> 4) & 7))];
      }
    } else if (t0 + 3 >= lo && t0 < hi) {
      uint8_t* const to = codes + (quad >> 2) * c.D * kSide + d * kSide + (t0 & 15);
      if (t0 >= lo && t0 + 4 <= hi) {
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<unsigned*>(to + j * kSide) = word[j];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t0 + i >= lo && t0 + i < hi)
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j * kSide + i] = (uint8_t)(word[j] >> (8 * i));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (t0 + i >= lo && t0 + i < hi)
        *reinterpret_cast<u32x2*>(codes + (t0 + i) * c.D + d) = code[i];
  }
  if (lo > 0 && e2 > before) {  // the same for the whole workgroup
    const float f = exp2i(max(before - e2, -126));
    for (int e = tid; e < lo * pieces; e += blockDim.x) {
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
// Eviction, first half: which tokens of a head stay.  Workgroup = (head, sequence).  The key of the
// last token that stays is searched for two bits at a time over the order-preserving 32-bit keys of
// the weights, which stay in registers (KEYS of them a thread; longer sequences are read again for
// each step): comparisons are counted by ballot, so equal weights cost no more than others (a
// histogram's atomics do), and the search ends as soon as a bound parts the right number.  Then
// every 64 tokens are counted once, the counts summed in token order, and what lies above the
// key, as many of its equals as are left, earliest first, and the recent ones written down.  Bound
// by its barriers (16 steps), a few microseconds.
// ---------------------------------------------------------------------------------
__device__ inline unsigned weight_key(float w) {
  unsigned b = __builtin_bit_cast(unsigned, w);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0;  // NaN: below every number
  if (b == 0x80000000u) b = 0;
  return (b >> 31) ? ~b : (b | 0x80000000u);
}

constexpr int kSelect = 1024, kSelectWaves = kSelect / 64;

template <int KEYS>
__global__ __launch_bounds__(kSelect) void evict_select_kernel(
    Cache c, const float* __restrict__ weights, int64_t w_seq, int64_t w_head, int w_tokens,
    int keep, int recent, int32_t* __restrict__ kept, float* __restrict__ new_weights,
    int32_t* __restrict__ new_lens) {
  constexpr int kChunk = KEYS * kSelect;  // tokens held at once
  __shared__ int counted[17][3];  // keys above the bounds of each step, all waves' together
  __shared__ int chunk_sums[2];
  __shared__ int2 before[KEYS * kSelectWaves];  // larger and equal keys before 64 tokens
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
  const int lane = tid & 63, wave = tid >> 6;
  const int n = min(min(max(c.lens[b], 0), c.capacity()), w_tokens);
  const float* const w = weights + b * w_seq + h * w_head;
  const int64_t out = ((int64_t)b * c.H + h) * keep;
  if (h == 0 && tid == 0) new_lens[b] = min(n, keep);
  const int m = max(n - recent, 0);       // the tokens that compete
  const int need = keep - min(recent, n); // for so many places
  const bool all = n <= keep;
  unsigned key[KEYS];
  float weight[KEYS];
  const auto load = [&](int t0) {  // all of them asked for before the first is used
#pragma unroll
    for (int j = 0; j < KEYS; ++j) weight[j] = w[min(t0 + j * kSelect + tid, max(n - 1, 0))];
#pragma unroll
    for (int j = 0; j < KEYS; ++j)
      key[j] = t0 + j * kSelect + tid < m ? weight_key(weight[j]) : 0u;
  };
  const int chunks = (n + kChunk - 1) / kChunk;
  load(0);
  for (int i = tid; i < 17 * 3; i += kSelect) counted[i / 3][i % 3] = 0;
  __syncthreads();
  // the largest `last` with at least `need` keys >= last (0: all of them; a key of 0 is a NaN's)
  unsigned last = 0;
  int reached = m;  // keys >= last
  if (!all && need > 0) {
    for (int shift = 30; shift >= 0 && reached != need; shift -= 2) {
      int found[3] = {0, 0, 0};
      for (int ch = 0; ch < chunks; ++ch) {
        if (chunks > 1) load(ch * kChunk);
#pragma unroll
        for (int j = 0; j < KEYS; ++j)
#pragma unroll
          for (int d = 0; d < 3; ++d)
            found[d] += __popcll(__ballot(key[j] >= (last | (unsigned)(d + 1) << shift)));
      }
      int(&total)[3] = counted[shift >> 1];
      if (lane < 3) atomicAdd(&total[lane], lane == 0 ? found[0] : lane == 1 ? found[1] : found[2]);
      __syncthreads();
      int digit = 0;
#pragma unroll
      for (int d = 0; d < 3; ++d) {
        const int sum = __builtin_amdgcn_readfirstlane(total[d]);
        if (sum >= need) {
          digit = d + 1;
          reached = sum;
        }
      }
      last |= (unsigned)digit << shift;
    }
  }
  // Where `reached` is the number needed, every key >= last stays; else last is a key that
  // several have, and of these the earliest stay.
  const bool exact = reached == need;
  const auto state = [&](int t, unsigned k, bool& more, bool& equal) {
    more = t < n && (all || t >= m || (need > 0 && (exact ? k >= last : k > last)));
    equal = t < m && !all && need > 0 && !exact && k == last;
  };
  int more_before = 0, equal_before = 0;  // in earlier chunks
  int equal_most = 0;
  if (!all && need > 0 && !exact) {
    int above = 0;
    for (int ch = 0; ch < chunks; ++ch) {
      if (chunks > 1) load(ch * kChunk);
#pragma unroll
      for (int j = 0; j < KEYS; ++j) above += __popcll(__ballot(key[j] > last));
    }
    if (lane == 0) atomicAdd(&counted[16][0], above);
    __syncthreads();
    above = counted[16][0];
    equal_most = need - above;
  }
  int written = 0;
  for (int t0 = 0; t0 < n; t0 += kChunk) {
    if (chunks > 1) load(t0);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      bool more, equal;
      state(t0 + j * kSelect + tid, key[j], more, equal);
      const int cm = __popcll(__ballot(more)), ce = __popcll(__ballot(equal));
      if (lane == 0) before[j * kSelectWaves + wave] = int2{cm, ce};
    }
    __syncthreads();
    if (wave == 0) {  // exclusive sums, 64 entries at a time
      int cm = more_before, ce = equal_before;
      for (int i0 = 0; i0 < KEYS * kSelectWaves; i0 += 64) {
        const int2 v = before[i0 + lane];
        int sm = v.x, se = v.y;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int pm = __shfl_up(sm, o), pe = __shfl_up(se, o);
          if (lane >= o) {
            sm += pm;
            se += pe;
          }
        }
        before[i0 + lane] = int2{cm + sm - v.x, ce + se - v.y};
        cm += __shfl(sm, 63);
        ce += __shfl(se, 63);
      }
      if (lane == 0) {
        chunk_sums[0] = cm;
        chunk_sums[1] = ce;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      const int t = t0 + j * kSelect + tid;
      bool more, equal;
      state(t, key[j], more, equal);
      const unsigned long long below = (1ull << lane) - 1;
      const unsigned long long bm = __ballot(more), be = __ballot(equal);
      const int2 base = before[j * kSelectWaves + wave];
      const int rank = base.y + __popcll(be & below);
      const int place = base.x + __popcll(bm & below) + min(rank, equal_most);
      if ((more || (equal && rank < equal_most)) && place < keep) {
        kept[out + place] = t;
        if (new_weights) new_weights[out + place] = weight[j];
      }
    }
    more_before = chunk_sums[0];
    equal_before = chunk_sums[1];
    written = more_before + min(equal_before, equal_most);
  }
  for (int i = written + tid; i < keep; i += kSelect) {
    kept[out + i] = -1;
    if (new_weights) new_weights[out + i] = 0.f;
  }
}

// ---------------------------------------------------------------------------------
// Second half: the kept tokens to their new pages.  Workgroup = (one new block, head, sequence),
// as an append of 32 tokens that are decoded from the cache.  Keys: 8 channels of a token a thread,
// as in the append.  Values: a thread has one channel of 16 new tokens, a side of the new block,
// which it writes in one piece; of each of its tokens it reads the 16 bytes of the channel's side
// (the others of which are its neighbours' for the other tokens there: a cache that turns values
// for the matrix cores is read whole where a quarter of it is kept).  What bounds it is the chain
// id, page, codes: keys, values and scales are asked for together.
// ---------------------------------------------------------------------------------
// WIDE: D is a multiple of 64, so a wave's rows of values are of one side and its tokens uniform.
// BIG: D is above 128.
template <bool WIDE, bool BIG>
__global__ __launch_bounds__(256, BIG ? 4 : WIDE ? 6 : 5) void evict_move_kernel(
    Cache c, Cache to, int keep, const int32_t* __restrict__ kept) {
  constexpr int KC = BIG ? 4 : 2, VC = BIG ? 2 : 1;  // pieces of keys, rows of values a thread
  __shared__ float red[2][4];
  __shared__ int64_t from_block[kBlock];  // of a token in the pool; -1: none
  __shared__ int from_slot[kBlock];
  __shared__ float from_scale[2][kBlock];
  const int tid = threadIdx.x, blk = blockIdx.x;
  const int h = blockIdx.y, b = blockIdx.z;
  const int32_t* const ids = kept + ((int64_t)b * c.H + h) * keep;
  const int place = blk * kBlock + tid;
  const int from = tid < kBlock && place < keep ? ids[place] : -1;
  int at;
  const int page = to.page_of(b, blk, at);
  int64_t src = -1;
  if (tid < kBlock) {
    int src_at, src_page = -1;
    if (from >= 0) src_page = c.page_of(b, from / kBlock, src_at);
    if (src_page >= 0) src = c.block_index(src_page, h, src_at);
    from_block[tid] = src;
    from_slot[tid] = from & (kBlock - 1);
  }
  // nothing to write: no token of the block is kept, or it has no page
  if (__syncthreads_or(from >= 0) == 0 || page < 0) return;
  int scale[2] = {0, 0};
  if (src >= 0) {
    scale[0] = c.ks[src];
    scale[1] = c.vs[src];
  }
  const int pieces = c.D / 8, total = kBlock * pieces;
  u32x2 key[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int e = tid + 256 * i, t = e / pieces, d = (e - t * pieces) * 8;
    key[i] = u32x2{0, 0};
    if (e < total && from_block[t] >= 0)
      key[i] = *reinterpret_cast<const u32x2*>(c.k + from_block[t] * kBlock * c.D +
                                               from_slot[t] * c.D + d);
  }
  // values: rows (side, channel) of the new block, 2 D of them
  u32x4 value[VC];
#pragma unroll
  for (int i = 0; i < VC; ++i) {
    const int e = tid + 256 * i;
    const int side = WIDE ? __builtin_amdgcn_readfirstlane(e / c.D) : e / c.D;
    const int d = e - side * c.D;
    value[i] = u32x4{0, 0, 0, 0};
    if (e >= 2 * c.D) continue;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      u32x4 row[8];
      int slot[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int k = side * kSide + half * 8 + t;
        int64_t block = from_block[k];
        slot[t] = from_slot[k];
        if (WIDE) {
          block = (int64_t)__builtin_amdgcn_readfirstlane((int)(block >> 32)) << 32 |
                  (unsigned)__builtin_amdgcn_readfirstlane((int)block);
          slot[t] = __builtin_amdgcn_readfirstlane(slot[t]);
        }
        row[t] = u32x4{0, 0, 0, 0};
        if (block >= 0)
          row[t] = *reinterpret_cast<const u32x4*>(
              c.v + block * kBlock * c.D + (slot[t] / kSide) * c.D * kSide + d * kSide);
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const unsigned word = slot[t] & 8 ? (slot[t] & 4 ? row[t][3] : row[t][2])
                                          : (slot[t] & 4 ? row[t][1] : row[t][0]);
        value[i][half * 2 + t / 4] |= (word >> (8 * (slot[t] & 3)) & 0xFFu) << (8 * (t & 3));
      }
      __builtin_amdgcn_sched_barrier(0);  // the registers of one half at a time
    }
  }
  if (tid < kBlock) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
      from_scale[x][tid] = src >= 0 ? exp2i(min(max(scale[x] - 127, -126), 127)) : 0.f;
  }
  __syncthreads();
  const auto key_values = [&](int i, float (&v)[8]) {
    const int t = min((tid + 256 * i) / pieces, kBlock - 1);
    decode8(key[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= from_scale[0][t];
  };
  const auto value_values = [&](int i, int half, float (&v)[8]) {
    const int t0 = min((tid + 256 * i) / c.D, 1) * kSide + half * 8;
    decode8(u32x2{value[i][2 * half], value[i][2 * half + 1]}, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= from_scale[1][t0 + j];
  };
  float amax[2] = {0.f, 0.f}, val[8];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    key_values(i, val);
#pragma unroll
    for (int j = 0; j < 8; ++j) amax[0] = fmaxf(amax[0], finite_abs(val[j]));
  }
#pragma unroll
  for (int i = 0; i < VC; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      value_values(i, half, val);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax[1] = fmaxf(amax[1], finite_abs(val[j]));
    }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    amax[0] = fmaxf(amax[0], __shfl_xor(amax[0], o));
    amax[1] = fmaxf(amax[1], __shfl_xor(amax[1], o));
  }
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = amax[0];
    red[1][tid >> 6] = amax[1];
  }
  __syncthreads();
  int e2[2];
  float inv[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    e2[x] = block_exp(fmaxf(fmaxf(red[x][0], red[x][1]), fmaxf(red[x][2], red[x][3])));
    inv[x] = exp2i(min(max(-e2[x], -126), 127));
  }
  const int64_t bi = to.block_index(page, h, at);
  if (tid == 0) {
    to.ks[bi] = (uint8_t)(e2[0] + 127);
    to.vs[bi] = (uint8_t)(e2[1] + 127);
  }
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int e = tid + 256 * i;
    if (e >= total) continue;
    key_values(i, val);
#pragma unroll
    for (int j = 0; j < 8; ++j) val[j] *= inv[0];
    *reinterpret_cast<u32x2*>(to.k + bi * kBlock * c.D + e * 8) = encode8(val);
  }
#pragma unroll
  for (int i = 0; i < VC; ++i) {
    const int e = tid + 256 * i;
    if (e >= 2 * c.D) continue;
    u32x2 w[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      value_values(i, half, val);
#pragma unroll
      for (int j = 0; j < 8; ++j) val[j] *= inv[1];
      w[half] = encode8(val);
    }
    *reinterpret_cast<u32x4*>(to.v + bi * kBlock * c.D + e * kSide) =
        u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
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
  const dim3 grid((unsigned)nx, (unsigned)ny), threads((unsigned)(c->head_dim + 63) / 64 * 64);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  if (dtype == FB_DT_F16)
    hipLaunchKernelGGL(cache_append_kernel<FB_DT_F16>, grid, threads, 0, hs, kc, x);
  else if (dtype == FB_DT_BF16)
    hipLaunchKernelGGL(cache_append_kernel<FB_DT_BF16>, grid, threads, 0, hs, kc, x);
  else
    hipLaunchKernelGGL(cache_append_kernel<FB_DT_F32>, grid, threads, 0, hs, kc, x);
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
  const int64_t nx = ((int64_t)keep + kBlock - 1) / kBlock;
  if (nx > INT32_MAX) return FB_ERR_SHAPE;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const auto select = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(c->heads, s->seqs), dim3(kSelect), 0, hs, kc, weights, w_seq,
                       w_head, w_tokens, keep, recent, kept, new_weights, new_lens);
  };
  // as many keys a thread as the longest sequence asks for, up to 32
  const int longest = std::min(s->max_len, w_tokens);
  if (longest <= 4 * kSelect)
    select(evict_select_kernel<4>);
  else if (longest <= 8 * kSelect)
    select(evict_select_kernel<8>);
  else
    select(evict_select_kernel<32>);
  if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  const bool big = c->head_dim > 128;
  hipLaunchKernelGGL(c->head_dim % 64
                         ? (big ? evict_move_kernel<false, true> : evict_move_kernel<false, false>)
                         : (big ? evict_move_kernel<true, true> : evict_move_kernel<true, false>),
                     dim3((unsigned)nx, c->heads, s->seqs), dim3(256), 0, hs, kc, to, keep, kept);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

}  // extern "C"
