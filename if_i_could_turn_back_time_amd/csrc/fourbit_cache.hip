// Writing to and evicting from the 8-bit key/value cache (layout: fourbit.h).
#include "fourbit_cache.h"

#include <algorithm>
#include <climits>

namespace {

using namespace fbc;

template <int CTRL, int ROWS>
__device__ inline unsigned moved(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xF, false);
}

// The wave's largest value, in every lane.
__device__ inline unsigned wave_max(unsigned v) {
  v = max(v, moved<0x111, 0xF>(v));  // row_shr:1, 2, 4, 8
  v = max(v, moved<0x112, 0xF>(v));
  v = max(v, moved<0x114, 0xF>(v));
  v = max(v, moved<0x118, 0xF>(v));
  v = max(v, moved<0x142, 0xA>(v));  // row_bcast:15, 31
  v = max(v, moved<0x143, 0xC>(v));
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// Largest of the workgroup's values; `lds` holds 4.  Every thread calls it, once for each `lds`.
__device__ inline unsigned block_max(unsigned v, unsigned* lds) {
  v = wave_max(v);
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
  int most;  // of a sequence
};

// ---------------------------------------------------------------------------------
// Append.  Workgroup = (sequence, head, keys or values) x (one block of 32 tokens that gets new
// ones), D threads rounded up to whole waves: the block's scale needs all of its new values, 32 D
// at most, which stay in registers as they came (4 tokens of 8 channels a thread) between the
// maximum, taken over their bits, and the codes.  Four tokens of a value's channel become one
// word; a full block's words go through LDS to whole 16-token sides.  Earlier codes are read only
// where the scale grows, and only a block that holds something not finite looks for it.  Bound by
// memory: 4 sequences of up to 2,048 tokens, 8 heads of 128, bf16 (44 MB): 10.6 us, 4.1 TB/s; by its
// launch for single tokens, 4.4 us.
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
  n = min(n, x.most);
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
// last token that stays is searched for eight bits at a time over the order-preserving 32-bit keys
// of the weights, which stay in registers (KEYS of them a thread; longer sequences are read again
// for each step): a histogram of the keys that share the bits found so far, in eight copies so
// that equal keys do not wait for each other, which every wave sums from the top by itself.  The
// search ends as soon as a bound parts the right number.  A wave's tokens lie together, so one
// exchange of the waves' counts gives every token its place: what lies above the key, as many of
// its equals as are left, earliest first, and the recent ones, in their order.  Bound by latency
// and by the instructions that 16 waves of one CU can issue: 4,096 tokens 9 us, 8,192 of 16
// sequences 12, 32,768 29 (with 512 threads 9, 13, 37; with four copies 9, 12, 32).
// ---------------------------------------------------------------------------------
// Order-preserving keys of weights: numbers have them from 0x7FFFFF (-inf) to 0xFF800000 (inf).
constexpr unsigned kNone = 0, kNan = 1, kNever = 2, kRecent = ~0u;

__device__ inline unsigned weight_key(float w) {
  unsigned b = __builtin_bit_cast(unsigned, w);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return kNan;  // below every number
  if (b == 0x80000000u) b = 0;
  return (b >> 31) ? ~b : (b | 0x80000000u);
}

constexpr int kSelect = 1024, kSelectWaves = kSelect / 64;
constexpr int kCopies = 8;  // of a histogram of 256 bins: a lane adds to copy lane % kCopies
constexpr int kCopy = 256 + 64 / kCopies;  // their bins are of different banks

// Bits of a ballot of lanes before this one.
__device__ inline int before_lane(unsigned long long bits) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(bits >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)bits, 0));
}

template <int KEYS>
__global__ __launch_bounds__(kSelect) void evict_select_kernel(
    Cache c, const float* __restrict__ weights, int64_t w_seq, int64_t w_head, int w_tokens,
    int keep, int recent, int32_t* __restrict__ kept, float* __restrict__ new_weights,
    int32_t* __restrict__ new_lens) {
  constexpr int kChunk = KEYS * kSelect;  // tokens held at once
  __shared__ __align__(16) int bins[4][kCopies * kCopy];
  __shared__ int2 totals[2][kSelectWaves];  // larger and equal keys of each wave
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
  const int lane = tid & 63, wave = tid >> 6;
  const int n = min(min(max(c.lens[b], 0), c.capacity()), w_tokens);
  const float* const w = weights + b * w_seq + h * w_head;
  const int64_t out = ((int64_t)b * c.H + h) * keep;
  if (h == 0 && tid == 0) new_lens[b] = min(n, keep);
  const bool all = n <= keep;
  unsigned key[KEYS];
  float weight[KEYS];
  // a wave's tokens lie together; all of them are asked for before the first is used
  const int own = wave * 64 * KEYS + lane;
  const auto load = [&](int t0) {
#pragma unroll
    for (int j = 0; j < KEYS; ++j) weight[j] = w[min(t0 + own + 64 * j, max(n - 1, 0))];
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      const int t = t0 + own + 64 * j;
      key[j] = t >= n ? kNone : t >= n - recent ? kRecent : weight_key(weight[j]);
    }
  };
  const int chunks = (n + kChunk - 1) / kChunk;
  load(0);
  for (int i = tid; i < kCopies * kCopy; i += kSelect)
    reinterpret_cast<u32x4*>(bins)[i] = u32x4{0, 0, 0, 0};
  __syncthreads();
  // the largest `last` with at least `keep` keys >= last, 8 bits at a time
  unsigned last = 0;
  int above = 0;          // keys whose bits so far are above last's
  int reached = INT_MAX;  // and those with last's among them
  if (!all) {
    for (int pass = 0; pass < 4 && reached != keep; ++pass) {
      const int shift = 24 - 8 * pass;
      int* const bin = bins[pass];
      for (int ch = 0; ch < chunks; ++ch) {
        if (chunks > 1) load(ch * kChunk);
        if (ch * kChunk + wave * 64 * KEYS >= n) break;
#pragma unroll
        for (int j = 0; j < KEYS; ++j)
          if (pass == 0 || ((key[j] ^ last) >> shift) < 256u)
            atomicAdd(bin + (key[j] >> shift & 255) + (lane & (kCopies - 1)) * kCopy, 1);
      }
      __syncthreads();
      // every wave for itself: lane l has the four bins from 255 - 4 l down
      u32x4 count = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        count += *reinterpret_cast<const u32x4*>(bin + i * kCopy + 252 - 4 * lane);
      const int four = (int)(count[0] + count[1] + count[2] + count[3]);
      const int upto = sum_to_lane(four);
      const int left = keep - above;  // at least 1, and at most all that are counted
      const int l = __builtin_ctzll(__ballot(upto >= left) | 1ull << 63);
      int run = upto - four, digit = 255 - 4 * lane, size = (int)count[3];
#pragma unroll
      for (int i = 1; i < 4; ++i)
        if (run + size < left) {
          run += size;
          size = (int)count[3 - i];
          digit = 255 - 4 * lane - i;
        }
      above += __builtin_amdgcn_readlane(run, l);
      reached = above + __builtin_amdgcn_readlane(size, l);
      last |= (unsigned)__builtin_amdgcn_readlane(digit, l) << shift;
    }
  }
  // Where `reached` is the number needed, every key >= last stays; else last is a key that
  // several have, and of these the earliest stay.
  const bool exact = all || reached == keep;
  const unsigned least = exact ? max(last, kNan) : last + 1, same = exact ? kNever : last;
  const int equal_most = exact ? 0 : keep - above;
  int more_before = 0, equal_before = 0;  // of earlier chunks
  for (int ch = 0; ch < chunks; ++ch) {
    if (chunks > 1) load(ch * kChunk);
    unsigned long long more[KEYS], equal[KEYS];
    int cm = 0, ce = 0;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      more[j] = __ballot(key[j] >= least);
      equal[j] = __ballot(key[j] == same);
      cm += __popcll(more[j]);
      ce += __popcll(equal[j]);
    }
    if (lane == 0) totals[ch & 1][wave] = int2{cm, ce};
    __syncthreads();  // (the next chunk's totals go elsewhere)
    const int2 v = lane < kSelectWaves ? totals[ch & 1][lane] : int2{0, 0};
    const int sm = sum_to_lane(v.x), se = sum_to_lane(v.y);
    cm = more_before + __builtin_amdgcn_readlane(sm, wave) - cm;
    ce = equal_before + __builtin_amdgcn_readlane(se, wave) - ce;
    more_before += __builtin_amdgcn_readlane(sm, 63);
    equal_before += __builtin_amdgcn_readlane(se, 63);
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      const int rank = ce + before_lane(equal[j]);
      const int place = cm + before_lane(more[j]) + min(rank, equal_most);
      if ((key[j] >= least || (key[j] == same && rank < equal_most)) && place < keep) {
        kept[out + place] = ch * kChunk + own + 64 * j;
        if (new_weights) new_weights[out + place] = weight[j];
      }
      cm += __popcll(more[j]);
      ce += __popcll(equal[j]);
    }
  }
  for (int i = more_before + min(equal_before, equal_most) + tid; i < keep; i += kSelect) {
    kept[out + i] = -1;
    if (new_weights) new_weights[out + i] = 0.f;
  }
}

// ---------------------------------------------------------------------------------
// Second half: the kept tokens to their new pages.  Workgroup = (one new block, head, sequence),
// as an append of 32 tokens that are decoded from the cache.  Keys: 8 channels of a token a thread,
// as they lie.  Values: a thread has one channel of 16 new tokens, a side of the new block, which it
// writes in one piece; it reads their bytes one by one, 16 bytes from its neighbours'.  Few blocks are
// bound by the chain id, page, codes, so all codes of a thread are asked for together (1,024 of 4,096
// tokens of 32 heads: 9 us); many by the values' strided bytes, 32 accesses of the first-level cache for
// 64 lanes, which is busy two thirds of the time (16 sequences of up to 8,192 cut to 2,048, 79 MB
// fetched for 67 MB kept: 46 to 50 us; 16-byte loads and a choice among their words took 64 for their
// registers, keys and values in workgroups of their own 91).
// ---------------------------------------------------------------------------------
// The codes of a word that are NaN: their top bits.
__device__ inline unsigned nan_codes(unsigned w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// Largest magnitude of eight numbers; NaN is passed over.
__device__ inline float largest(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j += 2)
    m = fmaxf(fmaxf(m, __builtin_fabsf(v[j])), __builtin_fabsf(v[j + 1]));
  return m;
}

// A token's scale over its new block's: 0 times it is 0, however far apart they are (what is not 0 is
// at most 448 times the new one).
__device__ inline float rescale(float from, float inv) { return fminf(from * inv, 0x1p126f); }

// WIDE: D is a multiple of 64, so a wave's rows of values are of one side and its tokens uniform.
// BIG: D is above 128.
template <bool WIDE, bool BIG>
__global__ __launch_bounds__(256, BIG ? 4 : 8) void evict_move_kernel(Cache c, Cache to, int keep,
                                                            const int32_t* __restrict__ kept) {
  constexpr int KC = BIG ? 4 : 2, VC = BIG ? 2 : 1;  // pieces of keys, rows of values a thread
  __shared__ float red[2][4];
  __shared__ int any_nan;
  __shared__ bool some, whole;
  __shared__ int64_t from_key[kBlock], from_value[kBlock];  // a token's first code; key -1: none
  __shared__ __align__(16) float from_scale[2][kBlock];
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
    const int slot = from & (kBlock - 1);
    const int64_t first = max(src, (int64_t)0) * kBlock * c.D;  // where there is none: any
    from_key[tid] = src >= 0 ? first + slot * c.D : -1;
    from_value[tid] = first + slot / kSide * c.D * kSide + slot % kSide;
  }
  if (tid < 64) {
    const unsigned long long held = __ballot(from >= 0), found = __ballot(src >= 0);
    if (tid == 0) {
      some = held != 0;
      whole = found == 0xFFFFFFFFull;
      any_nan = 0;
    }
  }
  __syncthreads();
  // nothing to write: no token of the block is kept, or it has no page
  if (!some || page < 0) return;
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
    if (e < total && from_key[t] >= 0)
      key[i] = *reinterpret_cast<const u32x2*>(c.k + from_key[t] + d);
  }
  // values: rows (side, channel) of the new block, 2 D of them
  u32x4 value[VC];
#pragma unroll
  for (int i = 0; i < VC; ++i) {
    const int e = min(tid + 256 * i, 2 * c.D - 1);
    const int side = WIDE ? __builtin_amdgcn_readfirstlane(e / c.D) : e / c.D;
    const unsigned d = (e - side * c.D) * kSide;
    unsigned byte[kSide];
#pragma unroll
    for (int t = 0; t < kSide; ++t) {
      int64_t row = from_value[side * kSide + t];
      if (WIDE)
        row = (int64_t)__builtin_amdgcn_readfirstlane((int)(row >> 32)) << 32 |
              (unsigned)__builtin_amdgcn_readfirstlane((int)row);
      byte[t] = (c.v + row)[d];
    }
    if (!whole) {
#pragma unroll
      for (int t = 0; t < kSide; ++t)
        if (from_key[side * kSide + t] < 0) byte[t] = 0;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w)
      value[i][w] = byte[4 * w] | byte[4 * w + 1] << 8 | byte[4 * w + 2] << 16 | byte[4 * w + 3] << 24;
  }
  if (tid < kBlock) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
      from_scale[x][tid] = src >= 0 ? exp2i(min(max(scale[x] - 127, -126), 127)) : 0.f;
  }
  __syncthreads();
  // Magnitudes by the tokens' scales; a NaN is seen in the codes.
  float amax[2] = {0.f, 0.f};
  unsigned nan = 0;
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    float v[8];
    decode8(key[i], v);
    nan |= nan_codes(key[i][0]) | nan_codes(key[i][1]);
    amax[0] = fmaxf(amax[0], largest(v) * from_scale[0][min((tid + 256 * i) / pieces, kBlock - 1)]);
  }
#pragma unroll
  for (int i = 0; i < 2 * VC; ++i) {
    const int t0 = min((tid + 256 * (i / 2)) / c.D, 1) * kSide + (i & 1) * 8;
    const u32x2 codes = {value[i / 2][2 * (i & 1)], value[i / 2][2 * (i & 1) + 1]};
    float v[8];
    decode8(codes, v);
    nan |= nan_codes(codes[0]) | nan_codes(codes[1]);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= from_scale[1][t0 + j];
    amax[1] = fmaxf(amax[1], largest(v));
  }
  if (__ballot(nan != 0) && (tid & 63) == 0) any_nan = 1;
#pragma unroll
  for (int x = 0; x < 2; ++x)  // not negative: in order as bits
    amax[x] = __builtin_bit_cast(float, wave_max(__builtin_bit_cast(unsigned, amax[x])));
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = amax[0];
    red[1][tid >> 6] = amax[1];
  }
  __syncthreads();
  const bool finite = __builtin_amdgcn_readfirstlane(any_nan) == 0;
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
    const float f = rescale(from_scale[0][e / pieces], inv[0]);
    float v[8];
    decode8(key[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    *reinterpret_cast<u32x2*>(to.k + bi * kBlock * c.D + e * 8) = finite ? encode8_finite(v) : encode8(v);
  }
#pragma unroll
  for (int i = 0; i < VC; ++i) {
    const int e = tid + 256 * i;
    if (e >= 2 * c.D) continue;
    const float* const f = from_scale[1] + e / c.D * kSide;
    u32x2 w[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float v[8];
      decode8(u32x2{value[i][2 * half], value[i][2 * half + 1]}, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= rescale(f[half * 8 + j], inv[1]);
      w[half] = finite ? encode8_finite(v) : encode8(v);
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
  const int nt = (c->head_dim + 63) / 64 * 64;
  if (ny > 65535 || !fits_grid(nx, nt)) return FB_ERR_SHAPE;
  const NewTokens x{k,      v,      k_token, k_head, v_token,
                    v_head, vec16(k, k_token, k_head, bytes), vec16(v, v_token, v_head, bytes),
                    s->max_new};
  const dim3 grid((unsigned)nx, (unsigned)ny), threads((unsigned)nt);
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
  if (!fits_grid(nx, 256)) return FB_ERR_SHAPE;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const auto select = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(c->heads, s->seqs), dim3(kSelect), 0, hs, kc, weights, w_seq,
                       w_head, w_tokens, keep, recent, kept, new_weights, new_lens);
  };
  // as many keys a thread as the longest sequence asks for, up to 32
  const int longest = std::min(s->max_len, w_tokens);
  if (longest <= 4096)
    select(evict_select_kernel<4096 / kSelect>);
  else if (longest <= 8192)
    select(evict_select_kernel<8192 / kSelect>);
  else if (longest <= 16384)
    select(evict_select_kernel<16384 / kSelect>);
  else
    select(evict_select_kernel<32768 / kSelect>);
  if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  const bool big = c->head_dim > 128;
  hipLaunchKernelGGL(c->head_dim % 64
                         ? (big ? evict_move_kernel<false, true> : evict_move_kernel<false, false>)
                         : (big ? evict_move_kernel<true, true> : evict_move_kernel<true, false>),
                     dim3((unsigned)nx, c->heads, s->seqs), dim3(256), 0, hs, kc, to, keep, kept);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

}  // extern "C"
