// Attention over the 8-bit key/value cache (layout: fourbit.h).
//
// Both kernels compute S^T = K Q^T and O^T = V^T P^T on the matrix cores, so that a lane's scores
// belong to one query row (a column of S^T) and the C layout of S^T is, with the cached tokens
// dealt to the rows of K's operand in the right order, the B layout that P^T needs: no score ever
// crosses lanes, except for the row maximum.  E4M3 codes are exact in fp16 and bf16, so products
// of q and a code are exact in fp32; a block's scale of K joins after the sum, in fp32.  P enters as
// fp16 (11 bits, relative to the row's largest score).  A block's scale of V joins where its codes
// are decoded, relative to the unit that the sums are in (Unit).
//
// A sequence's rows are its (new token, query head of the group) pairs, token-major: with shared
// heads a tile of rows reads a cached head once for the whole group.
#include "fourbit_cache.h"

#include <algorithm>
#include <type_traits>

// Host helper of fourbit_gemv.hip.  Not part of the library's ABI.
namespace fb_gpu {
__attribute__((visibility("hidden"))) int cu_count();
}

namespace {

using namespace fbc;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Attn {
  Cache c;
  const void* q;
  int64_t q_token, q_head;
  bool q_vec;
  int Hq, group;
  float scale2;       // scale * log2(e)
  void* out;
  float* lse;         // or null
  int splits, split_tokens;
  bool dealt;         // see find_part
  int chunk;          // tokens of a chunk: what parts are counted in
  int grain;          // chunks that a part has at least
  int most;           // parts that a sequence has at most
  int tiles;          // many rows: tiles of a sequence's rows that are dealt out; few: 0
  float* part;        // [splits][T * Hq][D]: averages over a part, which are no larger than v
  float2* part_ml;    // [splits][T * Hq]: what the weights' sum is relative to (base 2), the sum
  int per_shift;      // log2 of a page's blocks, -1: no power of two
  float* scores;      // or null: [B][H][score_rows][score_tokens], base 2
  int score_rows, score_tokens;
  unsigned div_mul, div_shift;

  // row / group, of rows below 2^31: (mulhi(row, m) + row) >> s with s = ceil(log2 group) and
  // m = floor(2^32 (2^s - group) / group) + 1
  __device__ int token_of(int row) const {
    return (int)((__umulhi((unsigned)row, div_mul) + (unsigned)row) >> div_shift);
  }
};

__device__ inline float exp2f_(float x) { return __builtin_amdgcn_exp2f(x); }

// What a block's sums of q and codes are multiplied by, for its scale's byte.  Positive and finite
// whatever the byte, which may be of a block that nobody wrote: a masked score of -inf stays that.
__device__ inline float key_scale(float scale2, int byte) {
  return __builtin_amdgcn_fmed3f(scale2 * exp2i(min(max(byte - 127, -126), 127)), 0x1p-149f,
                                 0x1.fffffep127f);
}

template <int DT>
struct Half;
template <>
struct Half<FB_DT_F16> {
  using x8 = h16x8;
  static __device__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // 8 E4M3 codes times a power of two: exactly from 2^-15 (a code's last bit is 2^-9, and
  // subnormal operands count in the products) to 2^7
  static __device__ x8 decode(unsigned lo, unsigned hi, float scale = 1.0f) {
    x8 r;
    const h16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, scale, false);
    const h16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, scale, true);
    const h16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, scale, false);
    const h16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, scale, true);
    r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1];
    r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
    return r;
  }
  static __device__ unsigned short round(float v) {
    return __builtin_bit_cast(unsigned short, (_Float16)v);
  }
};
template <>
struct Half<FB_DT_BF16> {
  using x8 = b16x8;
  static __device__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ x8 decode(unsigned lo, unsigned hi) {
    x8 r;
    const b16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false);
    const b16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true);
    const b16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false);
    const b16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true);
    r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1];
    r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
    return r;
  }
  static __device__ unsigned short round(float v) {
    return __builtin_bit_cast(unsigned short, (__bf16)v);
  }
};

// 8 channels of a query row as an operand; zeros where there are none.
template <int DT>
__device__ inline typename Half<DT>::x8 load_q(const Attn& a, bool there, int64_t at) {
  u32x4 w{0, 0, 0, 0};
  if (there) {
    const unsigned short* p = static_cast<const unsigned short*>(a.q) + at;
    if (a.q_vec) {
      w = *reinterpret_cast<const u32x4*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j / 2] |= (unsigned)p[j] << (16 * (j & 1));
    }
  }
  return __builtin_bit_cast(typename Half<DT>::x8, w);
}

// Rows in front of the first sequence's and behind the last one's get what a row gets that sees
// nothing.  Workgroup x of xs writes some of head h's.
__device__ inline void rows_of_none(const Attn& a, int h, int x, int xs) {
  const Cache& c = a.c;
  if (!c.cu) return;
  const int before = min(max(c.cu[0], 0), c.T);
  const int behind = c.T - min(max(c.cu[c.B], before), c.T), none = before + behind;
  const int pieces = a.group * c.D / 8;  // 16 bytes each: D is a multiple of 16
  for (int i = x; i < none; i += xs) {
    const int64_t row = (int64_t)(i < before ? i : c.T - none + i) * a.Hq + h * a.group;
    u32x4* const to = reinterpret_cast<u32x4*>(static_cast<unsigned short*>(a.out) + row * c.D);
    for (int p = threadIdx.x; p < pieces; p += blockDim.x) to[p] = u32x4{0, 0, 0, 0};
    if (a.lse)
      for (int p = threadIdx.x; p < a.group; p += blockDim.x) a.lse[row + p] = -__builtin_inff();
  }
}

// The bytes of the 4 codes from `at` on that lie before `limit`.
__device__ inline unsigned keep_bytes(int at, int limit) {
  const int n = limit - at;
  return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
}

// 0xFF in every byte that holds a NaN code.
__device__ inline unsigned nan_bytes(unsigned w) {
  const unsigned top = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  return (top >> 7) * 0xFFu;
}

// NaN codes as 1 (0x38), others as 0.
__device__ inline unsigned nan_ones(unsigned w) { return nan_bytes(w) & 0x38383838u; }

// The exponent of the unit that a wave's sums over the values are in.  It follows the blocks' scales
// up and down, each time by an exact scaling of the sums, so that neither a weight nor a decoded
// value loses bits to a block with another scale: two that are 2^22 apart share a unit, others take
// turns.  A row leaves it when no later block is seen by it, so what comes behind a row never
// touches its sums.  It stays within 2^60 of the largest it was, or sums could overflow: only
// values 2^75 below the scale of a block that counted lose bits.
struct Unit {
  static constexpr int kUp = 7, kDown = 15;  // what decode takes
  static constexpr int kFall = 60;
  int now = -1000, top = -1000;

  // A block's exponent as far as it is followed, and whether it can be decoded in this unit.
  __device__ int reach(int e) const { return max(e, top - kFall - kDown); }
  __device__ bool takes(int e) const { return (unsigned)(e - now + kDown) <= (unsigned)(kUp + kDown); }
  // The unit for blocks of exponents e0 and e1; false: none takes both.
  __device__ static bool shared(int e0, int e1, int& to) {
    const int hi = max(e0, e1), apart = hi - min(e0, e1);
    to = hi - max(apart - kDown, 0);
    return apart <= kUp + kDown;
  }
  // The unit that move(to) ends in: `to`, or as near as can be.
  __device__ int within(int to) const { return max(to, top - kFall); }
  // Returns what the sums are multiplied by.
  __device__ float move(int to) {
    to = within(to);
    const int by = now - to;  // at most kFall
    now = to;
    top = max(top, to);
    return by < -126 ? 0.f : exp2i(by);
  }
  // What the codes of a block of exponent e are multiplied by in unit `u`: e - u is within
  // [-kFall - kDown, kUp].
  __device__ static float scale(int e, int u) { return exp2i(e - u); }
};

// ---------------------------------------------------------------------------------
// Few rows (at most 16 a cached head and sequence: decoding).  Bound by reading the cache once,
// so nothing is staged: each wave takes 64 tokens at a time and reads keys and values straight
// into operands of 16x16x32 products.  The next keys are asked for when the scores are there, the
// next values when the sums are: a wave always has one of the two on its way.  Workgroup =
// (split of the tokens, head, sequence); its waves take chunks in turn and join their sums through
// LDS.
//  - K operand row r of product j: token 16 (r / 4) + 4 j + r % 4, channels 64 p + 16 q + 8 u.. of
//    lane group q: then a lane's scores are the tokens of side q, 4 j + i.
//  - V operand: channel 16 d + r, tokens 8 s.. of side q, which lie side by side.
//  - the sums are kept relative to a row's largest score of some earlier time.  It is looked for
//    again only where the weights relative to it become too large, which their sum tells: rare
//    after the first tile, and no maximum is taken in the others.
// Two workgroups of four waves a CU, one round of them (more, smaller ones had more to join); one
// above 128 channels, for its registers.
// Measured: 2 sequences of up to 100,003 tokens, 64 query heads over 8 of 128 (0.4 GB): 76 us, 5.3
// TB/s, and 6 to join; 16 of up to 8,192 with weights: 52 and 14 for joining and weights.  Short
// ones wait for the chain length, table, codes, join: 777 tokens of 32 heads 8 us and 3.  A head is
// worked on at 64, 128 or 256 channels: 4 sequences of up to 8,000, 32 heads over 8, take 14.7 us with
// 64, 17.3 with 80, 19.9 with 128, 27.5 with 144, 32.0 with 256.
// ---------------------------------------------------------------------------------
constexpr int kChunk = 64;
constexpr int kRows = 128, kTile = 64;  // of the kernel for many rows
// Weights enter the products as fp16 times 2^kLift, so that small ones keep their bits.
constexpr int kLift = 7;
// A tile's sum of them that asks for the row's largest score anew: none is above fp16's range.
constexpr float kMost = 32768.f;
// From here on a row's largest score, rounded, can be units away from itself, and its weight anything:
// such rows are weighed anew by rounded scores, of which the largest is equal to it.
constexpr float kFar = 4194304.f;

__device__ inline bool is_far(float m) {
  return __builtin_fabsf(m) >= kFar && m != -__builtin_inff();
}
// The weight's exponent, relative to m, for a sum of q and codes and their block's scale.
__device__ inline float exponent(float s, float ks, float m, float shift) {
#pragma clang fp contract(off)
  return is_far(m) ? (s * ks - m) + (float)kLift : __builtin_fmaf(s, ks, shift);
}

// Which sequence, tile of its rows (many rows have several) and part of its tokens a workgroup has.
// Up to 64 sequences are dealt out by their lengths: parts are about of one size, the least with
// which there are at most `a.splits` of them for all tiles, so that they all run side by side and
// none is much longer than the others.  More sequences have a.splits parts each.
struct Part {
  int b, tile, first, last, parts, slot;  // chunks [first, last); place of its sums
};

__device__ inline int held(const Cache& c, int b) { return min(max(c.lens[b], 0), c.capacity()); }

// What lane b's sequence has to be dealt out, and its parts of `size` chunks.
struct Load {
  int chunks, tiles;
  __device__ int parts(const Attn& a, int size) const {
    return tiles ? min(max(1, (chunks + size - 1) / size), a.most) : 0;
  }
};

__device__ inline Load load_of(const Attn& a, int b, int chunk) {
  if (b >= a.c.B) return Load{0, 0};
  Load x{(held(a.c, b) + chunk - 1) / chunk, 1};
  if (a.tiles) {
    int row0, n;
    a.c.rows(b, row0, n);
    x.tiles = min((n * a.group + kRows - 1) / kRows, a.tiles);
  }
  return x;
}

// The least size of a part (in chunks; found to a 32nd) with which the lanes' sequences have at most
// a.splits parts together, empty ones among them: one more would run after all the others.
__device__ inline int part_size(const Attn& a, Load mine) {
  const int tiles = a.tiles ? __builtin_amdgcn_readlane(sum_to_lane(mine.tiles), 63) : a.c.B;
  const unsigned all =
      (unsigned)__builtin_amdgcn_readlane(sum_to_lane(mine.chunks * mine.tiles), 63);
  const unsigned places = (unsigned)max(a.splits - tiles / 2, 1);  // half a part a tile is lost
  int size = max((int)((all + places - 1) / places), a.grain);
  for (;;) {
    const int n = mine.parts(a, size) * mine.tiles;
    // (a.splits is at least the tiles of all, so that one part each always does)
    if (__builtin_amdgcn_readlane(sum_to_lane(n), 63) <= a.splits || size > 0x3000000) return size;
    size += size / 32 + 1;
  }
}

// Every lane of a wave calls it; slot < 0: nothing to do.
__device__ inline Part find_part(const Attn& a, int x, int z, int chunk) {
  const Cache& c = a.c;
  Part p;
  p.tile = 0;
  if (!a.dealt) {
    p.b = z;
    p.slot = x;
    p.parts = a.splits;
    const int all = (held(c, z) + chunk - 1) / chunk;
    p.first = min(all, x * (a.split_tokens / chunk));
    p.last = x + 1 == a.splits ? all : min(all, p.first + a.split_tokens / chunk);
    return p;
  }
  const int lane = threadIdx.x & 63;
  const Load mine = load_of(a, lane, chunk);
  const int n = mine.parts(a, part_size(a, mine)), end = sum_to_lane(n * mine.tiles);
  const unsigned long long past = __ballot(lane < c.B && end <= x);
  const int b = __popcll(past);
  p.b = min(b, c.B - 1);
  p.parts = __shfl(n, p.b);
  const int chunks = __shfl(mine.chunks, p.b);
  int i = x - (__shfl(end, p.b) - p.parts * __shfl(mine.tiles, p.b));
  if (a.tiles && p.parts > 0) {
    p.tile = i / p.parts;
    i -= p.tile * p.parts;
  }
  p.slot = b < c.B ? i : -1;
  const int even = (chunks + p.parts - 1) / max(p.parts, 1);  // no more than size, or a.most of them
  p.first = min(chunks, i * even);
  p.last = min(chunks, p.first + even);
  return p;
}

constexpr int kFewWaves = 4;

template <int DT, int DP, bool EX>
__global__ __launch_bounds__(64 * kFewWaves, DP > 128 ? 1 : 2) void attn_few_kernel(Attn a) {
  using H = Half<DT>;
  using F = Half<FB_DT_F16>;
  constexpr int NP = DP / 64, ND = DP / 16, NW = kFewWaves;
  constexpr int PASS = 64;  // channels joined at a time
  __shared__ float join[NW][16][PASS + 4];
  __shared__ float wave_m[NW][16], wave_l[NW][16];
  __shared__ int wave_e[NW][16];
  const Cache& c = a.c;
  const int D = EX ? DP : c.D;  // known: the loads' addresses differ by constants
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q4 = lane >> 4;
  const int h = blockIdx.y;
  rows_of_none(a, h, blockIdx.x + gridDim.x * blockIdx.z, gridDim.x * gridDim.z);
  const Part part = find_part(a, blockIdx.x, blockIdx.z, kChunk);
  const int b = __builtin_amdgcn_readfirstlane(part.b);
  const int split = __builtin_amdgcn_readfirstlane(part.slot);
  if (split < 0) return;
  int row0, n;
  c.rows(b, row0, n);
  const int len = min(max(c.lens[b], 0), c.capacity());
  const int rows = n * a.group;
  const unsigned per = (unsigned)c.P / kBlock;
  const int32_t* const table = c.table + b * c.table_stride;
  // within a block: where the lane's keys and values begin
  const int k_from = (16 * ((r >> 2) & 1) + (r & 3)) * D + q4 * 16;
  const int v_from = ((q4 & 1) * D + r) * 16;
  for (int tile = 0; tile < rows; tile += 16) {
    const int row = tile + r, i = a.token_of(row);
    const bool there = row < rows;
    const int head = h * a.group + (row - i * a.group);
    const int sees = there ? min(max(len - n + i + 1, 0), len) : 0;
    const int least = min(max(len - n + a.token_of(tile) + 1, 0), len);  // of the tile's rows
    const int most = min(max(len - n + a.token_of(min(tile + 16, rows) - 1) + 1, 0), len);
    typename H::x8 qf[NP][2];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = 64 * p + 16 * q4 + 8 * u;
        qf[p][u] = load_q<DT>(a, there && d < D,
                              (int64_t)(row0 + i) * a.q_token + head * a.q_head + d);
      }
    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.f;  // m: what the sums are relative to
    bool far = false;                      // whether a row's m is
    Unit unit;
    int E = unit.now;                      // the row's: of the last block that it saw
    unsigned dead[(ND + 7) / 8] = {};      // bit 4 (d % 8) + k of d / 8: o[d][k] saw a NaN value

    const int first = __builtin_amdgcn_readfirstlane(part.first);
    const int last = __builtin_amdgcn_readfirstlane(part.last);
    // the two blocks of a chunk: entries of the table (read a chunk ahead) and places in the pages
    int id[2], at[2];
    const auto look = [&](int ch) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const unsigned blk = (unsigned)ch * 2 + y;
        const unsigned pg = a.per_shift >= 0 ? blk >> a.per_shift : blk / per;
        at[y] = (int)(blk - pg * per);
        id[y] = pg < (unsigned)c.max_pages ? table[pg] : 0;
      }
    };
    u32x4 kf[4][NP], vf[ND];
    int sk, sv;
    int64_t blk_k, blk_v;  // the lane's blocks in the pool
    const auto place = [&] {
      int64_t idx[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int pg = (unsigned)id[y] < (unsigned)c.pages ? id[y] : 0;
        idx[y] = c.block_index(pg, h, at[y]);
      }
      blk_k = r >> 3 ? idx[1] : idx[0];
      blk_v = q4 >> 1 ? idx[1] : idx[0];
    };
    const auto load_k = [&] {
      const uint8_t* const p0 = c.k + blk_k * kBlock * D + k_from;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          // pieces past D meet zeros of q: any others of the row
          const int off = 64 * p + 16 * q4 < D ? 64 * p : -16 * q4;
          kf[j][p] = *reinterpret_cast<const u32x4*>(p0 + 4 * j * D + off);
        }
      sk = c.ks[blk_v];
    };
    const auto load_v = [&] {
      const uint8_t* const p0 = c.v + blk_v * kBlock * D + v_from;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        vf[d] = 16 * d < D ? *reinterpret_cast<const u32x4*>(p0 + d * 256) : u32x4{0, 0, 0, 0};
      sv = c.vs[blk_v];
    };
    int ch = first + wave;
    if (ch < last) {
      look(ch);
      place();
      load_k();
      load_v();
      if (ch + NW < last) look(ch + NW);
    }
    for (; ch < last; ch += NW) {
      const bool masked = ch * kChunk + kChunk > least;  // the same for the wave
      // tokens of the lane's side that its row sees, and that are held
      const int seen = sees - ch * kChunk - q4 * 16, held = len - ch * kChunk - q4 * 16;
      f32x4 s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          s[j] = H::mfma16(H::decode(kf[j][p][0], kf[j][p][1]), qf[p][0], s[j]);
          s[j] = H::mfma16(H::decode(kf[j][p][2], kf[j][p][3]), qf[p][1], s[j]);
        }
      }
      const float ks = key_scale(a.scale2, sk);
      const bool more = ch + NW < last;
      if (more) {
        place();
        load_k();
        if (ch + 2 * NW < last) look(ch + 2 * NW);
      }
      if (masked) {
        asm volatile("");  // a branch, not selects in every chunk
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (4 * j + k >= seen) s[j][k] = -__builtin_inff();
      }
      if (a.scores && there && row < a.score_rows && ch * kChunk < a.score_tokens) {
        float* const to = a.scores +
                          (((int64_t)b * c.H + h) * a.score_rows + row) * a.score_tokens +
                          ch * kChunk + q4 * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(to + 4 * j) = s[j] * ks;
      }
      // of the lane's block, where a row sees it
      const bool block_seen = !masked || ch * kChunk + (q4 >> 1) * kBlock < most;
      const int e = unit.reach(block_seen ? sv - 127 : unit.now);
      bool apart = false;
      const auto move = [&](int to, int from) __attribute__((always_inline)) {
        const bool sees_it = sees > from;
        const float f = unit.move(to), mine = sees_it ? f : 1.f;
        E = sees_it ? unit.now : E;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= mine;
      };
      int e0 = 0, e1 = 0;
      if (__any(!unit.takes(e))) {
        asm volatile("");
        e0 = __builtin_amdgcn_readlane(e, 0);
        e1 = ch * kChunk + kBlock < most ? __builtin_amdgcn_readlane(e, 32) : e0;
        int to;
        apart = !Unit::shared(e0, e1, to);
        if (!apart) move(to, ch * kChunk);
      }
      const float vscale = Unit::scale(block_seen ? e : unit.now, unit.now);
      float sum;
      h16x8 pf[2];
      const auto weigh = [&](auto anew) __attribute__((always_inline)) {
        const float shift = (float)kLift - (m == -__builtin_inff() ? 0.f : m);
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float p = exp2f_(anew ? exponent(s[j][k], ks, m, shift)
                                        : __builtin_fmaf(s[j][k], ks, shift));
            sum += p;
            pf[j / 2][4 * (j & 1) + k] = (_Float16)p;
          }
      };
      weigh(std::false_type{});
      if (far || __any(m == -__builtin_inff() || sum > kMost)) {
        asm volatile("");
        float big = s[0][0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) big = fmaxf(big, s[j][k]);
        big *= ks;  // positive
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        const float up = fmaxf(m, big);
        const float alpha = up == -__builtin_inff() ? 0.f : exp2f_(m - up);
        l *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= alpha;
        m = up;
        far = __any(is_far(m));
        weigh(std::true_type{});
      }
      l += sum;
      if (masked) {
        asm volatile("");
        unsigned nan = 0;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            vf[d][w] &= keep_bytes(4 * w, held);  // what lies behind the end may be anything
            nan |= nan_bytes(vf[d][w]);
          }
        if (__any(nan != 0)) {
          // a NaN value reaches the rows that see its token, and no others: 0 * NaN must not
          // come up, so those channels are marked apart
          h16x8 see[2];
#pragma unroll
          for (int k = 0; k < 16; ++k) see[k / 8][k & 7] = k < seen ? (_Float16)1 : (_Float16)0;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            f32x4 bad{0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 2; ++x)
              bad = F::mfma16(F::decode(nan_ones(vf[d][2 * x]), nan_ones(vf[d][2 * x + 1])),
                              see[x], bad);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (bad[k] > 0.f) dead[d / 8] |= 1u << (4 * (d & 7) + k);
#pragma unroll
            for (int w = 0; w < 4; ++w) vf[d][w] &= ~nan_bytes(vf[d][w]);
          }
        }
      }
      if (!apart) {
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          o[d] = F::mfma16(F::decode(vf[d][0], vf[d][1], vscale), pf[0], o[d]);
          o[d] = F::mfma16(F::decode(vf[d][2], vf[d][3], vscale), pf[1], o[d]);
        }
      } else {
        // the blocks one after the other, each with the other's weights 0
#pragma unroll 1
        for (int y = 0; y < 2; ++y) {
          const int ey = unit.reach(y ? e1 : e0);
          move(ey, ch * kChunk + y * kBlock);
          const float scale = Unit::scale(ey, unit.now);
          const h16x8 none = {0, 0, 0, 0, 0, 0, 0, 0};
          const h16x8 p0 = (q4 >> 1) == y ? pf[0] : none, p1 = (q4 >> 1) == y ? pf[1] : none;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            o[d] = F::mfma16(F::decode(vf[d][0], vf[d][1], scale), p0, o[d]);
            o[d] = F::mfma16(F::decode(vf[d][2], vf[d][3], scale), p1, o[d]);
          }
        }
      }
      if (more) load_v();
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    l *= exp2i(-kLift);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (dead[d / 8] >> (4 * (d & 7) + k) & 1) o[d][k] = __builtin_nanf("");

    // the waves' sums, in wave order
    __syncthreads();
    if (q4 == 0) {
      wave_m[wave][r] = m;
      wave_l[wave][r] = l;
      wave_e[wave][r] = E;
    }
    __syncthreads();
    const auto unit_of = [&](int rr) {  // the largest of the waves'
      int x = wave_e[0][rr];
#pragma unroll
      for (int w = 1; w < NW; ++w) x = max(x, wave_e[w][rr]);
      return x;
    };
    const auto largest = [&](int rr) {
      float x = wave_m[0][rr];
#pragma unroll
      for (int w = 1; w < NW; ++w) x = fmaxf(x, wave_m[w][rr]);
      return x;
    };
    const auto share = [&](int w, int rr, float M) {
      return M == -__builtin_inff() ? 0.f : exp2f_(wave_m[w][rr] - M);
    };
    const float mine = __builtin_amdgcn_ldexpf(share(wave, r, largest(r)), E - unit_of(r));
    // of the row that this thread writes
    constexpr int TR = 4 * NW, E8 = PASS / TR;  // threads of a row, channels of a thread
    const int wr = threadIdx.x / TR, wi = a.token_of(tile + wr);
    const float M = largest(wr);
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) L += wave_l[w][wr] * share(w, wr, M);
    const bool writes = tile + wr < rows;
    const bool alone = part.parts == 1;  // no other part of the sequence: the result itself
    const int64_t orow = (int64_t)(row0 + wi) * a.Hq + h * a.group + (tile + wr - wi * a.group);
    const float out_scale =
        exp2i(min(max(unit_of(wr) - kLift, -126), 127)) * (L == 0.f ? 0.f : 1.f / L);
#pragma unroll
    for (int pass = 0; pass < DP / PASS; ++pass) {
      if (pass) __syncthreads();
#pragma unroll
      for (int d = 0; d < PASS / 16; ++d)
        *reinterpret_cast<f32x4*>(&join[wave][r][16 * d + 4 * q4]) =
            o[pass * (PASS / 16) + d] * mine;
      __syncthreads();
      const int dd = (threadIdx.x % TR) * E8, d = pass * PASS + dd;
      float v[E8];
#pragma unroll
      for (int x = 0; x < E8; ++x) {
        v[x] = join[0][wr][dd + x];
#pragma unroll
        for (int w = 1; w < NW; ++w) v[x] += join[w][wr][dd + x];
        v[x] *= out_scale;
      }
      if (!writes || d >= D) continue;
      if (!alone) {
        float* const to = a.part + ((int64_t)split * c.T * a.Hq + orow) * D + d;
#pragma unroll
        for (int x = 0; x < E8; ++x) to[x] = v[x];
      } else {
        unsigned* const to = reinterpret_cast<unsigned*>(static_cast<unsigned short*>(a.out) +
                                                         orow * D + d);
#pragma unroll
        for (int x = 0; x < E8; x += 2)
          to[x / 2] = (unsigned)H::round(v[x]) | (unsigned)H::round(v[x + 1]) << 16;
      }
    }
    if (writes && threadIdx.x % TR == 0) {
      if (!alone || a.scores) a.part_ml[(int64_t)split * c.T * a.Hq + orow] = float2{M, L};
      if (alone && a.lse)
        a.lse[orow] = L == 0.f ? -__builtin_inff() : (M + __builtin_log2f(L)) * kLn2;
    }
  }
}

// ---------------------------------------------------------------------------------
// Many rows (prompts).  Workgroup = (128 rows, head, sequence, split): wave w holds rows 32 w.. as
// the columns of 32x32x16 products.  128 tokens at a time go to LDS as codes, straight from memory
// (no registers between), the next ones while these are worked on, 64 at a time; each wave decodes
// its operands.
//  - K operand row 8 a + 4 x + y: token 16 x + 4 a + y of the block, in this order in LDS, the
//    16-byte pieces of a row exchanged by row number: a 16-byte LDS read serves lanes 0-3, 12-15,
//    20-27 together (and 4-11, 16-19, 28-31), and these rows' equal pieces then lie in different
//    banks.
//  - a lane's scores are then tokens 16 (lane / 32) + i of the block, i < 16; V operand: channel
//    32 d + lane % 32, tokens 16 (lane / 32) + 8 s..: one 16-byte side of the cache.
//  - the sums are brought up to date as above.
// Heads and sequences vary fastest over the workgroups, then the tiles, the longest first: the
// last ones to start are short, and where the heads are a multiple of 8 one XCD's L2 holds few.
// Bound by VALU issue: a wave's 32 rows by 64 tokens take 451 instructions, 355 of them vector and 32
// products; what hides behind a product is four others.  128 of them decode, which each of the four
// waves does for itself.  Measured: a prompt of 4,096, 64 heads over 8 of 128, bf16: 292 us, 940
// TFLOP/s; 2 x 333 rows of 4,001 tokens, 32 heads, dealt out to 480 places of 512: 65 us, 11 of them
// for the join.  Above 128 channels the registers are all taken, and 80 (256) or 252 bytes (others) are
// spilled, with 256 none of them between the products of a tile: 900 rows of 6,000 of 8 heads 45.5 us
// with 128 channels, 82 with 256, 133 with 192, which are worked on as 256 at run-time strides.
// ---------------------------------------------------------------------------------
// Tokens that are staged at once: a barrier for each, so two tiles where LDS has room for it.
template <int DP>
constexpr int stage_tokens() {
  return DP > 128 ? kTile : 2 * kTile;
}

__device__ inline void load_to_lds(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Before the barrier behind which all waves read what these loads bring: every wave has to wait
// for its own.  A barrier alone does not, and where else a wave waits the compiler decides.
__device__ inline void wait_for_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int DT, int DP, bool EX>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void attn_many_kernel(Attn a) {
  using H = Half<DT>;
  using F = Half<FB_DT_F16>;
  constexpr int NP = DP / 32, ND = DP / 32, NPC = DP / 16;
  constexpr int ST = stage_tokens<DP>(), SB = ST / kBlock;
  constexpr int RW = ST / 4;            // rows of K that a wave loads, and as much of V
  constexpr int NI = RW * NPC / 64;     // 16-byte loads of a lane for each
  // Arrays of their own: the compiler waits for a load to LDS before it reads where that may go.
  __shared__ __align__(16) uint8_t lk0[ST * DP], lv0[ST * DP], lk1[ST * DP], lv1[ST * DP];
  const Cache& c = a.c;
  const int D = EX ? DP : c.D;  // known: the loads' addresses differ by constants
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, x2 = lane >> 5;
  const int h = blockIdx.x % c.H, bs = blockIdx.x / c.H;
  rows_of_none(a, h, bs + gridDim.x / c.H * blockIdx.y, gridDim.x / c.H * gridDim.y);
  int b = bs / a.splits, split = bs - b * a.splits, parts = a.splits;
  int tile0 = blockIdx.y, tile_step = gridDim.y, part_stages = a.split_tokens / ST;
  if (a.dealt) {
    const Part part = find_part(a, bs, 0, ST);
    b = __builtin_amdgcn_readfirstlane(part.b);
    split = __builtin_amdgcn_readfirstlane(part.slot);
    if (split < 0) return;
    parts = __builtin_amdgcn_readfirstlane(part.parts);
    tile0 = __builtin_amdgcn_readfirstlane(part.tile);
    tile_step = a.tiles;
    const int stages = (held(c, b) + ST - 1) / ST;
    part_stages = (stages + parts - 1) / parts;
  }
  int row0, n;
  c.rows(b, row0, n);
  const int len = min(max(c.lens[b], 0), c.capacity());
  const int rows = n * a.group;
  const int tiles = (rows + kRows - 1) / kRows;
  const auto exchange = [](int row, int pc) {
    return pc ^ (NPC == 4 ? (row >> 2) & 3 : NPC == 8 ? (row >> 1) & 7 : row & 15);
  };
  // What a lane loads of the wave's block.  Pieces past D are others of the same row: they meet
  // zeros of q, or channels that are not written.
  const int wave_block = wave * RW / kBlock, wave_row = wave * RW % kBlock;
  const auto k_from = [&](int i) {
    const int piece = i * 64 + lane;
    const int rho = wave_row + piece / NPC;
    const int tok = ((rho & 4) << 2) | ((rho >> 1) & 12) | (rho & 3);
    const int pc = exchange(rho, piece % NPC);
    return tok * D + (pc * 16 < D ? pc : pc % (D / 16)) * 16;
  };
  const auto v_from = [&](int i) {
    const int piece = i * 64 + lane, side = wave_row / kSide + piece / DP;
    return (side * D + min(piece % DP, D - 1)) * 16;
  };
  const int k0 = k_from(0), v0 = v_from(0);
  // the i-th: where D is known it differs from the first by constants
  const auto k_at = [&](int i) {
    if constexpr (!EX) return k_from(i);
    if constexpr (NPC == 4) return k0 + 8 * i * DP;
    if constexpr (NPC == 8) return (k0 ^ (i & 1) * 64) + 4 * i * DP;
    return (k0 ^ i * 64) + (16 * (i & 1) + 4 * (i >> 1)) * DP;
  };
  const auto v_at = [&](int i) { return EX ? v0 + i * 1024 : v_from(i); };
  const unsigned per = (unsigned)c.P / kBlock;
  const int32_t* const table = c.table + b * c.table_stride;
  for (int ti = tile0; ti < tiles; ti += tile_step) {
    const int tile = (tiles - 1 - ti) * kRows;  // the longest first
    const int row = tile + wave * 32 + r, i = a.token_of(row);
    const bool there = row < rows;
    const int head = h * a.group + (row - i * a.group);
    const int sees = there ? min(max(len - n + i + 1, 0), len) : 0;
    // least and most that the wave's and the workgroup's rows see
    const int i_lo = a.token_of(tile + wave * 32);
    const int least = min(max(len - n + i_lo + 1, 0), len);
    const int least_wg = min(max(len - n + a.token_of(tile) + 1, 0), len);
    const int i_hi = a.token_of(min(tile + wave * 32 + 32, rows) - 1);
    const int wave_most = tile + wave * 32 < rows ? min(max(len - n + i_hi + 1, 0), len) : 0;
    const int j_hi = a.token_of(min(tile + kRows, rows) - 1);
    const int most = min(max(len - n + j_hi + 1, 0), len);
    typename H::x8 qf[NP][2];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = 32 * p + 16 * x2 + 8 * u;
        qf[p][u] = load_q<DT>(a, there && d < D,
                              (int64_t)(row0 + i) * a.q_token + head * a.q_head + d);
      }
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int k = 0; k < 16; ++k) o[d][k] = 0.f;
    float m = -__builtin_inff(), l = 0.f;  // m: what the sums are relative to
    bool far = false;                      // whether a row's m is
    Unit unit;
    int E = unit.now;                      // the row's: of the last block that it saw
    unsigned dead[(ND + 1) / 2] = {};      // bit 16 (d % 2) + k of d / 2: o[d][k] saw a NaN value

    const int first = split * part_stages;
    const int all = (most + ST - 1) / ST;
    const int last = split + 1 == parts ? all : min(all, first + part_stages);
    // lane j has block j % SB of the next stage: its page as the table has it (read a stage ahead)
    // and place in the page
    int id, at;
    const auto look = [&](int t) {
      const unsigned blk = (unsigned)t * SB + lane % SB;
      const unsigned pg = a.per_shift >= 0 ? blk >> a.per_shift : blk / per;
      at = (int)(blk - pg * per);
      id = pg < (unsigned)c.max_pages ? table[pg] : 0;
    };
    int scale_k, scale_v;  // lane j: of block j % SB of the stage that is on its way
    const auto fetch = [&](uint8_t* to_k, uint8_t* to_v, int t) __attribute__((always_inline)) {
      const int64_t bi = c.block_index((unsigned)id < (unsigned)c.pages ? id : 0, h, at);
      const int64_t mine =
          ((int64_t)__builtin_amdgcn_readlane((int)(bi >> 32), wave_block) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)bi, wave_block)) * kBlock * D;
#pragma unroll
      for (int k = 0; k < NI; ++k) {
        load_to_lds(c.k + mine + k_at(k), to_k + (wave * NI + k) * 1024);
        load_to_lds(c.v + mine + v_at(k), to_v + (wave * NI + k) * 1024);
      }
      scale_k = c.ks[bi];
      scale_v = c.vs[bi];
      if (t + 1 < last) look(t + 1);
    };
    __syncthreads();  // the buffers of the row tile before are free
    if (first < last) {
      look(first);
      fetch(lk0, lv0, first);
    }
    const auto run = [&](int st, const uint8_t* in_k, uint8_t* in_v, uint8_t* to_k,
                         uint8_t* to_v) __attribute__((always_inline)) {
      wait_for_loads();
      __syncthreads();  // this stage has arrived; everyone is done with the other buffers
      const int stage_k = scale_k, stage_v = scale_v;
      if (st + 1 < last) fetch(to_k, to_v, st + 1);
#pragma unroll 1
      for (int part = 0; part < ST / kTile; ++part) {
      const int t = st * (ST / kTile) + part;
      const uint8_t* const tk = in_k + part * kTile * DP;
      uint8_t* const tv = in_v + part * kTile * DP;
      // What is read from LDS differs by constants and exchanged bits; the asm keeps the compiler from
      // holding every address for the whole walk, which above 128 channels spills.
      int k_piece = (r * NPC + exchange(r, x2)) * 16, v_piece = (x2 * DP + r) * 16;
      asm volatile("" : "+v"(k_piece), "+v"(v_piece));
      const auto values = [&](int i) {  // block i / ND, channels 32 (i % ND)..
        return *reinterpret_cast<const u32x4*>(tv + v_piece + (2 * (i / ND) * DP + 32 * (i % ND)) * 16);
      };
      if (t * kTile + kTile > least_wg) {
        asm volatile("");
        // Some row does not see some token here.  A NaN value reaches the rows that see its token,
        // and no others, and what lies behind the end may be anything; but 0 * NaN must not come
        // up.  So NaNs are noted for the rows that see them, and taken out of the tile.  Every
        // wave looks at the same tile and comes to the same decision.
        const int seen = sees - t * kTile - x2 * 16, held = len - t * kTile - x2 * 16;
        unsigned nan = 0;
#pragma unroll 1
        for (int i = 0; i < 2 * ND; ++i) {
          const u32x4 w = values(i);
#pragma unroll
          for (int u = 0; u < 4; ++u) nan |= nan_bytes(w[u]);
        }
        if (__any(nan != 0)) {
          h16x8 see[2][2];
#pragma unroll
          for (int k = 0; k < 32; ++k)
            see[k / 16][k / 8 & 1][k & 7] =
                (k / 16) * kBlock + k % 16 < seen ? (_Float16)1 : (_Float16)0;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            f32x16 bad;
#pragma unroll
            for (int k = 0; k < 16; ++k) bad[k] = 0.f;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              u32x4 w = values(y * ND + d);
#pragma unroll
              for (int u = 0; u < 4; ++u)
                w[u] = nan_ones(w[u] & keep_bytes(y * kBlock + 4 * u, held));
              bad = F::mfma32(F::decode(w[0], w[1]), see[y][0], bad);
              bad = F::mfma32(F::decode(w[2], w[3]), see[y][1], bad);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (bad[k] > 0.f) dead[d / 2] |= 1u << (16 * (d & 1) + k);
          }
          __syncthreads();
          for (int i = tid; i < kTile * DP / 16; i += 256) {
            u32x4 w = *reinterpret_cast<const u32x4*>(tv + i * 16);
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] &= ~nan_bytes(w[u]);
            *reinterpret_cast<u32x4*>(tv + i * 16) = w;
          }
          __syncthreads();
        }
      }
      if (t * kTile >= wave_most) continue;  // the same for the wave
      float ks[2];
#pragma unroll
      for (int y = 0; y < 2; ++y)
        ks[y] = key_scale(a.scale2, __builtin_amdgcn_readlane(stage_k, 2 * part + y));
      const bool masked = t * kTile + kTile > least;  // the same for the wave
      const int seen = sees - t * kTile - x2 * 16;    // tokens of the lane's part
      // Keys: piece i is 16 channels of block i % 2.  A piece is read two ahead of its products, and
      // decoded between the products of the one before: left to itself the compiler reads,
      // waits, decodes and multiplies in turn, and a wave waits for LDS at every piece.
      f32x16 s[2];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int k = 0; k < 16; ++k) s[y][k] = 0.f;
      {
        const auto read = [&](int i) {
          return *reinterpret_cast<const u32x4*>(tk + (i & 1) * 32 * NPC * 16 +
                                                 (k_piece ^ (i & ~1) * 16));
        };
        u32x4 w[2] = {read(0), read(1)};
        typename H::x8 lo = H::decode(w[0][0], w[0][1]), hi = H::decode(w[0][2], w[0][3]);
#pragma unroll
        for (int i = 0; i < 2 * NP; ++i) {
          typename H::x8 next_lo = lo, next_hi = hi;
          if (i + 2 < 2 * NP) w[i & 1] = read(i + 2);
          const u32x4 n = w[(i + 1) & 1];
          __builtin_amdgcn_sched_barrier(0);
          s[i & 1] = H::mfma32(lo, qf[i / 2][0], s[i & 1]);
          if (i + 1 < 2 * NP) next_lo = H::decode(n[0], n[1]);
          __builtin_amdgcn_sched_barrier(0);
          s[i & 1] = H::mfma32(hi, qf[i / 2][1], s[i & 1]);
          if (i + 1 < 2 * NP) next_hi = H::decode(n[2], n[3]);
          __builtin_amdgcn_sched_barrier(0);
          lo = next_lo;
          hi = next_hi;
        }
      }
      u32x4 vw[2] = {values(0), values(1)};  // on their way during the weights
      if (masked) {
        asm volatile("");  // a branch, not selects in every tile
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (y * kBlock + k >= seen) s[y][k] = -__builtin_inff();
      }
      // The value blocks' unit, or one for each.  A row of the wave's sees the first; where none
      // sees the second, its weights are 0.
      const auto follow = [&](int e, int from) __attribute__((always_inline)) {
        const float f = unit.move(e);
        const bool sees_it = sees > from;
        E = sees_it ? unit.now : E;
        return sees_it ? f : 1.f;  // what the row's sums are multiplied by
      };
      const int e0 = unit.reach(__builtin_amdgcn_readlane(stage_v, 2 * part) - 127);
      const bool turn = !unit.takes(e0);  // the same for the wave
      float turned = 1.f;
      if (turn) turned = follow(e0, t * kTile);
      const int e1 = t * kTile + kBlock < wave_most
                         ? unit.reach(__builtin_amdgcn_readlane(stage_v, 2 * part + 1) - 127)
                         : unit.now;
      const float vscale[2] = {Unit::scale(e0, unit.now),
                               Unit::scale(e1, unit.takes(e1) ? unit.now : unit.within(e1))};
      float sum[2];
      h16x8 pf[2][2];
      const auto weigh = [&](auto anew) __attribute__((always_inline)) {
        const float shift = (float)kLift - (m == -__builtin_inff() ? 0.f : m);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          sum[y] = 0.f;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float p = exp2f_(anew ? exponent(s[y][k], ks[y], m, shift)
                                        : __builtin_fmaf(s[y][k], ks[y], shift));
            sum[y] += p;
            pf[y][k / 8][k & 7] = (_Float16)p;
          }
        }
      };
      weigh(std::false_type{});
      if (turn || far || __any(m == -__builtin_inff() || sum[0] + sum[1] > kMost)) {
        asm volatile("");
        float mx[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          mx[y] = s[y][0];
#pragma unroll
          for (int k = 1; k < 16; ++k) mx[y] = fmaxf(mx[y], s[y][k]);
        }
        float big = fmaxf(mx[0] * ks[0], mx[1] * ks[1]);  // the scales are positive
        big = fmaxf(big, __shfl_xor(big, 32));
        const float up = fmaxf(m, big);
        const float alpha = up == -__builtin_inff() ? 0.f : exp2f_(m - up), both = alpha * turned;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= both;
        m = up;
        far = __any(is_far(m));
        weigh(std::true_type{});
      }
      l += sum[0] + sum[1];
      {
        h16x8 lo = F::decode(vw[0][0], vw[0][1], vscale[0]);
        h16x8 hi = F::decode(vw[0][2], vw[0][3], vscale[0]);
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i) {
          const int y = i / ND, d = i % ND;
          const float scale = vscale[min(i + 1, 2 * ND - 1) / ND];
          h16x8 next_lo = lo, next_hi = hi;
          if (i + 2 < 2 * ND) vw[i & 1] = values(i + 2);
          const u32x4 n = vw[(i + 1) & 1];
          if (i == ND && !unit.takes(e1)) {  // the same for the wave
            asm volatile("");
            const float f = follow(e1, t * kTile + kBlock);
#pragma unroll
            for (int z = 0; z < ND; ++z) o[z] *= f;
          }
          __builtin_amdgcn_sched_barrier(0);
          o[d] = F::mfma32(lo, pf[y][0], o[d]);
          if (i + 1 < 2 * ND) next_lo = F::decode(n[0], n[1], scale);
          __builtin_amdgcn_sched_barrier(0);
          o[d] = F::mfma32(hi, pf[y][1], o[d]);
          if (i + 1 < 2 * ND) next_hi = F::decode(n[2], n[3], scale);
          __builtin_amdgcn_sched_barrier(0);
          lo = next_lo;
          hi = next_hi;
        }
      }
      }
    };
    for (int st = first; st < last; st += 2) {
      run(st, lk0, lv0, lk1, lv1);
      if (st + 1 < last) run(st + 1, lk1, lv1, lk0, lv0);
    }
    l += __shfl_xor(l, 32);
    l *= exp2i(-kLift);
#pragma unroll
    for (int d = 0; d < ND; ++d)
      if (dead[d / 2])
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (dead[d / 2] >> (16 * (d & 1) + k) & 1) o[d][k] = __builtin_nanf("");
    if (there) {
      const int64_t orow = (int64_t)(row0 + i) * a.Hq + head;
      const float factor = exp2i(min(max(E - kLift, -126), 127)) * (l == 0.f ? 0.f : 1.f / l);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
          const int ch = 32 * d + 2 * k + 4 * x2;
          if (ch >= D) continue;
          const f32x4 v = f32x4{o[d][k], o[d][k + 1], o[d][k + 2], o[d][k + 3]} * factor;
          if (parts > 1) {
            *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * c.T * a.Hq + orow) * D + ch) = v;
          } else {
            const u32x2 w{(unsigned)H::round(v[0]) | (unsigned)H::round(v[1]) << 16,
                          (unsigned)H::round(v[2]) | (unsigned)H::round(v[3]) << 16};
            *reinterpret_cast<u32x2*>(static_cast<unsigned short*>(a.out) + orow * D + ch) = w;
          }
        }
      if (x2 == 0) {
        if (parts > 1)
          a.part_ml[(int64_t)split * c.T * a.Hq + orow] = float2{m, l};
        else if (a.lse)
          a.lse[orow] = l == 0.f ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
      }
    }
  }
}

// How many parts sequence b has, as find_part deals them.
__device__ inline int parts_of(const Attn& a, int b, int chunk) {
  if (!a.dealt) return a.splits;
  const Load mine = load_of(a, threadIdx.x & 63, chunk);
  return __shfl(mine.parts(a, part_size(a, mine)), b);
}

// The parts' sums of a sequence's rows, in a fixed order.  D / 4 threads go over every `ways`-th part
// of a row, and the first of these groups adds up what the others found.  Workgroup: (some rows of
// the cached head's, head, sequence).
template <int DT>
__device__ void join_parts(const Attn& a, int ways, int x, int xs, int h, int b) {
  using H = Half<DT>;
  __shared__ f32x4 part_v[256];
  __shared__ float part_m[64], part_l[64];
  // The weights' sums are held 2^24 times smaller: times averages near fp32's range they would pass it.
  constexpr float kBelow = 24.f;
  const Cache& c = a.c;
  int row0, n;
  c.rows(b, row0, n);
  const int rows = n * a.group;
  const int parts = parts_of(a, b, a.chunk);
  if (a.dealt && parts == 1) return;  // written already
  const int64_t all = (int64_t)c.T * a.Hq;
  const int width = c.D / 4, groups = 256 / width / ways * ways, per = groups / ways;
  const int g = threadIdx.x / width, d = (threadIdx.x - g * width) * 4, way = g % ways;
  for (int r0 = x * per; r0 < rows; r0 += xs * per) {
    const int r = r0 + g / ways, i = a.token_of(r);
    const bool works = g < groups && r < rows;
    const int64_t row = (int64_t)(row0 + i) * a.Hq + h * a.group + (r - i * a.group);
    float M = -__builtin_inff(), L = 0.f;
    f32x4 v{0, 0, 0, 0};
    constexpr int kAhead = 4;  // parts that are read at once
    for (int s0 = way; works && s0 < parts; s0 += kAhead * ways) {
      float2 ml[kAhead];
      f32x4 w[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int s = s0 + j * ways, from = min(s, parts - 1);
        ml[j] = a.part_ml[from * all + row];
        w[j] = *reinterpret_cast<const f32x4*>(a.part + (from * all + row) * c.D + d);
        if (s >= parts) ml[j].y = 0.f;
      }
      float to = M;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) to = fmaxf(to, ml[j].y == 0.f ? M : ml[j].x);
      const float f0 = M == to ? 1.f : exp2f_(M - to);
      L *= f0;
      v *= f0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float g = ml[j].y == 0.f ? 0.f : ml[j].y * exp2f_(ml[j].x - to - kBelow);
        L += g;
        v += w[j] * g;
      }
      M = to;
    }
    if (ways > 1) {
      __syncthreads();
      part_v[threadIdx.x] = v;
      if (d == 0 && g < 64) {
        part_m[g] = M;
        part_l[g] = L;
      }
      __syncthreads();
      if (works && way == 0) {
        float to = M;
        for (int w = 1; w < ways; ++w) to = fmaxf(to, part_m[g + w]);
        const float f0 = M == to ? 1.f : exp2f_(M - to);
        L *= f0;
        v *= f0;
        for (int w = 1; w < ways; ++w) {
          const float f = part_l[g + w] == 0.f ? 0.f : exp2f_(part_m[g + w] - to);
          L += part_l[g + w] * f;
          v += part_v[threadIdx.x + w * width] * f;
        }
        M = to;
      }
    }
    if (!works || way) continue;
    v *= L == 0.f ? 0.f : 1.f / L;
    const u32x2 w{(unsigned)H::round(v[0]) | (unsigned)H::round(v[1]) << 16,
                  (unsigned)H::round(v[2]) | (unsigned)H::round(v[3]) << 16};
    *reinterpret_cast<u32x2*>(static_cast<unsigned short*>(a.out) + row * c.D + d) = w;
    if (d == 0 && a.lse)
      a.lse[row] = L == 0.f ? -__builtin_inff() : (M + (__builtin_log2f(L) + kBelow)) * kLn2;
  }
}

// ---------------------------------------------------------------------------------
// Accumulated weights of many rows: weights[t] += sum over the rows of exp(score - lse).  Workgroup =
// (head and sequence, 256 tokens, a run of the rows).  Each wave holds 64 tokens' keys (32 of the
// widest), decoded, as operands; the rows go to LDS, 128 at a time and straight from memory, and an
// operand that is read there meets both blocks of keys (with one block the LDS reads took as long as
// the products).  A lane's sums are of 16 tokens a block over the rows of its column, so nothing
// crosses lanes before the end.  Runs of rows leave their sums apart, which a last small kernel adds
// in order: no atomics.  Half the products of the attention itself.  Measured: a prompt of 4,096, 64
// heads over 8 of 128: 215 us, 640 TFLOP/s (5 more for the last kernel); what it waits for beside the
// products and one exponential a score was not looked into.
// ---------------------------------------------------------------------------------
struct Weights {
  float* to;
  int64_t seq, head;
  int tokens;
  float* part;   // or null: [runs][B][H][part_tokens]
  int part_tokens, runs, run_rows;
};

template <int DP>
constexpr int weight_rows() {  // that are staged at once
  return DP > 128 ? 32 : 128;
}

template <int DP>
constexpr int weight_blocks() {  // of a wave
  return DP > 128 ? 1 : 2;
}

template <int DT, int DP>
__global__ __launch_bounds__(256, 2) void attn_weights_kernel(Attn a, Weights w) {
  using H = Half<DT>;
  constexpr int NP = DP / 32, NQ = DP / 8;   // 16-byte pieces of a row of q
  constexpr int ROWS = weight_rows<DP>();
  constexpr int NL = ROWS * NQ / 256;        // of which a thread loads so many
  // arrays of their own, as in attn_many_kernel
  __shared__ __align__(16) uint8_t lq0[ROWS * DP * 2], lq1[ROWS * DP * 2];
  __shared__ float lse2[2][ROWS];
  constexpr int KB = weight_blocks<DP>(), TOKENS = 4 * KB * kBlock;
  const Cache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, x2 = lane >> 5;
  const int h = blockIdx.x % c.H, b = blockIdx.x / c.H, run = blockIdx.z;
  int row0, n;
  c.rows(b, row0, n);
  const int len = held(c, b), rows = n * a.group;
  const int end = min(len, w.tokens);
  // where piece pc of a row lies: the lanes that one LDS read serves (0-3, 12-15, 20-27) read
  // equal pieces of their rows from different banks
  const auto exchange = [](int row, int pc) {
    return pc ^ (NQ == 8 ? (row >> 1) & 7 : row & 15);
  };
  for (int tile = blockIdx.y * TOKENS; tile < end; tile += gridDim.y * TOKENS) {
    const int t0 = tile + wave * KB * kBlock;  // the wave's tokens
    typename H::x8 kf[KB][NP][2];
    float ks[KB], sum[KB][16];
#pragma unroll
    for (int z = 0; z < KB; ++z) {
      int at;
      const int page = max(c.page_of(b, t0 / kBlock + z, at), 0);
      const int64_t bi = c.block_index(page, h, at);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        // zeros past D: q's pieces there are others of the same row
        const int ch = 32 * p + 16 * x2;
        u32x4 k{0, 0, 0, 0};
        if (ch < c.D) k = *reinterpret_cast<const u32x4*>(c.k + (bi * kBlock + r) * c.D + ch);
        kf[z][p][0] = H::decode(k[0], k[1]);
        kf[z][p][1] = H::decode(k[2], k[3]);
      }
      ks[z] = key_scale(a.scale2, c.ks[bi]);
#pragma unroll
      for (int k = 0; k < 16; ++k) sum[z][k] = 0.f;
    }
    // the rows that see the tile's first token, of the run
    const int seeing = max(tile - (len - n), 0) * a.group;
    const int from = max(run * w.run_rows, seeing / ROWS * ROWS);
    const int to = run + 1 == w.runs ? rows : min(rows, (run + 1) * w.run_rows);
    float next_lse = 0.f;
    const auto fetch = [&](uint8_t* buf, int first) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < NL; ++x) {
        // a wave's 64 pieces lie side by side in LDS
        const int e = (wave * NL + x) * 64 + lane, at = e / NQ;
        const int row = min(first + at, to - 1), i = a.token_of(row);
        const int pc = exchange(at, e % NQ);
        load_to_lds(static_cast<const uint8_t*>(a.q) +
                        2 * ((int64_t)(row0 + i) * a.q_token +
                             (h * a.group + (row - i * a.group)) * a.q_head +
                             (pc * 8 < c.D ? pc : pc % (c.D / 8)) * 8),
                    buf + (wave * NL + x) * 1024);
      }
      if (tid < ROWS) {
        const int row = min(first + tid, to - 1), i = a.token_of(row);
        next_lse = a.lse[(int64_t)(row0 + i) * a.Hq + h * a.group + (row - i * a.group)];
      }
    };
    const auto stage = [&](int first, const uint8_t* buf, uint8_t* other, int parity)
        __attribute__((always_inline)) {
      // A row that sees nothing gives no weight.  One far from 0 (see kFar) has what its sum's rounding
      // may hide added, so that no weight is above 1.
      if (tid < ROWS) {
        const float l = next_lse * kLog2e;
        lse2[parity][tid] = next_lse == -__builtin_inff() ? __builtin_inff()
                            : is_far(l)                   ? l + __builtin_fabsf(l) * 0x1p-21f
                                                          : l;
      }
      wait_for_loads();
      __syncthreads();  // these rows are there; everyone is done with the other buffer
      if (first + ROWS < to) fetch(other, first + ROWS);
#pragma unroll 1
      for (int y = 0; y < ROWS / 32; ++y) {
        f32x16 s[KB];
#pragma unroll
        for (int z = 0; z < KB; ++z)
#pragma unroll
          for (int k = 0; k < 16; ++k) s[z][k] = 0.f;
        const int row = y * 32 + r;
        const auto read = [&](int i) {
          return *reinterpret_cast<const typename H::x8*>(
              buf + row * DP * 2 + exchange(row, 4 * (i / 2) + 2 * x2 + (i & 1)) * 16);
        };
        typename H::x8 q[3] = {read(0), read(1), read(2)};  // read three ahead
#pragma unroll
        for (int i = 0; i < 2 * NP; ++i) {
          const auto now = q[i % 3];
          if (i + 3 < 2 * NP) q[i % 3] = read(i + 3);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int z = 0; z < KB; ++z) s[z] = H::mfma32(kf[z][i / 2][i & 1], now, s[z]);
        }
        float l = lse2[parity][row];
        // the tile's least row against the wave's last token, its last against the run's end
        const bool masked = a.token_of(first + y * 32) + len - n + 1 < t0 + KB * kBlock ||
                            first + y * 32 + 32 > to;
        if (masked) {
          asm volatile("");  // a branch, not selects in every tile
          // a row of NaN gives nothing to what it does not see either: its scores have the NaN
          const float lost = l == l ? 0.f : l;
          l = l == l ? l : 0.f;
          const int seen = first + row < to
                               ? len - n + a.token_of(first + row) + 1 - t0 - 4 * x2
                               : INT32_MIN;
#pragma unroll
          for (int z = 0; z < KB; ++z)
#pragma unroll
            for (int k = 0; k < 16; ++k)
              s[z][k] = z * kBlock + 8 * (k / 4) + k % 4 < seen ? s[z][k] + lost : -__builtin_inff();
        }
#pragma unroll
        for (int z = 0; z < KB; ++z)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            sum[z][k] += exp2f_(__builtin_fmaf(s[z][k], ks[z], -l));
      }
    };
    __syncthreads();  // the buffers of the tile before are free
    if (from < to) fetch(lq0, from);
    for (int first = from; first < to; first += 2 * ROWS) {
      stage(first, lq0, lq1, 0);
      if (first + ROWS < to) stage(first + ROWS, lq1, lq0, 1);
    }
#pragma unroll
    for (int z = 0; z < KB; ++z)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float v = sum[z][k];
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor(v, o);
        const int t = t0 + z * kBlock + 8 * (k / 4) + 4 * x2 + k % 4;
        if (r == k && t < end) {
          if (w.part)
            w.part[((int64_t)(run * c.B + b) * c.H + h) * w.part_tokens + t] = v;
          else
            w.to[b * w.seq + h * w.head + t] += v;
        }
      }
  }
}

// Adds the runs' sums, in order.
__global__ __launch_bounds__(256) void attn_weights_join_kernel(Cache c, Weights w) {
  const int h = blockIdx.y, b = blockIdx.z, end = min(held(c, b), w.tokens);
  for (int t = blockIdx.x * 256 + threadIdx.x; t < end; t += gridDim.x * 256) {
    float v = 0.f;
#pragma unroll 4
    for (int run = 0; run < w.runs; ++run)
      v += w.part[((int64_t)(run * c.B + b) * c.H + h) * w.part_tokens + t];
    w.to[b * w.seq + h * w.head + t] += v;
  }
}

// Weights of few rows, from the scores that were written down: 4 tokens a thread.  Every row's sum
// comes from its parts here too, so that this need not wait for their being joined; the first 8 rows'
// scores and the old weights are asked for before it, 16 threads take a row's parts.
__device__ void add_few_weights(const Attn& a, const Weights& w, int x, int xs, int h, int b) {
  constexpr int kFirst = 8;
  __shared__ float part_m[16][16], part_l[16][16];
  __shared__ float lse2[16];
  const Cache& c = a.c;
  int row0, n;
  c.rows(b, row0, n);
  const int rows = min(n * a.group, a.score_rows), len = held(c, b);
  const int64_t all = (int64_t)c.T * a.Hq;
  const int end = min(len, w.tokens);
  const float* const s0 = a.scores + ((int64_t)b * c.H + h) * a.score_rows * a.score_tokens;
  float* const to = w.to + b * w.seq + h * w.head;
  int t = (x * 256 + threadIdx.x) * 4;
  f32x4 score[kFirst], old{0, 0, 0, 0};
  const auto load = [&] {
    if (t >= end) return;
#pragma unroll
    for (int row = 0; row < kFirst; ++row)
      if (row < rows)
        score[row] = *reinterpret_cast<const f32x4*>(s0 + (int64_t)row * a.score_tokens + t);
#pragma unroll
    for (int k = 0; k < 4; ++k) old[k] = to[min(t + k, end - 1)];
  };
  load();
  const int parts = parts_of(a, b, kChunk);
  const int mine = threadIdx.x & 15, first = threadIdx.x >> 4;
  float M = -__builtin_inff(), L = 0.f;
  if (mine < rows) {
    const int i = a.token_of(mine);
    const int64_t row = (int64_t)(row0 + i) * a.Hq + h * a.group + (mine - i * a.group);
    for (int s = first; s < parts; s += 16) {
      const float2 ml = a.part_ml[s * all + row];
      if (ml.y == 0.f) continue;
      const float to_m = fmaxf(M, ml.x);
      L = L * exp2f_(M - to_m) + ml.y * exp2f_(ml.x - to_m);
      M = to_m;
    }
  }
  part_m[first][mine] = M;
  part_l[first][mine] = L;
  __syncthreads();
  if ((int)threadIdx.x < rows) {  // in a fixed order
#pragma unroll
    for (int s = 1; s < 16; ++s) M = fmaxf(M, part_m[s][mine]);
    L = 0.f;
#pragma unroll
    for (int s = 0; s < 16; ++s)
      L += part_l[s][mine] == 0.f ? 0.f : part_l[s][mine] * exp2f_(part_m[s][mine] - M);
    lse2[mine] = L == 0.f ? 0.f : M + __builtin_log2f(L);  // 0: sees nothing
  }
  __syncthreads();
  while (t < end) {
    f32x4 sum{0, 0, 0, 0};
    if (t + 4 <= len - n + 1) {  // every row sees them
#pragma unroll
      for (int row = 0; row < kFirst; ++row)
        if (row < rows)
#pragma unroll
          for (int k = 0; k < 4; ++k) sum[k] += exp2f_(score[row][k] - lse2[row]);
#pragma unroll 4
      for (int row = kFirst; row < rows; ++row) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(s0 + (int64_t)row * a.score_tokens + t);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += exp2f_(s[k] - lse2[row]);
      }
    } else {  // seldom; a row of NaN gives nothing to what it does not see either
#pragma unroll 1
      for (int row = 0; row < rows; ++row) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(s0 + (int64_t)row * a.score_tokens + t);
        const int sees = len - n + a.token_of(row) + 1;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += t + k < sees ? exp2f_(s[k] - lse2[row]) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (t + k < end) to[t + k] = old[k] + sum[k];
    t += xs * 1024;
    load();
  }
}

// What is left after the parts: blocks x < joins join them, the others add the weights.  Bound by the
// parts' bytes where there are many rows (2 parts of 980 rows of 24 heads of 128: 11 us), by latency
// otherwise.
template <int DT>
__global__ __launch_bounds__(256) void attn_finish_kernel(Attn a, Weights w, int joins, int ways) {
  const int x = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  if (x < joins)
    join_parts<DT>(a, ways, x, joins, h, b);
  else
    add_few_weights(a, w, x - joins, gridDim.x - joins, h, b);
}

// ------------------------------------------------------------------ host side
struct Plan {
  bool few, dealt;
  int chunk, grain, most, tiles;
  int splits, split_tokens, ways;  // ways: of join_parts
  int score_rows, score_tokens;
  int runs, run_rows;              // of attn_weights_kernel
  size_t part, ml, total;
};

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// How a call is split.  It goes by host numbers alone, so that a captured call fits any lengths.
Plan plan(const fb_cache_t* c, const fb_seqs_t* s, int q_heads, int w_tokens) {
  Plan p{};
  const int group = q_heads / c->heads;
  const int64_t rows = (int64_t)std::max(1, std::min(s->max_new, s->tokens)) * group;
  p.few = rows <= 16;
  const int64_t capacity = std::min<int64_t>((int64_t)s->max_pages * c->page, 0x7FFFFFE0);
  const int64_t len = std::max<int64_t>(1, std::min<int64_t>(s->max_len, capacity));
  const int64_t tiles = p.few ? 1 : (rows + kRows - 1) / kRows;
  const int64_t units = tiles * c->heads * s->seqs;
  // The least part of few rows: a chunk a wave where that makes some but not many parts (one sequence
  // of 8 heads: 2,000 tokens 10.4 us, 12.6 with two; 8,000 11.1 and 12.7; 16,384 14.0 and 13.8, of one
  // head 11.7 and 13.1), two where one part could do (375 tokens of 160 heads: 9.2 us, 14.8 with two
  // parts to join) or many would be (100,000 tokens of one head: 17.9 us, 21.2 with 390).
  p.grain = len > 8 * kChunk && len <= 256 * kChunk ? 4 : 8;
  p.chunk = kChunk;
  if (!p.few) {
    p.chunk = c->head_dim > 128 ? stage_tokens<256>() : stage_tokens<128>();
    p.grain = 4 * kTile / p.chunk;
  }
  const int64_t least = (int64_t)p.grain * p.chunk;
  const int step = p.few ? 4 * kChunk : 4 * kTile;  // a part is a whole number of rounds or stages
  const int64_t most = (len + least - 1) / least;
  // Two workgroups a CU run side by side, of more than 128 channels one (900 rows of 6,000 tokens, 8
  // heads of 256: 101 us split for two, 82 so; one of 60,000, 4 heads: 39 and 34).
  const int64_t cus = fb_gpu::cu_count(), slots = c->head_dim <= 128 ? 2 * cus : cus;
  const int64_t want = std::min(std::max<int64_t>(1, slots / units), most);
  const int64_t steps = (len + step - 1) / step;
  const int64_t per = std::max((steps + want - 1) / want, least / step);
  p.split_tokens = (int)(per * step);
  p.splits = (int)((steps + per - 1) / per);
  int parts = p.splits;  // of one sequence, at most
  // Many rows are dealt out where parts are long: 2 x 333 rows of 4,001 tokens, 32 heads of 128, in
  // parts of 2,048 77 us, dealt out 66; but 3 x 100 of 2,000, 32 heads over 8, in parts of 512 34.6 and
  // 37.9, for the dealing and more parts to join.  A sequence has twice its even share at most, for
  // what joining reads.
  if (s->seqs > 1 && s->seqs <= 64 && p.splits > 1 &&
      (p.few || (int64_t)p.split_tokens * c->head_dim >= 1024 * 128)) {
    p.dealt = true;
    p.tiles = p.few ? 0 : (int)tiles;
    p.most = p.few ? INT32_MAX : 2 * p.splits;
    p.splits = (int)std::min<int64_t>(std::max<int64_t>(slots / c->heads, s->seqs),
                                      most * units / c->heads);
    parts = (int)std::min({(int64_t)p.splits, (int64_t)p.most, (capacity + least - 1) / least});
  }
  const size_t n = (size_t)s->tokens * q_heads;
  p.ways = 1;
  if (parts > 1) {
    p.part = align256((size_t)parts * n * c->head_dim * 4);
    // about 4 parts a thread
    while (p.ways * 4 < parts && p.ways * 2 * (c->head_dim / 4) <= 256) p.ways *= 2;
  }
  if (parts > 1 || (p.few && w_tokens > 0)) p.ml = align256((size_t)parts * n * 8);
  p.total = p.part + p.ml;
  if (p.few && w_tokens > 0) {
    p.score_rows = (int)rows;
    p.score_tokens = (w_tokens + kChunk - 1) / kChunk * kChunk;
    p.total += align256((size_t)s->seqs * c->heads * p.score_rows * p.score_tokens * 4);
  } else if (w_tokens > 0) {
    // Runs of rows until there are 12 workgroups a CU (a causal prompt leaves half of
    // them empty), of 512 rows or more; of one stage or more where that leaves places empty (82
    // rows of 60 heads over 152 tokens: 35 us with 60 workgroups, 26 with 240).
    const int tokens = c->head_dim > 128 ? 4 * kBlock : 8 * kBlock;  // of a workgroup
    const int64_t wgs = (len + tokens - 1) / tokens * c->heads * s->seqs;
    int64_t runs = std::min((12 * cus + wgs - 1) / wgs, (rows + 511) / 512);
    if (runs * wgs < 2 * cus) runs = std::min((2 * cus + wgs - 1) / wgs, (rows + 127) / 128);
    p.run_rows = (int)((rows + runs - 1) / runs + 127) / 128 * 128;  // whole stages
    p.runs = (int)((rows + p.run_rows - 1) / p.run_rows);
    p.score_tokens = w_tokens;
    if (p.runs > 1)
      p.total += align256((size_t)p.runs * s->seqs * c->heads * p.score_tokens * 4);
  }
  return p;
}

int check_attention(const fb_cache_t* c, const fb_seqs_t* s, int32_t q_heads, Cache& k) {
  const int st = check_cache(c, s, k);
  if (st != FB_OK) return st;
  if (q_heads < c->heads || q_heads % c->heads || (int64_t)s->tokens * q_heads > INT32_MAX ||
      (int64_t)s->max_new * (q_heads / c->heads) > INT32_MAX / 2)
    return FB_ERR_SHAPE;
  return FB_OK;
}

template <int DT, int DP, bool EX>
int launch(const Attn& a, const Plan& p, const fb_seqs_t* s, Weights w, hipStream_t hs) {
  const int64_t rows = (int64_t)std::max(1, std::min(s->max_new, s->tokens)) * a.group;
  if (p.few) {
    hipLaunchKernelGGL((attn_few_kernel<DT, DP, EX>), dim3(p.splits, a.c.H, p.dealt ? 1 : a.c.B),
                       dim3(64 * kFewWaves), 0, hs, a);
  } else {
    const int64_t nx = (int64_t)a.c.H * (p.dealt ? 1 : a.c.B) * p.splits;
    if (!fits_grid(nx, 256) || (w.to && !fits_grid((int64_t)a.c.H * a.c.B, 256))) return FB_ERR_SHAPE;
    const int64_t ny = p.dealt ? 1 : std::min<int64_t>((rows + kRows - 1) / kRows, 65535);
    hipLaunchKernelGGL((attn_many_kernel<DT, DP, EX>), dim3((unsigned)nx, (unsigned)ny), dim3(256),
                       0, hs, a);
  }
  if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  const int64_t cap = std::min<int64_t>((int64_t)a.c.max_pages * a.c.P, w.tokens);
  const int64_t len = std::max<int64_t>(1, std::min<int64_t>(cap, s->max_len));
  const int64_t per = 256 / (a.c.D / 4) / p.ways;  // rows of a joining workgroup
  const int joins = p.part ? (int)std::min<int64_t>((rows + per - 1) / per, 1 << 20) : 0;
  const int adds = a.scores ? (int)((len + 1023) / 1024) : 0;
  if (joins + adds) {
    hipLaunchKernelGGL(attn_finish_kernel<DT>, dim3(joins + adds, a.c.H, a.c.B), dim3(256), 0,
                       hs, a, w, joins, p.ways);
    if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  }
  if (w.to && !a.scores) {
    const int tokens = 4 * weight_blocks<DP>() * kBlock;
    const unsigned ny = (unsigned)std::min<int64_t>((len + tokens - 1) / tokens, 65535);
    hipLaunchKernelGGL((attn_weights_kernel<DT, DP>), dim3(a.c.H * a.c.B, ny, p.runs), dim3(256), 0,
                       hs, a, w);
    if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
    if (w.part) {
      hipLaunchKernelGGL(attn_weights_join_kernel, dim3((unsigned)((len + 255) / 256), a.c.H, a.c.B),
                         dim3(256), 0, hs, a.c, w);
      if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
    }
  }
  return FB_OK;
}

}  // namespace

extern "C" {

size_t fb_cache_attention_workspace_bytes(const fb_cache_t* c, const fb_seqs_t* s,
                                          int32_t q_heads, int32_t w_tokens) {
  Cache k;
  if (check_attention(c, s, q_heads, k) != FB_OK) return 0;
  return plan(c, s, q_heads, w_tokens).total;
}

int fb_cache_attention(const fb_cache_t* c, const fb_seqs_t* s, const void* q, int64_t q_token,
                       int64_t q_head, int32_t q_heads, int32_t dtype, float scale, void* out,
                       float* lse, float* weights, int64_t w_seq, int64_t w_head,
                       int32_t w_tokens, void* ws, size_t ws_bytes, void* stream) {
  Attn a{};
  const int st = check_attention(c, s, q_heads, a.c);
  if (st != FB_OK) return st;
  if (dtype != FB_DT_F16 && dtype != FB_DT_BF16) return FB_ERR_DTYPE;
  if (!(scale > 0.f) || !(scale < 1e30f)) return FB_ERR_VALUE;
  if (s->tokens == 0) return FB_OK;
  if (!q || !out || (weights && !lse)) return FB_ERR_NULL;
  if (weights && w_tokens < 1) return FB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(q) & 1u) || (reinterpret_cast<uintptr_t>(out) & 15u) ||
      (reinterpret_cast<uintptr_t>(lse) & 3u) || (reinterpret_cast<uintptr_t>(weights) & 3u) ||
      (reinterpret_cast<uintptr_t>(ws) & 255u))
    return FB_ERR_ALIGN;
  const Plan p = plan(c, s, q_heads, weights ? w_tokens : 0);
  // the rows of q go to LDS 16 bytes at a time there
  if (weights && !p.few &&
      ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(q_token * 2) | (uintptr_t)(q_head * 2)) & 15u))
    return FB_ERR_ALIGN;
  if (p.total && !ws) return FB_ERR_NULL;
  if (p.total > ws_bytes) return FB_ERR_WORKSPACE;
  a.q = q;
  a.q_token = q_token;
  a.q_head = q_head;
  a.q_vec = !((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(q_token * 2) | (uintptr_t)(q_head * 2)) &
              15u);
  a.Hq = q_heads;
  a.group = q_heads / c->heads;
  while ((1u << a.div_shift) < (unsigned)a.group) ++a.div_shift;
  a.div_mul = (unsigned)((((uint64_t)1 << 32) * (((uint64_t)1 << a.div_shift) - a.group)) / a.group) + 1;
  a.scale2 = scale * kLog2e;
  a.out = out;
  a.lse = lse;
  a.splits = p.splits;
  a.split_tokens = p.split_tokens;
  a.dealt = p.dealt;
  a.chunk = p.chunk;
  a.grain = p.grain;
  a.most = p.most;
  a.tiles = p.tiles;
  a.part = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + p.part);
  const int per = c->page / kBlock;
  a.per_shift = per & (per - 1) ? -1 : __builtin_ctz(per);
  float* const rest = reinterpret_cast<float*>(static_cast<char*>(ws) + p.part + p.ml);
  Weights w{weights, w_seq, w_head, w_tokens, nullptr, 0, p.runs, p.run_rows};
  if (p.score_rows) {
    a.scores = rest;
    a.score_rows = p.score_rows;
    a.score_tokens = p.score_tokens;
  } else if (p.runs > 1) {
    w.part = rest;
    w.part_tokens = p.score_tokens;
  }
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    switch (c->head_dim) {
      case 64:
        return launch<DT, 64, true>(a, p, s, w, hs);
      case 128:
        return launch<DT, 128, true>(a, p, s, w, hs);
      case 256:
        return launch<DT, 256, true>(a, p, s, w, hs);
      default:
        return c->head_dim < 64    ? launch<DT, 64, false>(a, p, s, w, hs)
               : c->head_dim < 128 ? launch<DT, 128, false>(a, p, s, w, hs)
                                   : launch<DT, 256, false>(a, p, s, w, hs);
    }
  };
  return dtype == FB_DT_F16 ? go(std::integral_constant<int, FB_DT_F16>{})
                            : go(std::integral_constant<int, FB_DT_BF16>{});
}

}  // extern "C"
