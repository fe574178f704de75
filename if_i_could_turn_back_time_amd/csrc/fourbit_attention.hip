// Attention over the 8-bit key/value cache (layout: fourbit.h).
//
// Both kernels compute S^T = K Q^T and O^T = V^T P^T on the matrix cores, so that a lane's scores
// belong to one query row (a column of S^T) and the C layout of S^T is, with the cached tokens
// dealt to the rows of K's operand in the right order, the B layout that P^T needs: no score ever
// crosses lanes, except for the row maximum.  E4M3 codes are exact in fp16 and bf16, so products
// of q and a code are exact in fp32; a block's scale joins after the sum, in fp32.  P enters as
// fp16 (11 bits, relative to the row's largest score), times the block's scale of V relative to
// the largest seen so far, which is a power of two.
//
// A sequence's rows are its (new token, query head of the group) pairs, token-major: with shared
// heads a tile of rows reads a cached head once for the whole group.
#include "fourbit_cache.h"

#include <algorithm>

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
  float* part;        // [splits][T * Hq][D]
  float2* part_ml;    // [splits][T * Hq]: largest score (base 2), sum
};

__device__ inline float exp2f_(float x) { return __builtin_amdgcn_exp2f(x); }

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
  // 8 E4M3 codes, exactly
  static __device__ x8 decode(unsigned lo, unsigned hi) {
    x8 r;
    const h16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false);
    const h16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
    const h16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false);
    const h16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
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

// ---------------------------------------------------------------------------------
// Few rows (at most 16 a cached head and sequence: decoding).  Bound by reading the cache once,
// so nothing is staged: each wave takes 128 tokens at a time and reads keys and values straight
// into operands of 16x16x32 products.  Workgroup = (split of the tokens, head, sequence), its 4
// waves take chunks in turn and join their sums through LDS.
//  - K operand row r of product j: token 32 (r / 4) + 4 j + r % 4, channels 64 p + 16 q + 8 u.. of
//    lane group q: then a lane's scores are the tokens of block q, 4 j + i.
//  - V operand: channel 16 d + r, tokens 8 s.. of block q, which lie side by side.
// ---------------------------------------------------------------------------------
constexpr int kChunk = 128;

template <int DT, int DP>
__global__ __launch_bounds__(256) void attn_few_kernel(Attn a) {
  using H = Half<DT>;
  constexpr int NP = DP / 64, ND = DP / 16;
  constexpr int PASS = DP < 128 ? DP : 128;  // channels joined at a time
  __shared__ float join[4][16][PASS + 4];
  __shared__ float wave_m[4][16], wave_l[4][16];
  __shared__ int wave_e[4];
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, q4 = lane >> 4;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  int row0, n;
  c.rows(b, row0, n);
  const int len = min(max(c.lens[b], 0), c.capacity());
  const int rows = n * a.group;
  for (int tile = 0; tile < rows; tile += 16) {
    const int row = tile + r, i = row / a.group;
    const bool there = row < rows;
    const int head = h * a.group + (row - i * a.group);
    const int sees = there ? min(max(len - n + i + 1, 0), len) : 0;
    const int least = min(max(len - n + tile / a.group + 1, 0), len);  // of the tile's rows
    typename H::x8 qf[NP][2];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = 64 * p + 16 * q4 + 8 * u;
        qf[p][u] = load_q<DT>(a, there && d < c.D,
                              (int64_t)(row0 + i) * a.q_token + head * a.q_head + d);
      }
    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.f;
    int E = kMinExp;  // the accumulators' unit is 2^E

    const int first = split * (a.split_tokens / kChunk);
    const int last = split + 1 == a.splits ? (len + kChunk - 1) / kChunk
                                           : min((len + kChunk - 1) / kChunk,
                                                 first + a.split_tokens / kChunk);
    for (int ch = first + wave; ch < last; ch += 4) {
      // keys: lane's rows are 4 j + r % 4 of block r / 4; values: block q4
      int at_k, at_v;
      const int pk = max(c.page_of(b, ch * 4 + (r >> 2), at_k), 0);
      const int pv = max(c.page_of(b, ch * 4 + q4, at_v), 0);
      const int64_t bk = c.block_index(pk, h, at_k), bv = c.block_index(pv, h, at_v);
      const uint8_t* const kp = c.k + bk * kBlock * c.D + (r & 3) * c.D + q4 * 16;
      const uint8_t* const vp = c.v + bv * kBlock * c.D + r * 16;
      u32x4 kf[8][NP], vf[ND][2];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          kf[j][p] = 64 * p + 16 * q4 < c.D
                         ? *reinterpret_cast<const u32x4*>(kp + 4 * j * c.D + 64 * p)
                         : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          vf[d][p] = 16 * d < c.D
                         ? *reinterpret_cast<const u32x4*>(vp + p * c.D * kSide + d * 256)
                         : u32x4{0, 0, 0, 0};
      const float ks = a.scale2 * exp2i(min(max((int)c.ks[bv] - 127, -126), 127));
      const bool held = ch * kChunk + q4 * kBlock < len;
      const int ev = held ? min(max((int)c.vs[bv] - 127, -126), 126) : kMinExp;

      f32x4 s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          s[j] = H::mfma16(H::decode(kf[j][p][0], kf[j][p][1]), qf[p][0], s[j]);
          s[j] = H::mfma16(H::decode(kf[j][p][2], kf[j][p][3]), qf[p][1], s[j]);
        }
      }
      const int t0 = ch * kChunk + q4 * kBlock;  // the lane's tokens: t0 + 4 j + i
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] *= ks;
      f32x4 bad[ND];
      bool any_bad = false;
      if (ch * kChunk + kChunk > least) {
        unsigned nan = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (t0 + 4 * j + k >= sees) s[j][k] = -__builtin_inff();
        // what lies behind the end may be anything: no NaN from there
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              vf[d][p][w] &= keep_bytes(t0 + 16 * p + 4 * w, len);
              nan |= nan_bytes(vf[d][p][w]);
            }
        any_bad = __any(nan != 0);
        if (any_bad) {
          // a NaN value reaches the rows that see its token, and no others: 0 * NaN must not
          // come up, so those channels are marked apart
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            bad[d] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              h16x8 see;
#pragma unroll
              for (int k = 0; k < 8; ++k) see[k] = t0 + 8 * x + k < sees ? (_Float16)1 : (_Float16)0;
              bad[d] = Half<FB_DT_F16>::mfma16(
                  Half<FB_DT_F16>::decode(nan_ones(vf[d][x / 2][2 * (x & 1)]),
                                          nan_ones(vf[d][x / 2][2 * (x & 1) + 1])),
                  see, bad[d]);
            }
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
              for (int w = 0; w < 4; ++w) vf[d][p][w] &= ~nan_bytes(vf[d][p][w]);
          }
        }
      }
      float mx = m;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = fmaxf(mx, s[j][k]);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      int e = max(ev, __shfl_xor(ev, 16));
      e = max(e, __shfl_xor(e, 32));
      e = max(e, E);
      const float base = mx == -__builtin_inff() ? 0.f : mx;
      const float alpha = exp2f_(m - base);
      const float fold = exp2i(max(ev - e, -64));
      const float unit = alpha * exp2i(max(E - e, -126));
      m = mx;
      E = e;
      float sum = 0.f;
      h16x8 pf[4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p = exp2f_(s[j][k] - base);
          sum += p;
          pf[j / 2][4 * (j & 1) + k] = (_Float16)(p * fold);
        }
      l = l * alpha + sum;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        o[d] *= unit;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          o[d] = Half<FB_DT_F16>::mfma16(
              Half<FB_DT_F16>::decode(vf[d][x / 2][2 * (x & 1)], vf[d][x / 2][2 * (x & 1) + 1]),
              pf[x], o[d]);
        if (any_bad)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (bad[d][k] > 0.f) o[d][k] = __builtin_nanf("");
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the four waves' sums, in wave order
    __syncthreads();
    if (q4 == 0) {
      wave_m[wave][r] = m;
      wave_l[wave][r] = l;
    }
    if (lane == 0) wave_e[wave] = E;
    __syncthreads();
    const int eM = max(max(wave_e[0], wave_e[1]), max(wave_e[2], wave_e[3]));
    const auto largest = [&](int rr) {
      return fmaxf(fmaxf(wave_m[0][rr], wave_m[1][rr]), fmaxf(wave_m[2][rr], wave_m[3][rr]));
    };
    const auto share = [&](int w, int rr, float M) {
      return M == -__builtin_inff() ? 0.f : exp2f_(wave_m[w][rr] - M);
    };
    const float mine = share(wave, r, largest(r)) * exp2i(max(E - eM, -126));
    // of the row that this thread writes
    const int wr = threadIdx.x >> 4, wi = (tile + wr) / a.group;
    const float M = largest(wr);
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += wave_l[w][wr] * share(w, wr, M);
    const bool writes = tile + wr < rows;
    const int64_t orow = (int64_t)(row0 + wi) * a.Hq + h * a.group + (tile + wr - wi * a.group);
    const float out_scale =
        exp2i(min(max(eM, -126), 127)) * (a.splits == 1 ? (L == 0.f ? 0.f : 1.f / L) : 1.f);
#pragma unroll
    for (int pass = 0; pass < DP / PASS; ++pass) {
      if (pass) __syncthreads();
#pragma unroll
      for (int d = 0; d < PASS / 16; ++d)
        *reinterpret_cast<f32x4*>(&join[wave][r][16 * d + 4 * q4]) =
            o[pass * (PASS / 16) + d] * mine;
      __syncthreads();
      constexpr int E8 = PASS / 16;  // channels of a thread
#pragma unroll
      for (int x = 0; x < E8; x += 4) {
        const int dd = (threadIdx.x & 15) * E8 + x, d = pass * PASS + dd;
        f32x4 v = *reinterpret_cast<const f32x4*>(&join[0][wr][dd]);
#pragma unroll
        for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(&join[w][wr][dd]);
        v *= out_scale;
        if (!writes || d >= c.D) continue;
        if (a.splits > 1) {
          *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * c.T * a.Hq + orow) * c.D + d) = v;
        } else {
          const u32x2 w{(unsigned)H::round(v[0]) | (unsigned)H::round(v[1]) << 16,
                        (unsigned)H::round(v[2]) | (unsigned)H::round(v[3]) << 16};
          *reinterpret_cast<u32x2*>(static_cast<unsigned short*>(a.out) + orow * c.D + d) = w;
        }
      }
    }
    if (writes && (threadIdx.x & 15) == 0) {
      if (a.splits > 1)
        a.part_ml[(int64_t)split * c.T * a.Hq + orow] = float2{M, L};
      else if (a.lse)
        a.lse[orow] = L == 0.f ? -__builtin_inff() : (M + __builtin_log2f(L)) * kLn2;
    }
  }
}

// ---------------------------------------------------------------------------------
// Many rows (prompts).  Workgroup = (128 rows, head, sequence, split): wave w holds rows 32 w.. as
// the columns of 32x32x16 products; 64 tokens at a time go through LDS as codes and are decoded by
// each wave.
//  - K operand row 8 a + 4 x + y: token 16 x + 4 a + y of the block, in this order in LDS.
//  - a lane's scores are then tokens 16 (lane / 32) + i of the block, i < 16; V operand: channel
//    32 d + lane % 32, tokens 16 (lane / 32) + 8 s..: one 16-byte side of the cache.
// ---------------------------------------------------------------------------------
constexpr int kRows = 128, kTile = 64;

template <int DT, int DP>
__global__ __launch_bounds__(256, 2) void attn_many_kernel(Attn a) {
  using H = Half<DT>;
  constexpr int NP = DP / 32, ND = DP / 32, KROW = DP + 16;
  constexpr int LK = kTile * DP / 16 / 256;  // 16-byte pieces a thread loads of each
  __shared__ __align__(16) uint8_t lk[kTile * KROW], lv[kTile * DP];
  __shared__ int lscale[2][2];
  const Cache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = lane & 31, x2 = lane >> 5;
  const int h = blockIdx.y, b = blockIdx.z / a.splits, split = blockIdx.z - b * a.splits;
  int row0, n;
  c.rows(b, row0, n);
  const int len = min(max(c.lens[b], 0), c.capacity());
  const int rows = n * a.group;
  const int tiles = (rows + kRows - 1) / kRows;
  for (int ti = blockIdx.x; ti < tiles; ti += gridDim.x) {
    const int tile = (tiles - 1 - ti) * kRows;  // the longest first
    const int row = tile + wave * 32 + r, i = row / a.group;
    const bool there = row < rows;
    const int head = h * a.group + (row - i * a.group);
    const int sees = there ? min(max(len - n + i + 1, 0), len) : 0;
    // least and most that the wave's and the workgroup's rows see
    const int i_lo = (tile + wave * 32) / a.group;
    const int least = min(max(len - n + i_lo + 1, 0), len);
    const int i_hi = (min(tile + wave * 32 + 32, rows) - 1) / a.group;
    const int wave_most =
        tile + wave * 32 < rows ? min(max(len - n + i_hi + 1, 0), len) : 0;
    const int j_hi = (min(tile + kRows, rows) - 1) / a.group;
    const int most = min(max(len - n + j_hi + 1, 0), len);
    typename H::x8 qf[NP][2];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = 32 * p + 16 * x2 + 8 * u;
        qf[p][u] = load_q<DT>(a, there && d < c.D,
                              (int64_t)(row0 + i) * a.q_token + head * a.q_head + d);
      }
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int k = 0; k < 16; ++k) o[d][k] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    int E = kMinExp;

    const int first = split * (a.split_tokens / kTile);
    const int all = (most + kTile - 1) / kTile;
    const int last = split + 1 == a.splits ? all : min(all, first + a.split_tokens / kTile);
    u32x4 gk[LK], gv[LK];
    int gs = 0;
    const auto fetch = [&](int t) {
#pragma unroll
      for (int x = 0; x < LK; ++x) {
        gk[x] = gv[x] = u32x4{0, 0, 0, 0};
        const int e = tid + 256 * x;
        {
          const int tok = e / (DP / 16), pc = e % (DP / 16);
          int at;
          const int page = max(c.page_of(b, t * 2 + tok / kBlock, at), 0);
          if (t * kTile + tok < len && pc * 16 < c.D)
            gk[x] = *reinterpret_cast<const u32x4*>(
                c.k + (c.block_index(page, h, at) * kBlock + tok % kBlock) * c.D + pc * 16);
        }
        {
          const int sub = e / DP, d = e % DP;
          int at;
          const int page = max(c.page_of(b, t * 2 + sub / 2, at), 0);
          const int tok = t * kTile + sub * kSide;
          if (tok < len && d < c.D) {
            gv[x] = *reinterpret_cast<const u32x4*>(
                c.v + c.block_index(page, h, at) * kBlock * c.D +
                ((int64_t)(sub & 1) * c.D + d) * kSide);
            if (tok + kSide > len)
#pragma unroll
              for (int w = 0; w < 4; ++w) gv[x][w] &= keep_bytes(tok + 4 * w, len);
          }
        }
      }
      if (tid < 4) {
        int at;
        const int page = max(c.page_of(b, t * 2 + (tid & 1), at), 0);
        const int64_t bi = c.block_index(page, h, at);
        gs = (int)(tid < 2 ? c.ks : c.vs)[bi] - 127;
      }
    };
    if (first < last) fetch(first);
    for (int t = first; t < last; ++t) {
      __syncthreads();
#pragma unroll
      for (int x = 0; x < LK; ++x) {
        const int e = tid + 256 * x;
        const int tok = e / (DP / 16), pc = e % (DP / 16);
        const int w = tok % kBlock;
        const int rho = ((w & 12) << 1) | ((w & 16) >> 2) | (w & 3);
        *reinterpret_cast<u32x4*>(lk + ((tok & kBlock) + rho) * KROW + pc * 16) = gk[x];
        *reinterpret_cast<u32x4*>(lv + e * 16) = gv[x];
      }
      if (tid < 4) lscale[tid >> 1][tid & 1] = gs;
      __syncthreads();
      if (t + 1 < last) fetch(t + 1);
      if (t * kTile >= wave_most) continue;  // the same for the wave; the barriers are above
      f32x16 s[2];
      float mx = m;
      const bool masked = t * kTile + kTile > least;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int k = 0; k < 16; ++k) s[y][k] = 0.f;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const u32x4 w =
              *reinterpret_cast<const u32x4*>(lk + (y * 32 + r) * KROW + p * 32 + x2 * 16);
          s[y] = H::mfma32(H::decode(w[0], w[1]), qf[p][0], s[y]);
          s[y] = H::mfma32(H::decode(w[2], w[3]), qf[p][1], s[y]);
        }
        const float ks = a.scale2 * exp2i(min(max(lscale[0][y], -126), 127));
        const int t0 = t * kTile + y * kBlock + x2 * 16;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          s[y][k] *= ks;
          if (masked && t0 + k >= sees) s[y][k] = -__builtin_inff();
          mx = fmaxf(mx, s[y][k]);
        }
      }
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const int ev0 = min(max(lscale[1][0], -126), 126);
      const int ev1 = t * kTile + kBlock < len ? min(max(lscale[1][1], -126), 126) : kMinExp;
      const int e = max(E, max(ev0, ev1));
      const float base = mx == -__builtin_inff() ? 0.f : mx;
      const float alpha = exp2f_(m - base);
      const float unit = alpha * exp2i(max(E - e, -126));
      m = mx;
      E = e;
      float sum = 0.f;
      h16x8 pf[2][2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float fold = exp2i(max((y ? ev1 : ev0) - e, -64));
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float p = exp2f_(s[y][k] - base);
          sum += p;
          pf[y][k / 8][k & 7] = (_Float16)(p * fold);
        }
      }
      l = l * alpha + sum;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        o[d] *= unit;
        f32x16 bad;
        bool any_bad = false;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          u32x4 w = *reinterpret_cast<const u32x4*>(lv + ((2 * y + x2) * DP + 32 * d + r) * 16);
          if (masked) {
            const unsigned nan = nan_bytes(w[0]) | nan_bytes(w[1]) | nan_bytes(w[2]) |
                                 nan_bytes(w[3]);
            if (__any(nan != 0)) {
              // a NaN value reaches the rows that see its token, and no others
              if (!any_bad)
#pragma unroll
                for (int k = 0; k < 16; ++k) bad[k] = 0.f;
              any_bad = true;
              const int t0 = t * kTile + y * kBlock + x2 * 16;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                h16x8 see;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  see[k] = t0 + 8 * u + k < sees ? (_Float16)1 : (_Float16)0;
                bad = Half<FB_DT_F16>::mfma32(
                    Half<FB_DT_F16>::decode(nan_ones(w[2 * u]), nan_ones(w[2 * u + 1])), see, bad);
              }
#pragma unroll
              for (int u = 0; u < 4; ++u) w[u] &= ~nan_bytes(w[u]);
            }
          }
          o[d] = Half<FB_DT_F16>::mfma32(Half<FB_DT_F16>::decode(w[0], w[1]), pf[y][0], o[d]);
          o[d] = Half<FB_DT_F16>::mfma32(Half<FB_DT_F16>::decode(w[2], w[3]), pf[y][1], o[d]);
        }
        if (any_bad)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (bad[k] > 0.f) o[d][k] = __builtin_nanf("");
      }
    }
    l += __shfl_xor(l, 32);
    if (there) {
      const int64_t orow = (int64_t)(row0 + i) * a.Hq + head;
      const float unit = exp2i(min(max(E, -126), 127)) *
                         (a.splits == 1 ? (l == 0.f ? 0.f : 1.f / l) : 1.f);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
          const int ch = 32 * d + 2 * k + 4 * x2;
          if (ch >= c.D) continue;
          const f32x4 v = f32x4{o[d][k], o[d][k + 1], o[d][k + 2], o[d][k + 3]} * unit;
          if (a.splits > 1) {
            *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * c.T * a.Hq + orow) * c.D + ch) = v;
          } else {
            const u32x2 w{(unsigned)H::round(v[0]) | (unsigned)H::round(v[1]) << 16,
                          (unsigned)H::round(v[2]) | (unsigned)H::round(v[3]) << 16};
            *reinterpret_cast<u32x2*>(static_cast<unsigned short*>(a.out) + orow * c.D + ch) = w;
          }
        }
      if (x2 == 0) {
        if (a.splits > 1)
          a.part_ml[(int64_t)split * c.T * a.Hq + orow] = float2{m, l};
        else if (a.lse)
          a.lse[orow] = l == 0.f ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
      }
    }
  }
}

// The splits' sums of a row, in order.  One wave a row.
template <int DT>
__global__ __launch_bounds__(256) void attn_join_kernel(Attn a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t rows = (int64_t)a.c.T * a.Hq;
  if (row >= rows) return;
  float M = -__builtin_inff(), L = 0.f;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.part_ml[s * rows + row].x);
  const int d = lane * 4;
  f32x4 v{0, 0, 0, 0};
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = a.part_ml[s * rows + row];
    if (ml.y == 0.f) continue;
    const float f = exp2f_(ml.x - M);
    L += ml.y * f;
    if (d < a.c.D) v += *reinterpret_cast<const f32x4*>(a.part + (s * rows + row) * a.c.D + d) * f;
  }
  v *= L == 0.f ? 0.f : 1.f / L;
  if (d < a.c.D) {
    using H = Half<DT>;
    const u32x2 w{(unsigned)H::round(v[0]) | (unsigned)H::round(v[1]) << 16,
                  (unsigned)H::round(v[2]) | (unsigned)H::round(v[3]) << 16};
    *reinterpret_cast<u32x2*>(static_cast<unsigned short*>(a.out) + row * a.c.D + d) = w;
  }
  if (lane == 0 && a.lse)
    a.lse[row] = L == 0.f ? -__builtin_inff() : (M + __builtin_log2f(L)) * kLn2;
}

// ---------------------------------------------------------------------------------
// Accumulated weights: weights[t] += sum over the rows of exp(score - lse).  Workgroup = (128
// tokens, head, sequence), each wave holds 32 tokens' keys as operands and walks over the rows
// that see them, so that every sum belongs to one wave and is added in row order.
// ---------------------------------------------------------------------------------
template <int DT, int DP>
__global__ __launch_bounds__(256) void attn_weights_kernel(Attn a, float* weights, int64_t w_seq,
                                                           int64_t w_head, int w_tokens) {
  using H = Half<DT>;
  constexpr int NP = DP / 32;
  const Cache& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, x2 = lane >> 5;
  const int h = blockIdx.y, b = blockIdx.z;
  int row0, n;
  c.rows(b, row0, n);
  const int len = min(max(c.lens[b], 0), c.capacity());
  const int rows = n * a.group;
  const int end = min(len, w_tokens);
  for (int blk = blockIdx.x * 4 + wave; blk * kBlock < end; blk += gridDim.x * 4) {
    int at;
    const int page = max(c.page_of(b, blk, at), 0);
    const int64_t bi = c.block_index(page, h, at);
    u32x4 kf[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p)
      kf[p] = 32 * p + 16 * x2 < c.D ? *reinterpret_cast<const u32x4*>(
                                           c.k + (bi * kBlock + r) * c.D + 32 * p + 16 * x2)
                                     : u32x4{0, 0, 0, 0};
    const float ks = a.scale2 * exp2i(min(max((int)c.ks[bi] - 127, -126), 127));
    f32x16 sum;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum[k] = 0.f;
    // the first row that sees the block's first token
    const int from = max(blk * kBlock - (len - n), 0) * a.group / 32 * 32;
    for (int tile = from; tile < rows; tile += 32) {
      const int row = tile + r, i = row / a.group;
      const bool there = row < rows;
      const int head = h * a.group + (row - i * a.group);
      const int sees = there ? min(max(len - n + i + 1, 0), len) : 0;
      const float lse = there ? a.lse[(int64_t)(row0 + i) * a.Hq + head] * kLog2e : 0.f;
      f32x16 s;
#pragma unroll
      for (int k = 0; k < 16; ++k) s[k] = 0.f;
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int d = 32 * p + 16 * x2 + 8 * u;
          const auto qf = load_q<DT>(a, there && d < c.D,
                                     (int64_t)(row0 + i) * a.q_token + head * a.q_head + d);
          s = H::mfma32(H::decode(kf[p][2 * u], kf[p][2 * u + 1]), qf, s);
        }
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int t = blk * kBlock + 8 * (k / 4) + 4 * x2 + k % 4;
        if (t < sees) sum[k] += exp2f_(s[k] * ks - lse);
      }
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float v = sum[k];
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor(v, o);
      const int t = blk * kBlock + 8 * (k / 4) + 4 * x2 + k % 4;
      if (r == k && t < end) weights[b * w_seq + h * w_head + t] += v;
    }
  }
}

// ------------------------------------------------------------------ host side
struct Plan {
  bool few;
  int splits, split_tokens;
  size_t part, total;
};

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// How a call is split.  It goes by host numbers alone, so that a captured call fits any lengths.
Plan plan(const fb_cache_t* c, const fb_seqs_t* s, int q_heads) {
  Plan p{};
  const int group = q_heads / c->heads;
  const int64_t rows = (int64_t)std::max(1, std::min(s->max_new, s->tokens)) * group;
  p.few = rows <= 16;
  const int64_t capacity = std::min<int64_t>((int64_t)s->max_pages * c->page, 0x7FFFFFE0);
  const int64_t len = std::max<int64_t>(1, std::min<int64_t>(s->max_len, capacity));
  const int64_t tiles = p.few ? 1 : (rows + kRows - 1) / kRows;
  const int64_t units = tiles * c->heads * s->seqs;
  const int step = p.few ? 4 * kChunk : 4 * kTile;
  const int64_t most = (len + step - 1) / step;
  const int64_t want = std::max<int64_t>(1, 4 * (int64_t)fb_gpu::cu_count() / units);
  const int64_t per = (most + std::min(want, most) - 1) / std::min(want, most);
  p.split_tokens = (int)(per * step);
  p.splits = (int)((most + per - 1) / per);
  const size_t n = (size_t)s->tokens * q_heads;
  if (p.splits > 1) {
    p.part = align256((size_t)p.splits * n * c->head_dim * 4);
    p.total = p.part + align256((size_t)p.splits * n * 8);
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

template <int DT, int DP>
int launch(const Attn& a, const Plan& p, const fb_seqs_t* s, float* weights, int64_t w_seq,
           int64_t w_head, int w_tokens, hipStream_t hs) {
  const int64_t rows = (int64_t)std::min(s->max_new, s->tokens) * a.group;
  if (p.few) {
    hipLaunchKernelGGL((attn_few_kernel<DT, DP>), dim3(p.splits, a.c.H, a.c.B), dim3(256), 0, hs, a);
  } else {
    if ((int64_t)p.splits * a.c.B > 65535) return FB_ERR_SHAPE;
    hipLaunchKernelGGL((attn_many_kernel<DT, DP>),
                       dim3((unsigned)((rows + kRows - 1) / kRows), a.c.H, a.c.B * p.splits),
                       dim3(256), 0, hs, a);
  }
  if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  if (p.splits > 1) {
    const int64_t n = (int64_t)a.c.T * a.Hq;
    hipLaunchKernelGGL(attn_join_kernel<DT>, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, hs, a);
    if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  }
  if (weights) {
    const int64_t cap = std::min<int64_t>((int64_t)a.c.max_pages * a.c.P, w_tokens);
    const int64_t len = std::max<int64_t>(1, std::min<int64_t>(cap, s->max_len));
    const int64_t nx = std::min<int64_t>((len + 127) / 128, 1 << 20);
    hipLaunchKernelGGL((attn_weights_kernel<DT, DP>), dim3((unsigned)nx, a.c.H, a.c.B), dim3(256), 0,
                       hs, a, weights, w_seq, w_head, w_tokens);
    if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  }
  return FB_OK;
}

}  // namespace

extern "C" {

size_t fb_cache_attention_workspace_bytes(const fb_cache_t* c, const fb_seqs_t* s,
                                          int32_t q_heads) {
  Cache k;
  if (check_attention(c, s, q_heads, k) != FB_OK) return 0;
  return plan(c, s, q_heads).total;
}

int fb_cache_attention(const fb_cache_t* c, const fb_seqs_t* s, const void* q, int64_t q_token,
                       int64_t q_head, int32_t q_heads, int32_t dtype, float scale, void* out,
                       float* lse, float* weights, int64_t w_seq, int64_t w_head,
                       int32_t w_tokens, void* ws, size_t ws_bytes, void* stream) {
  Attn a{};
  const int st = check_attention(c, s, q_heads, a.c);
  if (st != FB_OK) return st;
  if (dtype != FB_DT_F16 && dtype != FB_DT_BF16) return FB_ERR_DTYPE;
  if (s->tokens == 0 || s->max_new == 0) return FB_OK;
  if (!q || !out || (weights && !lse)) return FB_ERR_NULL;
  if (weights && w_tokens < 1) return FB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(q) & 1u) || (reinterpret_cast<uintptr_t>(out) & 15u) ||
      (reinterpret_cast<uintptr_t>(lse) & 3u) || (reinterpret_cast<uintptr_t>(weights) & 3u) ||
      (reinterpret_cast<uintptr_t>(ws) & 255u))
    return FB_ERR_ALIGN;
  const Plan p = plan(c, s, q_heads);
  if (p.total && !ws) return FB_ERR_NULL;
  if (p.total > ws_bytes) return FB_ERR_WORKSPACE;
  a.q = q;
  a.q_token = q_token;
  a.q_head = q_head;
  a.q_vec = !((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(q_token * 2) | (uintptr_t)(q_head * 2)) &
              15u);
  a.Hq = q_heads;
  a.group = q_heads / c->heads;
  a.scale2 = scale * kLog2e;
  a.out = out;
  a.lse = lse;
  a.splits = p.splits;
  a.split_tokens = p.split_tokens;
  a.part = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + p.part);
  const int dp = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel) {
    return kernel(a, p, s, weights, w_seq, w_head, w_tokens, hs);
  };
  if (dtype == FB_DT_F16)
    return dp == 64    ? go(launch<FB_DT_F16, 64>)
           : dp == 128 ? go(launch<FB_DT_F16, 128>)
                       : go(launch<FB_DT_F16, 256>);
  return dp == 64    ? go(launch<FB_DT_BF16, 64>)
         : dp == 128 ? go(launch<FB_DT_BF16, 128>)
                     : go(launch<FB_DT_BF16, 256>);
}

}  // extern "C"
