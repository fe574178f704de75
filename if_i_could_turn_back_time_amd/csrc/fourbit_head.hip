// Log probabilities of given tokens, and entropies, under a head of 16-bit weights, whose logits are
// never kept; and the gradients of the hidden states and of the weights.
//
//   l = x W^T,  logprob = l[token] - log sum exp l,  entropy = -sum p log p
//   G[r, v] = g_r [v = token_r] - p (g_r + h_r (log p + entropy_r)),  grad_x = G W,  grad_w = G^T x
//
// Four products on the matrix cores, all by product_kernel:
//   kStats    a tile of logits is reduced where it was summed, to (largest, sum of exponentials, sum of
//             exponentials times distance) for each of its rows; head_join makes a row's results of them.
//   kGradient the same logits again, bit for bit (a logit's products are added in the same order
//             whatever the tile), turned into G, rounded to the weights' type, for a piece of the
//             vocabulary: 1 GiB of G at most, or 256 tokens where rows are more than 2^21.
//   kProduct  grad_x: G times W over the vocabulary, pieces and parts of which are added in fp32;
//             grad_w: G^T times x over the rows.
// G in 16 bits costs each of its values half a step; products and all sums are fp32.  Of a log
// probability's gradient one value of a row stands out, the given token's, wherever no other token is
// likely: what it lost is kept in fp32 and goes into both results, times its row of W (head_sum) or of x
// (grad_w's tiles end with the rows whose token they hold, which a sort by token finds).  The others'
// roundings stay: those of an entropy's gradient, and of likely tokens that were not given.  They add up as
// their terms do, so that their part of a result is at most as large as the result's own rounding, and the
// error at most 1.4 times that (8000 x 1024, bf16, 256 rows: 1.67e-3 of the gradients' norms for log
// probabilities where logits are of a few units, 2.0e-3 where they are of 20, 2.37e-3 for entropies,
// rounding alone 1.66e-3; fp16 2.10e-4, 2.5e-4, 3.04e-4 and 2.08e-4).  G in two parts would take it
// off, for 4 M V K operations more beside these 8.  In fp16 each row of G has
// a power of two of its own that brings it near the type's largest values, and grad_w's x one that takes
// it off again, times a common one that brings the largest of them near the type's largest values too: a
// row's x keeps its bits as far as 2^-30 of the largest row's g x, which is the distance between the least
// and the largest values that the result may have in fp16.
// The logits are worked out twice rather than kept: 2 of the 8 M V K operations, for M V values that are
// never in memory beyond a piece.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fourbit.h"
#include "fourbit_decode.h"
#include "fourbit_layout.h"
#include "fourbit_tokens.h"

namespace fb_gpu {
__attribute__((visibility("hidden"))) int cu_count();
}  // namespace fb_gpu

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // rows of odd widths begin anywhere

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLow = -200.f;  // exp of it is 0, and its product with a sum stays finite
constexpr int kChunk = 64;      // contraction values staged at a time

enum Mode { kStats, kGradient, kProduct };

struct ProductArgs {
  const uint8_t* p;  // the side whose index is contiguous in the result
  const uint8_t* q;
  int64_t ldp, ldq;  // elements
  int np, nq, k;
  int tiles_p, tiles_q;
  int chunks;        // of a part
  // kStats
  float *pm, *pz, *pw;  // [tiles_p, nq]
  float* given;         // [nq]: the given token's logit
  const int64_t* token;
  int v0;  // p's first row is this token
  // kGradient
  const float* stats;  // [nq, 2] as head_join writes them, or (three) [nq, 3] as fb_token_logprobs does
  int three;
  const float *entropy, *g_logprob, *g_entropy, *scale;
  uint16_t* g;
  int64_t ldg;
  int vocab;
  float* lost;  // [nq]: what the given token's value lost in rounding
  // kProduct
  void* out;   // [nq, np] of 16 bits, or null
  float* acc;  // [parts, nq, np] otherwise
  int add;     // to what acc holds
  const float* out_scale;  // null, or of one value
  // and for QT: the rows by token (key, place), from which of them on each 128 tokens' lie, and what to
  // add of each
  const unsigned *key, *place, *start;
  int starts;
};

// By what the 32-byte units of contraction row k are permuted (TR, below): the rows that 32 lanes read
// at a time, 0 to 3 and 8 to 11 of 16 or 4 to 7 and 12 to 15, get all of 0 to 7.
__device__ inline int row_mask(int k) { return (k & 3) | ((((k >> 3) ^ (k >> 4)) & 1) << 2); }

// One operand's tile of T values by kChunk of the contraction in LDS, T / 8 requests of 1 KiB.
// Rows of the contraction side by side (TR = false): [T][64], a row's eight 16-byte units permuted by
// its number, so that the 16 lanes that LDS serves at a time read 16 different ones.
// The contraction along memory's rows (TR): [64][T], 32 bytes of 16 values permuted by the row, read
// by the transposing LDS reads: 16 lanes read 4 rows of 16 values and get a column of 4 each.
template <bool TR, int T, int WAVES>
struct Side {
  static constexpr int kRequests = (T / 8 + WAVES - 1) / WAVES;
  static constexpr bool kEven = T / 8 % WAVES == 0;
  unsigned off[kRequests];  // of this lane's request j
  int ku;                   // TR = false: the lane's first contraction value (of even requests)
  unsigned rd;              // where this lane reads
  __device__ void init(int wave, int lane, int64_t ld) {
    ku = 0;
#pragma unroll
    for (int j = 0; j < kRequests; ++j) {
      const int i = wave * kRequests + j;
      if constexpr (TR) {
        constexpr int PER = T / 8;  // lanes of a row
        const int k = i * (64 / PER) + lane / PER;
        const int w = ((lane % PER) >> 1) ^ row_mask(k);
        off[j] = (unsigned)(k * ld + w * 16 + (lane & 1) * 8) * 2u;
      } else {
        const int row = i * 8 + (lane >> 3);
        const int u = (lane & 7) ^ ((row >> 1) & 7);
        off[j] = (unsigned)(row * ld + u * 8) * 2u;
        if (j == 0) ku = u * 8;
      }
    }
    const int r = lane & 15, g = lane >> 4;
    if constexpr (TR) {
      const int k = 8 * g + (r >> 2);
      rd = k * (2 * T) + row_mask(k) * 32 + (r & 3) * 8;
    } else {
      rd = r * 128 + ((g ^ ((r >> 1) & 7)) << 4);
    }
  }
  // Requests chunk c of the tile at t0.
  __device__ void stage(const uint8_t* base, int64_t ld, int n, int k, int t0, int c, int wave,
                        uint8_t* buf) const {
    const int rows = min(T, n - t0), left = k - c * kChunk;
    rsrc_t rs;  // up to the last whole unit of 8 values
    if constexpr (TR)
      rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(base) + ((int64_t)c * kChunk * ld + t0) * 2, (short)0,
          (int)(((min(left, kChunk) - 1) * ld + ((rows + 7) & ~7)) * 2), kRsrcWord3);
    else
      rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base) + (int64_t)t0 * ld * 2,
                                             (short)0, (int)(((rows - 1) * ld + ((k + 7) & ~7)) * 2),
                                             kRsrcWord3);
#pragma unroll
    for (int j = 0; j < kRequests; ++j) {
      const int i = wave * kRequests + j;
      if (!kEven && i >= T / 8) break;
      unsigned o = off[j];
      if constexpr (!TR) {
        // requests of a wave differ by 8 rows, which changes the unit by 4
        const int kv = j & 1 ? ku ^ 32 : ku;
        o = kv < left ? o + (unsigned)c * (kChunk * 2) : kXOutOfRange;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_byte*)(buf + i * 1024), 16, o, 0, 0, 0);
    }
  }
  // The matrix operand of 16 values (tile i) and contraction values 32 s .. 32 s + 31.
  __device__ u32x4 read(const uint8_t* buf, int i, int s) const {
    if constexpr (TR) {
      typedef __attribute__((address_space(3))) s16x4* lds4;
      const uint8_t* at = buf + (rd ^ (i * 32)) + s * 32 * 2 * T;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 4 * 2 * T));
      const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
      return u32x4{a.x, a.y, b.x, b.y};
    } else {
      return *reinterpret_cast<const u32x4*>(buf + (rd ^ (s * 64)) + i * 2048);
    }
  }
};

// Workgroup barrier once this wave has received all that it asked for.  Builtins, because the compiler
// counts them: after waits it cannot see it has every LDS read wait for the requests before it.
__device__ inline void arrive() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int DT>
__device__ inline unsigned pack2(float a, float b) {
  if constexpr (DT == FB_DT_F16)
    return __builtin_bit_cast(unsigned short, (_Float16)a) |
           (unsigned)__builtin_bit_cast(unsigned short, (_Float16)b) << 16;
  else
    return __builtin_bit_cast(unsigned short, (__bf16)a) |
           (unsigned)__builtin_bit_cast(unsigned short, (__bf16)b) << 16;
}

template <int DT>
__device__ inline float rounded(float v) {
  if constexpr (DT == FB_DT_F16) return (float)(_Float16)v;
  else return (float)(__bf16)v;
}

// Sums of exp(l - m) and of exp(l - m) (l - m).
struct Sums {
  float m = -__builtin_inff(), z = 0.f, w = 0.f;
  __device__ void add(float m2, float z2, float w2) {
    if (z2 == 0.f) return;  // of nothing but -inf
    const float to = fmaxf(m, m2), d1 = m - to, d2 = m2 - to;
    const float f1 = z == 0.f ? 0.f : __builtin_amdgcn_exp2f(d1 * kLog2e);
    const float f2 = __builtin_amdgcn_exp2f(d2 * kLog2e);
    w = f1 * __builtin_fmaf(fmaxf(d1, kLow), z, w) + f2 * __builtin_fmaf(fmaxf(d2, kLow), z2, w2);
    z = f1 * z + f2 * z2;
    m = to;
  }
};

// A tile of TP x TQ of p q^T, WP x WQ waves, D chunks staged at a time.  Operands go from memory straight
// to LDS, a chunk ahead, and from there to registers half a chunk ahead of the products.  What bounds
// the large tiles is requests: 4096 x 131072 x 4096 takes 3.3 ms (1.32 PFLOP/s, matrix instructions two
// thirds of the cycles) as kStats, 3.5 as kGradient, 3.1 for grad_x and 3.5 for grad_w, where 128 x 128
// takes 4.0 to 4.4; without its requests the loop runs at 1.7 to 2.2 PFLOP/s.  With D > 1 (few rows: the
// weight's bytes are the work) the tiles begin at chunks of their own and go round: all at the same
// columns of rows of a power of two of bytes, the requests meet in few of the memory's channels (16 x
// 32000 x 4096: 61 us, 49 so with D = 2).
template <int DT, bool PT, bool QT, int TP, int TQ, int WP, int WQ, int D, int MODE>
__global__ __launch_bounds__(WP* WQ * 64, D * TP * TQ == 32768 ? 1 : 2) void product_kernel(ProductArgs a) {
  constexpr int WAVES = WP * WQ;
  constexpr int RP = TP / WP / 16, RQ = TQ / WQ / 16;
  constexpr bool kTurned = D > 1;
  static_assert(!kTurned || (!PT && !QT && MODE != kProduct), "no parts, and rows of the contraction");
  __shared__ __align__(1024) uint8_t p0[TP * 128 * D], p1[TP * 128 * D], q0[TQ * 128 * D],
      q1[TQ * 128 * D];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wp = wave % WP, wq = wave / WP;

  // Workgroups go round-robin over the 8 XCDs: each takes a contiguous run of tiles, 4 of q by many
  // of p at a time, which share operands in its L2.
  int id = blockIdx.x;
  {
    const int n = gridDim.x >> 3, r = gridDim.x & 7, xcd = id & 7, i = id >> 3;
    id = (xcd < r ? xcd * (n + 1) : r * (n + 1) + (xcd - r) * n) + i;
  }
  const int per = a.tiles_p * a.tiles_q, part = id / per;
  id -= part * per;
  const int group = id / (4 * a.tiles_p), gq = min(4, a.tiles_q - group * 4);
  const int in = id - group * 4 * a.tiles_p;
  const int tp = in / gq, tq = group * 4 + in % gq;
  const int tp0 = tp * TP, tq0 = tq * TQ;
  const int c0 = part * a.chunks;
  const int n = (min(a.chunks, (a.k + kChunk - 1) / kChunk - c0) + D - 1) / D;  // stages
  // the same for a token in every call: its logits are the same sums in both passes
  const int turn = kTurned ? (a.v0 + tp0) / 256 % n : 0;

  Side<PT, TP, WAVES> sp;
  Side<QT, TQ, WAVES> sq;
  sp.init(wave, lane, a.ldp);
  sq.init(wave, lane, a.ldq);
  // grad_w: the rows whose given tokens are of this tile, sorted places s0 to s1.  What is needed of
  // the first 64 of them after the products is asked for before them.
  constexpr bool kLost = MODE == kProduct && QT;
  constexpr int kParts = WAVES * 64 / kChunk;  // threads of a row
  __shared__ int place_lds[kLost ? kChunk : 1];
  const int s0 = kLost ? a.start[min((a.v0 + tq0) / 128, a.starts)] : 0;
  const int s1 = kLost ? a.start[min((a.v0 + tq0 + TQ) / 128, a.starts)] : 0;
  int key = 0, place = 0;
  float lost = 0.f;
  const auto request = [&](int c, uint8_t* pb, uint8_t* qb) {
    if (kTurned) {
      c += turn;
      if (c >= n) c -= n;
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      sp.stage(a.p, a.ldp, a.np, a.k, tp0, c0 + c * D + d, wave, pb + d * (TP * 128));
      sq.stage(a.q, a.ldq, a.nq, a.k, tq0, c0 + c * D + d, wave, qb + d * (TQ * 128));
    }
  };
  f32x4 acc[RP][RQ];
#pragma unroll
  for (int i = 0; i < RP; ++i)
#pragma unroll
    for (int j = 0; j < RQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  u32x4 pa[2][RP], qa[2][RQ];
  // Item i of what a half chunk reads: one of p first, then q, then the rest of p.
  const auto read = [&](const uint8_t* pb, const uint8_t* qb, int s, int to, int i) {
    if (i >= 1 && i <= RQ)
      qa[to][i - 1] = sq.read(qb, wq * RQ + i - 1, s);
    else
      pa[to][i ? i - RQ : 0] = sp.read(pb, wp * RP + (i ? i - RQ : 0), s);
  };
  // The products of a half chunk, with the next one's operands read between them.
  const auto half = [&](const uint8_t* pb, const uint8_t* qb, int s, int from) {
    constexpr int G = RP > 2 ? RP - 2 : 1, I = RP + RQ;
#pragma unroll
    for (int i = 0; i < RP; ++i) {
#pragma unroll
      for (int t = i * I / G; t < (i + 1) * I / G && t < I; ++t) read(pb, qb, s, from ^ 1, t);
#pragma unroll
      for (int j = 0; j < RQ; ++j) acc[i][j] = mfma<DT>(pa[from][i], qa[from][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const auto step = [&](int c, uint8_t* pb, uint8_t* qb, const uint8_t* pn, const uint8_t* qn) {
#pragma unroll
    for (int h = 1; h < 2 * D; ++h)
      half(pb + (h >> 1) * (TP * 128), qb + (h >> 1) * (TQ * 128), h & 1, (h & 1) ^ 1);
    // the next stage is there, and no wave reads this one any more
    arrive();
    if (c + 2 < n) request(c + 2, pb, qb);
    half(pn, qn, 0, 1);
  };
  if (n > 0) {
    request(0, p0, q0);
    if (kLost && s1 > s0) {
      const int i = min(s0 + (int)threadIdx.x / kParts, s1 - 1);
      key = a.key[i];
      place = a.place[i];
    }
    arrive();
    if (kLost && s1 > s0) {
      lost = a.lost[place];
      place_lds[threadIdx.x / kParts] = place;
    }
    if (n > 1) request(1, p1, q1);
#pragma unroll
    for (int i = 0; i < RP + RQ; ++i) read(p0, q0, 0, 0, i);
    for (int c = 0; c < n; c += 2) {
      step(c, p0, q0, p1, q1);
      if (c + 1 < n) step(c + 1, p1, q1, p0, q0);
    }
  }

  if constexpr (kLost) {
    // What they lost, as chunks of 64 rows more, with one value of q in each.
    for (int at = s0; at < s1; at += kChunk) {
      const int k = threadIdx.x / kParts;
      if (at != s0) {
        const int i = min(at + k, s1 - 1);
        key = a.key[i];
        place = a.place[i];
        lost = a.lost[place];
      }
      __syncthreads();  // no wave reads a tile, or places, any more
      if (at != s0) {
        place_lds[k] = place;
        __syncthreads();
      }
#pragma unroll
      for (int j = 0; j < sp.kRequests; ++j) {
        constexpr int PER = TP / 8;
        const int i = wave * sp.kRequests + j, r = i * (64 / PER) + lane / PER;
        const int w = ((lane % PER) >> 1) ^ row_mask(r);
        const int64_t col = tp0 + w * 16 + (lane & 1) * 8;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(a.p + (place_lds[r] * a.ldp +
                                                                   (col < a.ldp ? col : 0)) * 2),
            (__attribute__((address_space(3))) void*)(p0 + i * 1024), 16, 0, 0);
      }
      const int v = key - a.v0 - tq0;
      const unsigned value = at + k < s1 ? pack2<DT>(lost, 0.f) << (16 * (v & 1)) : 0u;
#pragma unroll
      for (int e = 0; e < TQ / 8 / kParts; ++e) {
        const int u = threadIdx.x % kParts * (TQ / 8 / kParts) + e;  // 8 values
        const bool here = (u >> 1) == ((v >> 4) ^ row_mask(k)) && (u & 1) == ((v >> 3) & 1);
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = here && ((v >> 1) & 3) == j ? value : 0u;
        *reinterpret_cast<u32x4*>(q0 + k * (TQ * 2) + u * 16) = o;
      }
      arrive();
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < RP + RQ; ++i) read(p0, q0, s, 0, i);
#pragma unroll
        for (int i = 0; i < RP; ++i)
#pragma unroll
          for (int j = 0; j < RQ; ++j) acc[i][j] = mfma<DT>(pa[0][i], qa[0][j], acc[i][j]);
      }
    }
  }

  // lane: q's row lane % 16 of tile j, p's rows 4 (lane / 16) .. + 3 of tile i
  const int pl = tp0 + wp * (TP / WP) + (lane >> 4) * 4;
  const int ql = tq0 + wq * (TQ / WQ) + (lane & 15);

  // 16-bit results go through LDS, a wave's part of the tile each, so that a store writes whole runs of a
  // row: straight from the accumulators (32 bytes of 16 rows each) they took 92 of 486 us of grad_w of
  // 2048 x 32000 x 4096.  The 16-byte units of a row are permuted by its number.
  constexpr int kUnits = RP * 2, kWaveBytes = RP * RQ * 512, kPer = TP * 128 / kWaveBytes;
  static_assert(kPer >= 1 && (kPer * 2 >= WAVES || (TP == TQ && kPer * 4 >= WAVES)), "all waves' parts fit");
  uint8_t* const mine_lds = (wave / kPer == 0   ? p0
                             : wave / kPer == 1 ? p1
                             : wave / kPer == 2 ? q0
                                                : q1) +
                            wave % kPer * kWaveBytes;
  const auto put = [&](int i, int j, unsigned lo, unsigned hi) {
    const int row = j * 16 + (lane & 15), u = i * 2 + (lane >> 5);
    *reinterpret_cast<uint2*>(mine_lds + row * (kUnits * 16) + ((u ^ (row & (kUnits - 1))) << 4) +
                              ((lane >> 4) & 1) * 8) = make_uint2(lo, hi);
  };
  const auto put_one = [&](int i, int j, int e, uint16_t v) {
    const int row = j * 16 + (lane & 15), u = i * 2 + (lane >> 5);
    *reinterpret_cast<uint16_t*>(mine_lds + row * (kUnits * 16) + ((u ^ (row & (kUnits - 1))) << 4) +
                                 ((lane >> 4) & 1) * 8 + e * 2) = v;
  };
  // The wave's part to rows of `out`, ld values apart, of which the first n columns and rows are there.
  const auto write = [&](void* out, int64_t ld, int n, int rows) {
    constexpr int R = 64 / kUnits;  // rows of a store
    asm volatile("" ::: "memory");
#pragma unroll
    for (int k = 0; k < RQ * 16 / R; ++k) {
      const int row = k * R + lane / kUnits, u = lane % kUnits;
      const u32x4 v = *reinterpret_cast<const u32x4*>(mine_lds + row * (kUnits * 16) +
                                                      ((u ^ (row & (kUnits - 1))) << 4));
      const int64_t r = tq0 + wq * (TQ / WQ) + row;
      const int c = tp0 + wp * (TP / WP) + u * 8;
      uint16_t* const to = static_cast<uint16_t*>(out) + r * ld + c;
      if (r < rows && c + 8 <= n) {
        *reinterpret_cast<u32x4_any*>(to) = v;
      } else if (r < rows) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < n) to[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
      }
    }
  };
  if constexpr (MODE != kStats) __syncthreads();  // no wave reads a tile any more
  if constexpr (MODE == kStats) {
    const bool whole = tp0 + TP <= a.np;
    float* const part = reinterpret_cast<float*>(p0);  // [WP, TQ, 3]
    static_assert(WP * TQ * 12 <= TP * 128, "the waves' sums take the place of a tile");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RQ; ++j) {
      const int r = ql + j * 16;
      float m = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < RP; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!whole && pl + i * 16 + e >= a.np) acc[i][j][e] = -__builtin_inff();
          m = fmaxf(m, acc[i][j][e]);
        }
      }
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const float to = m == -__builtin_inff() ? 0.f : m;
      float z = 0.f, w = 0.f;
#pragma unroll
      for (int i = 0; i < RP; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = acc[i][j][e] - to, x = __builtin_amdgcn_exp2f(d * kLog2e);
          z += x;
          w = __builtin_fmaf(x, fmaxf(d, kLow), w);
        }
      z += __shfl_xor(z, 16);
      w += __shfl_xor(w, 16);
      z += __shfl_xor(z, 32);
      w += __shfl_xor(w, 32);
      if (r < a.nq) {
        const int64_t t = a.token[r] - a.v0 - pl;  // from this lane's first token on
        if (t >= 0 && t < TP && (t & 15) < 4) {
#pragma unroll
          for (int i = 0; i < RP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t == i * 16 + e && pl + i * 16 + e < a.np) a.given[r] = acc[i][j][e];
        }
      }
      if (lane < 16) {
        float* const to_wave = part + ((wp * TQ) + r - tq0) * 3;
        to_wave[0] = m;
        to_wave[1] = z;
        to_wave[2] = w;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TQ && tq0 + i < a.nq; i += WAVES * 64) {
      Sums t;
#pragma unroll
      for (int w = 0; w < WP; ++w) {
        const float* const v = part + (w * TQ + i) * 3;
        t.add(v[0], v[1], v[2]);
      }
      const int64_t at = (int64_t)tp * a.nq + tq0 + i;
      a.pm[at] = t.m;
      a.pz[at] = t.z;
      a.pw[at] = t.w;
    }
  } else if constexpr (MODE == kGradient) {
    const bool whole = tp0 + TP <= a.np;
    const auto rows = [&](auto with_entropy) {
      constexpr bool ENT = decltype(with_entropy)::value;
#pragma unroll
      for (int j = 0; j < RQ; ++j) {
        const int r = min(ql + j * 16, a.nq - 1);
        const bool mine = ql + j * 16 < a.nq;
        const int64_t token = a.token[r];
        const bool any = token >= 0 && token < a.vocab;
        const float g = any && a.g_logprob ? a.g_logprob[r] : 0.f;
        const float ge = ENT ? a.g_entropy[r] : 0.f;
        float m, l2z;  // log2 p = (l - m) log2(e) - l2z
        if (a.three) {
          // (l - a) log2(e) - R - b, relative to a logit near the largest instead
          const float off = a.stats[3 * r + 1] * kLn2;
          m = a.stats[3 * r] + off;
          l2z = a.stats[3 * r + 2] + __builtin_fmaf(-off, kLog2e, a.stats[3 * r + 1]);
        } else {
          m = a.stats[2 * r];
          l2z = a.stats[2 * r + 1];
        }
        const float up = a.scale[r];
        const float all = -up * (g + (ENT ? ge * a.entropy[r] : 0.f));
        const float slope = -up * ge * kLn2;
        const auto value = [&](float l) {
          const float y = __builtin_fmaf(l - m, kLog2e, -l2z), p = __builtin_amdgcn_exp2f(y);
          return p * (ENT ? __builtin_fmaf(slope, fmaxf(y, kLow), all) : all);
        };
        // a row without a gradient is 0 whatever its logits are
        const unsigned keep = up == 0.f ? 0u : ~0u;
#pragma unroll
        for (int i = 0; i < RP; ++i) {
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[e] = value(acc[i][j][e]);
            if (!whole && pl + i * 16 + e >= a.np) o[e] = 0.f;
          }
          put(i, j, pack2<DT>(o[0], o[1]) & keep, pack2<DT>(o[2], o[3]) & keep);
        }
        const int64_t t = token - a.v0 - pl;  // the given token, from this lane's first one on
        if (any && keep && t >= 0 && t < RP * 16 && (t & 15) < 4) {
#pragma unroll
          for (int i = 0; i < RP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t == i * 16 + e) {
                const float v = __builtin_fmaf(up, g, value(acc[i][j][e]));
                put_one(i, j, e, (uint16_t)pack2<DT>(v, 0.f));
                if (mine) a.lost[r] = v - rounded<DT>(v);
              }
        }
      }
    };
    if (a.g_entropy)
      rows(std::true_type{});
    else
      rows(std::false_type{});
    write(a.g, a.ldg, (int)a.ldg, a.nq);
  } else {
    if (a.acc) {
      const bool vec = (a.np & 3) == 0;
#pragma unroll
      for (int j = 0; j < RQ; ++j) {
        const int r = ql + j * 16;
        if (r >= a.nq) continue;
#pragma unroll
        for (int i = 0; i < RP; ++i) {
          const int at = pl + i * 16;
          float* const dst = a.acc + ((int64_t)part * a.nq + r) * a.np + at;
          if (vec && at < a.np) {
            f32x4 s = acc[i][j];
            if (a.add) s += *reinterpret_cast<const f32x4*>(dst);
            *reinterpret_cast<f32x4*>(dst) = s;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (at + e < a.np) dst[e] = a.add ? dst[e] + acc[i][j][e] : acc[i][j][e];
          }
        }
      }
    } else {
      const float up = a.out_scale ? a.out_scale[0] : 1.f;
#pragma unroll
      for (int j = 0; j < RQ; ++j)
#pragma unroll
        for (int i = 0; i < RP; ++i) {
          const f32x4 v = acc[i][j] * up;
          put(i, j, pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
        }
      write(a.out, a.np, a.np, a.nq);
    }
  }
}

// A row's results from its parts: 16 rows by 64 threads each.  2048 rows of 125 parts take 5 us, 4096 of
// 512 12.
__global__ __launch_bounds__(1024) void head_join(const float* __restrict__ pm,
                                                  const float* __restrict__ pz,
                                                  const float* __restrict__ pw, int parts, int rows,
                                                  const float* __restrict__ given,
                                                  const int64_t* __restrict__ token, int vocab,
                                                  float* __restrict__ logprob,
                                                  float* __restrict__ entropy,
                                                  float* __restrict__ stats) {
  __shared__ float red[3][64][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, r = blockIdx.x * 16 + x;
  Sums s;
  for (int p0 = y; p0 < parts; p0 += 256) {
    float m[4], z[4], w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + j * 64;
      const int64_t at = (int64_t)p * rows + r;
      const bool on = p < parts && r < rows;
      m[j] = on ? pm[at] : 0.f;
      z[j] = on ? pz[at] : 0.f;
      w[j] = on ? pw[at] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s.add(m[j], z[j], w[j]);
  }
  // halves, so that the order is the same whatever the machine does
  for (int half = 32; half >= 1; half >>= 1) {
    if (y >= half && y < 2 * half) {
      red[0][y][x] = s.m;
      red[1][y][x] = s.z;
      red[2][y][x] = s.w;
    }
    __syncthreads();
    if (y < half) s.add(red[0][y + half][x], red[1][y + half][x], red[2][y + half][x]);
  }
  if (y || r >= rows) return;
  const int64_t t = token[r];
  const bool none = s.z == 0.f;
  const float l2z = __builtin_log2f(s.z);
  const bool any = t >= 0 && t < vocab;
  logprob[r] = !any ? 0.f : none ? -__builtin_inff() : given[r] - s.m - kLn2 * l2z;
  entropy[r] = none ? 0.f : __builtin_fmaf(kLn2, l2z, -s.w / s.z);
  if (stats) {
    stats[2 * r] = none ? 0.f : s.m;
    stats[2 * r + 1] = none ? __builtin_inff() : l2z;
  }
}

// start[i] = the first sorted place of a token from 128 i on, for i up to `tiles` (beyond the last).
__global__ __launch_bounds__(256) void head_starts(const unsigned* __restrict__ key, int rows,
                                                   int vocab, int tiles, unsigned* __restrict__ start) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i > tiles) return;
  const unsigned from = min((unsigned)vocab, 128u * i);
  int lo = 0, hi = rows;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (key[mid] < from) lo = mid + 1;
    else hi = mid;
  }
  start[i] = lo;
}

// A packed weight in 16 bits, [N, K], a block of 16 rows by 512 columns a wave: lane L has row L % 16 of
// its 128 columns L / 16.  Through LDS, so that rows are written 1 KiB at a time.  32000 x 4096: 53 us,
// 6.2 TB/s read and written.
template <int FMT, int DT>
__global__ __launch_bounds__(256) void head_decode(const uint8_t* __restrict__ w, int N, int K, int spans,
                                                   int64_t blocks, uint16_t* __restrict__ out) {
  constexpr int BB = FMT == FB_FMT_GF4 ? fb::kGf4BlockBytes : fb::kE2m1BlockBytes;
  __shared__ __align__(16) u32x4 rows[4][16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, item = lane >> 4;
  const int64_t b = (int64_t)blockIdx.x * 4 + wave;
  if (b >= blocks) return;
  Rec<FMT> r;
  load_rec_global<FMT>(w + b * BB, lane, r);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      u32x4 v;
      if constexpr (FMT == FB_FMT_GF4)
        v = gf4_decode8(r.nib[c][d], r.t0, r.t1);
      else
        v = e2m1_decode8<DT>(r.nib[c][d],
                             __builtin_bit_cast(float, ((r.t0.x >> (8 * c)) & 0xFFu) << 23));
      rows[wave][row][(item * 16 + c * 4 + d) ^ row] = v;
    }
  asm volatile("" ::: "memory");
  const int64_t n0 = b / spans * 16;
  const int col = (int)(b % spans) * 512 + lane * 8;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (n0 + i < N && col < K)
      *reinterpret_cast<u32x4*>(out + (n0 + i) * K + col) = rows[wave][i][lane ^ i];
}

// What bounds |G| in row r: 0 where no gradient comes in.  The entropy's part is p |log p + H|: at most
// 1 / e + log 2^24 = 17.1 times its gradient, for p <= 1 and at most 2^24 tokens.
__device__ inline float row_bound(int64_t r, const int64_t* token, int vocab, const float* g,
                                  const float* ge) {
  const int64_t t = token[r];
  float b = g && t >= 0 && t < vocab ? __builtin_fabsf(g[r]) : 0.f;
  if (ge) b += 24.f * __builtin_fabsf(ge[r]);
  return b;
}
// The least exponent with bound < 2^e, from -100 to 127.
__device__ inline int bound_exp(float b) {
  const int e = (int)(__builtin_bit_cast(unsigned, b) >> 23) - 126;
  return e < -100 ? -100 : e > 127 ? 127 : e;
}
constexpr int kF16Exp = 14;
constexpr float kLeastReach = -200.f;  // of all rows

// fp16: reach[r] = the exponent of what bounds the row's g x; -1000 without a gradient.  777 x 1000: 5 us.
__global__ __launch_bounds__(256) void head_reach(const uint8_t* __restrict__ x, int64_t ldx, int K8,
                                                  const int64_t* __restrict__ token, int vocab,
                                                  const float* __restrict__ g,
                                                  const float* __restrict__ ge,
                                                  float* __restrict__ reach) {
  __shared__ unsigned red[4];
  const int64_t r = blockIdx.x;
  const u32x4* const src = reinterpret_cast<const u32x4*>(x + r * ldx * 2);
  unsigned most = 0;  // of the values' bits, without their signs
  for (int i = threadIdx.x; i < K8; i += 256) {
    const u32x4 v = src[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) most = max(most, max(v[j] & 0x7FFFu, v[j] >> 16 & 0x7FFFu));
  }
  for (int s = 32; s; s >>= 1) most = max(most, __shfl_xor(most, s));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x) return;
  most = min(max(max(red[0], red[1]), max(red[2], red[3])), 0x7BFFu);  // infinities: as the largest number
  const float b = row_bound(r, token, vocab, g, ge);
  reach[r] = b == 0.f ? -1000.f
                      : (float)(bound_exp(b) +
                                bound_exp((float)__builtin_bit_cast(_Float16, (unsigned short)most)));
}

// top[1] = the largest reach, top[0] = what grad_w's sums are multiplied by.  Up to kTopRows rows
// head_rows does that by itself: a launch, 5 us of 90 of a small call with its gradients.
constexpr int kTopRows = 1024;
__global__ __launch_bounds__(1024) void head_top(const float* __restrict__ reach, int rows,
                                                 float* __restrict__ top) {
  __shared__ float red[1024];
  float e = kLeastReach;
  for (int r = threadIdx.x; r < rows; r += 1024) e = fmaxf(e, reach[r]);
  red[threadIdx.x] = e;
  __syncthreads();
  for (int s = 512; s; s >>= 1) {
    if ((int)threadIdx.x < s) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + s]);
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    top[0] = __builtin_ldexpf(1.f, (int)red[0] - kF16Exp - 16);
    top[1] = red[0];
  }
}

// A row's power of two and x as grad_w takes it: times what makes G x of all rows 2^(30 - the largest
// reach) times what they are, so that the largest x is just below 2^16; 0 where the row has no gradient
// (whatever x holds there).
template <int DT>
__global__ __launch_bounds__(256) void head_rows(const uint8_t* __restrict__ x, int64_t ldx, int K8,
                                                 const int64_t* __restrict__ token, int vocab,
                                                 const float* __restrict__ g,
                                                 const float* __restrict__ ge,
                                                 const float* __restrict__ reach, int rows,
                                                 float* __restrict__ top, float* __restrict__ scale,
                                                 float* __restrict__ undo, float* __restrict__ lost,
                                                 uint8_t* __restrict__ xs) {
  const int64_t r = blockIdx.x;
  const float b = row_bound(r, token, vocab, g, ge);
  float up = b == 0.f ? 0.f : 1.f, down = up, f = up;
  if constexpr (DT == FB_DT_F16) {
    float most = kLeastReach;
    if (xs && rows <= kTopRows) {
      __shared__ float red[4];
      for (int i = threadIdx.x; i < rows; i += 256) most = fmaxf(most, reach[i]);
      for (int s = 32; s; s >>= 1) most = fmaxf(most, __shfl_xor(most, s));
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
      __syncthreads();
      most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      if (r == 0 && threadIdx.x == 0) top[0] = __builtin_ldexpf(1.f, (int)most - kF16Exp - 16);
    } else if (xs) {
      most = top[1];
    }
    if (b != 0.f) {
      const int e = bound_exp(b);
      up = __builtin_ldexpf(1.f, kF16Exp - e);
      down = __builtin_ldexpf(1.f, e - kF16Exp);
      f = __builtin_ldexpf(1.f, 16 + e - (int)most);
    }
  }
  if (threadIdx.x == 0) {
    scale[r] = up;
    undo[r] = down;
    lost[r] = 0.f;
  }
  if (!xs) return;
  const u32x4* const src = reinterpret_cast<const u32x4*>(x + r * ldx * 2);
  u32x4* const dst = reinterpret_cast<u32x4*>(xs + r * K8 * 16);
  for (int i = threadIdx.x; i < K8; i += 256) {
    u32x4 v = b == 0.f ? u32x4{0, 0, 0, 0} : src[i];
    if constexpr (DT == FB_DT_F16) {
      half8_t h = __builtin_bit_cast(half8_t, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (_Float16)((float)h[e] * f);
      v = __builtin_bit_cast(u32x4, h);
    }
    dst[i] = v;
  }
}

// out = (the parts' sums added in their order + what the given token's value lost times its row of W)
// times the row's power of two, rounded once.  2048 x 4096 of 2 parts: 26 us, for the rows of W are
// wherever their tokens are.
template <int DT>
__global__ __launch_bounds__(256) void head_sum(const float* __restrict__ acc, int parts, int rows,
                                                int K, const float* __restrict__ undo,
                                                const float* __restrict__ lost,
                                                const int64_t* __restrict__ token, int vocab,
                                                const uint16_t* __restrict__ w, int64_t ldw,
                                                void* __restrict__ out, int odt) {
  const int64_t n = (int64_t)rows * K, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const auto value = [](unsigned h) {
    if constexpr (DT == FB_DT_F16) return (float)__builtin_bit_cast(_Float16, (unsigned short)h);
    else return __builtin_bit_cast(float, h << 16);
  };
  if (i >= n) return;
  if ((K & 3) == 0) {
    const int64_t r = i / K, t = token[r];
    f32x4 s = *reinterpret_cast<const f32x4*>(acc + i);
#pragma unroll 8
    for (int p = 1; p < parts; ++p) s += *reinterpret_cast<const f32x4*>(acc + p * n + i);
    const float l = lost[r];
    if (l != 0.f && t >= 0 && t < vocab) {
      const uint2 v = *reinterpret_cast<const uint2*>(w + t * ldw + (i - r * K));
      s += f32x4{l * value(v.x & 0xFFFFu), l * value(v.x >> 16), l * value(v.y & 0xFFFFu),
                 l * value(v.y >> 16)};
    }
    s *= undo[r];
    store4(out, i, s, odt);
  } else {
    for (int64_t at = i; at < n && at < i + 4; ++at) {
      const int64_t r = at / K, t = token[r];
      float s = acc[at];
#pragma unroll 8
      for (int p = 1; p < parts; ++p) s += acc[p * n + at];
      if (lost[r] != 0.f && t >= 0 && t < vocab) s += lost[r] * value(w[t * ldw + (at - r * K)]);
      store_y(out, at, s * undo[r], odt);
    }
  }
}

// Rows of 16-bit values, zeros behind them: `rows_of` rows of `units` 8 values a workgroup.  102177 x 3002:
// 248 us, 4.9 TB/s.
__global__ __launch_bounds__(256) void head_pad(const uint16_t* __restrict__ src, int64_t stride,
                                                int64_t rows, int K, uint16_t* __restrict__ dst,
                                                int64_t ld, unsigned units, unsigned rows_of) {
  const int64_t r0 = (int64_t)blockIdx.x * rows_of;
  for (unsigned i = threadIdx.x; i < units * rows_of; i += 256) {
    const unsigned y = i / units, u = i - y * units;
    if (r0 + y >= rows) break;
    const uint16_t* const from = src + (r0 + y) * stride + u * 8;
    u32x4 v{0, 0, 0, 0};
    if ((int)(u * 8 + 8) <= K) {
      v = *reinterpret_cast<const u32x4_any*>(from);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((int)(u * 8) + e < K) v[e / 2] |= (unsigned)from[e] << (16 * (e & 1));
    }
    *reinterpret_cast<u32x4*>(dst + (r0 + y) * ld + u * 8) = v;
  }
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------
constexpr int64_t kMostG = 1ll << 30;       // bytes of G at once
constexpr int64_t kMostRows = 1 << 23;      // 256 threads each stay below a launch's 2^32
constexpr int64_t kStatRows = 1 << 14;      // rows of logits whose parts are held at once

// Tiles to choose from: two for any product, two for few rows of grad_x, four for few rows of logits.
// With what a workgroup takes in us, of those that are chosen by it: a chunk of the contraction with all of
// a CU's workgroups running and with one, where the contraction lies along rows and where (TR) not, and the
// rest.  Fitted to timings of the four products of 2048 x 32000 x 4096, 1024 x 32000 x 4096, 4096 x
// 131072 x 4096 and 777 x 50001 x 1000.
struct Shape {
  int tp, tq, slots;  // workgroups of a CU
  double full, alone, full_tr, alone_tr, rest;
};
constexpr Shape kShapes[] = {{256, 256, 1, 1.55, 1.55, 1.5, 1.5, 9},
                             {128, 128, 2, 0.95, 0.75, 1.13, 0.85, 7},
                             {128, 64, 2, 0.8, 0.6, 0.9, 0.7, 6},
                             {128, 16, 4, 0.8, 0.4, 0.8, 0.4, 5},
                             {64, 64, 2, 0, 0, 0, 0, 0},
                             {128, 16, 2, 0, 0, 0, 0, 0},
                             {64, 16, 4, 0, 0, 0, 0, 0},
                             {128, 128, 1, 0, 0, 0, 0, 0}};

double product_us(int shape, bool tr, int64_t np, int64_t nq, int64_t k, int parts, int cus) {
  const Shape& s = kShapes[shape];
  const int64_t wgs = (np + s.tp - 1) / s.tp * ((nq + s.tq - 1) / s.tq) * parts, slots = cus * s.slots;
  const int64_t chunks = ((k + kChunk - 1) / kChunk + parts - 1) / parts, left = wgs % slots;
  const double full = tr ? s.full_tr : s.full, alone = tr ? s.alone_tr : s.alone;
  return wgs / slots * (chunks * full + s.rest) +
         (left ? chunks * (left <= cus ? alone : full) + s.rest : 0.0);
}

int pick_wide(bool tr, int64_t np, int64_t nq, int64_t k, int cus) {
  return nq <= 128 || product_us(1, tr, np, nq, k, 1, cus) < product_us(0, tr, np, nq, k, 1, cus);
}

// Of logits.  Tiles of 64 tokens up to one of 128 a CU: 16 x 32000 x 4096 44.4 us, by 128 tokens 48.8;
// 16 x 131072 x 4096 182 and 171.  Two chunks of 128 x 128 at a time, one tile a CU, where there are no
// more: 128 x 32000 x 4096 58 us, one chunk 71; 128 x 131072 x 4096 231 and 186.
int pick_shape(int64_t np, int64_t nq, int64_t k, int cus) {
  const bool few = (np + 127) / 128 <= cus;
  if (nq <= 16) return few ? 6 : 5;
  if (nq <= 64) return 4;
  if (nq <= 128 && few) return 7;
  return pick_wide(false, np, nq, k, cus);
}

template <int DT, bool PT, bool QT, int MODE>
int launch_product(ProductArgs a, int shape, int parts, hipStream_t hs) {
  const Shape s = kShapes[shape];
  a.tiles_p = (a.np + s.tp - 1) / s.tp;
  a.tiles_q = (a.nq + s.tq - 1) / s.tq;
  a.chunks = ((a.k + kChunk - 1) / kChunk + parts - 1) / parts;
  const int64_t grid = (int64_t)a.tiles_p * a.tiles_q * parts;
  if (grid > (1 << 22)) return FB_ERR_SHAPE;
  const auto go = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), 0, hs, a);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  };
  if (shape == 0) return go(product_kernel<DT, PT, QT, 256, 256, 2, 4, 1, MODE>, 512);
  if (shape == 1) return go(product_kernel<DT, PT, QT, 128, 128, 2, 2, 1, MODE>, 256);
  if constexpr (MODE == kProduct && !QT) {
    if (shape == 2) return go(product_kernel<DT, PT, QT, 128, 64, 4, 1, 1, MODE>, 256);
    if (shape == 3) return go(product_kernel<DT, PT, QT, 128, 16, 4, 1, 1, MODE>, 256);
  }
  if constexpr (MODE != kProduct) {
    if (shape == 7) return go(product_kernel<DT, PT, QT, 128, 128, 2, 2, 2, MODE>, 256);
    if (shape == 4) return go(product_kernel<DT, PT, QT, 64, 64, 2, 2, 2, MODE>, 256);
    if (shape == 5) return go(product_kernel<DT, PT, QT, 128, 16, 4, 1, 2, MODE>, 256);
    if (shape == 6) return go(product_kernel<DT, PT, QT, 64, 16, 2, 1, 2, MODE>, 128);
  }
  return FB_ERR_SHAPE;
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

struct StatPlan {
  int64_t rows;  // at once
  int shape, parts;
  size_t part_bytes, bytes;
};
StatPlan stat_plan(int64_t rows, int K, int vocab, int cus) {
  StatPlan p{};
  p.rows = std::min(rows, kStatRows);
  p.shape = pick_shape(vocab, p.rows, K, cus);
  const Shape s = kShapes[p.shape];
  p.parts = (vocab + s.tp - 1) / s.tp;
  p.part_bytes = up256((size_t)p.parts * p.rows * 4);
  p.bytes = 3 * p.part_bytes + up256(p.rows * 4);
  return p;
}

struct GradPlan {
  int64_t piece;  // tokens of the vocabulary at once
  int gshape, xshape, wshape, parts;
  size_t at_scale, at_undo, at_lost, at_top, at_reach, at_x, at_g, at_acc;
  size_t at_key, at_place, at_start, at_sort, bytes;
};
GradPlan grad_plan(int64_t rows, int K, int vocab, bool gx, bool gw, int cus) {
  GradPlan p{};
  const int64_t v256 = ((int64_t)vocab + 255) / 256 * 256;
  p.piece = std::min(v256, std::max<int64_t>(256, kMostG / (rows * 2) / 256 * 256));
  const int64_t most = std::min<int64_t>(p.piece, vocab);
  p.gshape = pick_shape(most, rows, K, cus);
  p.wshape = pick_wide(true, K, most, rows, cus);
  p.parts = 1;
  if (gx) {
    const int64_t chunks = (most + kChunk - 1) / kChunk;
    const int least = rows <= 16 ? 3 : rows <= 64 ? 2 : rows <= 128 ? 1 : 0;
    double best = 0;
    for (int shape = least; shape <= std::max(1, least); ++shape)
      for (int n = 1; n <= 64 && n <= chunks; ++n) {
        if (n > 1 && (int64_t)n * rows * K * 4 > kMostG) break;
        // and the parts' sums, written and read at 5 TB/s
        const double us = product_us(shape, true, K, rows, most, n, cus) + n * (double)rows * K * 8 / 5e6;
        if (best == 0 || us < best) {
          best = us;
          p.parts = n;
          p.xshape = shape;
        }
      }
    const int64_t per = (chunks + p.parts - 1) / p.parts;
    p.parts = (int)((chunks + per - 1) / per);
  }
  size_t at = 0;
  const auto take = [&](size_t n) {
    const size_t was = at;
    at += up256(n);
    return was;
  };
  p.at_scale = take(rows * 4);
  p.at_undo = take(rows * 4);
  p.at_lost = take(rows * 4);
  p.at_top = take(8);
  p.at_reach = take(gw ? rows * 4 : 0);
  p.at_x = take(gw ? (size_t)rows * ((K + 7) / 8) * 16 : 0);
  p.at_g = take((size_t)rows * p.piece * 2);
  p.at_acc = take(gx ? (size_t)p.parts * rows * K * 4 : 0);
  if (gw) {
    p.at_key = take(rows * 4);
    p.at_place = take(rows * 4);
    p.at_start = take(((size_t)vocab / 128 + 2) * 4);
    p.at_sort = take(fb_gpu::sort_bytes(rows, vocab));
  }
  p.bytes = at;
  return p;
}

bool bad_align(std::initializer_list<const void*> ps, unsigned mask) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & mask) return true;
  return false;
}

constexpr int64_t kMostSums = 1ll << 33;    // rows x K of grad_x

int head_check(int32_t dtype, int64_t rows, int32_t K, int32_t vocab, int64_t ldx, int64_t ldw) {
  if (dtype != FB_DT_F16 && dtype != FB_DT_BF16) return FB_ERR_DTYPE;
  const int64_t k8 = ((int64_t)K + 7) / 8 * 8;
  if (rows < 0 || rows > kMostRows || K < 1 || K > (1 << 20) || vocab < 1 || vocab > (1 << 24) ||
      ldx < k8 || ldw < k8 || ldx > (1 << 20) || ldw > (1 << 20))
    return FB_ERR_SHAPE;
  if ((ldx | ldw) & 7) return FB_ERR_ALIGN;
  return FB_OK;
}

template <int DT>
int run_stats(ProductArgs a, const StatPlan& p, int64_t rows, int32_t vocab, float* logprob,
              float* entropy, float* stats, uint8_t* ws, hipStream_t hs) {
  for (int64_t r = 0; r < rows; r += p.rows) {
    ProductArgs b = a;
    b.q = a.q + r * a.ldq * 2;
    b.nq = (int)std::min(rows - r, p.rows);
    b.token = a.token + r;
    b.pm = reinterpret_cast<float*>(ws);
    b.pz = reinterpret_cast<float*>(ws + p.part_bytes);
    b.pw = reinterpret_cast<float*>(ws + 2 * p.part_bytes);
    b.given = reinterpret_cast<float*>(ws + 3 * p.part_bytes);
    const int st = launch_product<DT, false, false, kStats>(b, p.shape, 1, hs);
    if (st != FB_OK) return st;
    hipLaunchKernelGGL(head_join, dim3((b.nq + 15) / 16), dim3(1024), 0, hs, b.pm, b.pz, b.pw, p.parts,
                       b.nq, b.given, b.token, vocab, logprob + r, entropy + r,
                       stats ? stats + 2 * r : nullptr);
    if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  }
  return FB_OK;
}

template <int DT>
int run_grad(const ProductArgs& in, const GradPlan& p, int64_t rows, int32_t K, int32_t vocab,
             void* grad_x, int32_t grad_x_dtype, void* grad_w, uint8_t* ws, hipStream_t hs) {
  float* const scale = reinterpret_cast<float*>(ws + p.at_scale);
  float* const undo = reinterpret_cast<float*>(ws + p.at_undo);
  float* const lost = reinterpret_cast<float*>(ws + p.at_lost);
  float* const top = reinterpret_cast<float*>(ws + p.at_top);
  float* const reach = reinterpret_cast<float*>(ws + p.at_reach);
  uint8_t* const xs = ws + p.at_x;
  float* const acc = reinterpret_cast<float*>(ws + p.at_acc);
  const int K8 = (K + 7) / 8;
  if (DT == FB_DT_F16 && grad_w) {
    hipLaunchKernelGGL(head_reach, dim3((unsigned)rows), dim3(256), 0, hs, in.q, in.ldq, K8, in.token,
                       vocab, in.g_logprob, in.g_entropy, reach);
    if (rows > kTopRows)
      hipLaunchKernelGGL(head_top, dim3(1), dim3(1024), 0, hs, reach, (int)rows, top);
  }
  hipLaunchKernelGGL(head_rows<DT>, dim3((unsigned)rows), dim3(256), 0, hs, in.q, in.ldq, K8,
                     in.token, vocab, in.g_logprob, in.g_entropy, reach, (int)rows, top, scale, undo,
                     lost, grad_w ? xs : nullptr);
  if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  unsigned* const key = reinterpret_cast<unsigned*>(ws + p.at_key);
  unsigned* const place = reinterpret_cast<unsigned*>(ws + p.at_place);
  unsigned* const start = reinterpret_cast<unsigned*>(ws + p.at_start);
  const int starts = (vocab + 127) / 128;
  if (grad_w) {
    const int st = fb_gpu::sort_tokens(in.token, rows, vocab, key, place, nullptr, 0, ws + p.at_sort, hs);
    if (st != FB_OK) return st;
    hipLaunchKernelGGL(head_starts, dim3((unsigned)(starts / 256 + 1)), dim3(256), 0, hs, key, (int)rows,
                       vocab, starts, start);
    if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  }
  for (int64_t v = 0; v < vocab; v += p.piece) {
    const int nv = (int)std::min<int64_t>(p.piece, vocab - v);
    ProductArgs g = in;
    g.p = in.p + v * in.ldp * 2;
    g.np = nv;
    g.nq = (int)rows;
    g.k = K8 * 8;
    g.v0 = (int)v;
    g.scale = scale;
    g.g = reinterpret_cast<uint16_t*>(ws + p.at_g);
    g.ldg = ((int64_t)nv + 63) / 64 * 64;
    g.vocab = vocab;
    g.lost = lost;
    int st = launch_product<DT, false, false, kGradient>(g, p.gshape, 1, hs);
    if (st != FB_OK) return st;
    if (grad_x) {
      ProductArgs b{};
      b.p = in.p + v * in.ldp * 2;
      b.ldp = in.ldp;
      b.np = K;
      b.q = ws + p.at_g;
      b.ldq = g.ldg;
      b.nq = (int)rows;
      b.k = nv;
      b.acc = acc;
      b.add = v > 0;
      st = launch_product<DT, true, false, kProduct>(b, p.xshape, p.parts, hs);
      if (st != FB_OK) return st;
    }
    if (grad_w) {
      ProductArgs b{};
      b.p = xs;
      b.ldp = K8 * 8;
      b.np = K;
      b.q = ws + p.at_g;
      b.ldq = g.ldg;
      b.nq = nv;
      b.k = (int)rows;
      b.out = static_cast<uint8_t*>(grad_w) + v * K * 2;
      b.out_scale = DT == FB_DT_F16 ? top : nullptr;
      b.v0 = (int)v;
      b.key = key;
      b.place = place;
      b.start = start;
      b.starts = starts;
      b.lost = lost;
      st = launch_product<DT, true, true, kProduct>(b, p.wshape, 1, hs);
      if (st != FB_OK) return st;
    }
  }
  if (grad_x) {
    const int64_t n = ((int64_t)rows * K + 1023) / 1024;
    hipLaunchKernelGGL(head_sum<DT>, dim3((unsigned)n), dim3(256), 0, hs, acc, p.parts, (int)rows, K,
                       undo, lost, in.token, vocab, reinterpret_cast<const uint16_t*>(in.p), in.ldp,
                       grad_x, grad_x_dtype);
    if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  }
  return FB_OK;
}

}  // namespace

extern "C" {

size_t fb_head_logprobs_workspace_bytes(int64_t rows, int32_t K, int32_t vocab) {
  if (rows < 1 || rows > kMostRows || K < 1 || vocab < 1) return 0;
  return stat_plan(rows, K, vocab, fb_gpu::cu_count()).bytes;
}

int fb_head_logprobs(const void* x, int64_t x_stride, const void* w, int64_t w_stride, int32_t dtype,
                     int64_t rows, int32_t K, int32_t vocab, const int64_t* token, float* logprob,
                     float* entropy, float* stats, void* ws, size_t ws_bytes, void* stream) {
  const int st = head_check(dtype, rows, K, vocab, x_stride, w_stride);
  if (st != FB_OK) return st;
  if (rows == 0) return FB_OK;
  if (!x || !w || !token || !logprob || !entropy || !ws) return FB_ERR_NULL;
  if (bad_align({x, w}, 15) || bad_align({token}, 7) || bad_align({logprob, entropy, stats}, 3) ||
      bad_align({ws}, 255))
    return FB_ERR_ALIGN;
  const StatPlan p = stat_plan(rows, K, vocab, fb_gpu::cu_count());
  if (ws_bytes < p.bytes) return FB_ERR_WORKSPACE;
  ProductArgs a{};
  a.p = static_cast<const uint8_t*>(w);
  a.ldp = w_stride;
  a.np = vocab;
  a.q = static_cast<const uint8_t*>(x);
  a.ldq = x_stride;
  a.k = (K + 7) / 8 * 8;
  a.token = token;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  return dtype == FB_DT_F16 ? run_stats<FB_DT_F16>(a, p, rows, vocab, logprob, entropy, stats,
                                                   static_cast<uint8_t*>(ws), hs)
                            : run_stats<FB_DT_BF16>(a, p, rows, vocab, logprob, entropy, stats,
                                                    static_cast<uint8_t*>(ws), hs);
}

size_t fb_head_logprobs_grad_workspace_bytes(int64_t rows, int32_t K, int32_t vocab,
                                             int32_t want_x, int32_t want_w) {
  if (rows < 1 || rows > kMostRows || K < 1 || vocab < 1) return 0;
  return grad_plan(rows, K, vocab, want_x, want_w, fb_gpu::cu_count()).bytes;
}

int fb_head_logprobs_grad(const void* x, int64_t x_stride, const void* w, int64_t w_stride,
                          int32_t dtype, int64_t rows, int32_t K, int32_t vocab,
                          const int64_t* token, const float* stats, const float* entropy,
                          const float* g_logprob, const float* g_entropy, void* grad_x, void* grad_w,
                          void* ws, size_t ws_bytes, void* stream) {
  const int st = head_check(dtype, rows, K, vocab, x_stride, w_stride);
  if (st != FB_OK) return st;
  if (grad_x && rows * K > kMostSums) return FB_ERR_SHAPE;
  if (rows == 0 || (!grad_x && !grad_w)) return FB_OK;
  if (!x || !w || !token || !stats || (g_entropy && !entropy) || !ws) return FB_ERR_NULL;
  if (bad_align({x, w}, 15) || bad_align({token}, 7) || bad_align({grad_x, grad_w}, 7) ||
      bad_align({stats, entropy, g_logprob, g_entropy}, 3) || bad_align({ws}, 255))
    return FB_ERR_ALIGN;
  const GradPlan p = grad_plan(rows, K, vocab, grad_x, grad_w, fb_gpu::cu_count());
  if (ws_bytes < p.bytes) return FB_ERR_WORKSPACE;
  ProductArgs a{};
  a.p = static_cast<const uint8_t*>(w);
  a.ldp = w_stride;
  a.q = static_cast<const uint8_t*>(x);
  a.ldq = x_stride;
  a.token = token;
  a.stats = stats;
  a.entropy = entropy;
  a.g_logprob = g_logprob;
  a.g_entropy = g_entropy;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  return dtype == FB_DT_F16
             ? run_grad<FB_DT_F16>(a, p, rows, K, vocab, grad_x, dtype, grad_w, static_cast<uint8_t*>(ws),
                                   hs)
             : run_grad<FB_DT_BF16>(a, p, rows, K, vocab, grad_x, dtype, grad_w, static_cast<uint8_t*>(ws),
                                    hs);
}

int fb_pad_rows(const void* src, int64_t src_stride, int64_t rows, int32_t K, void* dst,
                int64_t dst_stride, void* stream) {
  if (!src || !dst) return FB_ERR_NULL;
  if (rows < 1 || rows > (1 << 24) || K < 1 || K > (1 << 20) || src_stride < 0 ||
      src_stride > (1ll << 40) || dst_stride < K || dst_stride > (1 << 20) || dst_stride % 8)
    return FB_ERR_SHAPE;
  if (bad_align({src}, 1) || bad_align({dst}, 15)) return FB_ERR_ALIGN;
  // a launch has fewer than 2^32 threads: at most 2^22 workgroups
  const unsigned units = (unsigned)(K + 7) / 8;
  const unsigned rows_of = std::max({1u, 1024 / units, (unsigned)((rows + (1 << 22) - 1) >> 22)});
  hipLaunchKernelGGL(head_pad, dim3((unsigned)((rows + rows_of - 1) / rows_of)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<const uint16_t*>(src), src_stride,
                     rows, K, static_cast<uint16_t*>(dst), dst_stride, units, rows_of);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

size_t fb_packed_head_grad_workspace_bytes(const fb_shape_t* s) {
  if (!s || s->B < 1 || s->B > kMostRows || fb_validate(s) != FB_OK) return 0;
  return up256((size_t)s->N * s->K * 2) +
         grad_plan(s->B, s->K, s->N, true, false, fb_gpu::cu_count()).bytes;
}

int fb_packed_head_grad(const void* wdev, const void* x, const fb_shape_t* s, const int64_t* token,
                        const float* stats, const float* entropy, const float* g_logprob,
                        const float* g_entropy, void* grad_x, int32_t grad_x_dtype, void* ws,
                        size_t ws_bytes, void* stream) {
  if (!s || !wdev || !x || !token || !stats || (g_entropy && !entropy) || !grad_x || !ws)
    return FB_ERR_NULL;
  int st = fb_validate(s);
  if (st != FB_OK) return st;
  if (s->fwht_block) return FB_ERR_FWHT;
  if (s->x_dtype != FB_DT_F16 && s->x_dtype != FB_DT_BF16) return FB_ERR_DTYPE;
  if (s->fmt == FB_FMT_GF4 && s->x_dtype != FB_DT_F16) return FB_ERR_DTYPE;
  if (grad_x_dtype != FB_DT_F16 && grad_x_dtype != FB_DT_BF16 && grad_x_dtype != FB_DT_F32)
    return FB_ERR_DTYPE;
  st = head_check(s->x_dtype, s->B, s->K, s->N, s->K, s->K);
  if (st != FB_OK) return st;
  if ((int64_t)s->B * s->K > kMostSums) return FB_ERR_SHAPE;
  if (bad_align({wdev, x, grad_x}, 15) || bad_align({token}, 7) ||
      bad_align({stats, entropy, g_logprob, g_entropy}, 3) || bad_align({ws}, 255))
    return FB_ERR_ALIGN;
  const size_t decoded = up256((size_t)s->N * s->K * 2);
  const GradPlan p = grad_plan(s->B, s->K, s->N, true, false, fb_gpu::cu_count());
  if (ws_bytes < decoded + p.bytes) return FB_ERR_WORKSPACE;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const int spans = (s->K / 128 + 3) / 4;
  const int64_t blocks = (int64_t)((s->N + 15) / 16) * spans;
  if ((blocks + 3) / 4 > (1 << 23)) return FB_ERR_SHAPE;
  const auto decode = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((blocks + 3) / 4)), dim3(256), 0, hs,
                       static_cast<const uint8_t*>(wdev), s->N, s->K, spans, blocks,
                       static_cast<uint16_t*>(ws));
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  };
  st = s->fmt == FB_FMT_GF4         ? decode(head_decode<FB_FMT_GF4, FB_DT_F16>)
       : s->x_dtype == FB_DT_F16 ? decode(head_decode<FB_FMT_E2M1, FB_DT_F16>)
                                 : decode(head_decode<FB_FMT_E2M1, FB_DT_BF16>);
  if (st != FB_OK) return st;
  ProductArgs a{};
  a.p = static_cast<const uint8_t*>(ws);
  a.ldp = s->K;
  a.q = static_cast<const uint8_t*>(x);
  a.ldq = s->K;
  a.token = token;
  a.stats = stats;
  a.three = 1;
  a.entropy = entropy;
  a.g_logprob = g_logprob;
  a.g_entropy = g_entropy;
  uint8_t* const rest = static_cast<uint8_t*>(ws) + decoded;
  return s->x_dtype == FB_DT_F16
             ? run_grad<FB_DT_F16>(a, p, s->B, s->K, s->N, grad_x, grad_x_dtype, nullptr, rest, hs)
             : run_grad<FB_DT_BF16>(a, p, s->B, s->K, s->N, grad_x, grad_x_dtype, nullptr, rest, hs);
}

}  // extern "C"
