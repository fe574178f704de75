// The seam between two blocks of a decoder: a block's output is normalised, gated and scaled, added to
// the residual stream, and the sum is normalised for the next block; and the gradient of all of it.
//
//   b' = b rsqrt(mean b^2 + eps) wb (or b),  h = x + s g b',  y = h rsqrt(mean h^2 + eps) w
//
// with n = h r2, dn = dy w, q = s g wb n_b and n_b = b r1:
//   dx = dh + r2 (dn - n mean(dn n)),  t = s dx,  dg = t b',  db = r1 (wb g t - n_b mean(wb g t n_b))
//   dw = sum dy n,  dwb = sum t g n_b
// Everything in fp32 from the 16-bit inputs, each result rounded once: y is of the sum h before h's own
// rounding, and the gradient works that sum out again from x and b.
// A row is a group's of T threads (a wave's, or a workgroup's), kept in registers between its one read
// and one write.  The gradient's three row sums are one reduction: mean(wb g t n_b) follows from
// sum (dh + r2 dn) q and sum n q.
// Bound by memory: 8192 x 8192 in bf16 with a branch and both norms 98 us (5.5 TB/s), 8192 x 4096 52 us
// and its gradient 86 (4.7 TB/s of six arrays) with 10 for the sums of its parts.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fourbit.h"
#include "fourbit_rows.h"

namespace fb_gpu {
__attribute__((visibility("hidden"))) int cu_count();
}  // namespace fb_gpu

namespace {

// load and store of a vector that may be fp32 instead.
template <int DT, bool EVEN>
__device__ inline void load_vec(const void* p, int f32, int64_t from, int at, int n,
                                float (&o)[Of<DT>::V]) {
  constexpr int V = Of<DT>::V;
  if (DT == FB_DT_F32 || !f32) return load<DT, EVEN>(p, from, at, n, o);
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    float v[4];
    load<FB_DT_F32, EVEN>(p, from, at + h, n - h, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[h + i] = v[i];
  }
}
template <int DT, bool EVEN>
__device__ inline void store_vec(void* p, int f32, int64_t at, int n, const float (&o)[Of<DT>::V]) {
  constexpr int V = Of<DT>::V;
  if (DT == FB_DT_F32 || !f32) return store<DT, EVEN>(p, at, n, o);
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    const float v[4] = {o[h], o[h + 1], o[h + 2], o[h + 3]};
    store<FB_DT_F32, EVEN>(p, at + h, n - h, v);
  }
}

// V fp32 values to p[at] on, of d.
template <bool EVEN, int V>
__device__ inline void store_part(float* p, int at, int d, const float (&v)[V]) {
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    const float o[4] = {v[h], v[h + 1], v[h + 2], v[h + 3]};
    store<FB_DT_F32, EVEN>(p, at + h, d - at - h, o);
  }
}

template <int CTRL, int ROWS>
__device__ inline float moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL,
                                                               ROWS, 0xF, false));
}
__device__ inline float wave_sum(float v) {
  v += moved<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);  // row_bcast:15, 31
  v += moved<0x143, 0xC>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// The instruction takes numbers below 2^-126 for 0: they are brought above first.
__device__ inline float rsqrt_of(float v) {
  const bool low = v < 0x1p-100f;
  return __builtin_amdgcn_rsqf(low ? v * 0x1p60f : v) * (low ? 0x1p30f : 1.f);
}
// N sums over a group of T threads.  Calls take turns with two `red`: one barrier a call is enough then.
template <int T, int N>
__device__ inline void group_sum(float (&v)[N], float (*red)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (T > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[0][i];
#pragma unroll
      for (int w = 1; w < T / 64; ++w) v[i] += red[w][i];
    }
  }
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct NormArgs {
  fb_norm_t n;
  int bf32, wf32, gf32;  // branch_weight, weight, gate are fp32 beside 16-bit rows
  void *h, *y;
  float* stats;
  // gradient
  const void *dh, *dy;
  void *dx, *db, *dgate;
  float *pw, *pwb, *pg;  // [units, width], [units, width], [units, 2, width]
  int rows_per_unit;
  void *dw, *dwb;
  int units;
};

template <int T>
constexpr int kBlock = T == 64 ? 256 : T;  // waves that share a row share no workgroup with another

template <int DT, int T, int NV, bool EVEN>
__global__ __launch_bounds__(kBlock<T>, 4) void norm_kernel(NormArgs a) {
  constexpr int V = Of<DT>::V, G = kBlock<T> / T;
  __shared__ float red[2][T / 64][1];
  int turn = 0;
  const int t = threadIdx.x % T, group = threadIdx.x / T, d = a.n.width;
  float w[NV][V], wb[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * T + t) * V;
    load_vec<DT, EVEN>(a.n.weight, a.wf32, 0, at, d - at, w[j]);
    if (a.n.branch_weight) load_vec<DT, EVEN>(a.n.branch_weight, a.bf32, 0, at, d - at, wb[j]);
  }
  const float inv = 1.f / (float)d;
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.n.rows; r0 += (int64_t)gridDim.x * G) {
    const int64_t r = min(r0 + group, a.n.rows - 1);  // all groups take part in the barriers
    const bool mine = r0 + group < a.n.rows;
    float x[NV][V], b[NV][V], r1 = 0.f;
    u32x4 xr[NV], br[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      xr[j] = raw<DT, EVEN>(a.n.x, r * a.n.x_stride, at, d - at);
      if (a.n.branch) br[j] = raw<DT, EVEN>(a.n.branch, r * a.n.branch_stride, at, d - at);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      unpack<DT>(settled<DT, EVEN>(xr[j], at, d - at), x[j]);
      if (a.n.branch) unpack<DT>(settled<DT, EVEN>(br[j], at, d - at), b[j]);
    }
    if (a.n.branch) {
      if (a.n.branch_weight) {
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) s[0] = __builtin_fmaf(b[j][i], b[j][i], s[0]);
        group_sum<T>(s, red[turn ^= 1]);
        r1 = rsqrt_of(__builtin_fmaf(s[0], inv, a.n.eps));
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) b[j][i] = b[j][i] * r1 * wb[j][i];
      }
      const int64_t g0 = a.n.gate ? r / a.n.gate_rows * d : 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * T + t) * V;
        float g[V];
        if (a.n.gate) load_vec<DT, EVEN>(a.n.gate, a.gf32, g0, at, d - at, g);
#pragma unroll
        for (int i = 0; i < V; ++i)
          x[j][i] = __builtin_fmaf(a.n.gate ? a.n.scale * g[i] : a.n.scale, b[j][i], x[j][i]);
        if (mine) store<DT, EVEN>(a.h, r * d + at, d - at, x[j]);
      }
    }
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] = __builtin_fmaf(x[j][i], x[j][i], s[0]);
    group_sum<T>(s, red[turn ^= 1]);
    const float r2 = rsqrt_of(__builtin_fmaf(s[0], inv, a.n.eps));
    if (!mine) continue;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = x[j][i] * r2 * w[j][i];
      store<DT, EVEN>(a.y, r * d + at, d - at, y);
    }
    if (a.stats && t == 0) {
      a.stats[2 * r] = r1;
      a.stats[2 * r + 1] = r2;
    }
  }
}

// 16 bytes of a row's values, or the two pieces that as many take in fp32.
struct Raw2 {
  u32x4 lo, hi;
};
template <int DT, bool EVEN>
__device__ inline Raw2 raw_vec(const void* p, int f32, int64_t from, int at, int n) {
  if (DT == FB_DT_F32 || !f32) return {raw<DT, EVEN>(p, from, at, n), u32x4{0, 0, 0, 0}};
  return {raw<FB_DT_F32, EVEN>(p, from, at, n), raw<FB_DT_F32, EVEN>(p, from, at + 4, n - 4)};
}
template <int DT, bool EVEN>
__device__ inline void unpack_vec(const Raw2& r, int f32, int at, int n, float (&o)[Of<DT>::V]) {
  if (DT == FB_DT_F32 || !f32) return unpack<DT>(settled<DT, EVEN>(r.lo, at, n), o);
  const u32x4 lo = settled<FB_DT_F32, EVEN>(r.lo, at, n), hi = settled<FB_DT_F32, EVEN>(r.hi, at + 4, n - 4);
#pragma unroll
  for (int i = 0; i < Of<DT>::V; ++i) {
    const unsigned u = i < 4 ? lo[i & 3] : hi[i & 3];
    o[i] = __builtin_bit_cast(float, u);
  }
}

// A unit is the rows_per_unit consecutive rows of a group of threads, which keeps their sums for the
// weights and, over runs of rows that share a gate, for the gate.  A gate whose rows are all one
// unit's is written; else the unit leaves its part, in place 0 where the gate's first row of it is the
// unit's first, in place 1 otherwise (its last gate).  A row is asked for while the one before it is
// worked on, and kept as it came: what is needed again after the sums is unpacked again.
//
// KIND -1: any call.  From 0 on: rows of whole pieces with a branch, kPost and kGate as bits of it say
// (the code of what is not there costs registers, and they are what bounds the rows in flight).
constexpr int kAny = -1, kPost = 1, kGate = 2;
template <int DT, int T, int NV, int KIND>
__global__ __launch_bounds__(kBlock<T>) void norm_grad_kernel(NormArgs a) {
  constexpr bool EVEN = KIND != kAny;
  constexpr int V = Of<DT>::V, G = kBlock<T> / T;
  // Wide rows: no room to keep what the sums are made of, or the next row; and as many of the weights' and
  // the gate's sums as LDS holds are there.
  constexpr bool LEAN = T == 1024;
  constexpr int kInLds = !LEAN ? 0 : NV * V <= 8 ? 3 : NV * V <= 16 ? 2 : 1;
  __shared__ f32x4 lds_sums[kInLds ? kInLds : 1][kInLds ? NV * V / 4 : 1][kInLds ? T : 1];
  __shared__ float red[2][T / 64][3];
  const int t = threadIdx.x % T, group = threadIdx.x / T, d = a.n.width;
  const int unit = blockIdx.x * G + group;
  const int64_t first = (int64_t)unit * a.rows_per_unit;
  const int64_t end = min(first + a.rows_per_unit, a.n.rows);
  const bool branch = KIND != kAny || a.n.branch;
  const bool post = KIND != kAny ? KIND & kPost : a.n.branch_weight != nullptr;
  const bool gate = KIND != kAny ? KIND & kGate : a.n.gate != nullptr;
  if (first >= end) return;  // the whole group
  float sums[3][NV][V], kept_w[NV][V], kept_wb[NV][V];
  // Sums 0 (weight), 1 (branch weight), 2 (gate) of piece j: the value of one of its values ...
  const auto sum_at = [&](int k, int j, int i) __attribute__((always_inline)) -> float {
    return k < kInLds ? lds_sums[k < kInLds ? k : 0][(j * V + i) / 4][t][i & 3] : sums[k][j][i];
  };
  // ... grows by the products of two, or is cleared
  const auto grow = [&](int k, int j, const float (&p)[V], const float (&q)[V])
      __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < V; h += 4) {
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(p[h + i], q[h + i], sum_at(k, j, h + i));
      if (k < kInLds)
        lds_sums[k < kInLds ? k : 0][(j * V + h) / 4][t] = v;
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[k][j][h + i] = v[i];
    }
  };
  const auto clear = [&](int k, int j) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < V; h += 4) {
      if (k < kInLds) lds_sums[k < kInLds ? k : 0][(j * V + h) / 4][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[k][j][h + i] = 0.f;
    }
  };
  const auto sums_of = [&](int k, int j, float (&o)[V]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = sum_at(k, j, i);
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * T + t) * V;
    if (!LEAN) {
      load_vec<DT, EVEN>(a.n.weight, a.wf32, 0, at, d - at, kept_w[j]);
      if (post) load_vec<DT, EVEN>(a.n.branch_weight, a.bf32, 0, at, d - at, kept_wb[j]);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) clear(k, j);
  }
  const float inv = 1.f / (float)d;
  int64_t gi = gate ? first / a.n.gate_rows : 0;
  int64_t left = gate ? (gi + 1) * a.n.gate_rows - first : 0;  // rows of this gate from here on
  int turn = 0;
  u32x4 x[NV], b[NV], gy[NV], gh[NV];
  Raw2 g[NV];
  float r1, r2;
  const auto fetch = [&](int64_t r, int64_t of) {
    r1 = a.stats[2 * r];
    r2 = a.stats[2 * r + 1];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      x[j] = raw<DT, EVEN>(a.n.x, r * a.n.x_stride, at, d - at);
      if (branch) b[j] = raw<DT, EVEN>(a.n.branch, r * a.n.branch_stride, at, d - at);
      if (gate) g[j] = raw_vec<DT, EVEN>(a.n.gate, a.gf32, of * d, at, d - at);
      gy[j] = gh[j] = u32x4{0, 0, 0, 0};
      if (a.dy) gy[j] = raw<DT, EVEN>(a.dy, r * d, at, d - at);
      if (a.dh) gh[j] = raw<DT, EVEN>(a.dh, r * d, at, d - at);
    }
  };
  // Piece j: n, u = dh + r2 dn, the branch (n_b after a norm), f = scale gate, q, dn, dy, the weights.
  struct Piece {
    float n[V], u[V], nb[V], f[V], q[V], dn[V], dy[V], wb[V];
  };
  const auto piece = [&](int j) __attribute__((always_inline)) {
    Piece p;
    const int at = (j * T + t) * V;
    float w[V];
    unpack<DT>(settled<DT, EVEN>(x[j], at, d - at), p.n);
    unpack<DT>(settled<DT, EVEN>(gy[j], at, d - at), p.dy);
    unpack<DT>(settled<DT, EVEN>(gh[j], at, d - at), p.u);
    if (branch) {
      unpack<DT>(settled<DT, EVEN>(b[j], at, d - at), p.nb);
      if (gate) unpack_vec<DT, EVEN>(g[j], a.gf32, at, d - at, p.f);
    }
    if (LEAN) {
      load_vec<DT, EVEN>(a.n.weight, a.wf32, 0, at, d - at, w);
      if (post) load_vec<DT, EVEN>(a.n.branch_weight, a.bf32, 0, at, d - at, p.wb);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!LEAN) {
        w[i] = kept_w[j][i];
        if (post) p.wb[i] = kept_wb[j][i];
      }
      p.q[i] = 0.f;
      if (branch) {
        if (post) p.nb[i] *= r1;
        p.f[i] = gate ? a.n.scale * p.f[i] : a.n.scale;
        p.q[i] = post ? p.f[i] * p.wb[i] * p.nb[i] : p.f[i] * p.nb[i];
      }
      p.n[i] = (p.n[i] + p.q[i]) * r2;
      p.dn[i] = p.dy[i] * w[i];
      p.u[i] = __builtin_fmaf(r2, p.dn[i], p.u[i]);
    }
    return p;
  };
  fetch(first, gi);
  for (int64_t r = first; r < end; ++r) {
    float s[3] = {0.f, 0.f, 0.f};
    Piece kept[LEAN ? 1 : NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Piece p = piece(j);
      if (!LEAN) kept[j] = p;
      grow(0, j, p.dy, p.n);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[0] = __builtin_fmaf(p.dn[i], p.n[i], s[0]);
        s[1] = __builtin_fmaf(p.u[i], p.q[i], s[1]);
        s[2] = __builtin_fmaf(p.n[i], p.q[i], s[2]);
      }
      if (LEAN) __builtin_amdgcn_sched_barrier(0);
    }
    const int64_t of = gi;
    const float ra = r1, rb = r2;
    const bool flush = gate && (--left == 0 || r + 1 == end);
    if (gate && left == 0) {
      ++gi;
      left = a.n.gate_rows;
    }
    if (!LEAN && r + 1 < end) fetch(r + 1, gi);
    group_sum<T>(s, red[turn ^= 1]);
    const float m1 = s[0] * inv * rb;           // dx = u - m1 n
    const float m2 = (s[1] - m1 * s[2]) * inv;  // mean of wb g t n_b
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (LEAN)  // or the compiler keeps what it worked out before
        asm volatile("" : "+v"(x[j]), "+v"(b[j]), "+v"(gy[j]), "+v"(gh[j]), "+v"(g[j].lo), "+v"(g[j].hi));
      Piece p = LEAN ? piece(j) : kept[LEAN ? 0 : j];
      const int at = (j * T + t) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) p.u[i] = __builtin_fmaf(-m1, p.n[i], p.u[i]);
      if (a.dx) store<DT, EVEN>(a.dx, r * d + at, d - at, p.u);
      if (branch) {
        if (gate) {
          float tt[V], b2[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            tt[i] = a.n.scale * p.u[i];
            b2[i] = post ? p.wb[i] * p.nb[i] : p.nb[i];
          }
          grow(2, j, tt, b2);
        }
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = p.u[i] * p.f[i];  // g t
        if (post) {
          grow(1, j, o, p.nb);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] = ra * __builtin_fmaf(-m2, p.nb[i], o[i] * p.wb[i]);
        }
        if (a.db) store<DT, EVEN>(a.db, r * d + at, d - at, o);
      }
      if (LEAN) __builtin_amdgcn_sched_barrier(0);
    }
    if (LEAN && r + 1 < end) fetch(r + 1, gi);
    if (flush) {
      const int64_t g0 = of * a.n.gate_rows, g1 = min(g0 + a.n.gate_rows, a.n.rows);
      const bool whole = g0 >= first && g1 <= end;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * T + t) * V;
        float o[V];
        sums_of(2, j, o);
        clear(2, j);
        if (a.dgate && whole)
          store_vec<DT, EVEN>(a.dgate, a.gf32, of * d + at, d - at, o);
        else if (a.dgate)
          store_part<EVEN>(a.pg + ((int64_t)unit * 2 + (g0 > first)) * d, at, d, o);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * T + t) * V;
    float o[V];
    if (a.dw) {
      sums_of(0, j, o);
      store_part<EVEN>(a.pw + (int64_t)unit * d, at, d, o);
    }
    if (a.dwb) {
      sums_of(1, j, o);
      store_part<EVEN>(a.pwb + (int64_t)unit * d, at, d, o);
    }
  }
}

// Sums of the units' parts, in their order within 16 shares: blockIdx.y 0: weight, 1: branch weight,
// from 2 on gates.
template <int DT>
__global__ __launch_bounds__(1024) void norm_grad_sum(NormArgs a, int64_t gates) {
  __shared__ float red[16][64];
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6, d = a.n.width;
  const int c = blockIdx.x * 64 + x;
  for (int64_t what = blockIdx.y; what < 2 + gates; what += gridDim.y) {
    const float* p;
    void* out;
    int f32, u0 = 0, u1 = a.units;
    int64_t at = c;
    if (what == 0) {
      p = a.pw;
      out = a.dw;
      f32 = a.wf32;
    } else if (what == 1) {
      p = a.pwb;
      out = a.dwb;
      f32 = a.bf32;
    } else {
      const int64_t g = what - 2, g0 = g * a.n.gate_rows;
      u0 = (int)(g0 / a.rows_per_unit);
      u1 = (int)((min(g0 + a.n.gate_rows, a.n.rows) - 1) / a.rows_per_unit) + 1;
      p = a.pg;
      out = u1 - u0 > 1 ? a.dgate : nullptr;  // else written already
      f32 = a.gf32;
      at = g * d + c;
    }
    if (!out) continue;
    float s = 0.f;
    if (c < d) {
#pragma unroll 4
      for (int u = u0 + y; u < u1; u += 16) {
        const int64_t row =
            what < 2 ? u
                     : (int64_t)u * 2 + ((what - 2) * a.n.gate_rows > (int64_t)u * a.rows_per_unit);
        s += p[row * d + c];
      }
    }
    red[y][x] = s;
    __syncthreads();
    if (y == 0 && c < d) {
      for (int i = 1; i < 16; ++i) s += red[i][x];
      if (f32 || DT == FB_DT_F32)
        static_cast<float*>(out)[at] = s;
      else
        static_cast<typename Of<DT>::T*>(out)[at] = (typename Of<DT>::T)s;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------
constexpr int kMaxWidth = 32768;

int norm_check(const fb_norm_t* n) {
  if (!n) return FB_ERR_NULL;
  if (n->dtype != FB_DT_F16 && n->dtype != FB_DT_BF16 && n->dtype != FB_DT_F32) return FB_ERR_DTYPE;
  if (n->rows < 0 || n->rows > INT32_MAX || n->width < 1 || n->width > kMaxWidth ||
      n->x_stride < 0 || n->branch_stride < 0)
    return FB_ERR_SHAPE;
  if (!n->branch && (n->gate || n->branch_weight)) return FB_ERR_NULL;
  if (!n->weight || (n->rows && !n->x)) return FB_ERR_NULL;
  const auto other = [&](const void* p, int32_t dt) {
    return p && dt != n->dtype && dt != FB_DT_F32;
  };
  if (other(n->weight, n->weight_dtype) || other(n->branch_weight, n->branch_weight_dtype) ||
      other(n->gate, n->gate_dtype))
    return FB_ERR_DTYPE;
  if (n->gate && (n->gate_rows < 1 || n->gate_rows > INT32_MAX)) return FB_ERR_SHAPE;
  const auto off = [](const void* p, int32_t dt) {
    return reinterpret_cast<uintptr_t>(p) & (dt == FB_DT_F32 ? 3u : 1u);
  };
  if (off(n->x, n->dtype) || off(n->branch, n->dtype) || off(n->weight, n->weight_dtype) ||
      (n->branch_weight && off(n->branch_weight, n->branch_weight_dtype)) ||
      (n->gate && off(n->gate, n->gate_dtype)))
    return FB_ERR_ALIGN;
  if (!(n->eps >= 0.f)) return FB_ERR_VALUE;
  return FB_OK;
}

bool off_row(const void* p, int32_t dt) {
  return reinterpret_cast<uintptr_t>(p) & (dt == FB_DT_F32 ? 3u : 1u);
}

NormArgs norm_args(const fb_norm_t* n) {
  NormArgs a{};
  a.n = *n;
  const bool narrow = n->dtype != FB_DT_F32;
  a.wf32 = narrow && n->weight_dtype == FB_DT_F32;
  a.bf32 = narrow && n->branch_weight_dtype == FB_DT_F32;
  a.gf32 = narrow && n->gate_dtype == FB_DT_F32;
  return a;
}

// Threads of a row, and its values a thread.
struct Split {
  int threads, values;
};
Split split_of(int width) {
  if (width <= 512) return {64, 8};
  for (int t = 64; t <= 1024; t *= 2)
    if (width <= t * 16) return {t, 16};
  return {1024, 32};
}
// The gradient keeps three sums for each value: half as many of them a thread.
Split grad_split_of(int width) {
  for (int t = 64; t <= 1024; t *= 2)
    if (width <= t * 8) return {t, 8};
  return {1024, width <= 16384 ? 16 : 32};
}

// Units of the gradient: as many as fill the device once, for each leaves sums to be added.
int rows_per_unit(const fb_norm_t* n, int cus) {
  const int64_t units = (int64_t)cus * std::min(8, std::max(1, 1024 / grad_split_of(n->width).threads));
  return (int)std::max<int64_t>(1, (n->rows + units - 1) / units);
}

struct NormPlan {
  int per, units;
  size_t at_w, at_wb, at_g, bytes;
};
NormPlan norm_plan(const fb_norm_t* n, int cus) {
  NormPlan p{};
  p.per = rows_per_unit(n, cus);
  p.units = (int)((n->rows + p.per - 1) / p.per);
  const size_t one = ((size_t)p.units * n->width * 4 + 255) & ~size_t(255);
  p.at_w = 0;
  p.at_wb = one;
  p.at_g = p.at_wb + (n->branch_weight ? one : 0);
  p.bytes = p.at_g + (n->gate && n->gate_rows > 1 ? 2 * one : 0);
  return p;
}

template <int T, int VALUES, int DT>
struct Config {
  static constexpr int kThreads = T, kVecs = VALUES / Of<DT>::V;
};
template <int DT>
int run_norm(const NormArgs& a, hipStream_t hs) {
  const auto go = [&](auto c) {
    constexpr int T = decltype(c)::kThreads, NV = decltype(c)::kVecs, G = kBlock<T> / T;
    const int64_t groups = (a.n.rows + G - 1) / G;
    const int64_t most = (int64_t)fb_gpu::cu_count() * (2048 / kBlock<T>);
    const dim3 grid((unsigned)std::min(groups, most)), block(kBlock<T>);
    if (a.n.width % 8 == 0)
      hipLaunchKernelGGL((norm_kernel<DT, T, NV, true>), grid, block, 0, hs, a);
    else
      hipLaunchKernelGGL((norm_kernel<DT, T, NV, false>), grid, block, 0, hs, a);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  };
  const Split s = split_of(a.n.width);
  if (s.values == 8) return go(Config<64, 8, DT>{});
  if (s.values == 32) return go(Config<1024, 32, DT>{});
  switch (s.threads) {
    case 64: return go(Config<64, 16, DT>{});
    case 128: return go(Config<128, 16, DT>{});
    case 256: return go(Config<256, 16, DT>{});
    case 512: return go(Config<512, 16, DT>{});
    default: return go(Config<1024, 16, DT>{});
  }
}

template <int DT>
int run_norm_grad(const NormArgs& a, hipStream_t hs) {
  const auto go = [&](auto c) {
    constexpr int T = decltype(c)::kThreads, NV = decltype(c)::kVecs, G = kBlock<T> / T;
    const dim3 grid((unsigned)((a.units + G - 1) / G)), block(kBlock<T>);
    const int kind = !a.n.branch || a.n.width % 8 ? kAny
                                                  : (a.n.branch_weight ? kPost : 0) + (a.n.gate ? kGate : 0);
    if constexpr (NV * Of<DT>::V <= 16) {
      if (kind == 0) hipLaunchKernelGGL((norm_grad_kernel<DT, T, NV, 0>), grid, block, 0, hs, a);
      if (kind == 1) hipLaunchKernelGGL((norm_grad_kernel<DT, T, NV, 1>), grid, block, 0, hs, a);
      if (kind == 2) hipLaunchKernelGGL((norm_grad_kernel<DT, T, NV, 2>), grid, block, 0, hs, a);
      if (kind == 3) hipLaunchKernelGGL((norm_grad_kernel<DT, T, NV, 3>), grid, block, 0, hs, a);
    }
    if (NV * Of<DT>::V > 16 || kind == kAny)
      hipLaunchKernelGGL((norm_grad_kernel<DT, T, NV, kAny>), grid, block, 0, hs, a);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  };
  const Split s = grad_split_of(a.n.width);
  int st;
  if (s.values == 32) st = go(Config<1024, 32, DT>{});
  else if (s.values == 16) st = go(Config<1024, 16, DT>{});
  else if (s.threads == 1024) st = go(Config<1024, 8, DT>{});
  else if (s.threads == 512) st = go(Config<512, 8, DT>{});
  else if (s.threads == 256) st = go(Config<256, 8, DT>{});
  else if (s.threads == 128) st = go(Config<128, 8, DT>{});
  else st = go(Config<64, 8, DT>{});
  if (st != FB_OK) return st;
  int64_t gates = 0;
  if (a.dgate && a.n.gate_rows > 1) gates = (a.n.rows + a.n.gate_rows - 1) / a.n.gate_rows;
  if (!a.dw && !a.dwb && !gates) return FB_OK;
  hipLaunchKernelGGL(norm_grad_sum<DT>,
                     dim3((a.n.width + 63) / 64, (unsigned)std::min<int64_t>(2 + gates, 32768)),
                     dim3(1024), 0, hs, a, gates);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

}  // namespace

extern "C" {

int fb_residual_norm(const fb_norm_t* n, void* h, void* y, float* stats, void* stream) {
  const int st = norm_check(n);
  if (st != FB_OK) return st;
  if (n->rows == 0) return FB_OK;
  if (!y || (n->branch && !h)) return FB_ERR_NULL;
  if (off_row(y, n->dtype) || off_row(h, n->dtype) || off_row(stats, FB_DT_F32)) return FB_ERR_ALIGN;
  NormArgs a = norm_args(n);
  a.h = h;
  a.y = y;
  a.stats = stats;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  return n->dtype == FB_DT_F16    ? run_norm<FB_DT_F16>(a, hs)
         : n->dtype == FB_DT_BF16 ? run_norm<FB_DT_BF16>(a, hs)
                                  : run_norm<FB_DT_F32>(a, hs);
}

size_t fb_residual_norm_grad_workspace_bytes(const fb_norm_t* n) {
  if (norm_check(n) != FB_OK || n->rows == 0) return 0;
  return norm_plan(n, fb_gpu::cu_count()).bytes;
}

int fb_residual_norm_grad(const fb_norm_t* n, const float* stats, const void* g_h, const void* g_y,
                          void* grad_x, void* grad_branch, void* grad_weight,
                          void* grad_branch_weight, void* grad_gate, void* ws, size_t ws_bytes,
                          void* stream) {
  const int st = norm_check(n);
  if (st != FB_OK) return st;
  if (n->rows == 0) return FB_OK;
  if (!stats || (!n->branch && grad_branch) || (!n->branch_weight && grad_branch_weight) ||
      (!n->gate && grad_gate))
    return FB_ERR_NULL;
  for (const void* p : {g_h, g_y, (const void*)grad_x, (const void*)grad_branch})
    if (off_row(p, n->dtype)) return FB_ERR_ALIGN;
  if (off_row(grad_weight, n->weight_dtype) || off_row(grad_branch_weight, n->branch_weight_dtype) ||
      off_row(grad_gate, n->gate_dtype) || off_row(stats, FB_DT_F32))
    return FB_ERR_ALIGN;
  const NormPlan p = norm_plan(n, fb_gpu::cu_count());
  if (!ws) return FB_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(ws) & 255u) return FB_ERR_ALIGN;
  if (ws_bytes < p.bytes) return FB_ERR_WORKSPACE;
  NormArgs a = norm_args(n);
  a.stats = const_cast<float*>(stats);
  a.dh = g_h;
  a.dy = g_y;
  a.dx = grad_x;
  a.db = grad_branch;
  a.dw = grad_weight;
  a.dwb = grad_branch_weight;
  a.dgate = grad_gate;
  uint8_t* const w = static_cast<uint8_t*>(ws);
  a.pw = reinterpret_cast<float*>(w + p.at_w);
  a.pwb = reinterpret_cast<float*>(w + p.at_wb);
  a.pg = reinterpret_cast<float*>(w + p.at_g);
  a.rows_per_unit = p.per;
  a.units = p.units;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  return n->dtype == FB_DT_F16    ? run_norm_grad<FB_DT_F16>(a, hs)
         : n->dtype == FB_DT_BF16 ? run_norm_grad<FB_DT_BF16>(a, hs)
                                  : run_norm_grad<FB_DT_F32>(a, hs);
}

}  // extern "C"
