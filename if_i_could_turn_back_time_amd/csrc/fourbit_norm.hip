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
// sum (dh + r2 dn) q and sum n q.  Bound by memory.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fourbit.h"

namespace fb_gpu {
__attribute__((visibility("hidden"))) int cu_count();
}  // namespace fb_gpu

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

// V values from p on, of which the first `n` are there (0 beyond them).
template <int DT>
__device__ inline void load(const void* p, int64_t at, int n, float (&o)[Of<DT>::V]) {
  using T = typename Of<DT>::T;
  constexpr int V = Of<DT>::V;
  const T* s = static_cast<const T*>(p) + at;
  if (n >= V) {
    const u32x4 w = *reinterpret_cast<const u32x4_any*>(s);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (DT == FB_DT_F32) {
        const unsigned u = w[i];
        o[i] = __builtin_bit_cast(float, u);
      } else {
        const unsigned u = w[i / 2];
        if constexpr (DT == FB_DT_F16)
          o[i] = (float)__builtin_bit_cast(_Float16, (unsigned short)(u >> (16 * (i & 1))));
        else
          o[i] = __builtin_bit_cast(float, i & 1 ? u & 0xFFFF0000u : u << 16);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = i < n ? (float)s[i] : 0.f;
  }
}
template <int DT>
__device__ inline void store(void* p, int64_t at, int n, const float (&v)[Of<DT>::V]) {
  using T = typename Of<DT>::T;
  constexpr int V = Of<DT>::V;
  T* d = static_cast<T*>(p) + at;
  if (n >= V) {
    T o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (T)v[i];
    u32x4 w;
    __builtin_memcpy(&w, o, 16);
    *reinterpret_cast<u32x4_any*>(d) = w;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) d[i] = (T)v[i];
  }
}
// The same of a vector that may be fp32 instead.
template <int DT>
__device__ inline void load_vec(const void* p, int f32, int64_t at, int n, float (&o)[Of<DT>::V]) {
  constexpr int V = Of<DT>::V;
  if (DT == FB_DT_F32 || !f32) return load<DT>(p, at, n, o);
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    float v[4];
    load<FB_DT_F32>(p, at + h, n - h, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[h + i] = v[i];
  }
}
template <int DT>
__device__ inline void store_vec(void* p, int f32, int64_t at, int n, const float (&o)[Of<DT>::V]) {
  constexpr int V = Of<DT>::V;
  if (DT == FB_DT_F32 || !f32) return store<DT>(p, at, n, o);
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    const float v[4] = {o[h], o[h + 1], o[h + 2], o[h + 3]};
    store<FB_DT_F32>(p, at + h, n - h, v);
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

template <int DT, int T, int NV>
__global__ __launch_bounds__(kBlock<T>) void norm_kernel(NormArgs a) {
  constexpr int V = Of<DT>::V, G = kBlock<T> / T;
  __shared__ float red[2][T / 64][1];
  int turn = 0;
  const int t = threadIdx.x % T, group = threadIdx.x / T, d = a.n.width;
  float w[NV][V], wb[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * T + t) * V;
    load_vec<DT>(a.n.weight, a.wf32, at, d - at, w[j]);
    if (a.n.branch_weight) load_vec<DT>(a.n.branch_weight, a.bf32, at, d - at, wb[j]);
  }
  const float inv = 1.f / (float)d;
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.n.rows; r0 += (int64_t)gridDim.x * G) {
    const int64_t r = min(r0 + group, a.n.rows - 1);  // all groups take part in the barriers
    const bool mine = r0 + group < a.n.rows;
    float x[NV][V], b[NV][V], r1 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      load<DT>(a.n.x, r * a.n.x_stride + at, d - at, x[j]);
      if (a.n.branch) load<DT>(a.n.branch, r * a.n.branch_stride + at, d - at, b[j]);
    }
    if (a.n.branch) {
      if (a.n.branch_weight) {
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) s[0] = __builtin_fmaf(b[j][i], b[j][i], s[0]);
        group_sum<T>(s, red[turn ^= 1]);
        r1 = __builtin_amdgcn_rsqf(__builtin_fmaf(s[0], inv, a.n.eps));
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
        if (a.n.gate) load_vec<DT>(a.n.gate, a.gf32, g0 + at, d - at, g);
#pragma unroll
        for (int i = 0; i < V; ++i)
          x[j][i] = __builtin_fmaf(a.n.gate ? a.n.scale * g[i] : a.n.scale, b[j][i], x[j][i]);
        if (mine) store<DT>(a.h, r * d + at, d - at, x[j]);
      }
    }
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] = __builtin_fmaf(x[j][i], x[j][i], s[0]);
    group_sum<T>(s, red[turn ^= 1]);
    const float r2 = __builtin_amdgcn_rsqf(__builtin_fmaf(s[0], inv, a.n.eps));
    if (!mine) continue;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = x[j][i] * r2 * w[j][i];
      store<DT>(a.y, r * d + at, d - at, y);
    }
    if (a.stats && t == 0) {
      a.stats[2 * r] = r1;
      a.stats[2 * r + 1] = r2;
    }
  }
}

// A unit is the rows_per_unit consecutive rows of a group of threads, which keeps their sums for the
// weights and, over runs of rows that share a gate, for the gate.  A gate whose rows are all one
// unit's is written; else the unit leaves its part, in place 0 where the gate's first row of it is the
// unit's first, in place 1 otherwise (its last gate).
template <int DT, int T, int NV>
__global__ __launch_bounds__(kBlock<T>) void norm_grad_kernel(NormArgs a) {
  constexpr int V = Of<DT>::V, G = kBlock<T> / T;
  __shared__ float red[2][T / 64][3];
  const int t = threadIdx.x % T, group = threadIdx.x / T, d = a.n.width;
  const int unit = blockIdx.x * G + group;
  const int64_t first = (int64_t)unit * a.rows_per_unit;
  const int64_t end = min(first + a.rows_per_unit, a.n.rows);
  const bool branch = a.n.branch, post = a.n.branch_weight, gate = a.n.gate;
  float sw[NV][V], swb[NV][V], sg[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) sw[j][i] = swb[j][i] = sg[j][i] = 0.f;
  const float inv = 1.f / (float)d;
  int64_t gi = gate ? first / a.n.gate_rows : 0;
  int turn = 0;
  for (int64_t k = 0; k < a.rows_per_unit; ++k) {
    const int64_t r = first + k;
    if (r >= end) break;  // the same for the whole group
    const float r1 = a.stats[2 * r], r2 = a.stats[2 * r + 1];
    float x[NV][V], b[NV][V], gy[NV][V], u[NV][V];  // u: dh + r2 dn
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      load<DT>(a.n.x, r * a.n.x_stride + at, d - at, x[j]);
      if (branch) load<DT>(a.n.branch, r * a.n.branch_stride + at, d - at, b[j]);
      if (a.dy) load<DT>(a.dy, r * d + at, d - at, gy[j]);
      if (a.dh) load<DT>(a.dh, r * d + at, d - at, u[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      float w[V], wb[V], g[V];
      load_vec<DT>(a.n.weight, a.wf32, at, d - at, w);
      if (post) load_vec<DT>(a.n.branch_weight, a.bf32, at, d - at, wb);
      if (gate) load_vec<DT>(a.n.gate, a.gf32, gi * d + at, d - at, g);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float q = 0.f;
        if (branch) {
          if (post) b[j][i] *= r1;  // n_b
          const float f = gate ? a.n.scale * g[i] : a.n.scale;
          q = post ? f * wb[i] * b[j][i] : f * b[j][i];
        }
        const float n = (x[j][i] + q) * r2;
        const float dy = a.dy ? gy[j][i] : 0.f, dn = dy * w[i];
        u[j][i] = __builtin_fmaf(r2, dn, a.dh ? u[j][i] : 0.f);
        x[j][i] = n;
        sw[j][i] = __builtin_fmaf(dy, n, sw[j][i]);
        s[0] = __builtin_fmaf(dn, n, s[0]);
        if (post) {
          s[1] = __builtin_fmaf(u[j][i], q, s[1]);
          s[2] = __builtin_fmaf(n, q, s[2]);
        }
      }
    }
    group_sum<T>(s, red[turn ^= 1]);
    const float m1 = s[0] * inv * r2;               // dx = u - m1 n
    const float m2 = (s[1] - m1 * s[2]) * inv;      // mean of wb g t n_b
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * T + t) * V;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = u[j][i] = __builtin_fmaf(-m1, x[j][i], u[j][i]);
      if (a.dx) store<DT>(a.dx, r * d + at, d - at, o);
      if (branch) {
        float wb[V], g[V];
        if (post) load_vec<DT>(a.n.branch_weight, a.bf32, at, d - at, wb);
        if (gate) load_vec<DT>(a.n.gate, a.gf32, gi * d + at, d - at, g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float tt = a.n.scale * u[j][i], nb = b[j][i];
          sg[j][i] = __builtin_fmaf(tt, post ? wb[i] * nb : nb, sg[j][i]);
          const float f = gate ? tt * g[i] : tt;
          o[i] = f;
          if (post) {
            swb[j][i] = __builtin_fmaf(f, nb, swb[j][i]);
            o[i] = r1 * __builtin_fmaf(-m2, nb, f * wb[i]);
          }
        }
        if (a.db) store<DT>(a.db, r * d + at, d - at, o);
      }
    }
    if (gate) {
      const int64_t g0 = gi * a.n.gate_rows, g1 = min(g0 + a.n.gate_rows, a.n.rows);
      if (r + 1 == g1 || r + 1 == end) {
        const bool whole = g0 >= first && g1 <= end;
        if (a.dgate) {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const int at = (j * T + t) * V;
            if (whole) {
              store_vec<DT>(a.dgate, a.gf32, gi * d + at, d - at, sg[j]);
            } else {
              float* const p = a.pg + ((int64_t)unit * 2 + (g0 > first)) * d;
#pragma unroll
              for (int i = 0; i < V; ++i)
                if (at + i < d) p[at + i] = sg[j][i];
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) sg[j][i] = 0.f;
        gi += r + 1 == g1;
      }
    }
  }
  if (first >= a.n.rows) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * T + t) * V;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (at + i < d) {
        if (a.dw) a.pw[(int64_t)unit * d + at + i] = sw[j][i];
        if (a.dwb) a.pwb[(int64_t)unit * d + at + i] = swb[j][i];
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

// Units of the gradient: two rounds of workgroups at most, or the parts' sums cost as much as rows.
int rows_per_unit(const fb_norm_t* n, int cus) {
  const Split s = split_of(n->width);
  const int64_t units = (int64_t)cus * std::max(1, 512 / s.threads);
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

template <int DT, typename F>
int with_split(int width, F&& go) {
  constexpr int V = Of<DT>::V;
  const Split s = split_of(width);
  if (s.values == 8) return go(std::integral_constant<int, 64>{}, std::integral_constant<int, 8 / V>{});
  if (s.values == 32)
    return go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 32 / V>{});
  constexpr std::integral_constant<int, 16 / V> nv{};
  switch (s.threads) {
    case 64: return go(std::integral_constant<int, 64>{}, nv);
    case 128: return go(std::integral_constant<int, 128>{}, nv);
    case 256: return go(std::integral_constant<int, 256>{}, nv);
    case 512: return go(std::integral_constant<int, 512>{}, nv);
    default: return go(std::integral_constant<int, 1024>{}, nv);
  }
}

template <int DT>
int run_norm(const NormArgs& a, hipStream_t hs) {
  return with_split<DT>(a.n.width, [&](auto t, auto nv) {
    constexpr int T = decltype(t)::value, NV = decltype(nv)::value, G = kBlock<T> / T;
    const int64_t groups = (a.n.rows + G - 1) / G;
    const int64_t most = (int64_t)fb_gpu::cu_count() * (2048 / kBlock<T>);
    hipLaunchKernelGGL((norm_kernel<DT, T, NV>), dim3((unsigned)std::min(groups, most)),
                       dim3(kBlock<T>), 0, hs, a);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  });
}

template <int DT>
int run_norm_grad(const NormArgs& a, hipStream_t hs) {
  const int st = with_split<DT>(a.n.width, [&](auto t, auto nv) {
    constexpr int T = decltype(t)::value, NV = decltype(nv)::value, G = kBlock<T> / T;
    hipLaunchKernelGGL((norm_grad_kernel<DT, T, NV>), dim3((unsigned)((a.units + G - 1) / G)),
                       dim3(kBlock<T>), 0, hs, a);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  });
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
