// Log probabilities of given tokens, entropy and the likeliest alternatives of rows of logits, and
// their gradient.
//
// In base 2: with y = x log2(e) - R for a whole number R near the row's largest, z = sum 2^y and
// w = sum 2^y y come from one walk over the row:  log p_i = ln 2 (y_i - log2 z), entropy =
// ln 2 (log2 z - w / z).  Each thread has its own R, raised when a value passes it by 2^kSlack; a
// whole R is subtracted without rounding (one fma) and threads are joined by exact powers of two.
// That holds while R, itself rounded from a product, is within 8 of it: between -2^27 (where it
// starts, so that anything lower counts as 0) and 2^27.  Rows beyond are walked again relative to
// their largest value.
// The alternatives: lane l's largest value over all waves is one of 64 different values of the
// row, so the top-th largest of these 64 bounds the row's top-th largest from below.  Only threads
// whose own largest reaches the bound hold candidates (about as many as are wanted), and only
// their shares of the row, 1 KiB or so each, are read again, a wave a share; the collected
// ones are ranked by (value, lowest id).  Where more qualify than the list holds (many equal
// values), those above the bound are taken and the equal ones in the order of their ids; where
// even those above it are too many, a radix select over all 32 key bits takes their place.
// One walk bounds it: 7 to 8 VALU instructions a value, fewer cycles than its bytes take.  Measured,
// bf16: 1,024 rows of 131,072 with 20 alternatives 65 us, 4.1 TB/s; 2,048 of 32,000 38 us, 3.4
// (27 where the logits come out of the last-level cache); 16 of 32,000 with 5 8 us and of 131,072 14, a
// row's latency on one CU.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fourbit.h"

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kList = 1024;

template <int DT>
struct Type;
template <>
struct Type<FB_DT_F32> {
  using T = float;
  static constexpr int V = 4;
};
template <>
struct Type<FB_DT_F16> {
  using T = _Float16;
  static constexpr int V = 8;
};
template <>
struct Type<FB_DT_BF16> {
  using T = __bf16;
  static constexpr int V = 8;
};

// Order-preserving key of a value: NaN above all, -0 as +0.
__device__ inline unsigned key_of(float v) {
  unsigned b = __builtin_bit_cast(unsigned, v);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  if (b == 0x80000000u) b = 0;
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ inline float value_of(unsigned key) {
  if (key == 0xFFFFFFFFu) return __builtin_nanf("");
  return __builtin_bit_cast(float, key >> 31 ? key & 0x7FFFFFFFu : ~key);
}

// A row's 16-byte vectors, from its first aligned element on: vector v belongs to thread
// v % kThreads; what is left at both ends (fewer than 2 V values) goes one by one to the first
// threads.
template <int DT>
struct Row {
  using T = typename Type<DT>::T;
  static constexpr int V = Type<DT>::V;
  const T* p;
  int n, head, vecs;
  __device__ Row(const void* row, int vocab) : p(static_cast<const T*>(row)), n(vocab) {
    head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (int)sizeof(T));
    vecs = (n - head) / V;
  }
  __device__ int first(int v) const { return head + v * V; }  // id of vector v's first value
  __device__ int rest() const { return n - vecs * V; }
  __device__ int rest_id(int i) const { return i < head ? i : vecs * V + i; }
  __device__ u32x4 raw(int v) const { return *reinterpret_cast<const u32x4*>(p + first(v)); }
  __device__ static void unpack(u32x4 w, float (&x)[V]) {
    if constexpr (DT == FB_DT_F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned u = w[j];  // a bit cast of a vector's element takes the first one
        x[j] = __builtin_bit_cast(float, u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned u = w[j / 2];
        if constexpr (DT == FB_DT_F16)
          x[j] = (float)__builtin_bit_cast(_Float16, (unsigned short)(u >> (16 * (j & 1))));
        else
          x[j] = __builtin_bit_cast(float, j & 1 ? u & 0xFFFF0000u : u << 16);
      }
    }
  }
  // Calls f(id, value) for the thread's whole share.
  template <typename F>
  __device__ void walk(F&& f) const {
    for (int v = threadIdx.x; v < vecs; v += kThreads) {
      float x[V];
      unpack(raw(v), x);
#pragma unroll
      for (int j = 0; j < V; ++j) f(first(v) + j, x[j]);
    }
    if ((int)threadIdx.x < rest()) f(rest_id(threadIdx.x), (float)p[rest_id(threadIdx.x)]);
  }
};

// Largest of three, NaN passed over.  (fmaxf would first copy every value that comes from bits, for
// signalling NaNs; here such a NaN may only cost a maximum of values that a NaN outranks anyway.)
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 24.f;     // a thread's sums stay below 2^24 * its values
constexpr float kLow = -200.f;     // 2^y is 0 from here on, and y itself may be -inf
constexpr float kFar = 0x1p27f;    // of R, see above
constexpr float kHuge = 0x1p100f;  // keeps a difference of two R finite

// Sums of 2^y and 2^y y relative to R.
struct Sums {
  float R, z, w;
  __device__ void add(float y) {
    const float e = __builtin_amdgcn_exp2f(y);
    z += e;
    w = __builtin_fmaf(e, fmaxf(y, kLow), w);
  }
  __device__ void rebase(float to) {  // to >= R
    const float d = R - to, f = __builtin_amdgcn_exp2f(d);
    w = f * __builtin_fmaf(fmaxf(d, -kHuge), z, w);
    z *= f;
    R = to;
  }
};

// The wave's sum and largest value, in every lane.
template <int CTRL, int ROWS>
__device__ inline float moved(float v, float old) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
      __builtin_bit_cast(int, old), __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
}
__device__ inline float last_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ inline float wave_sum(float v) {
  v += moved<0x111, 0xF>(v, 0.f);  // row_shr:1, 2, 4, 8
  v += moved<0x112, 0xF>(v, 0.f);
  v += moved<0x114, 0xF>(v, 0.f);
  v += moved<0x118, 0xF>(v, 0.f);
  v += moved<0x142, 0xA>(v, 0.f);  // row_bcast:15, 31
  v += moved<0x143, 0xC>(v, 0.f);
  return last_lane(v);
}
__device__ inline float wave_max(float v) {
  v = fmaxf(v, moved<0x111, 0xF>(v, v));
  v = fmaxf(v, moved<0x112, 0xF>(v, v));
  v = fmaxf(v, moved<0x114, 0xF>(v, v));
  v = fmaxf(v, moved<0x118, 0xF>(v, v));
  v = fmaxf(v, moved<0x142, 0xA>(v, v));
  v = fmaxf(v, moved<0x143, 0xC>(v, v));
  return last_lane(v);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(
    const void* __restrict__ logits, int64_t stride, int vocab, const int64_t* __restrict__ token,
    int top, float* __restrict__ logprob, float* __restrict__ entropy,
    float* __restrict__ top_logprobs, int64_t* __restrict__ top_ids, float* __restrict__ stats) {
  using T = typename Type<DT>::T;
  constexpr int V = Type<DT>::V;
  __shared__ float red[kWaves][3];
  __shared__ float lane_max[kWaves][64];
  __shared__ int count, shares;
  __shared__ unsigned list_key[kList];
  __shared__ int list_id[kList];
  __shared__ int share[kThreads];
  __shared__ unsigned hist[256], chosen[2];
  __shared__ int wave_count[kWaves];
  const int64_t r = blockIdx.x;
  const Row<DT> row(static_cast<const T*>(logits) + r * stride, vocab);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inf = __builtin_inff();

  const int64_t t = token[r];  // early: read while the row is on its way
  const bool given = t >= 0 && t < vocab;
  const float at_token = given ? (float)row.p[t] : 0.f;
  float m = -inf;  // the thread's largest value
  Sums s{-kFar, 0.f, 0.f};
  const auto raise = [&](float x) {  // to a whole number near x
    const float to = fminf(__builtin_rintf(x * kLog2e), 3e38f);
    if (to > s.R + kSlack) s.rebase(to);
  };
  constexpr int U = 8;  // vectors on their way at once
  for (int v0 = tid; v0 < row.vecs; v0 += U * kThreads) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * kThreads < row.vecs) raw[u] = row.raw(v0 + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v0 + u * kThreads >= row.vecs) break;
      float x[V];
      row.unpack(raw[u], x);
      float big = max3(x[0], x[1], x[2]);
#pragma unroll
      for (int j = 3; j + 1 < V; j += 2) big = max3(big, x[j], x[j + 1]);
      big = max3(big, x[V - 1], x[V - 1]);
      m = fmaxf(m, big);
      raise(big);
#pragma unroll
      for (int j = 0; j < V; ++j) s.add(__builtin_fmaf(x[j], kLog2e, -s.R));
    }
  }
  if (tid < row.rest()) {
    const float x = (float)row.p[row.rest_id(tid)];
    m = fmaxf(m, x);
    raise(x);
    s.add(__builtin_fmaf(x, kLog2e, -s.R));
  }
  const float mine = m;
  lane_max[wave][lane] = m;
  s.rebase(wave_max(s.R));
  s.z = wave_sum(s.z);
  s.w = wave_sum(s.w);
  if (lane == 0) {
    red[wave][0] = s.R;
    red[wave][1] = s.z;
    red[wave][2] = s.w;
  }
  if (tid == 0) count = shares = 0;
  __syncthreads();
  float to = red[0][0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) to = fmaxf(to, red[i][0]);
  s = Sums{to, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    Sums o{red[i][0], red[i][1], red[i][2]};
    o.rebase(to);
    s.z += o.z;
    s.w += o.w;
  }
  // Far from 0, or nothing but -inf: relative to the largest itself, then scaled.  (The sums may be
  // NaN for being far; of a row that holds a NaN they come out so again.)
  float shift = 0.f;  // y = (x - shift) log2(e) - R
  if (!(s.z > 0.f) || __builtin_fabsf(s.R) >= kFar) {
    m = -inf;
    for (int i = 0; i < kWaves; ++i) m = fmaxf(m, lane_max[i][lane]);
    m = wave_max(m);
    if (__builtin_fabsf(m) < inf) {
      shift = m;
      s = Sums{0.f, 0.f, 0.f};
      row.walk([&](int, float x) { s.add((x - shift) * kLog2e); });
      s.z = wave_sum(s.z);
      s.w = wave_sum(s.w);
      __syncthreads();
      if (lane == 0) {
        red[wave][1] = s.z;
        red[wave][2] = s.w;
      }
      __syncthreads();
      s.z = s.w = 0.f;
      for (int i = 0; i < kWaves; ++i) {
        s.z += red[i][1];
        s.w += red[i][2];
      }
    }
  }
  if (m == inf || s.z == inf) s.z = __builtin_nanf("");  // of a logit of +inf
  const float log2z = __builtin_log2f(s.z);
  const auto logp = [&](float x) {
    const float y = __builtin_fmaf(x - shift, kLog2e, -s.R) - log2z;
    // a masked logit of the type's least value passes the range in base 2 only
    return s.z == 0.f ? -inf : y < -kHuge ? (x - shift) - kLn2 * (s.R + log2z) : kLn2 * y;
  };
  if (tid == 0) {
    logprob[r] = given ? logp(at_token) : 0.f;
    entropy[r] = s.z == 0.f ? 0.f : kLn2 * (log2z - s.w / s.z);
    if (stats) {
      stats[3 * r] = shift;
      stats[3 * r + 1] = s.z == 0.f ? 0.f : s.R;  // p = 2^-inf = 0 then
      stats[3 * r + 2] = s.z == 0.f ? 0.f : log2z;
    }
  }
  if (!top) return;

  // the bound, by every wave for itself and to 16 bits of the key: a little low costs candidates only
  unsigned least = 0;
  {
    float x = -inf;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) x = fmaxf(x, lane_max[i][lane]);
    const unsigned k = key_of(x);
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
      const unsigned more = least | 1u << bit;
      if (__popcll(__ballot(k >= more)) >= top) least = more;
    }
  }
  // NaN counts as the largest, but no maximum shows it: then every share is looked at
  const bool all = s.z != s.z;
  if (all || key_of(mine) >= least) share[atomicAdd(&shares, 1)] = tid;
  __syncthreads();
  const auto take = [&](int id, float x, unsigned from) {
    const unsigned k = key_of(x);
    if (k >= from) {
      const int at = atomicAdd(&count, 1);
      if (at < kList) {
        list_key[at] = k;
        list_id[at] = id;
      }
    }
  };
  // The shares with candidates, a wave each: what is at least `from`.
  const auto collect = [&](unsigned from) {
    for (int i = wave; i < shares; i += kWaves) {
      const int owner = share[i];
#pragma unroll 2
      for (int v = owner + lane * kThreads; v < row.vecs; v += 64 * kThreads) {
        float x[V];
        row.unpack(row.raw(v), x);
#pragma unroll
        for (int j = 0; j < V; ++j) take(row.first(v) + j, x[j], from);
      }
      if (lane == 0 && owner < row.rest())
        take(row.rest_id(owner), (float)row.p[row.rest_id(owner)], from);
    }
    __syncthreads();
  };
  collect(least);
  int found = count;
  if (found > kList) {  // many equal values, or large ones side by side
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    unsigned last = least;  // the key of which not all may be taken
    collect(last + 1);      // last is no NaN's: a bound of NaN has fewer than the list holds
    int above = count;
    __syncthreads();
    if (above >= top) {
      unsigned prefix = 0, mask = 0;
      int left = top;
      for (int b = 24; b >= 0; b -= 8) {
        for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
        __syncthreads();
        row.walk([&](int, float x) {
          const unsigned k = key_of(x);
          if ((k & mask) == prefix) atomicAdd(&hist[(k >> b) & 255u], 1u);
        });
        __syncthreads();
        if (tid == 0) {
          int d = 255;
          unsigned sum = 0;
          while (d > 0 && sum + hist[d] < (unsigned)left) sum += hist[d--];
          chosen[0] = d;
          chosen[1] = sum;
          count = 0;
        }
        __syncthreads();
        prefix |= chosen[0] << b;
        mask |= 255u << b;
        left -= (int)chosen[1];
        __syncthreads();
      }
      last = prefix;
      if (last != 0xFFFFFFFFu) collect(last + 1);  // fewer than top
      above = top - left;
    }
    int have = above;  // then equal ones in the order of their ids
    for (int i0 = 0; i0 < vocab && have < top; i0 += kThreads) {
      const int id = i0 + tid;
      const bool equal = id < vocab && key_of((float)row.p[id]) == last;
      const unsigned long long eq = __ballot(equal);
      if (lane == 0) wave_count[wave] = __popcll(eq);
      __syncthreads();
      int at = have + __popcll(eq & ((1ull << lane) - 1)), sum = 0;
      for (int i = 0; i < kWaves; ++i) {
        if (i < wave) at += wave_count[i];
        sum += wave_count[i];
      }
      if (equal && at < top) {
        list_key[at] = last;
        list_id[at] = id;
      }
      have += sum;
      __syncthreads();
    }
    __syncthreads();
    found = min(have, top);
  }
  for (int i = tid; i < found; i += kThreads) {
    const unsigned k = list_key[i];
    const int id = list_id[i];
    int better = 0;
#pragma unroll 4
    for (int j = 0; j < found; ++j)
      better += list_key[j] > k || (list_key[j] == k && list_id[j] < id);
    if (better < top) {
      top_ids[r * top + better] = id;
      top_logprobs[r * top + better] = logp(value_of(k));
    }
  }
}

// ---------------------------------------------------------------------------------
// The gradient: elementwise but for the given token and the alternatives, which the thread that
// holds them adds.  Workgroup = (a run of a row's values, row).  Bound by memory, one read and one
// write: 2,048 rows of 32,000, bf16, 41 us, 6.4 TB/s (the logits come out of the last-level cache).
// With alternatives by their list, which every value is compared with: 1 alternative 4 us more, 5
// alternatives 62, 20 alternatives 312.
// ---------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(
    const void* __restrict__ logits, int64_t stride, int vocab, int span,
    const int64_t* __restrict__ token, int top, const int64_t* __restrict__ top_ids,
    const float* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ g_logprob, const float* __restrict__ g_entropy,
    const float* __restrict__ g_top, void* __restrict__ grad, int64_t rows) {
  using T = typename Type<DT>::T;
  constexpr int V = Type<DT>::V;
  const int tid = threadIdx.x;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const T* const row = static_cast<const T*>(logits) + r * stride;
    T* const out = static_cast<T*>(grad) + r * vocab;
    const float shift = stats[3 * r], R = stats[3 * r + 1], log2z = stats[3 * r + 2];
    const int64_t t = token ? token[r] : -1;
    const float g = g_logprob && t >= 0 && t < vocab ? g_logprob[r] : 0.f;
    const float ge = g_entropy ? g_entropy[r] : 0.f;
    float all = g + (g_entropy ? ge * entropy[r] : 0.f);
    if (g_top)
      for (int j = 0; j < top; ++j) all += g_top[r * top + j];
    all = -__builtin_fmaf(0.f, log2z, all);  // NaN throughout where the row has one
    const float slope = -ge * kLn2;
    const auto one = [&](int i, float x) {
      const float y = __builtin_fmaf(x - shift, kLog2e, -R) - log2z;
      const float p = __builtin_amdgcn_exp2f(y);
      float v = p * __builtin_fmaf(slope, fmaxf(y, kLow), all);
      if (i == t) v += g;
      return v;
    };
    const auto with_top = [&](int i, float v) {
      if (g_top)
        for (int j = 0; j < top; ++j)
          if (top_ids[r * top + j] == i) v += g_top[r * top + j];
      return v;
    };
    const int i0 = blockIdx.x * span, i1 = min(vocab, i0 + span);
    const bool vec = !((reinterpret_cast<uintptr_t>(row + i0) |
                        reinterpret_cast<uintptr_t>(out + i0)) & 15u);
    if (vec) {
      for (int i = i0 + tid * V; i + V <= i1; i += 256 * V) {
        float v[V];
        Row<DT>::unpack(*reinterpret_cast<const u32x4*>(row + i), v);
        T o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (T)with_top(i + j, one(i + j, v[j]));
        u32x4 w;
        __builtin_memcpy(&w, o, 16);
        *reinterpret_cast<u32x4*>(out + i) = w;
      }
      for (int i = i0 + (i1 - i0) / V * V + tid; i < i1; i += 256)
        out[i] = (T)with_top(i, one(i, (float)row[i]));
    } else {
      for (int i = i0 + tid; i < i1; i += 256) out[i] = (T)with_top(i, one(i, (float)row[i]));
    }
  }
}

bool known(int32_t dtype) {
  return dtype == FB_DT_F16 || dtype == FB_DT_BF16 || dtype == FB_DT_F32;
}

int check_logits(const void* logits, int32_t dtype, int64_t stride, int64_t rows, int32_t vocab,
                 int32_t top) {
  if (!known(dtype)) return FB_ERR_DTYPE;
  if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > (1 << 30) || top < 0 ||
      top > FB_LOGPROBS_TOP_MAX || top > vocab || stride < 0)
    return FB_ERR_SHAPE;
  if (rows && !logits) return FB_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == FB_DT_F32 ? 3u : 1u)) return FB_ERR_ALIGN;
  return FB_OK;
}

bool misaligned(std::initializer_list<const void*> ps, unsigned mask) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & mask) return true;
  return false;
}

}  // namespace

extern "C" {

int fb_token_logprobs(const void* logits, int32_t dtype, int64_t stride, int64_t rows,
                      int32_t vocab, const int64_t* token, int32_t top, float* logprob,
                      float* entropy, float* top_logprobs, int64_t* top_ids, float* stats,
                      void* stream) {
  const int st = check_logits(logits, dtype, stride, rows, vocab, top);
  if (st != FB_OK) return st;
  if (rows == 0) return FB_OK;
  if (!token || !logprob || !entropy || (top && (!top_logprobs || !top_ids))) return FB_ERR_NULL;
  if (misaligned({logprob, entropy, top_logprobs, stats}, 3) || misaligned({token, top_ids}, 7))
    return FB_ERR_ALIGN;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const int64_t row_bytes = stride * (dtype == FB_DT_F32 ? 4 : 2);
  const auto go = [&](auto kernel) {
    // a grid has fewer than 2^32 threads in a direction: beyond that rows would go missing
    constexpr int64_t kMost = 1 << 22;
    for (int64_t r = 0; r < rows; r += kMost) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(rows - r, kMost)), dim3(kThreads), 0, hs,
                         static_cast<const char*>(logits) + r * row_bytes, stride, vocab, token + r,
                         top, logprob + r, entropy + r, top ? top_logprobs + r * top : nullptr,
                         top ? top_ids + r * top : nullptr, stats ? stats + 3 * r : nullptr);
      if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
    }
    return FB_OK;
  };
  return dtype == FB_DT_F16    ? go(logprobs_kernel<FB_DT_F16>)
         : dtype == FB_DT_BF16 ? go(logprobs_kernel<FB_DT_BF16>)
                               : go(logprobs_kernel<FB_DT_F32>);
}

int fb_token_logprobs_grad(const void* logits, int32_t dtype, int64_t stride, int64_t rows,
                           int32_t vocab, const int64_t* token, int32_t top,
                           const int64_t* top_ids, const float* stats, const float* entropy,
                           const float* g_logprob, const float* g_entropy, const float* g_top,
                           void* grad, void* stream) {
  const int st = check_logits(logits, dtype, stride, rows, vocab, top);
  if (st != FB_OK) return st;
  if (rows == 0) return FB_OK;
  if (!token || !stats || !grad || (g_entropy && !entropy) || (g_top && (!top_ids || !top)))
    return FB_ERR_NULL;
  if (misaligned({stats, entropy, g_logprob, g_entropy, g_top}, 3) ||
      misaligned({token, top_ids}, 7) || misaligned({grad}, dtype == FB_DT_F32 ? 3 : 1))
    return FB_ERR_ALIGN;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const int span = 8192;
  const dim3 grid((vocab + span - 1) / span, (unsigned)std::min<int64_t>(rows, 65535));
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, hs, logits, stride, vocab, span, token, top,
                       top_ids, stats, entropy, g_logprob, g_entropy, g_top, grad, rows);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  };
  return dtype == FB_DT_F16    ? go(logprobs_grad_kernel<FB_DT_F16>)
         : dtype == FB_DT_BF16 ? go(logprobs_grad_kernel<FB_DT_BF16>)
                               : go(logprobs_grad_kernel<FB_DT_F32>);
}

}  // extern "C"
