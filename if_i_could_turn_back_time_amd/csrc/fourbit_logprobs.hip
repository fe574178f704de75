// Log probabilities of given tokens, entropy and the likeliest alternatives of rows of logits, and
// their gradient.
//
// With m the largest logit, Z = sum exp(x - m) and W = sum exp(x - m) (x - m) come from one walk
// over the row with a running maximum:  log p_i = x_i - m - log Z,  entropy = log Z - W / Z.
// The alternatives: lane l's largest value over all waves is one of 64 different values of the
// row, so the top-th largest of these 64 bounds the row's top-th largest from below.  A second
// walk collects what is not below the bound (about as many as are wanted, plus ties), and the
// collected ones are ranked by (value, lowest id).  Where more qualify than the list holds (many
// equal values), a radix select over all 32 key bits and a walk in id order take its place.
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

template <int DT>
__device__ inline void load_vec(const void* row, int i, float* v) {
  using T = typename Type<DT>::T;
  const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const T*>(row) + i);
  if constexpr (DT == FB_DT_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned u = w[j];  // a bit cast of a vector's element takes the first one
      v[j] = __builtin_bit_cast(float, u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned short u = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
      v[j] = DT == FB_DT_F16 ? (float)__builtin_bit_cast(_Float16, u)
                             : __builtin_bit_cast(float, (unsigned)u << 16);
    }
  }
}

// Calls f(id, value) for the thread's share of a row; 16 bytes at a time where the row allows it.
// The first `head` elements (up to the first aligned one) and the tail go one by one.
template <int DT, typename F>
__device__ inline void walk(const void* row, int n, F&& f) {
  using T = typename Type<DT>::T;
  constexpr int V = Type<DT>::V;
  const int tid = threadIdx.x;
  const int head =
      min(n, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (int)sizeof(T));
  const int body = (n - head) / V * V;
  float v[V];
  for (int i = tid * V; i < body; i += kThreads * V) {
    load_vec<DT>(static_cast<const T*>(row) + head, i, v);
#pragma unroll
    for (int j = 0; j < V; ++j) f(head + i + j, v[j]);
  }
  const int rest = n - body;  // head and tail, fewer than 2 V
  if (tid < rest) {
    const int i = tid < head ? tid : body + tid;
    f(i, (float)static_cast<const T*>(row)[i]);
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(
    const void* __restrict__ logits, int64_t stride, int vocab, const int64_t* __restrict__ token,
    int top, float* __restrict__ logprob, float* __restrict__ entropy,
    float* __restrict__ top_logprobs, int64_t* __restrict__ top_ids, float* __restrict__ stats) {
  using T = typename Type<DT>::T;
  __shared__ float red[kWaves][3];
  __shared__ float lane_max[kWaves][64];
  __shared__ unsigned bound;
  __shared__ int count;
  __shared__ unsigned list_key[kList];
  __shared__ int list_id[kList];
  __shared__ unsigned hist[256], chosen[2];
  __shared__ int wave_count[2][kWaves];
  const int64_t r = blockIdx.x;
  const T* const row = static_cast<const T*>(logits) + r * stride;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float inf = __builtin_inff();

  float m = -inf, z = 0.f, w = 0.f;
  const auto merge = [&](float om, float oz, float ow) {
    const float big = fmaxf(m, om);
    const float base = big == -inf ? 0.f : big;
    const float a = __expf(m - base), b = __expf(om - base);
    // (m - base) z: 0 where nothing is there yet
    w = a * (w + (z == 0.f ? 0.f : (m - base) * z)) + b * (ow + (oz == 0.f ? 0.f : (om - base) * oz));
    z = a * z + b * oz;
    m = big;
  };
  walk<DT>(row, vocab, [&](int, float x) {
    if (x > m) {
      const float a = m == -inf ? 0.f : __expf(m - x);
      w = a * (w + (z == 0.f ? 0.f : (m - x) * z));
      z *= a;
      m = x;
    }
    const float d = x - (m == -inf ? 0.f : m);
    const float e = __expf(d);
    z += e;
    w += d == -inf ? 0.f : e * d;
  });
  lane_max[wave][lane] = m;
  for (int o = 32; o; o >>= 1) {
    const float om = __shfl_xor(m, o), oz = __shfl_xor(z, o), ow = __shfl_xor(w, o);
    merge(om, oz, ow);
  }
  if (lane == 0) {
    red[wave][0] = m;
    red[wave][1] = z;
    red[wave][2] = w;
  }
  if (tid == 0) count = 0;
  __syncthreads();
  m = red[0][0];
  z = red[0][1];
  w = red[0][2];
  for (int i = 1; i < kWaves; ++i) merge(red[i][0], red[i][1], red[i][2]);
  const float base = m == -inf ? 0.f : m;
  const float logz = logf(z);
  if (tid == 0) {
    const int64_t t = token ? token[r] : -1;
    if (logprob)
      logprob[r] = t >= 0 && t < vocab ? (z == 0.f ? -inf : ((float)row[t] - base) - logz) : 0.f;
    if (entropy) entropy[r] = z == 0.f ? 0.f : logz - w / z;
    if (stats) {
      stats[2 * r] = base;
      stats[2 * r + 1] = z == 0.f ? 0.f : logz;  // p = exp(-inf) = 0 then
    }
  }
  if (!top) return;

  if (wave == 0) {
    float x = -inf;
    for (int i = 0; i < kWaves; ++i) x = fmaxf(x, lane_max[i][lane]);
    const unsigned k = key_of(x);
    int better = 0;  // lanes with a larger value, or an equal one and a lower number
    for (int i = 0; i < 64; ++i) {
      const unsigned o = (unsigned)__builtin_amdgcn_readlane((int)k, i);
      better += o > k || (o == k && i < lane);
    }
    if (better == top - 1) bound = k;
  }
  __syncthreads();
  const unsigned least = bound;
  walk<DT>(row, vocab, [&](int id, float x) {
    const unsigned k = key_of(x);
    if (k >= least) {
      const int at = atomicAdd(&count, 1);
      if (at < kList) {
        list_key[at] = k;
        list_id[at] = id;
      }
    }
  });
  __syncthreads();
  int found = count;
  if (found > kList) {
    unsigned prefix = 0, mask = 0;
    int left = top, above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
      __syncthreads();
      walk<DT>(row, vocab, [&](int, float x) {
        const unsigned k = key_of(x);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
      });
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
    if (tid == 0) count = 0;
    __syncthreads();
    walk<DT>(row, vocab, [&](int id, float x) {  // fewer than top
      const unsigned k = key_of(x);
      if (k > prefix) {
        const int at = atomicAdd(&count, 1);
        list_key[at] = k;
        list_id[at] = id;
      }
    });
    int have = above;  // then the first `left` equal ones in id order
    for (int i0 = 0; i0 < vocab && have < top; i0 += kThreads) {
      const int id = i0 + tid;
      const bool equal = id < vocab && key_of((float)row[id]) == prefix;
      const unsigned long long eq = __ballot(equal);
      if (lane == 0) wave_count[0][wave] = __popcll(eq);
      __syncthreads();
      int at = have + __popcll(eq & ((1ull << lane) - 1)), all = 0;
      for (int i = 0; i < kWaves; ++i) {
        if (i < wave) at += wave_count[0][i];
        all += wave_count[0][i];
      }
      if (equal && at < top) {
        list_key[at] = prefix;
        list_id[at] = id;
      }
      have += all;
      __syncthreads();
    }
    __syncthreads();
    found = top;
  }
  for (int i = tid; i < found; i += kThreads) {
    const unsigned k = list_key[i];
    const int id = list_id[i];
    int better = 0;
    for (int j = 0; j < found; ++j) better += list_key[j] > k || (list_key[j] == k && list_id[j] < id);
    if (better < top) {
      top_ids[r * top + better] = id;
      top_logprobs[r * top + better] =
          z == 0.f ? -inf : ((float)row[id] - base) - logz;
    }
  }
}

// ---------------------------------------------------------------------------------
// The gradient: elementwise but for the given token and the alternatives, which the thread that
// holds them adds.  Workgroup = (a run of a row's values, row).
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
    const float base = stats[2 * r], logz = stats[2 * r + 1];
    const int64_t t = token ? token[r] : -1;
    const float g = g_logprob && t >= 0 && t < vocab ? g_logprob[r] : 0.f;
    const float ge = g_entropy ? g_entropy[r] : 0.f, H = g_entropy ? entropy[r] : 0.f;
    float all = g;
    if (g_top)
      for (int j = 0; j < top; ++j) all += g_top[r * top + j];
    const auto one = [&](int i, float x) {
      const float lp = (x - base) - logz;
      const float p = __expf(lp);
      float v = p == 0.f ? 0.f : -p * (all + ge * (lp + H));
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
        load_vec<DT>(row, i, v);
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
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(kThreads), 0, hs, logits, stride, vocab,
                       token, top, logprob, entropy, top_logprobs, top_ids, stats);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
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
