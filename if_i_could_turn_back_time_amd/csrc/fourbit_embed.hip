// Embedding: rows of a table by token, scaled, and the table's gradient.
//
//   out[i] = scale W[t_i] (0 for a token outside the vocabulary)
//   grad[v] = scale sum_{i: t_i = v} g_i, for every v, those without a token too
//
// The gradient sorts the places by token (stably, so that a token's places keep their order): then a
// token's rows are a run.  Runs are summed in fp32 and in a fixed order, whatever the device does:
// kShare sorted places that lie within one run are summed by themselves first (a padding or stop token
// may have most of the batch), and the run's workgroup adds those sums and the places before and
// behind them.  The table's zeros, most of the bytes, are written beside the sort.  Up to
// kSmall places are sorted in one workgroup's LDS, 6 bits a pass; more by passes of 8 bits over memory.
// Bound by memory: the table's gradient written, and the rows read, once.
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

// Workgroup: `across` threads of a row's vectors, 256 / across rows.
template <int DT>
__global__ __launch_bounds__(256) void embed_kernel(const void* __restrict__ w, int64_t stride,
                                                    int vocab, int K,
                                                    const int64_t* __restrict__ token, int64_t rows,
                                                    float scale, void* __restrict__ out, int across) {
  constexpr int V = Of<DT>::V;
  const int x = threadIdx.x % across, y = threadIdx.x / across;
  const int at = (blockIdx.x * across + x) * V;
  if (at >= K) return;
  const int per = 256 / across;
  for (int64_t r = (int64_t)blockIdx.y * per + y; r < rows; r += (int64_t)gridDim.y * per) {
    const int64_t t = token[r];
    float v[V];
    if (t >= 0 && t < vocab) {
      load<DT>(w, t * stride + at, K - at, v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] *= scale;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = 0.f;
    }
    store<DT>(out, r * K + at, K - at, v);
  }
}

constexpr int kSmall = 16384;  // places of one workgroup's sort
constexpr int kSmallBits = 18;
constexpr int kShare = 32;     // sorted places of a sum of their own

__device__ inline unsigned key_of(int64_t t, int vocab) {
  return t >= 0 && t < vocab ? (unsigned)t : (unsigned)vocab;  // the others, together, last
}

// Lanes of the wave with the same digit as this one (of `bits` bits), of those that are `on`.
template <int BITS>
__device__ inline unsigned long long same_digit(unsigned digit, bool on) {
  unsigned long long m = __ballot(on);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const unsigned long long s = __ballot(digit >> b & 1);
    m &= digit >> b & 1 ? s : ~s;
  }
  return m;
}

// Workgroup 0 sorts up to kSmall places by token: key and place in one word.  The others clear the
// gradient, whose zeros need not wait.
__global__ __launch_bounds__(1024) void embed_sort_small(const int64_t* __restrict__ token, int rows,
                                                         int vocab, int bits,
                                                         unsigned* __restrict__ key,
                                                         unsigned* __restrict__ place,
                                                         u32x4* __restrict__ grad, int64_t units,
                                                         uint8_t* __restrict__ tail, int tail_bytes) {
  if (blockIdx.x) {
    const u32x4 zero{0, 0, 0, 0};
    const int64_t step = (int64_t)(gridDim.x - 1) * 1024;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x; i < units; i += step)
      __builtin_nontemporal_store(zero, grad + i);
    if (blockIdx.x == 1 && (int)threadIdx.x < tail_bytes) tail[threadIdx.x] = 0;
    return;
  }
  constexpr int WAVES = 16, BINS = 64;
  __shared__ unsigned item[2][kSmall];
  __shared__ unsigned count[WAVES][BINS];  // of a wave's places, then where they go
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < rows; i += 1024) item[0][i] = key_of(token[i], vocab) << 14 | (unsigned)i;
  // a wave's places: a run of whole rounds of 64, so that the order is the waves', then the rounds'
  const int rounds = ((rows + 1023) / 1024), first = wave * rounds * 64;
  int from = 0;
  for (int shift = 14; shift < 14 + bits; shift += 6) {
    for (int b = lane; b < BINS; b += 64) count[wave][b] = 0;
    __syncthreads();
    for (int i = 0; i < rounds; ++i) {
      const int at = first + i * 64 + lane;
      if (at < rows) atomicAdd(&count[wave][item[from][at] >> shift & 63], 1u);
    }
    __syncthreads();
    if (tid < BINS) {  // one wave: bins before this one, then waves before
      unsigned sum = 0;
      for (int w = 0; w < WAVES; ++w) sum += count[w][tid];
      unsigned before = sum;
      for (int s = 1; s < 64; s <<= 1) {
        const unsigned o = __shfl_up(before, s);
        if (lane >= s) before += o;
      }
      before -= sum;
      for (int w = 0; w < WAVES; ++w) {
        const unsigned c = count[w][tid];
        count[w][tid] = before;
        before += c;
      }
    }
    __syncthreads();
    for (int i = 0; i < rounds; ++i) {
      const int at = first + i * 64 + lane;
      const bool on = at < rows;
      const unsigned v = on ? item[from][at] : 0, d = v >> shift & 63;
      const unsigned long long m = same_digit<6>(d, on);
      if (on) {
        const int rank = __popcll(m & ((1ull << lane) - 1));
        const unsigned base = count[wave][d];
        item[from ^ 1][base + rank] = v;
        // the last of them moves the bin on; all have read it (the wave runs in step)
        if (rank + 1 == __popcll(m)) count[wave][d] = base + rank + 1;
      }
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    from ^= 1;
  }
  for (int i = tid; i < rows; i += 1024) {
    key[i] = item[from][i] >> 14;
    place[i] = item[from][i] & (kSmall - 1);
  }
}

// ---- more places: passes of 8 bits, kTile places a workgroup ----
constexpr int kTile = 4096, kBins = 256;

// (key, place) of the places, and the gradient cleared beside it.
__global__ __launch_bounds__(256) void embed_keys(const int64_t* __restrict__ token, int64_t rows,
                                                  int vocab, uint2* __restrict__ item,
                                                  u32x4* __restrict__ grad, int64_t units,
                                                  uint8_t* __restrict__ tail, int tail_bytes) {
  const int64_t step = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = i0; i < rows; i += step)
    item[i] = make_uint2(key_of(token[i], vocab), (unsigned)i);
  const u32x4 zero{0, 0, 0, 0};
  for (int64_t i = i0; i < units; i += step) __builtin_nontemporal_store(zero, grad + i);
  if (i0 < tail_bytes) tail[i0] = 0;
}

__global__ __launch_bounds__(256) void embed_count(const uint2* __restrict__ item, int64_t rows,
                                                   int shift, unsigned* __restrict__ count,
                                                   int tiles) {
  __shared__ unsigned bin[kBins];
  bin[threadIdx.x] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kTile;
  for (int i = threadIdx.x; i < kTile; i += 256)
    if (i0 + i < rows) atomicAdd(&bin[item[i0 + i].x >> shift & 255], 1u);
  __syncthreads();
  count[(int64_t)threadIdx.x * tiles + blockIdx.x] = bin[threadIdx.x];
}

// Sums before each of n counts, one workgroup.
__global__ __launch_bounds__(1024) void embed_scan(unsigned* __restrict__ count, int n) {
  __shared__ unsigned wave_sum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned carry = 0;
  for (int i0 = 0; i0 < n; i0 += 4096) {
    unsigned v[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = i0 + tid * 4 + j;
      v[j] = at < n ? count[at] : 0;
      sum += v[j];
    }
    unsigned run = sum;
    for (int s = 1; s < 64; s <<= 1) {
      const unsigned o = __shfl_up(run, s);
      if (lane >= s) run += o;
    }
    if (lane == 63) wave_sum[wave] = run;
    __syncthreads();
    unsigned at = carry + run - sum, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) at += wave_sum[w];
      all += wave_sum[w];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + tid * 4 + j < n) count[i0 + tid * 4 + j] = at;
      at += v[j];
    }
    carry += all;
    __syncthreads();
  }
}

__global__ __launch_bounds__(256) void embed_move(const uint2* __restrict__ item, int64_t rows,
                                                  int shift, const unsigned* __restrict__ start,
                                                  int tiles, uint2* __restrict__ to,
                                                  unsigned* __restrict__ key,
                                                  unsigned* __restrict__ place) {
  __shared__ unsigned count[4][kBins];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int w = 0; w < 4; ++w) count[w][tid] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kTile + wave * (kTile / 4);
  for (int i = lane; i < kTile / 4; i += 64)
    if (i0 + i < rows) atomicAdd(&count[wave][item[i0 + i].x >> shift & 255], 1u);
  __syncthreads();
  unsigned at = start[(int64_t)tid * tiles + blockIdx.x];
  for (int w = 0; w < 4; ++w) {
    const unsigned c = count[w][tid];
    count[w][tid] = at;
    at += c;
  }
  __syncthreads();
  for (int i = lane; i < kTile / 4; i += 64) {
    const bool on = i0 + i < rows;
    const uint2 v = on ? item[i0 + i] : make_uint2(0, 0);
    const unsigned d = v.x >> shift & 255;
    const unsigned long long m = same_digit<8>(d, on);
    if (on) {
      const int rank = __popcll(m & ((1ull << lane) - 1));
      const unsigned base = count[wave][d];
      if (key) {  // the last pass
        key[base + rank] = v.x;
        place[base + rank] = v.y;
      } else {
        to[base + rank] = v;
      }
      if (rank + 1 == __popcll(m)) count[wave][d] = base + rank + 1;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- sums over the sorted places ----
struct SumArgs {
  const unsigned *key, *place;
  const void* g;
  int64_t g_stride, rows;
  int vocab, K;
  float scale;
  float* part;  // [rows / kShare, K]
  void* grad;
};

// Adds rows from .. to - 1 of the sorted places to s, four in flight.
template <int DT>
__device__ inline void add_rows(const SumArgs& a, int64_t from, int64_t to, int at,
                                float (&s)[Of<DT>::V]) {
  constexpr int V = Of<DT>::V;
  int64_t i = from;
  for (; i + 4 <= to; i += 4) {
    float v[4][V];
#pragma unroll
    for (int j = 0; j < 4; ++j) load<DT>(a.g, (int64_t)a.place[i + j] * a.g_stride + at, a.K - at, v[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += v[j][e];
  }
  for (; i < to; ++i) {
    float v[V];
    load<DT>(a.g, (int64_t)a.place[i] * a.g_stride + at, a.K - at, v);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += v[e];
  }
}

// How many of the n <= kShare sorted places from `from` on have key k, which none before has not.
__device__ inline int run_length(const SumArgs& a, int64_t from, int64_t n, unsigned k) {
  int c = 0;
#pragma unroll
  for (int j = 0; j < kShare; ++j)
    if (j < n && from + j < a.rows) c += a.key[from + j] == k;
  return c;
}

// Shares of kShare sorted places that are one token's.
template <int DT>
__global__ __launch_bounds__(256) void embed_shares(SumArgs a, int across) {
  constexpr int V = Of<DT>::V;
  const int x = threadIdx.x % across, y = threadIdx.x / across, per = 256 / across;
  const int at = (blockIdx.x * across + x) * V;
  if (at >= a.K) return;
  const int64_t shares = a.rows / kShare;
  for (int64_t c = (int64_t)blockIdx.y * per + y; c < shares; c += (int64_t)gridDim.y * per) {
    const unsigned k = a.key[c * kShare];
    if (k == (unsigned)a.vocab || k != a.key[c * kShare + kShare - 1]) continue;
    float s[V] = {};
    add_rows<DT>(a, c * kShare, (c + 1) * kShare, at, s);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (at + e < a.K) a.part[c * a.K + at + e] = s[e];
  }
}

// The run that begins at a sorted place, if one does.
template <int DT>
__global__ __launch_bounds__(256) void embed_runs(SumArgs a, int across) {
  constexpr int V = Of<DT>::V;
  const int x = threadIdx.x % across, y = threadIdx.x / across, per = 256 / across;
  const int at = (blockIdx.x * across + x) * V;
  if (at >= a.K) return;
  for (int64_t i = (int64_t)blockIdx.y * per + y; i < a.rows; i += (int64_t)gridDim.y * per) {
    const unsigned k = a.key[i];
    if (k == (unsigned)a.vocab || (i && a.key[i - 1] == k)) continue;
    float s[V] = {};
    const int64_t share = (i + kShare - 1) / kShare;  // the first whole one
    int64_t end = i + run_length(a, i, share * kShare - i, k);
    add_rows<DT>(a, i, end, at, s);
    if (end == share * kShare) {
      int64_t c = share;
      for (; (c + 1) * kShare <= a.rows && a.key[(c + 1) * kShare - 1] == k; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (at + e < a.K) s[e] += a.part[c * a.K + at + e];
      end = c * kShare + run_length(a, c * kShare, kShare, k);
      add_rows<DT>(a, c * kShare, end, at, s);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] *= a.scale;
    store<DT>(a.grad, (int64_t)k * a.K + at, a.K - at, s);
  }
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------
constexpr int64_t kMostRows = 1ll << 30;

int elem(int32_t dtype) { return dtype == FB_DT_F32 ? 4 : 2; }

int embed_check(int32_t dtype, int64_t stride, int64_t rows, int32_t vocab, int32_t K) {
  if (dtype != FB_DT_F16 && dtype != FB_DT_BF16 && dtype != FB_DT_F32) return FB_ERR_DTYPE;
  if (rows < 0 || rows > kMostRows || vocab < 1 || vocab > (1 << 30) || K < 1 || K > (1 << 20) ||
      stride < 0)
    return FB_ERR_SHAPE;
  return FB_OK;
}

// Threads of a row: a power of two that its vectors fill, 256 at most.
int across_of(int K, int32_t dtype) {
  const int vecs = (K * elem(dtype) + 15) / 16;
  int t = 8;
  while (t < 256 && t < vecs) t *= 2;
  return t;
}
dim3 grid_of(int K, int32_t dtype, int64_t rows) {
  const int across = across_of(K, dtype), V = 16 / elem(dtype);
  const int64_t y = (rows + 256 / across - 1) / (256 / across);
  return dim3((K + across * V - 1) / (across * V), (unsigned)std::min<int64_t>(y, 65535));
}

int bits_of(int32_t vocab) {  // of the keys 0 .. vocab
  int b = 1;
  while (b < 31 && vocab >> b) ++b;
  return b;
}
bool small_sort(int64_t rows, int32_t vocab) { return rows <= kSmall && bits_of(vocab) <= kSmallBits; }

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

struct EmbedPlan {
  int tiles;
  size_t at_key, at_place, at_part, at_item[2], at_count, bytes;
};
EmbedPlan embed_plan(int64_t rows, int32_t vocab, int32_t K) {
  EmbedPlan p{};
  size_t at = 0;
  const auto take = [&](size_t n) {
    const size_t was = at;
    at += up256(n);
    return was;
  };
  p.at_key = take(rows * 4);
  p.at_place = take(rows * 4);
  p.at_part = take((size_t)(rows / kShare) * K * 4);
  if (!small_sort(rows, vocab)) {
    p.tiles = (int)((rows + kTile - 1) / kTile);
    p.at_item[0] = take(rows * 8);
    p.at_item[1] = take(rows * 8);
    p.at_count = take((size_t)p.tiles * kBins * 4);
  }
  p.bytes = at;
  return p;
}

template <int DT>
int run_sums(const SumArgs& a, int across, hipStream_t hs) {
  const int32_t dt = DT;
  if (a.rows >= kShare)
    hipLaunchKernelGGL(embed_shares<DT>, grid_of(a.K, dt, a.rows / kShare), dim3(256), 0, hs, a, across);
  hipLaunchKernelGGL(embed_runs<DT>, grid_of(a.K, dt, a.rows), dim3(256), 0, hs, a, across);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

bool off(const void* p, unsigned mask) { return reinterpret_cast<uintptr_t>(p) & mask; }

}  // namespace

extern "C" {

int fb_embed(const void* w, int64_t w_stride, int32_t dtype, int32_t vocab, int32_t K,
             const int64_t* token, int64_t rows, float scale, void* out, void* stream) {
  const int st = embed_check(dtype, w_stride, rows, vocab, K);
  if (st != FB_OK) return st;
  if (rows == 0) return FB_OK;
  if (!w || !token || !out) return FB_ERR_NULL;
  if (off(w, elem(dtype) - 1) || off(out, elem(dtype) - 1) || off(token, 7)) return FB_ERR_ALIGN;
  const int across = across_of(K, dtype);
  const dim3 grid = grid_of(K, dtype, rows);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, hs, w, w_stride, vocab, K, token, rows, scale, out,
                       across);
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  };
  return dtype == FB_DT_F16    ? go(embed_kernel<FB_DT_F16>)
         : dtype == FB_DT_BF16 ? go(embed_kernel<FB_DT_BF16>)
                               : go(embed_kernel<FB_DT_F32>);
}

size_t fb_embed_grad_workspace_bytes(int64_t rows, int32_t vocab, int32_t K) {
  if (rows < 1 || rows > kMostRows || vocab < 1 || vocab > (1 << 30) || K < 1 || K > (1 << 20)) return 0;
  return embed_plan(rows, vocab, K).bytes;
}

int fb_embed_grad(const void* g, int64_t g_stride, int32_t dtype, int32_t vocab, int32_t K,
                  const int64_t* token, int64_t rows, float scale, void* grad, void* ws,
                  size_t ws_bytes, void* stream) {
  const int st = embed_check(dtype, g_stride, rows, vocab, K);
  if (st != FB_OK) return st;
  if (!grad || (rows && (!g || !token || !ws))) return FB_ERR_NULL;
  if (off(grad, 15) || off(g, elem(dtype) - 1) || off(token, 7) || off(ws, 255)) return FB_ERR_ALIGN;
  const EmbedPlan p = embed_plan(rows, vocab, K);
  if (ws_bytes < p.bytes) return FB_ERR_WORKSPACE;
  hipStream_t hs = static_cast<hipStream_t>(stream);
  uint8_t* const w = static_cast<uint8_t*>(ws);
  const int64_t bytes = (int64_t)vocab * K * elem(dtype), units = bytes / 16;
  uint8_t* const tail = static_cast<uint8_t*>(grad) + units * 16;
  u32x4* const zeros = static_cast<u32x4*>(grad);
  unsigned* const key = reinterpret_cast<unsigned*>(w + p.at_key);
  unsigned* const place = reinterpret_cast<unsigned*>(w + p.at_place);
  const int bits = bits_of(vocab), cus = fb_gpu::cu_count();
  if (small_sort(rows, vocab)) {
    const int64_t fill = std::min<int64_t>((units + 4095) / 4096 + 1, 2 * cus);
    hipLaunchKernelGGL(embed_sort_small, dim3((unsigned)(1 + fill)), dim3(1024), 0, hs, token, (int)rows,
                       vocab, bits, key, place, zeros, units, tail, (int)(bytes & 15));
  } else {
    uint2* item[2] = {reinterpret_cast<uint2*>(w + p.at_item[0]),
                      reinterpret_cast<uint2*>(w + p.at_item[1])};
    unsigned* const count = reinterpret_cast<unsigned*>(w + p.at_count);
    hipLaunchKernelGGL(embed_keys, dim3(8 * cus), dim3(256), 0, hs, token, rows, vocab, item[0], zeros,
                       units, tail, (int)(bytes & 15));
    int from = 0;
    for (int shift = 0; shift < bits; shift += 8, from ^= 1) {
      const bool last = shift + 8 >= bits;
      hipLaunchKernelGGL(embed_count, dim3(p.tiles), dim3(256), 0, hs, item[from], rows, shift, count,
                         p.tiles);
      hipLaunchKernelGGL(embed_scan, dim3(1), dim3(1024), 0, hs, count, p.tiles * kBins);
      hipLaunchKernelGGL(embed_move, dim3(p.tiles), dim3(256), 0, hs, item[from], rows, shift, count,
                         p.tiles, item[from ^ 1], last ? key : nullptr, last ? place : nullptr);
    }
  }
  if (hipGetLastError() != hipSuccess) return FB_ERR_HIP;
  if (rows == 0) return FB_OK;
  SumArgs a{key, place, g, g_stride, rows, vocab, K, scale,
            reinterpret_cast<float*>(w + p.at_part), grad};
  const int across = across_of(K, dtype);
  return dtype == FB_DT_F16    ? run_sums<FB_DT_F16>(a, across, hs)
         : dtype == FB_DT_BF16 ? run_sums<FB_DT_BF16>(a, across, hs)
                               : run_sums<FB_DT_F32>(a, across, hs);
}

}  // extern "C"
