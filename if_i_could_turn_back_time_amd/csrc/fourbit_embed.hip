// Embedding: rows of a table by token, scaled, and the table's gradient.
//
//   out[i] = scale W[t_i] (0 for a token outside the vocabulary)
//   grad[v] = scale sum_{i: t_i = v} g_i, for every v, those without a token too
//
// The gradient sorts the places by token (stably, so that a token's places keep their order): then a
// token's rows are a run.  Runs are summed in fp32 and in a fixed order, whatever the device does:
// kShare sorted places that lie within one run are summed by themselves first (a padding or stop token
// may have most of the batch), and a long run's wave adds those sums and the places before and
// behind them.  The table's zeros, most of the bytes, are written beside the sort.  Up to
// kSmall places are sorted in one workgroup's LDS, 6 bits a pass; more by passes of 8 bits over memory.
// Bound by memory: the table's gradient written, and the rows read, once.  4096 rows of 32000 x 4096 in
// bf16: 15 us; the gradient 39 (sort and zeros, 6.7 TB/s), 21 (sums) and 11 (long runs).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fourbit.h"
#include "fourbit_rows.h"
#include "fourbit_tokens.h"

namespace fb_gpu {
__attribute__((visibility("hidden"))) int cu_count();
}  // namespace fb_gpu

namespace {

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
      load<DT>(w, t * stride, at, K - at, v);
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

// Zeros, by 256 threads of each of `groups` workgroups.  As many as there are CUs, and plain stores: 1 GiB
// in 165 us (6.5 TB/s), with 1,024 threads 188, with non-temporal stores of 512 such workgroups 225.
__device__ inline void clear(u32x4* to, int64_t units, uint8_t* tail, int tail_bytes, int group,
                             int groups) {
  if (threadIdx.x >= 256) return;
  for (int64_t i = (int64_t)group * 256 + threadIdx.x; i < units; i += (int64_t)groups * 256)
    to[i] = u32x4{0, 0, 0, 0};
  if (group == 0 && (int)threadIdx.x < tail_bytes) tail[threadIdx.x] = 0;
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
    clear(grad, units, tail, tail_bytes, blockIdx.x - 1, gridDim.x - 1);
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
  clear(grad, units, tail, tail_bytes, blockIdx.x, gridDim.x);
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
constexpr int kShare = 16;  // sorted places of a sum of their own

struct SumArgs {
  const unsigned *key, *place;
  const void* g;
  int64_t g_stride, rows;
  int vocab, K;
  float scale;
  float* part;  // [rows / kShare, K]
  void* grad;
};
constexpr int kVecs = 2;  // 16-byte pieces of a row a lane

// Adds the n rows whose places lanes l0 .. l0 + n - 1 hold to s, U in flight.
template <int DT, int U>
__device__ inline void add_rows(const SumArgs& a, unsigned place, int l0, int n, int at,
                                float (&s)[kVecs][Of<DT>::V]) {
  constexpr int V = Of<DT>::V;
  for (int i = 0; i < n; i += U) {
    u32x4 w[U][kVecs];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t r = __builtin_amdgcn_readlane((int)place, min(l0 + i + j, 63));
      if (i + j < n)
#pragma unroll
        for (int k = 0; k < kVecs; ++k)
          w[j][k] = raw<DT>(a.g, r * a.g_stride, at + k * 64 * V, a.K - at - k * 64 * V);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (i + j >= n) break;
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        float v[V];
        unpack<DT>(settled<DT>(w[j][k], at + k * 64 * V, a.K - at - k * 64 * V), v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[k][e] += v[e];
      }
    }
  }
}

// Shares of kShare sorted places that are one token's, a wave (and its columns) each.
template <int DT>
__device__ inline void token_shares(const SumArgs& a, int64_t group, int64_t groups) {
  constexpr int V = Of<DT>::V;
  const int lane = threadIdx.x & 63, at = (blockIdx.x * kVecs * 64 + lane) * V;
  const int64_t shares = a.rows / kShare;
  for (int64_t c = group * 4 + (threadIdx.x >> 6); c < shares; c += groups * 4) {
    const int64_t i = c * kShare + min(lane, kShare - 1);
    const unsigned k = a.key[i], place = a.place[i];
    const unsigned k0 = __builtin_amdgcn_readfirstlane(k);
    if (k0 == (unsigned)a.vocab || k0 != (unsigned)__builtin_amdgcn_readlane((int)k, kShare - 1)) continue;
    float s[kVecs][V] = {};
    add_rows<DT, 8>(a, place, 0, kShare, at, s);
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (at + j * 64 * V + e < a.K) a.part[c * a.K + at + j * 64 * V + e] = s[j][e];
  }
}

template <int DT>
__device__ inline void store_run(const SumArgs& a, unsigned k, int at, float (&s)[kVecs][Of<DT>::V]) {
  constexpr int V = Of<DT>::V;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
#pragma unroll
    for (int e = 0; e < V; ++e) s[j][e] *= a.scale;
    const int col = at + j * 64 * V;
    if (col < a.K) store<DT>(a.grad, (int64_t)k * a.K + col, a.K - col, s[j]);
  }
}

// The run of fewer than kLong places that begins at a sorted place, if one does, a wave (and its columns)
// each.
constexpr int kLong = 32;
template <int DT>
__device__ inline void token_runs(const SumArgs& a, int64_t group, int64_t groups) {
  constexpr int V = Of<DT>::V;
  const int lane = threadIdx.x & 63, at = (blockIdx.x * kVecs * 64 + lane) * V;
  const unsigned none = 0xFFFFFFFFu;
  for (int64_t i = group * 4 + (threadIdx.x >> 6); i < a.rows; i += groups * 4) {
    const unsigned before = i ? a.key[i - 1] : none;
    const unsigned key = i + lane < a.rows ? a.key[i + lane] : none;
    const unsigned place = i + lane < a.rows ? a.place[i + lane] : 0;
    const unsigned k = __builtin_amdgcn_readfirstlane(key);
    if (k == (unsigned)a.vocab || __builtin_amdgcn_readfirstlane(before) == k) continue;
    const unsigned long long other = __ballot(key != k || lane >= kLong);
    if (__builtin_ctzll(other) == kLong) continue;
    float s[kVecs][V] = {};
    add_rows<DT, 8>(a, place, 0, __builtin_ctzll(other), at, s);
    store_run<DT>(a, k, at, s);
  }
}

// Both in one launch: the first `shares` workgroups of a column sum shares.
template <int DT>
__global__ __launch_bounds__(256) void token_sums(SumArgs a, int shares) {
  if ((int)blockIdx.y < shares)
    token_shares<DT>(a, blockIdx.y, shares);
  else
    token_runs<DT>(a, blockIdx.y - shares, gridDim.y - shares);
}

// The longer runs, 16 waves each: every wave adds a row before the first whole share, each 16th of the
// shares and a row behind the last, and the waves' sums are joined in pairs.  A run is its first place's
// that kLong divides, of which it has one.  (By one wave, runs of 270 rows took 50 us.)
template <int DT>
__global__ __launch_bounds__(1024) void token_long_runs(SumArgs a) {
  constexpr int V = Of<DT>::V;
  __shared__ float red[8][kVecs * V][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int at = (blockIdx.x * kVecs * 64 + lane) * V;
  for (int64_t q = (int64_t)blockIdx.y * kLong; q < a.rows; q += (int64_t)gridDim.y * kLong) {
    const unsigned k = a.key[q];
    // places before q of this run, fewer than kLong where it is the run's first such place
    const unsigned long long same = __ballot(q - 1 - lane >= 0 && a.key[max(q - 1 - lane, (int64_t)0)] == k);
    const int ahead = ~same ? __builtin_ctzll(~same) : 64;
    const int64_t start = q - ahead;
    if (k == (unsigned)a.vocab || ahead >= kLong || start + kLong > a.rows ||
        a.key[start + kLong - 1] != k)
      continue;
    float s[kVecs][V] = {};
    int64_t c = (start + kShare - 1) / kShare;
    const auto row = [&](int64_t i) { add_rows<DT, 1>(a, a.place[i], 0, 1, at, s); };
    if (start + wave < c * kShare) row(start + wave);
    for (bool more = true; more;) {  // 64 shares at a time
      const int64_t last = (c + lane + 1) * kShare - 1;
      const unsigned long long end = __ballot(last >= a.rows || a.key[min(last, a.rows - 1)] != k);
      const int n = end ? __builtin_ctzll(end) : 64;
      u32x4 v[4][kVecs][V / 4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int p = 0; p < kVecs; ++p)
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            const int col = at + p * 64 * V + e;
            v[j][p][e / 4] = wave + 16 * j < n
                                 ? raw<FB_DT_F32>(a.part, (c + wave + 16 * j) * a.K, col, a.K - col)
                                 : u32x4{0, 0, 0, 0};
          }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int p = 0; p < kVecs; ++p)
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            const int col = at + p * 64 * V + e;
            float o[4];
            unpack<FB_DT_F32>(settled<FB_DT_F32>(v[j][p][e / 4], col, a.K - col), o);
#pragma unroll
            for (int m = 0; m < 4; ++m) s[p][e + m] += o[m];
          }
      c += n;
      more = n == 64;
    }
    const int64_t rest = c * kShare + wave;
    if (rest < a.rows && a.key[rest] == k) row(rest);
    for (int half = 8; half; half >>= 1) {
      if (wave >= half && wave < 2 * half)
#pragma unroll
        for (int p = 0; p < kVecs; ++p)
#pragma unroll
          for (int e = 0; e < V; ++e) red[wave - half][p * V + e][lane] = s[p][e];
      __syncthreads();
      if (wave < half)
#pragma unroll
        for (int p = 0; p < kVecs; ++p)
#pragma unroll
          for (int e = 0; e < V; ++e) s[p][e] += red[wave][p * V + e][lane];
      __syncthreads();
    }
    if (wave == 0) store_run<DT>(a, k, at, s);
  }
}

inline int elem(int32_t dtype) { return dtype == FB_DT_F32 ? 4 : 2; }

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

template <int DT>
int run_sums(const SumArgs& a, hipStream_t hs) {
  constexpr int kColumns = 64 * kVecs * Of<DT>::V;
  const unsigned x = (a.K + kColumns - 1) / kColumns;
  const auto groups = [](int64_t n, int64_t each) {
    return (int)std::min<int64_t>((n + each - 1) / each, 32767);
  };
  const bool any_long = a.rows >= kLong;
  const int shares = any_long ? groups(a.rows / kShare, 4) : 0, runs = groups(a.rows, 4);
  hipLaunchKernelGGL(token_sums<DT>, dim3(x, shares + runs), dim3(256), 0, hs, a, shares);
  if (any_long)
    hipLaunchKernelGGL(token_long_runs<DT>, dim3(x, groups(a.rows, kLong)), dim3(1024), 0, hs, a);
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------
constexpr int64_t kMostRows = 1ll << 30;

int embed_check(int32_t dtype, int64_t stride, int64_t rows, int32_t vocab, int32_t K) {
  if (dtype != FB_DT_F16 && dtype != FB_DT_BF16 && dtype != FB_DT_F32) return FB_ERR_DTYPE;
  if (rows < 0 || rows > kMostRows || vocab < 1 || vocab > (1 << 30) || K < 1 || K > (1 << 20) ||
      stride < 0)
    return FB_ERR_SHAPE;
  return FB_OK;
}

int bits_of(int32_t vocab) {  // of the keys 0 .. vocab
  int b = 1;
  while (b < 31 && vocab >> b) ++b;
  return b;
}
bool small_sort(int64_t rows, int32_t vocab) { return rows <= kSmall && bits_of(vocab) <= kSmallBits; }

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

struct SortPlan {
  int tiles;
  size_t at_item[2], at_count, bytes;
};
SortPlan sort_plan(int64_t rows, int32_t vocab) {
  SortPlan p{};
  if (small_sort(rows, vocab)) return p;
  p.tiles = (int)((rows + kTile - 1) / kTile);
  p.at_item[1] = up256(rows * 8);
  p.at_count = 2 * p.at_item[1];
  p.bytes = p.at_count + up256((size_t)p.tiles * kBins * 4);
  return p;
}

struct EmbedPlan {
  size_t at_place, at_part, at_sort, bytes;
};
EmbedPlan embed_plan(int64_t rows, int32_t vocab, int32_t K) {
  EmbedPlan p{};
  p.at_place = up256(rows * 4);
  p.at_part = 2 * p.at_place;
  p.at_sort = p.at_part + up256((size_t)(rows / kShare) * K * 4);
  p.bytes = p.at_sort + sort_plan(rows, vocab).bytes;
  return p;
}

bool off(const void* p, unsigned mask) { return reinterpret_cast<uintptr_t>(p) & mask; }

}  // namespace

size_t fb_gpu::sort_bytes(int64_t rows, int32_t vocab) { return sort_plan(rows, vocab).bytes; }

int fb_gpu::sort_tokens(const int64_t* token, int64_t rows, int32_t vocab, unsigned* key,
                        unsigned* place, void* clear, int64_t bytes, void* ws, hipStream_t hs) {
  const SortPlan p = sort_plan(rows, vocab);
  const int64_t units = bytes / 16;
  u32x4* const zeros = static_cast<u32x4*>(clear);
  uint8_t* const tail = static_cast<uint8_t*>(clear) + units * 16;
  const int bits = bits_of(vocab), cus = cu_count();
  if (small_sort(rows, vocab)) {
    const int64_t fill = std::min<int64_t>(units / 1024 + 1, cus);
    hipLaunchKernelGGL(embed_sort_small, dim3((unsigned)(1 + fill)), dim3(1024), 0, hs, token, (int)rows,
                       vocab, bits, key, place, zeros, units, tail, (int)(bytes & 15));
    return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
  }
  uint8_t* const w = static_cast<uint8_t*>(ws);
  uint2* const item[2] = {reinterpret_cast<uint2*>(w), reinterpret_cast<uint2*>(w + p.at_item[1])};
  unsigned* const count = reinterpret_cast<unsigned*>(w + p.at_count);
  hipLaunchKernelGGL(embed_keys, dim3(cus), dim3(256), 0, hs, token, rows, vocab, item[0], zeros,
                     units, tail, (int)(bytes & 15));
  int from = 0;
  for (int shift = 0; rows && shift < bits; shift += 8, from ^= 1) {
    const bool last = shift + 8 >= bits;
    hipLaunchKernelGGL(embed_count, dim3(p.tiles), dim3(256), 0, hs, item[from], rows, shift, count,
                       p.tiles);
    hipLaunchKernelGGL(embed_scan, dim3(1), dim3(1024), 0, hs, count, p.tiles * kBins);
    hipLaunchKernelGGL(embed_move, dim3(p.tiles), dim3(256), 0, hs, item[from], rows, shift, count,
                       p.tiles, item[from ^ 1], last ? key : nullptr, last ? place : nullptr);
  }
  return hipGetLastError() == hipSuccess ? FB_OK : FB_ERR_HIP;
}

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
  unsigned* const key = reinterpret_cast<unsigned*>(w);
  unsigned* const place = reinterpret_cast<unsigned*>(w + p.at_place);
  const int rc = fb_gpu::sort_tokens(token, rows, vocab, key, place, grad,
                                     (int64_t)vocab * K * elem(dtype), w + p.at_sort, hs);
  if (rc != FB_OK || rows == 0) return rc;
  SumArgs a{};
  a.key = key;
  a.place = place;
  a.g = g;
  a.g_stride = g_stride;
  a.rows = rows;
  a.vocab = vocab;
  a.K = K;
  a.scale = scale;
  a.part = reinterpret_cast<float*>(w + p.at_part);
  a.grad = grad;
  return dtype == FB_DT_F16    ? run_sums<FB_DT_F16>(a, hs)
         : dtype == FB_DT_BF16 ? run_sums<FB_DT_BF16>(a, hs)
                               : run_sums<FB_DT_F32>(a, hs);
}

}  // extern "C"
