// Log probabilities of given tokens, the entropy and the likeliest tokens of
// rows of logits, and the gradient.
//
//   s = sum e^(l - m),  u = sum e^(l - m) (l - m)  with the largest logit m
//   log p_t = (l_t - m) - log s,   H = log s - u / s
//   d l_i = a (1[i = t] - p_i) - b p_i (log p_i + H)   for gradients a, b
//
// One pass over the logits: each workgroup of a row keeps m, s and u of its
// part and its part's best entries; a second kernel joins the parts.  Bound by
// memory.  Entries of -inf are tokens that are not allowed: p = 0, and they add
// nothing anywhere.
#pragma clang fp contract(fast)
#include <algorithm>

#include "clear.hpp"
#include "clear_tile.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_SPLITS = 64;  // workgroups of a row
constexpr int THREADS = 256, TILE = 16 * THREADS;  // logits of a workgroup at a time

// Sums relative to a maximum.
struct Stats {
  float m, s, u;
};

__device__ __forceinline__ Stats join(Stats a, Stats b) {
  if (b.m > a.m) {
    const Stats t = a;
    a = b;
    b = t;
  }
  // a holds the larger maximum (or one of them is NaN, which the sums carry on)
  const float gap = b.m - a.m;
  if (b.m == -INFINITY && b.s == 0.0f) return a;
  const float f = __builtin_amdgcn_exp2f(gap * LOG2E);
  // f = 0 where b's terms are nothing beside a's; gap may be infinite then
  a.s += f * b.s;
  a.u += f == 0.0f ? 0.0f : f * (b.u + gap * b.s);
  return a;
}

__device__ __forceinline__ Stats wave_join(Stats a) {
#pragma unroll
  for (int d = 32; d; d /= 2) a = join(a, {__shfl_xor(a.m, d), __shfl_xor(a.s, d), __shfl_xor(a.u, d)});
  return a;
}

// An entry as a number that orders by value, then by the lower index.
__device__ __forceinline__ uint64_t to_key(float v, uint32_t index) {
  uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 is 0
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)b << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  uint32_t b = (uint32_t)(k >> 32);
  b = b & 0x80000000u ? b & 0x7fffffffu : ~b;
  return __builtin_bit_cast(float, b);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

struct RowArgs {
  Logprob l;
  LogprobOut o;
  int splits, tiles;  // workgroups a row; tiles of each
  Stats* stats;       // [rows][splits]
  uint64_t* best;     // [rows][splits][top]
};

// Sixteen logits of a thread in a tile that begins at column `base` (a multiple
// of 16 bytes; it may be negative), as they lie in memory.  -inf outside of the
// row.
template <class T>
struct Sixteen {
  static constexpr int VEC = Num<T>::VEC, PIECES = 16 / VEC;
  union {
    u32x4 w[PIECES];
    T e[16];
  };
  // column of element j
  static __device__ __forceinline__ int64_t column(int64_t base, int j) {
    return base + (int64_t)(j / VEC) * THREADS * VEC + threadIdx.x * VEC + j % VEC;
  }
  __device__ __forceinline__ void read(const T* row, int64_t base, int64_t vocab) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int64_t c = column(base, p * VEC);
      if (c >= 0 && c + VEC <= vocab) {
        w[p] = *reinterpret_cast<const u32x4*>(row + c);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[p * VEC + i] = c + i >= 0 && c + i < vocab ? row[c + i] : (T)-INFINITY;
      }
    }
  }
  __device__ __forceinline__ void widen(float* v) const {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = (float)e[j];
  }
};

// Elements by which a row starts after a multiple of 16 bytes.
template <class T>
__device__ __forceinline__ int row_lead(const T* row) {
  return (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
}

__device__ __forceinline__ Stats add16(Stats a, const float* v) {
  float m = a.m;
#pragma unroll
  for (int j = 0; j < 16; ++j) m = fmaxf(m, v[j]);  // passes over NaN, which the sums carry
  if (m == -INFINITY) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (v[j] != v[j]) a = {NAN, NAN, NAN};
    return a;
  }
  Stats b{m, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float d = v[j] - m, e = __builtin_amdgcn_exp2f(d * LOG2E);
    b.s += e;
    b.u += e * fmaxf(d, -1e3f);  // 0 where e is, and not 0 times infinity
  }
  return join(b, a);
}

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The `top` largest of this tile's keys and the `top` that `best` holds (0: an
// empty place), in order, to `best`.  The threads are 64 groups of four, one of
// each wavefront; the top-th largest of the groups' maxima bounds the entry wanted
// from below, and only the `top` groups at or over it can hold entries that
// large: the candidates are at most 64 top, and hardly more than top.
struct TopLds {
  uint64_t maxima[THREADS], best[MAX_TOP], candidate[64 * MAX_TOP + MAX_TOP];
  int count;
};

template <class T>
__device__ void keep_best(TopLds& lds, const float* v, int64_t base, int64_t vocab, int top) {
  uint64_t mine = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int64_t c = Sixteen<T>::column(base, j);
    if (c >= 0 && c < vocab) mine = max64(mine, to_key(v[j], (uint32_t)c));
  }
  lds.maxima[threadIdx.x] = mine;
  if (threadIdx.x == 0) lds.count = 0;
  __syncthreads();
  const int lane = lane_id();
  uint64_t group = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) group = max64(group, lds.maxima[64 * w + lane]);
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)group, i);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(group >> 32), i);
    rank += ((uint64_t)hi << 32 | lo) > group;
  }
  // fewer than `top` groups with entries: all are candidates
  const uint64_t found = __ballot(group && rank == top - 1);
  uint64_t bound = lds.best[top - 1];
  if (found) {
    const int at = __builtin_ctzll(found);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)group, at);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(group >> 32), at);
    bound = max64(bound, (uint64_t)hi << 32 | lo);
  }
  if (mine && mine >= bound) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t c = Sixteen<T>::column(base, j);
      if (c < 0 || c >= vocab) continue;
      const uint64_t k = to_key(v[j], (uint32_t)c);
      if (k >= bound) lds.candidate[atomicAdd(&lds.count, 1)] = k;
    }
  }
  if ((int)threadIdx.x < top && lds.best[threadIdx.x])
    lds.candidate[atomicAdd(&lds.count, 1)] = lds.best[threadIdx.x];
  __syncthreads();
  // their order does not depend on the order in which they came
  const int count = lds.count;
  for (int i = threadIdx.x; i < count; i += THREADS) {
    const uint64_t k = lds.candidate[i];
    int r = 0;
    for (int j = 0; j < count; ++j) r += lds.candidate[j] > k;
    if (r < top) lds.best[r] = k;
  }
  __syncthreads();
}

template <class T, bool TOP>
__global__ __launch_bounds__(THREADS) void k_row_parts(RowArgs a) {
  __shared__ Stats waves[THREADS / 64];
  __shared__ TopLds lds;
  const int64_t row_i = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  const T* row = (const T*)a.l.logits + row_i * a.l.row_stride;
  const int lead = row_lead(row);
  if constexpr (TOP) {
    if (threadIdx.x < MAX_TOP) lds.best[threadIdx.x] = 0;
    __syncthreads();
  }
  Stats st{-INFINITY, 0.0f, 0.0f};
  const int64_t start = (int64_t)split * a.tiles * TILE - lead;
  Sixteen<T> x;
  x.read(row, start, a.l.vocab);
  for (int t = 0; t < a.tiles; ++t) {
    const int64_t base = start + (int64_t)t * TILE;
    if (base >= a.l.vocab) break;
    float v[16];
    x.widen(v);
    if (t + 1 < a.tiles) x.read(row, base + TILE, a.l.vocab);  // in flight meanwhile
    st = add16(st, v);
    if constexpr (TOP) keep_best<T>(lds, v, base, a.l.vocab, a.l.top);
  }
  st = wave_join(st);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) st = join(st, waves[w]);
    a.stats[row_i * a.splits + split] = st;
  }
  if constexpr (TOP) {
    if ((int)threadIdx.x < a.l.top)
      a.best[(row_i * a.splits + split) * a.l.top + threadIdx.x] = lds.best[threadIdx.x];
  }
}

// A workgroup a row.
template <class T>
__global__ __launch_bounds__(THREADS) void k_row_join(RowArgs a) {
  __shared__ Stats waves[THREADS / 64];
  __shared__ float peak, log_sum;
  const int64_t row_i = blockIdx.x;
  Stats st{-INFINITY, 0.0f, 0.0f};
  for (int i = threadIdx.x; i < a.splits; i += THREADS) st = join(st, a.stats[row_i * a.splits + i]);
  st = wave_join(st);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) st = join(st, waves[w]);
    const bool none = st.m == -INFINITY;  // no token is allowed
    const float log_s = none ? 0.0f : logf(st.s);
    // apart, since their sum would round off what large logits differ by
    a.o.peak[row_i] = peak = st.m;
    a.o.log_sum[row_i] = log_sum = log_s;
    a.o.entropy[row_i] = none ? 0.0f : log_s - st.u / st.s;
    const int64_t t = a.l.targets ? a.l.targets[row_i] : -1;
    float lp = 0.0f;  // a target below 0 is left out
    if (t >= a.l.vocab) lp = NAN;
    else if (t >= 0) {
      const float v = (float)((const T*)a.l.logits)[row_i * a.l.row_stride + t];
      lp = none ? -INFINITY : (v - st.m) - log_s;
    }
    a.o.logprob[row_i] = lp;
  }
  if (!a.l.top) return;
  __syncthreads();
  __shared__ uint64_t best[MAX_SPLITS * MAX_TOP];
  const int count = a.splits * a.l.top;
  for (int i = threadIdx.x; i < count; i += THREADS) best[i] = a.best[row_i * count + i];
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += THREADS) {
    const uint64_t k = best[i];
    if (!k) continue;
    int r = 0;
    for (int j = 0; j < count; ++j) r += best[j] > k;
    if (r < a.l.top) {
      const float v = key_value(k);
      a.o.top_logprob[row_i * a.l.top + r] = v == -INFINITY ? -INFINITY : (v - peak) - log_sum;
      a.o.top_index[row_i * a.l.top + r] = (int)key_index(k);
    }
  }
}

struct BackArgs {
  Logprob l;
  const float *peak, *log_sum, *entropy, *dlogprob, *dentropy;
  void* out;
  int splits;
};

template <class T>
__global__ __launch_bounds__(THREADS) void k_row_back(BackArgs a) {
  constexpr int VEC = Num<T>::VEC;
  // the last rows first: the forward call read them last, and what of them is
  // still in the last-level cache is read from there
  const uint32_t block = gridDim.x - 1 - blockIdx.x;
  const int64_t row_i = block / a.splits;
  const int split = block % a.splits;
  const T* row = (const T*)a.l.logits + row_i * a.l.row_stride;
  T* out = (T*)a.out + row_i * a.l.vocab;
  const int lead = row_lead(row);
  // the gradients' rows start as the logits' do, or are written one by one
  const bool wide = row_lead(out) == lead;
  const int64_t base = (int64_t)split * TILE - lead;
  const float peak = a.peak[row_i], log_sum = a.log_sum[row_i], entropy = a.entropy[row_i];
  const int64_t t = a.l.targets ? a.l.targets[row_i] : -1;
  const float ga = t >= 0 && t < a.l.vocab && a.dlogprob ? a.dlogprob[row_i] : 0.0f;
  const float gb = a.dentropy ? a.dentropy[row_i] : 0.0f;
  const bool none = peak == -INFINITY;
  Sixteen<T> x;
  x.read(row, base, a.l.vocab);
  float v[16];
  x.widen(v);
#pragma unroll
  for (int p = 0; p < Sixteen<T>::PIECES; ++p) {
    const int64_t c = Sixteen<T>::column(base, p * VEC);
    union {
      u32x4 w;
      T e[VEC];
    } u;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float lp = (v[p * VEC + i] - peak) - log_sum, e = none ? 0.0f : __builtin_amdgcn_exp2f(lp * LOG2E);
      float d = c + i == t ? ga : 0.0f;
      d -= ga * e;
      if (e != 0.0f) d -= gb * e * (lp + entropy);
      u.e[i] = (T)(none ? 0.0f : d);
    }
    if (wide && c >= 0 && c + VEC <= a.l.vocab) {
      *reinterpret_cast<u32x4*>(out + c) = u.w;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c + i >= 0 && c + i < a.l.vocab) out[c + i] = u.e[i];
    }
  }
}

// Tiles of a row's longest reach: a row may start up to a piece before its
// first tile's end.
int64_t tiles_of(const Logprob& l) { return (l.vocab + 7 + TILE - 1) / TILE; }

// Workgroups of a row: one a tile while that is at most 64 of a row or about
// four a CU in all; the parts' best entries are joined by comparing all pairs.
int splits_of(const Logprob& l) {
  const int64_t tiles = tiles_of(l), want = std::max<int64_t>(1, 4096 / l.rows);
  return (int)std::min<int64_t>({tiles, want, MAX_SPLITS});
}

}  // namespace

size_t logprob_workspace(const Logprob& l) {
  return (size_t)l.rows * splits_of(l) * (sizeof(Stats) + 8 * (size_t)l.top) + 256;
}

void logprob(const Logprob& l, const LogprobOut& o, void* workspace, hipStream_t stream) {
  RowArgs a{l, o, splits_of(l), 0, nullptr, nullptr};
  a.tiles = (int)((tiles_of(l) + a.splits - 1) / a.splits);
  a.best = (uint64_t*)workspace;
  a.stats = (Stats*)(a.best + (size_t)l.rows * a.splits * l.top);
  auto run = [&](auto zero) {
    using T = decltype(zero);
    const uint32_t grid = (uint32_t)(l.rows * a.splits);
    if (l.top) k_row_parts<T, true><<<grid, THREADS, 0, stream>>>(a);
    else k_row_parts<T, false><<<grid, THREADS, 0, stream>>>(a);
    hip_check(hipGetLastError(), "log probabilities");
    k_row_join<T><<<(uint32_t)l.rows, THREADS, 0, stream>>>(a);
    hip_check(hipGetLastError(), "log probabilities join");
  };
  if (l.dtype == BF16) run(bf16{});
  else run(float{});
}

void logprob_backward(const Logprob& l, const float* peak, const float* log_sum, const float* entropy,
                      const float* dlogprob, const float* dentropy, void* dlogits, hipStream_t stream) {
  BackArgs a{l, peak, log_sum, entropy, dlogprob, dentropy, dlogits, (int)tiles_of(l)};
  const uint32_t grid = (uint32_t)(l.rows * a.splits);
  if (l.dtype == BF16) k_row_back<bf16><<<grid, THREADS, 0, stream>>>(a);
  else k_row_back<float><<<grid, THREADS, 0, stream>>>(a);
  hip_check(hipGetLastError(), "log probability gradient");
}

}  // namespace fhe::clear
