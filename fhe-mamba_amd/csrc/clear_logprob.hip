// Log probabilities of given tokens, the entropy and the likeliest tokens of
// rows of logits, and the gradient.
//
//   s = sum e^(l - m),  u = sum e^(l - m) (l - m)  with the largest logit m
//   log p_t = (l_t - m) - log s,   H = log s - u / s
//   d l_i = a (1[i = t] - p_i) - b p_i (log p_i + H)   for gradients a, b
//
// One pass over the logits: each workgroup of a row keeps m, s and u of its
// part; a second kernel joins the parts.  Bound by memory where there are many
// rows: 4095 of 50280 in 16 bits take 102 + 7 us forward (4.0 TB/s, a plain sum's
// rate) and 141 for the gradient (5.8 TB/s, part of it from the last-level
// cache).  A row alone takes 13 us, the waits of two launches.  Entries of -inf are
// tokens that are not allowed: p = 0, and they add nothing anywhere.
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
  if (b.m > a.m || b.m != b.m) {
    const Stats t = a;
    a = b;
    b = t;
  }
  // a holds the larger maximum, or NaN if either is: that of entries of which all
  // others are masked, so that a maximum of -inf says that there is no entry
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

struct RowArgs {
  Logprob l;
  LogprobOut o;
  int splits, tiles;  // workgroups a row; tiles of each
  int64_t all_tiles;  // of a row
  Stats* stats;       // [rows][splits]
  uint64_t* keys;     // [rows][all_tiles][SETS]
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

// An entry's value as a number that orders as it, above 0; equal for the zeros.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
// Ordered by value, then by the lower index.
__device__ __forceinline__ uint64_t to_key(uint32_t order, uint32_t index) {
  return (uint64_t)order << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

template <int CTRL>
__device__ __forceinline__ uint32_t quad_swap(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}

// The likeliest entries are found in two steps.  The 64 entries that four
// neighbouring threads hold of a tile are a set, and the first kernel writes the
// largest key of each.  An entry among the `top` largest lies in one of the `top`
// sets with the largest keys: were it in another, each of these had a larger
// entry.  The second kernel picks those sets and reads only their entries again.
// Keeping the `top` best in the first kernel instead, tile by tile, takes it from
// 13.6 to 28 us for 20 of 250 rows of 50280.  In those 13.6 us the vector units work
// in 25 of a CU's 26 thousand cycles: the sets' keys and the statistics, a twentieth
// of the instructions exponentials.
constexpr int SET = 64, SETS = TILE / SET;  // entries of a set, sets of a tile

// The largest key of the set of this thread, 0 if all of it lies outside of the row.
template <class T>
__device__ __forceinline__ uint64_t set_key(const float* v, int64_t base, int64_t vocab) {
  uint32_t order[16], most = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) order[j] = order_of(v[j]);
  if (base < 0 || base + TILE > vocab) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t c = Sixteen<T>::column(base, j);
      if (c < 0 || c >= vocab) order[j] = 0;
    }
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) most = max(most, order[j]);
  most = max(most, quad_swap<0xb1>(most));  // of lanes 1, 0, 3, 2
  most = max(most, quad_swap<0x4e>(most));  // 2, 3, 0, 1
  if (!most) return 0;
  uint32_t first = 0xffffffffu;
#pragma unroll
  for (int j = 15; j >= 0; --j)
    if (order[j] == most) first = (uint32_t)Sixteen<T>::column(base, j);
  first = min(first, quad_swap<0xb1>(first));
  first = min(first, quad_swap<0x4e>(first));
  return to_key(most, first);
}

// Column of entry e of the set that holds column c.
template <class T>
__device__ __forceinline__ int64_t set_column(int64_t c, int lead, int e) {
  constexpr int RUN = 4 * Num<T>::VEC;  // a set's entries in a row
  const int64_t at = c + lead, tile = at / TILE * TILE;
  const int run = (int)(at - tile) / RUN % SETS;
  return tile - lead + (e / RUN * SETS + run) * RUN + e % RUN;
}

constexpr int HELD = 8;  // keys of a thread
struct TopLds {
  uint64_t maxima[THREADS], best[MAX_TOP], candidate[4 * HELD * MAX_TOP + MAX_TOP];
  int count;
};

// The `top` largest of the threads' keys and of the `top` that `best` holds (0:
// none), in order, to `best`.  No two of them are equal.  The threads are 64
// groups of four, one of each wavefront; the top-th largest of the groups' maxima
// bounds the keys wanted from below, and only the `top` groups at or over it can
// hold keys that large: the candidates are at most 32 top, and hardly more than top.
__device__ void keep_best(TopLds& lds, const uint64_t (&key)[HELD], int top) {
  uint64_t mine = 0;
#pragma unroll
  for (int j = 0; j < HELD; ++j) mine = max64(mine, key[j]);
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
  // fewer than `top` groups with keys: all are candidates
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
    for (int j = 0; j < HELD; ++j)
      if (key[j] && key[j] >= bound) lds.candidate[atomicAdd(&lds.count, 1)] = key[j];
  }
  if ((int)threadIdx.x < top && lds.best[threadIdx.x])
    lds.candidate[atomicAdd(&lds.count, 1)] = lds.best[threadIdx.x];
  __syncthreads();
  // their order does not depend on the order in which they came
  const int count = lds.count;
  for (int i = threadIdx.x; i < count; i += THREADS) {
    const uint64_t k = lds.candidate[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) r += lds.candidate[j] > k;
    if (r < top) lds.best[r] = k;
  }
  __syncthreads();
}

template <class T, bool TOP>
__global__ __launch_bounds__(THREADS) void k_row_parts(RowArgs a) {
  __shared__ Stats waves[THREADS / 64];
  const int64_t row_i = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  const T* row = (const T*)a.l.logits + row_i * a.l.row_stride;
  const int lead = row_lead(row);
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
    if constexpr (TOP) {
      const uint64_t key = set_key<T>(v, base, a.l.vocab);
      const int64_t tile = row_i * a.all_tiles + (int64_t)split * a.tiles + t;
      if (threadIdx.x % 4 == 0) a.keys[tile * SETS + threadIdx.x / 4] = key;
    }
  }
  st = wave_join(st);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) st = join(st, waves[w]);
    a.stats[row_i * a.splits + split] = st;
  }
}

// A workgroup a row.
template <class T, bool TOP>
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
  if constexpr (TOP) {
    const int top = a.l.top;
    const T* row = (const T*)a.l.logits + row_i * a.l.row_stride;
    const int lead = row_lead(row);
    const int64_t count = (a.l.vocab + lead + TILE - 1) / TILE * SETS;  // at most all_tiles SETS
    const uint64_t* keys = a.keys + row_i * a.all_tiles * SETS;
    __shared__ TopLds lds;
    __shared__ uint64_t sets[MAX_TOP];
    if (threadIdx.x < MAX_TOP) lds.best[threadIdx.x] = 0;
    __syncthreads();
    uint64_t key[HELD];
    for (int64_t first = 0; first < count; first += THREADS * HELD) {
#pragma unroll
      for (int j = 0; j < HELD; ++j) {
        const int64_t at = first + j * THREADS + threadIdx.x;
        key[j] = at < count ? keys[at] : 0;
      }
      keep_best(lds, key, top);
    }
    if (threadIdx.x < MAX_TOP) {
      sets[threadIdx.x] = (int)threadIdx.x < top ? lds.best[threadIdx.x] : 0;
      lds.best[threadIdx.x] = 0;
    }
    __syncthreads();
    static_assert(MAX_TOP * SET <= THREADS * HELD);
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int at = j * THREADS + threadIdx.x;
      const uint64_t set = sets[at / SET];
      const int64_t c = set_column<T>(key_index(set), lead, at % SET);
      key[j] = set && c >= 0 && c < a.l.vocab ? to_key(order_of((float)row[c]), (uint32_t)c) : 0;
    }
    keep_best(lds, key, top);
    if ((int)threadIdx.x < top) {
      const uint64_t k = lds.best[threadIdx.x];
      const float v = key_value(k);
      a.o.top_logprob[row_i * top + threadIdx.x] = (v == -INFINITY ? v : v - peak) - log_sum;
      a.o.top_index[row_i * top + threadIdx.x] = k ? (int)key_index(k) : 0;  // a row of NaN may have none
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

// Workgroups of a row: one a tile, but at most 64, and more than one only up to
// sixteen a CU in all.
int splits_of(const Logprob& l) {
  const int64_t tiles = tiles_of(l), want = std::max<int64_t>(1, 4096 / l.rows);
  return (int)std::min<int64_t>({tiles, want, MAX_SPLITS});
}

}  // namespace

size_t logprob_workspace(const Logprob& l) {
  const size_t keys = l.top ? (size_t)tiles_of(l) * SETS * sizeof(uint64_t) : 0;
  return (size_t)l.rows * (keys + splits_of(l) * sizeof(Stats));
}

void logprob(const Logprob& l, const LogprobOut& o, void* workspace, hipStream_t stream) {
  RowArgs a{l, o, splits_of(l), 0, tiles_of(l), nullptr, nullptr};
  a.tiles = (int)((a.all_tiles + a.splits - 1) / a.splits);
  a.keys = (uint64_t*)workspace;
  a.stats = (Stats*)(a.keys + (l.top ? (size_t)l.rows * a.all_tiles * SETS : 0));
  auto run = [&](auto zero) {
    using T = decltype(zero);
    const uint32_t grid = (uint32_t)(l.rows * a.splits);
    if (l.top) k_row_parts<T, true><<<grid, THREADS, 0, stream>>>(a);
    else k_row_parts<T, false><<<grid, THREADS, 0, stream>>>(a);
    hip_check(hipGetLastError(), "log probabilities");
    if (l.top) k_row_join<T, true><<<(uint32_t)l.rows, THREADS, 0, stream>>>(a);
    else k_row_join<T, false><<<(uint32_t)l.rows, THREADS, 0, stream>>>(a);
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
