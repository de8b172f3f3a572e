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
#include "clear_logits.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

constexpr int MAX_SPLITS = 64;  // workgroups of a row

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
  x.template read<true>(row, start, a.l.vocab);
  for (int t = 0; t < a.tiles; ++t) {
    const int64_t base = start + (int64_t)t * TILE;
    if (base >= a.l.vocab) break;
    float v[16];
    x.widen(v);
    if (t + 1 < a.tiles) x.template read<true>(row, base + TILE, a.l.vocab);  // in flight meanwhile
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
    __shared__ TopLds lds;
    best_of_row(row, a.l.vocab, row_lead(row), a.keys + row_i * a.all_tiles * SETS, top, lds);
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
  x.template read<true>(row, base, a.l.vocab);
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

// Workgroups of a row: one a tile, but at most 64, and more than one only up to
// sixteen a CU in all.
int splits_of(const Logprob& l) {
  const int64_t tiles = tiles_of(l.vocab), want = std::max<int64_t>(1, 4096 / l.rows);
  return (int)std::min<int64_t>({tiles, want, MAX_SPLITS});
}

}  // namespace

size_t logprob_workspace(const Logprob& l) {
  const size_t keys = l.top ? (size_t)tiles_of(l.vocab) * SETS * sizeof(uint64_t) : 0;
  return (size_t)l.rows * (keys + splits_of(l) * sizeof(Stats));
}

void logprob(const Logprob& l, const LogprobOut& o, void* workspace, hipStream_t stream) {
  RowArgs a{l, o, splits_of(l), 0, tiles_of(l.vocab), nullptr, nullptr};
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
  BackArgs a{l, peak, log_sum, entropy, dlogprob, dentropy, dlogits, (int)tiles_of(l.vocab)};
  const uint32_t grid = (uint32_t)(l.rows * a.splits);
  if (l.dtype == BF16) k_row_back<bf16><<<grid, THREADS, 0, stream>>>(a);
  else k_row_back<float><<<grid, THREADS, 0, stream>>>(a);
  hip_check(hipGetLastError(), "log probability gradient");
}

}  // namespace fhe::clear
