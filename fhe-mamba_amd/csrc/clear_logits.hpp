// Rows of logits: reading them in tiles, and their largest entries in order.
#pragma once

#include "clear.hpp"
#include "clear_tile.hpp"

namespace fhe::clear {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 256, TILE = 16 * THREADS;  // logits of a workgroup at a time

// Sixteen logits of a thread in a tile that begins at column `base` (it may be
// negative; ALIGNED: at a multiple of 16 bytes), as they lie in memory.  -inf outside of the
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
  template <bool ALIGNED>
  __device__ __forceinline__ void read(const T* row, int64_t base, int64_t vocab) {
    if (!ALIGNED && base >= 0 && base + TILE <= vocab) {  // all pieces on their way at once
#pragma unroll
      for (int p = 0; p < PIECES; ++p) __builtin_memcpy(&w[p], row + column(base, p * VEC), 16);
      return;
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int64_t c = column(base, p * VEC);
      if (c >= 0 && c + VEC <= vocab) {
        if constexpr (ALIGNED) w[p] = *reinterpret_cast<const u32x4*>(row + c);
        else __builtin_memcpy(&w[p], row + c, 16);
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
  uint64_t maxima[THREADS], best[MAX_TOP], sets[MAX_TOP], candidate[4 * HELD * MAX_TOP + MAX_TOP];
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

// The `top` largest entries of a row, in order, to lds.best, from the largest keys
// of its sets; the first tile begins `lead` columns before the row.
template <class T>
__device__ void best_of_row(const T* row, int64_t vocab, int lead, const uint64_t* keys, int top, TopLds& lds) {
  const int64_t count = (vocab + lead + TILE - 1) / TILE * SETS;  // at most tiles_of(vocab) SETS
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
    lds.sets[threadIdx.x] = (int)threadIdx.x < top ? lds.best[threadIdx.x] : 0;
    lds.best[threadIdx.x] = 0;
  }
  __syncthreads();
  static_assert(MAX_TOP * SET <= THREADS * HELD);
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int at = j * THREADS + threadIdx.x;
    const uint64_t set = lds.sets[at / SET];
    const int64_t c = set_column<T>(key_index(set), lead, at % SET);
    key[j] = set && c >= 0 && c < vocab ? to_key(order_of((float)row[c]), (uint32_t)c) : 0;
  }
  keep_best(lds, key, top);
}

// Tiles of a row's longest reach: a row may start up to a piece before its
// first tile's end.
inline int64_t tiles_of(int64_t vocab) { return (vocab + 7 + TILE - 1) / TILE; }

}  // namespace fhe::clear
