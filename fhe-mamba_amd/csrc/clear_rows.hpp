// Rows of contiguous elements at any alignment, and sums over a wavefront, for
// the operators in the clear that work row by row.
#pragma once

#include "clear_tile.hpp"

namespace fhe::clear {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Four elements from p on as 32-bit numbers, zeros past `count`.  p needs the
// alignment of its type alone: memory takes wide accesses at any address, and
// one that crosses a line costs that line's second access.
__device__ __forceinline__ f32x4 get4(const float* p, int count) {
  f32x4 v{};
  if (count >= 4) {
    __builtin_memcpy(&v, p, 16);
    return v;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < count ? p[i] : 0.0f;
  return v;
}
__device__ __forceinline__ f32x4 get4(const bf16* p, int count) {
  if (count >= 4) {
    u32x2 u;
    __builtin_memcpy(&u, p, 8);
    return f32x4{low2(u[0]), high2(u[0]), low2(u[1]), high2(u[1])};
  }
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < count ? (float)p[i] : 0.0f;
  return v;
}

// The same in two steps, so that loads can all be on their way before the first is widened.
__device__ __forceinline__ f32x4 raw4(const float* p, int count) { return get4(p, count); }
__device__ __forceinline__ u32x2 raw4(const bf16* p, int count) {
  u32x2 u{};
  if (count >= 4) {
    __builtin_memcpy(&u, p, 8);
    return u;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) u[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << 16 * (i % 2);
  return u;
}
__device__ __forceinline__ f32x4 widen(f32x4 v) { return v; }
__device__ __forceinline__ f32x4 widen(u32x2 u) { return {low2(u[0]), high2(u[0]), low2(u[1]), high2(u[1])}; }
template <class T>
using Raw4 = decltype(raw4((const T*)nullptr, 4));

__device__ __forceinline__ void put4(float* p, f32x4 v, int count) {
  if (count >= 4) {
    __builtin_memcpy(p, &v, 16);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) p[i] = v[i];
}
__device__ __forceinline__ void put4(bf16* p, f32x4 v, int count) {
  if (count >= 4) {
    const u32x2 u{pack2(v[0], v[1]), pack2(v[2], v[3])};
    __builtin_memcpy(p, &u, 8);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) p[i] = (bf16)v[i];
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d; d /= 2) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// A row lies in the registers of W wavefronts, PER pieces of four elements a lane.  One
// wavefront as long as they hold it: it needs no barrier, and leaves no lane idle that
// more would (4096 gated norms of 1536 channels take 8 us with one, 15 with four).
constexpr int MAX_ROW = 16 * 256 * 8;
constexpr int threads_of(int w) { return w == 16 ? 1024 : 256; }
inline int rows_at_once(int channels) { return channels <= 6 * 256 ? 4 : 1; }  // of a workgroup

// How the pieces of the lanes cover a row: just so; with a last piece moved back to the
// row's end, over elements of the piece before it; or a row shorter than a piece.
enum Cover { WHOLE, MOVED, SHORT };

// A lane's piece of four elements that begins at element c.
template <int COVER>
struct Piece {
  int at;   // where it lies
  int own;  // how many of its elements are no other piece's: the last ones, or of a short row the first

  __device__ __forceinline__ Piece(int c, int channels)
      : at(COVER == MOVED ? min(c, channels - 4) : c), own(COVER == WHOLE ? 4 : max(0, min(4, channels - c))) {}
  Piece() = default;

  template <class T>
  __device__ __forceinline__ f32x4 get(const T* row) const {
    return get4(row + at, COVER == SHORT ? own : 4);
  }
  template <class T>
  __device__ __forceinline__ Raw4<T> raw(const T* row) const {
    return raw4(row + at, COVER == SHORT ? own : 4);
  }
  // A moved piece writes its neighbour's elements too: the same values from the same inputs.
  template <class T>
  __device__ __forceinline__ void put(T* row, f32x4 v) const {
    if (COVER == WHOLE || own > 0) put4(row + at, v, COVER == SHORT ? own : 4);
  }
  // v where element i is the piece's own, else 0
  __device__ __forceinline__ float mine(int i, float v) const { return COVER == MOVED && i < 4 - own ? 0.0f : v; }
};

// f(W, PER, COVER) for rows of at most MAX_ROW.
template <class F>
void by_shape(int channels, F&& f) {
  auto go = [&](auto w, auto per) {
    if (channels == 256 * w() * per()) f(w, per, std::integral_constant<int, WHOLE>{});
    else f(w, per, std::integral_constant<int, MOVED>{});
  };
  const int pieces = (channels + 255) / 256;  // of 64 lanes
  std::integral_constant<int, 1> one;
  std::integral_constant<int, 2> two;
  std::integral_constant<int, 3> three;
  std::integral_constant<int, 4> four;
  std::integral_constant<int, 6> six;
  std::integral_constant<int, 8> eight;
  std::integral_constant<int, 16> sixteen;
  if (channels < 4) f(one, one, std::integral_constant<int, SHORT>{});
  else if (pieces <= 1) go(one, one);
  else if (pieces <= 2) go(one, two);
  else if (pieces <= 3) go(one, three);
  else if (pieces <= 4) go(one, four);
  else if (pieces <= 6) go(one, six);
  else if (pieces <= 16) go(four, four);
  else if (pieces <= 32) go(four, eight);
  else if (pieces <= 64) go(sixteen, four);
  else go(sixteen, eight);
}

}  // namespace fhe::clear
