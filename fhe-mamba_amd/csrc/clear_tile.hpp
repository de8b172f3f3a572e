// Matrix-unit fragments of 16 x 16 tiles for the operators that run in the
// clear, in bfloat16 and in 32 bits.
//
// A wavefront's lane is (q, l) = (lane / 16, lane % 16).  An accumulator tile
// holds column l and rows 4 q + r, r = 0..3.  An operand fragment covers 32
// values of the summed index: lane (q, l) holds row (or column) l at the
// indices 4 q + j and 16 + 4 q + j, j = 0..3.  The order of the summed index is
// free as long as both operands share it, and in this one two accumulator
// tiles, one below the other, ARE the fragment of their transposed product: a
// state or a matrix of pairs goes from one product into the next without
// leaving its registers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace fhe::clear {

typedef __bf16 bf16;
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define LDS_PTR(type) __attribute__((address_space(3))) type*

// Orders LDS accesses of one wavefront's lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// No instruction is moved across: keeps the scheduler from starting a step's
// loads while the registers still hold the last one's.
__device__ __forceinline__ void step_end() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// The lane's number, of which the compiler knows nothing: what is computed from it
// is computed there, and not kept in registers through a loop around it.
__device__ __forceinline__ int lane_here() {
  int lane = lane_id();
  asm volatile("" : "+v"(lane));
  return lane;
}

template <class T>
struct Num;

template <>
struct Num<bf16> {
  using Frag = bf16x8;
  static constexpr int VEC = 8;  // elements of a 16-byte access
  // bfloat16 pieces that a 32-bit value is split into for a product: 8 bits each,
  // up to all 24.  FULL is for what ends in results of 32 bits: states, and the
  // gates' gradients.  FAIR is for what ends in bfloat16.  One piece would do for
  // sums of many terms of random sign (y of 30011 tokens 1.9e-3 off for 1.7e-3, in
  // 131 us for 149), but not where few terms cancel.
  static constexpr int FULL = 3, FAIR = 2;

  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Num<float> {
  using Frag = f32x8;
  static constexpr int VEC = 4;
  static constexpr int FULL = 1, FAIR = 1;

  // One index a lane group and instruction: the j-th takes 4 q + j.
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// A row-major tile of 64 rows and SPAN columns in LDS, and its fragments: rows()
// of 16 rows and 32 columns, whose summed index is the column, and cols() of 16
// columns and 32 rows, whose summed index is the row.
template <class T, int SPAN>
struct Tile;

// 16-byte pieces; 16 rows begin in banks four apart, so that the 8-byte reads of
// rows() do not meet.  Turning pieces by the row's number instead keeps cols()
// apart too and saves the padding, but its addresses take 20 registers more: the
// reverse value sweep of 8192 tokens took 103 us for 73, the others the same.
template <int SPAN>
struct Tile<bf16, SPAN> {
  static constexpr int PITCH = SPAN + 8;

  static __device__ __forceinline__ int at(int row, int piece) { return row * PITCH + piece * 8; }
  static __device__ __forceinline__ bf16x8 rows(const bf16* tile, int r0, int c0) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const bf16* at = tile + (r0 + l) * PITCH + c0 + 4 * q;
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(at);
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(at + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // The transposing read gives lane l of each sixteen column l of four rows,
  // whose 8-byte parts its lanes address.
  static __device__ __forceinline__ bf16x8 cols(const bf16* tile, int r0, int c0) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const bf16* at = tile + (r0 + 4 * q + (l >> 2)) * PITCH + c0 + 4 * (l & 3);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))at);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(at + 16 * PITCH));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// Rows begin four banks apart.
template <int SPAN>
struct Tile<float, SPAN> {
  static constexpr int PITCH = SPAN + 4;

  static __device__ __forceinline__ int at(int row, int piece) { return row * PITCH + piece * 4; }
  static __device__ __forceinline__ f32x8 rows(const float* tile, int r0, int c0) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const float* at = tile + (r0 + l) * PITCH + c0 + 4 * q;
    const f32x4 a = *reinterpret_cast<const f32x4*>(at);
    const f32x4 b = *reinterpret_cast<const f32x4*>(at + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ f32x8 cols(const float* tile, int r0, int c0) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const float* at = tile + (r0 + 4 * q) * PITCH + c0 + l;
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = at[j * PITCH];
      f[4 + j] = at[(16 + j) * PITCH];
    }
    return f;
  }
};

// A 32-bit fragment in NS pieces of T whose sum it is (to 8 NS bits).
template <class T, int NS>
struct Split {
  typename Num<T>::Frag f[NS];
};

// Two numbers rounded to bfloat16 in one instruction, and back.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ float low2(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float high2(uint32_t u) { return __builtin_bit_cast(float, u & 0xffff0000u); }

template <class T, int NS>
__device__ __forceinline__ Split<T, NS> split(f32x8 v) {
  Split<T, NS> s;
  if constexpr (std::is_same_v<T, float>) {
    s.f[0] = v;
  } else {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      u32x4 u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u[j] = pack2(v[2 * j], v[2 * j + 1]);
        if (n + 1 < NS) {
          v[2 * j] -= low2(u[j]);
          v[2 * j + 1] -= high2(u[j]);
        }
      }
      s.f[n] = __builtin_bit_cast(bf16x8, u);
    }
  }
  return s;
}

// A fragment as 32-bit numbers.
__device__ __forceinline__ f32x8 widen(f32x8 f) { return f; }
__device__ __forceinline__ f32x8 widen(bf16x8 f) {
  const u32x4 u = __builtin_bit_cast(u32x4, f);
  f32x8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = low2(u[j]);
    v[2 * j + 1] = high2(u[j]);
  }
  return v;
}

template <class T, int NS>
__device__ __forceinline__ f32x4 mma(const Split<T, NS>& a, typename Num<T>::Frag b, f32x4 c) {
#pragma unroll
  for (int n = NS - 1; n >= 0; --n) c = Num<T>::mma(a.f[n], b, c);
  return c;
}
template <class T, int NS>
__device__ __forceinline__ f32x4 mma(typename Num<T>::Frag a, const Split<T, NS>& b, f32x4 c) {
#pragma unroll
  for (int n = NS - 1; n >= 0; --n) c = Num<T>::mma(a, b.f[n], c);
  return c;
}

__device__ __forceinline__ f32x8 join(f32x4 a, f32x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// `count` of the elements at `p`, zeros after them, as 16 bytes.  `wide`: p is
// 16-byte aligned.  Nothing past the count is read.
template <class T>
__device__ __forceinline__ u32x4 load16(const T* p, int count, bool wide) {
  constexpr int VEC = Num<T>::VEC;
  if (wide && count >= VEC) return *reinterpret_cast<const u32x4*>(p);
  union {
    T e[VEC];
    u32x4 v;
  } u;
#pragma unroll
  for (int i = 0; i < VEC; ++i) u.e[i] = i < count ? p[i] : (T)0.0f;
  return u.v;
}

template <class T>
using Four = T __attribute__((ext_vector_type(4)));

// The same for four elements; `wide`: p is aligned to four.
template <class T>
__device__ __forceinline__ Four<T> load4(const T* p, int count, bool wide) {
  if (wide && count >= 4) return *reinterpret_cast<const Four<T>*>(p);
  Four<T> v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < count ? p[i] : (T)0.0f;
  return v;
}
template <class T>
__device__ __forceinline__ void store4(T* p, f32x4 v, int count, bool wide) {
  if (wide && count >= 4) {
    if constexpr (std::is_same_v<T, float>) {
      *reinterpret_cast<f32x4*>(p) = v;
    } else {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      *reinterpret_cast<u32x2*>(p) = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) p[i] = (T)v[i];
}

// Rows l of 16 rows of contiguous elements, `row` elements apart, as a fragment
// straight from memory: `first` the first of them, `rows` how many there are,
// `count` their elements; zeros past both.  FULL: 32 elements, aligned to 16
// bytes, and offsets of 32 bits.
template <class T, bool FULL>
__device__ __forceinline__ typename Num<T>::Frag row_frag(const T* first, int64_t row, int rows, int count,
                                                          bool wide) {
  const int q = lane_id() >> 4, l = lane_id() & 15;
  if (FULL && rows >= 16) {
    const uint32_t at = ((uint32_t)l * (uint32_t)row + 4 * q) * (uint32_t)sizeof(T);
    const T* p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(first) + at);
    const Four<T> a = *reinterpret_cast<const Four<T>*>(p), b = *reinterpret_cast<const Four<T>*>(p + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  const T* p = first + l * row + 4 * q;
  if (l >= rows) count = 0;
  const Four<T> a = load4(p, count - 4 * q, FULL || wide), b = load4(p + 16, count - 4 * q - 16, FULL || wide);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Its elements of tile `half` (0 or 1) as 32-bit numbers.
template <class Frag>
__device__ __forceinline__ f32x4 half_of(const Frag& f, int half) {
  const f32x8 v = widen(f);
  return half ? __builtin_shufflevector(v, v, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 0, 1, 2, 3);
}

}  // namespace fhe::clear
