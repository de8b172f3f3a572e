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

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

template <class T>
struct Num;

template <>
struct Num<bf16> {
  using Frag = bf16x8;
  static constexpr int VEC = 8;  // elements of a 16-byte access
  // Elements added to an LDS row: 16-byte rows, 16 of which start in banks
  // four apart, so that the 8-byte reads of a fragment do not conflict.
  static constexpr int PAD = 8;
  // bfloat16 pieces that a 32-bit value is split into for a product.  Two keep
  // 16 bits, which is below the rounding of a bfloat16 result; three keep 24,
  // for results in 32 bits.
  static constexpr int FINE = 3, FAIR = 2;

  // Rows l of a row-major tile, 32 columns from `p`.
  static __device__ __forceinline__ Frag rows(const bf16* p, int stride) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const bf16* at = p + l * stride + 4 * q;
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(at);
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(at + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // Columns l of a row-major tile in LDS, 32 rows from `p`: the transposing
  // read gives lane l of each sixteen column l of four rows, whose 8-byte
  // pieces its lanes address.
  static __device__ __forceinline__ Frag cols(const bf16* p, int stride) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const bf16* at = p + (4 * q + (l >> 2)) * stride + 4 * (l & 3);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))at);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(at + 16 * stride));
    return __builtin_bit_cast(Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Num<float> {
  using Frag = f32x8;
  static constexpr int VEC = 4, PAD = 4;
  static constexpr int FINE = 1, FAIR = 1;

  static __device__ __forceinline__ Frag rows(const float* p, int stride) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const float* at = p + l * stride + 4 * q;
    const f32x4 a = *reinterpret_cast<const f32x4*>(at);
    const f32x4 b = *reinterpret_cast<const f32x4*>(at + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ Frag cols(const float* p, int stride) {
    const int q = lane_id() >> 4, l = lane_id() & 15;
    const float* at = p + 4 * q * stride + l;
    Frag f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = at[j * stride];
      f[4 + j] = at[(16 + j) * stride];
    }
    return f;
  }
  // One index a lane group and instruction: the j-th takes 4 q + j.
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// A 32-bit fragment in NS pieces of T whose sum it is (to 8 NS bits).
template <class T, int NS>
struct Split {
  typename Num<T>::Frag f[NS];
};

template <class T, int NS>
__device__ __forceinline__ Split<T, NS> split(f32x8 v) {
  Split<T, NS> s;
  if constexpr (std::is_same_v<T, float>) {
    s.f[0] = v;
  } else {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s.f[n][j] = (bf16)v[j];
      if (n + 1 < NS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] -= (float)s.f[n][j];
      }
    }
  }
  return s;
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
__device__ __forceinline__ void store16(T* p, u32x4 v, int count, bool wide) {
  constexpr int VEC = Num<T>::VEC;
  if (wide && count >= VEC) {
    *reinterpret_cast<u32x4*>(p) = v;
    return;
  }
  union {
    T e[VEC];
    u32x4 v;
  } u;
  u.v = v;
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < count) p[i] = u.e[i];
}

}  // namespace fhe::clear
