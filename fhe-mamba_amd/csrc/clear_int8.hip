// Matrix product in 8-bit integers:
//   a_m = max_k |x_mk| / 127,   q_mk = the integer nearest to x_mk / a_m
//   y_mn = a_m b_n sum_k q_mk W_nk + bias_n
// The sums are of 32-bit integers and exact.  The quotient is rounded to 32 bits
// before it is rounded to an integer (even among equals), so that q is the same
// on any machine with IEEE division.  Few rows are bound by the weights' bytes,
// many by the bytes of y and the matrix units.
//
// Both operands lie with the summed index contiguous, as the matrix instruction
// (16 x 16, 64 indices) takes them: lane (q, l) holds 16 bytes of row l from
// index 16 q on.  The weights are its first operand, so that a lane ends with
// four neighbouring outputs of one row of y.
#pragma clang fp contract(fast)
#include <algorithm>

#include "clear.hpp"
#include "clear_rows.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int STEP = 128;  // bytes of a row at a time; rows of q are whole steps, zeros behind the inputs

int64_t pitch_of(int64_t inputs) { return (inputs + STEP - 1) / STEP * STEP; }

// ----------------------------------------------------------------- rounding rows
template <class T, int W, int PER>
__global__ __launch_bounds__(threads_of(W)) void k_quantize(const T* x, int64_t x_row, int64_t rows, int channels,
                                                            int8_t* q, int64_t pitch, float* scales) {
  constexpr int LANES = 64 * W, ROWS = threads_of(W) / LANES;
  __shared__ uint32_t lds[W];
  const int lane = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (row >= rows) return;  // with W > 1 a workgroup has one row
  x += row * x_row;
  q += row * pitch;
  f32x4 v[PER];
  uint32_t most = 0;  // |x| as a number orders as its bits do, infinity and NaN above all
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = (k * LANES + lane) * 4;
    v[k] = get4(x + c, channels - c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = v[k][i];  // a cast of the vector's element itself takes its first
      most = max(most, __builtin_bit_cast(uint32_t, e) & 0x7fffffffu);
    }
  }
#pragma unroll
  for (int d = 32; d; d /= 2) most = max(most, (uint32_t)__shfl_xor((int)most, d));
  if constexpr (W > 1) {
    if (lane_id() == 0) lds[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) most = max(most, lds[w]);
  }
  const bool finite = most < 0x7f800000u;
  const float scale = finite ? __builtin_bit_cast(float, most) / 127.0f : NAN;
  const bool some = finite && scale > 0.0f;
  if (lane == 0) scales[row] = scale;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = (k * LANES + lane) * 4;
    if (c >= pitch) continue;
    uint32_t bytes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = some ? fminf(fmaxf(rintf(v[k][i] / scale), -127.0f), 127.0f) : 0.0f;
      bytes |= (uint32_t)((int)r & 255) << 8 * i;
    }
    if (c + 4 <= pitch) {
      __builtin_memcpy(q + c, &bytes, 4);
    } else {
      for (int i = c; i < pitch; ++i) q[i] = (int8_t)(bytes >> 8 * (i - c));
    }
  }
}

void quantize(const Quantize& z, int8_t* values, int64_t pitch, float* scale, hipStream_t stream) {
  if (!z.rows) return;
  auto run = [&](auto zero) {
    using T = decltype(zero);
    by_shape((int)pitch, [&](auto w, auto per, auto) {
      const int at = threads_of(w()) / (64 * w());
      k_quantize<T, w(), per()><<<(uint32_t)((z.rows + at - 1) / at), threads_of(w()), 0, stream>>>(
          (const T*)z.x.p, z.x.row, z.rows, z.channels, values, pitch, scale);
    });
  };
  if (z.dtype == BF16) run(bf16{});
  else run(float{});
  hip_check(hipGetLastError(), "rounding of rows");
}

// ----------------------------------------------------------------- products
struct ProductArgs {
  const int8_t* q;        // [rows][pitch]
  const float* row_scale;
  int64_t pitch, rows;
  const int8_t* weight;   // [outputs][inputs]
  const float *scale, *bias;
  int inputs, outputs;
  void* y;                // [rows][outputs]
  int row_tiles, out_tiles;
};

// 16 bytes of a weight's row from k on.  Where q is zero, any bytes of the table do.
template <bool WIDE>
__device__ __forceinline__ i32x4 weight16(const int8_t* row, int k, int inputs) {
  if constexpr (WIDE) {
    return *reinterpret_cast<const i32x4*>(row + (k < inputs ? k : 0));
  } else {
    i32x4 v{};
    if (k + 16 <= inputs) {
      __builtin_memcpy(&v, row + k, 16);
    } else {
      uint32_t u[4] = {};
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k + i < inputs) u[i / 4] |= (uint32_t)(uint8_t)row[k + i] << 8 * (i % 4);
      v = i32x4{(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
    }
    return v;
  }
}

// Four neighbouring outputs of a row.
template <class O>
__device__ __forceinline__ void put_outputs(const ProductArgs& p, int64_t m, int n, i32x4 sum) {
  const int count = p.outputs - n;
  if (m >= p.rows || count <= 0) return;
  const float a = p.row_scale[m];
  const f32x4 b = get4(p.scale + n, count);
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)sum[i] * (a * b[i]);
  if (p.bias) v += get4(p.bias + n, count);
  put4((O*)p.y + m * p.outputs + n, v, count);
}

// Few rows: a workgroup has 16 outputs and MT times 16 rows, its four wavefronts
// a part of the summed index each; operands straight from memory.
template <class O, int MT, bool WIDE>
__global__ __launch_bounds__(256) void k_few(ProductArgs p) {
  __shared__ i32x4 lds[3][MT][64];
  const int wave = threadIdx.x >> 6, lane = lane_id(), q = lane >> 4, l = lane & 15;
  const int n0 = (blockIdx.x / p.row_tiles) * 16;
  const int64_t m0 = (int64_t)(blockIdx.x % p.row_tiles) * 16 * MT;
  const int8_t* w = p.weight + (int64_t)min(n0 + l, p.outputs - 1) * p.inputs;
  const int8_t* x[MT];
  i32x4 sum[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    x[i] = p.q + min(m0 + 16 * i + l, p.rows - 1) * p.pitch + 16 * q;
    sum[i] = i32x4{};
  }
  for (int k = 64 * wave; k < p.inputs; k += 256) {
    const i32x4 a = weight16<WIDE>(w, k + 16 * q, p.inputs);
#pragma unroll
    for (int i = 0; i < MT; ++i)
      sum[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *reinterpret_cast<const i32x4*>(x[i] + k), sum[i], 0, 0, 0);
  }
  if (wave) {
#pragma unroll
    for (int i = 0; i < MT; ++i) lds[wave - 1][i][lane] = sum[i];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int o = 0; o < 3; ++o) sum[i] += lds[o][i][lane];
    put_outputs<O>(p, m0 + 16 * i + l, n0 + 4 * q, sum[i]);
  }
}

// Many rows: tiles of 128 rows and 128 outputs, 64 x 64 a wavefront.  A row of a
// tile in LDS is 128 bytes in 16-byte pieces, whose place is turned by a number
// that differs between the rows that eight neighbouring lanes read.
constexpr int TILE = 128;

__device__ __forceinline__ int turn_of_row(int row) { return row & 7; }
__device__ __forceinline__ int turn_of_out(int row) { return (row & 3) | (row >> 2 & 4); }

template <class O, bool WIDE>
__global__ __launch_bounds__(256) void k_many(ProductArgs p) {
  __shared__ int8_t rows[TILE * STEP], outs[TILE * STEP];
  const int wave = threadIdx.x >> 6, lane = lane_id(), q = lane >> 4, l = lane & 15;
  const int64_t m0 = (int64_t)(blockIdx.x / p.out_tiles) * TILE;
  const int n0 = (blockIdx.x % p.out_tiles) * TILE;
  const int wm = wave >> 1, wn = wave & 1;
  i32x4 sum[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = i32x4{};
  // piece `part` of row threadIdx.x / 8 + 32 j
  const int part = threadIdx.x & 7, at = threadIdx.x >> 3;
  i32x4 x[4], w[4];
  auto load = [&](int k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = at + 32 * j;
      x[j] = *reinterpret_cast<const i32x4*>(p.q + min(m0 + r, p.rows - 1) * p.pitch + k + 16 * part);
      w[j] = weight16<WIDE>(p.weight + (int64_t)min(n0 + r, p.outputs - 1) * p.inputs, k + 16 * part, p.inputs);
    }
  };
  load(0);
  for (int k = 0; k < p.inputs; k += STEP) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = at + 32 * j;
      *reinterpret_cast<i32x4*>(rows + r * STEP + 16 * (part ^ turn_of_row(r))) = x[j];
      *reinterpret_cast<i32x4*>(outs + r * STEP + 16 * (part ^ turn_of_out(r))) = w[j];
    }
    __syncthreads();
    if (k + STEP < p.inputs) load(k + STEP);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      i32x4 a[4], b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = wm * 64 + 16 * j + l, n = wn * 64 + 16 * (l >> 2) + 4 * j + (l & 3);
        b[j] = *reinterpret_cast<const i32x4*>(rows + r * STEP + 16 * ((4 * s + q) ^ turn_of_row(r)));
        a[j] = *reinterpret_cast<const i32x4*>(outs + n * STEP + 16 * ((4 * s + q) ^ turn_of_out(n)));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], b[i], sum[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      put_outputs<O>(p, m0 + wm * 64 + 16 * i + l, n0 + wn * 64 + 16 * q + 4 * j, sum[i][j]);
}

constexpr int FEW = 64;  // rows

}  // namespace

void quantize_rows(const Quantize& z, int8_t* values, float* scale, hipStream_t stream) {
  quantize(z, values, z.channels, scale, stream);
}

size_t int8_workspace(const Int8& p) { return (size_t)p.rows * (pitch_of(p.inputs) + sizeof(float)); }

void int8_linear(const Int8& p, void* y, void* workspace, hipStream_t stream) {
  if (!p.rows) return;
  ProductArgs a{};
  a.pitch = pitch_of(p.inputs);
  int8_t* q = (int8_t*)workspace;
  float* row_scale = (float*)(q + p.rows * a.pitch);
  quantize({p.dtype, p.rows, p.inputs, p.x}, q, a.pitch, row_scale, stream);
  a.q = q;
  a.row_scale = row_scale;
  a.rows = p.rows;
  a.weight = p.weight;
  a.scale = p.scale;
  a.bias = p.bias;
  a.inputs = p.inputs;
  a.outputs = p.outputs;
  a.y = y;
  const bool wide = p.inputs % 16 == 0 && reinterpret_cast<uintptr_t>(p.weight) % 16 == 0;
  const bool few = p.rows <= FEW || (int64_t)p.rows * p.outputs < 256 * TILE * TILE;
  auto run = [&](auto zero, auto wide) {
    using O = decltype(zero);
    if (few) {
      auto go = [&](auto mt) {
        a.row_tiles = (int)((p.rows + 16 * mt() - 1) / (16 * mt()));
        const int64_t grid = (int64_t)a.row_tiles * ((p.outputs + 15) / 16);
        k_few<O, mt(), wide()><<<(uint32_t)grid, 256, 0, stream>>>(a);
      };
      if (p.rows <= 16) go(std::integral_constant<int, 1>{});
      else if (p.rows <= 32) go(std::integral_constant<int, 2>{});
      else go(std::integral_constant<int, 4>{});
    } else {
      a.row_tiles = (int)((p.rows + TILE - 1) / TILE);
      a.out_tiles = (p.outputs + TILE - 1) / TILE;
      k_many<O, wide()><<<(uint32_t)((int64_t)a.row_tiles * a.out_tiles), 256, 0, stream>>>(a);
    }
  };
  auto by_width = [&](auto zero) {
    if (wide) run(zero, std::true_type{});
    else run(zero, std::false_type{});
  };
  if (p.dtype == BF16) by_width(bf16{});
  else by_width(float{});
  hip_check(hipGetLastError(), "8-bit product");
}

}  // namespace fhe::clear
