// Matrix product in 8-bit integers:
//   a_m = max_k |x_mk| / 127,   q_mk = the integer nearest to x_mk / a_m
//   y_mn = a_m b_n sum_k q_mk W_nk + bias_n
// The sums are of 32-bit integers and exact.  The quotient is rounded to 32 bits
// before it is rounded to an integer (even among equals), so that q is the same
// on any machine with IEEE division.  Few rows are bound by the weights' bytes: one
// row of 768 inputs and 50280 outputs takes 11 us (3.5 TB/s).  Many are bound by the
// way through LDS, the matrix units and the bytes of y together: 30011 rows of 768
// inputs and 3352 outputs in bfloat16 take 20 us to round (3.5 TB/s) and 104 to
// multiply (1.48 POP/s), 8192 rows of 8192 inputs and outputs 476 (2.31 POP/s).
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

typedef __attribute__((address_space(3))) void lds_bytes;
typedef __attribute__((address_space(1))) const void global_bytes;

// BYTES of each lane from memory to LDS, one lane's behind the other's.
template <int BYTES>
__device__ __forceinline__ void load_lds(const void* from, void* to) {
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds((global_bytes*)from, (lds_bytes*)to, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds((global_bytes*)from, (lds_bytes*)to, 4, 0, 0);
}
// Waits until at most the N youngest of this wavefront's loads and stores are in flight.
template <int N>
__device__ __forceinline__ void wait_memory() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr int STEP = 128;  // bytes of a row at a time; rows of q are whole steps, zeros behind the inputs

int64_t pitch_of(int64_t inputs) { return (inputs + STEP - 1) / STEP * STEP; }

// ----------------------------------------------------------------- rounding rows
template <class T, int LANES, int PER>
__device__ __forceinline__ void load_row(f32x4 (&v)[PER], const T* x, int channels, int lane) {
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = (k * LANES + lane) * 4;
    v[k] = get4(x + c, channels - c);
  }
}

// A row in registers as integers, to bytes c .. of q for c below `pitch`; its scale.
// `all`: the largest of the lanes' numbers for the whole row.
//
// A product with the reciprocal is within 2^-15 of the quotient, so both round to
// the same integer unless the product lies that near to the middle of two: then, or
// for a scale whose reciprocal is no good, the quotient itself is taken.  Dividing
// each takes 30011 rows of 768 from 20 to 22 us.
template <int LANES, int PER, class All>
__device__ __forceinline__ float round_row(const f32x4 (&v)[PER], int lane, int8_t* q, int64_t pitch, All&& all) {
  uint32_t most = 0;  // |x| as a number orders as its bits do, infinity and NaN above all
#pragma unroll
  for (int k = 0; k < PER; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = v[k][i];  // a cast of the vector's element itself takes its first
      most = max(most, __builtin_bit_cast(uint32_t, e) & 0x7fffffffu);
    }
  }
#pragma unroll
  for (int d = 32; d; d /= 2) most = max(most, (uint32_t)__shfl_xor((int)most, d));
  most = all(most);
  const bool finite = most < 0x7f800000u;
  const float scale = finite ? __builtin_bit_cast(float, most) / 127.0f : NAN;
  const bool some = finite && scale > 0.0f, plain = scale >= 1e-30f;
  const float inverse = plain ? 1.0f / scale : 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = (k * LANES + lane) * 4;
    if (c >= pitch) continue;
    // 1.5 2^23 + r in 32 bits rounds to an integer as the quotient would be rounded,
    // and holds it in its low byte
    float off = 0.0f;
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sum = __builtin_fmaf(v[k][i], inverse, 0x1.8p23f);
      t[i] = __builtin_bit_cast(uint32_t, sum);
      off = fmaxf(off, fabsf(__builtin_fmaf(v[k][i], inverse, 0x1.8p23f - sum)));
    }
    uint32_t bytes = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400) | __builtin_amdgcn_perm(t[3], t[2], 0x04000c0c);
    if (!plain || off > 0.4998f) {
      bytes = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float r = some ? fminf(fmaxf(rintf(v[k][i] / scale), -127.0f), 127.0f) : 0.0f;
        bytes |= (uint32_t)((int)r & 255) << 8 * i;
      }
    }
    if (c + 4 <= pitch) {
      __builtin_memcpy(q + c, &bytes, 4);
    } else {
      for (int i = c; i < pitch; ++i) q[i] = (int8_t)(bytes >> 8 * (i - c));
    }
  }
  return scale;
}

template <class T, int W, int PER>
__global__ __launch_bounds__(threads_of(W)) void k_quantize(const T* x, int64_t x_row, int64_t rows, int channels,
                                                            int8_t* q, int64_t pitch, float* scales) {
  constexpr int LANES = 64 * W, ROWS = threads_of(W) / LANES;
  __shared__ uint32_t lds[W];
  const int lane = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (row >= rows) return;  // with W > 1 a workgroup has one row
  auto all = [&](uint32_t most) {
    if constexpr (W > 1) {
      if (lane_id() == 0) lds[threadIdx.x >> 6] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) most = max(most, lds[w]);
    }
    return most;
  };
  f32x4 v[PER];
  load_row<T, LANES>(v, x + row * x_row, channels, lane);
  const float scale = round_row<LANES>(v, lane, q + row * pitch, pitch, all);
  if (lane == 0) scales[row] = scale;
}

void quantize(const Quantize& z, int8_t* values, int64_t pitch, float* scale, hipStream_t stream) {
  constexpr int64_t MOST = 1 << 20;  // rows of a launch, which has fewer than 2^32 threads
  auto run = [&](auto zero, int64_t first) {
    using T = decltype(zero);
    const int64_t rows = std::min(z.rows - first, MOST);
    by_shape((int)pitch, [&](auto w, auto per, auto) {
      const int at = threads_of(w()) / (64 * w());
      k_quantize<T, w(), per()><<<(uint32_t)((rows + at - 1) / at), threads_of(w()), 0, stream>>>(
          (const T*)z.x.p + first * z.x.row, z.x.row, rows, z.channels, values + first * pitch, pitch, scale + first);
    });
  };
  for (int64_t first = 0; first < z.rows; first += MOST) {
    if (z.dtype == BF16) run(bf16{}, first);
    else run(float{}, first);
    hip_check(hipGetLastError(), "rounding of rows");
  }
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
__device__ __forceinline__ void put_outputs(const ProductArgs& p, int64_t m, int n, i32x4 sum, float a) {
  const int count = p.outputs - n;
  if (count <= 0) return;
  const f32x4 b = get4(p.scale + n, count);
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)sum[i] * (a * b[i]);
  if (p.bias) v += get4(p.bias + n, count);
  put4((O*)p.y + m * p.outputs + n, v, count);
}

// The fewest rows, of at most 1536 inputs: every workgroup rounds them itself, which
// saves a launch, while its weights are on their way.  A wavefront has 16 outputs, and
// all of their weights in its registers.
constexpr int FEWEST = 16;

// EACH: rows of a wavefront.
template <class O, int PER, int EACH, bool WIDE>
__global__ __launch_bounds__(256) void k_fewest(ProductArgs p, const O* x, int64_t x_row) {
  constexpr int WIDTH = PER * 256, PITCH = WIDTH + 16;  // rows begin in banks four apart
  __shared__ alignas(16) int8_t rows[4 * EACH * PITCH];
  __shared__ float scales[4 * EACH];
  const int wave = threadIdx.x >> 6, lane = lane_id(), q = lane >> 4, l = lane & 15;
  const int n0 = (blockIdx.x * 4 + wave) * 16, count = (int)p.rows;
  const int8_t* w = p.weight + (int64_t)min(n0 + l, p.outputs - 1) * p.inputs;
  i32x4 a[4 * PER];
#pragma unroll
  for (int s = 0; s < 4 * PER; ++s) {
    const int k = 64 * s + 16 * q;
    a[s] = k < p.inputs ? weight16<WIDE>(w, k, p.inputs) : i32x4{};
  }
  f32x4 v[EACH][PER];
#pragma unroll
  for (int i = 0; i < EACH; ++i)  // rows past the last are the last again
    load_row<O, 64>(v[i], x + min(wave + 4 * i, count - 1) * x_row, p.inputs, lane);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int r = wave + 4 * i;
    const float scale = round_row<64>(v[i], lane, rows + r * PITCH, WIDTH, [](uint32_t most) { return most; });
    if (lane == 0) scales[r] = scale;
  }
  __syncthreads();
  i32x4 sum[2] = {};
  const int8_t* row = rows + min(l, count - 1) * PITCH;
#pragma unroll
  for (int s = 0; s < 4 * PER; ++s) {
    const i32x4 b = *reinterpret_cast<const i32x4*>(row + 64 * s + 16 * q);
    sum[s % 2] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], b, sum[s % 2], 0, 0, 0);
  }
  if (l < count) put_outputs<O>(p, l, n0 + 4 * q, sum[0] + sum[1], scales[l]);
}

// Few rows: a workgroup has 16 outputs and MT times 16 rows, its four wavefronts
// a part of the summed index each; operands straight from memory.  A step's operands
// are waited for before its products, in a chain of six for 1536 inputs: 250 rows of
// those and 768 outputs take 7.6 us, their bytes 0.5.
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
    const int64_t m = m0 + 16 * i + l;
    if (m < p.rows) put_outputs<O>(p, m, n0 + 4 * q, sum[i], p.row_scale[m]);
  }
}

// ----------------------------------------------------------------- many rows
// Tiles of WM WN wavefronts, 16 MI rows and 64 outputs each, STEP indices at a time.
// 256 x 256 in eight wavefronts need the fewest bytes from the caches and from LDS for
// a product.  With the rows' rounding, in bfloat16: 30011 x 768 x 3352 takes 122 - 125 us
// in them, 128 in 192 x 256, 131 - 133 in 256 x 128 or 128 x 256, 125 in 128 x 128 in
// four wavefronts; 8192 x 8192 x 8192 494, 539, 606 - 618 and 587.
template <int WM, int WN, int MI>
struct Shape {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, ROWS = 16 * WM * MI, OUTS = 64 * WN;
  // loads of a wavefront that fill its part of a step's rows, and of its weights
  static constexpr int ROW_LOADS = ROWS / 8 / WAVES, OUT_LOADS = OUTS / 8 / WAVES;
  static constexpr int BYTES = (ROWS + OUTS) * STEP;
};

// Which output a lane's sums of its j-th tile begin at, of 64.  For 16-bit results two
// tiles share 32 outputs, so that a lane has eight in a row, 16 bytes.
template <class O>
__device__ __forceinline__ int first_output(int j, int q) {
  return sizeof(O) == 2 ? 32 * (j >> 1) + 8 * q + 4 * (j & 1) : 16 * j + 4 * q;
}
// and which output's weights lane l holds of it
template <class O>
__device__ __forceinline__ int weight_row(int j, int l) {
  return first_output<O>(j, l >> 2) + (l & 3);
}

// A row of a tile in LDS is 128 bytes in 16-byte pieces, whose place is turned by a
// number that differs between the eight rows that neighbouring lanes read.
__device__ __forceinline__ int turn_of_row(int row) { return row & 7; }
template <class O>
__device__ __forceinline__ int turn_of_out(int row) {
  return sizeof(O) == 2 ? (row & 3) | (row >> 1 & 4) : row & 7;
}

// The workgroup's i-th tile.  An XCD has an eighth of the tiles, in groups of 8 row
// tiles for all outputs, so that its cache holds the rows and reads the weights once
// a group.
__device__ __forceinline__ bool tile_of(const ProductArgs& p, int i, int* row_tile, int* out_tile) {
  constexpr uint32_t GROUP = 8;
  const uint32_t all = (uint32_t)p.row_tiles * p.out_tiles, share = (all + 7) / 8;
  const uint32_t at = blockIdx.x / 8 + i * (gridDim.x / 8), t = blockIdx.x % 8 * share + at;
  if (at >= share || t >= all) return false;
  const uint32_t group = t / (GROUP * p.out_tiles), in = t - group * GROUP * p.out_tiles;
  const uint32_t size = min(GROUP, p.row_tiles - group * GROUP);
  *row_tile = (int)(group * GROUP + in % size);
  *out_tile = (int)(in / size);
  return true;
}

// One step's products, from the tiles in LDS.
template <class O, class S, int WN, int MI>
__device__ __forceinline__ void multiply(const int8_t* rows, i32x4 (&sum)[MI][4]) {
  const int wave = threadIdx.x >> 6, lane = lane_id(), q = lane >> 4, l = lane & 15;
  const int8_t* outs = rows + S::ROWS * STEP;
#pragma unroll
  for (int k = 0; k < STEP / 16; k += 4) {
    i32x4 a[4], b[MI];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = wave % WN * 64 + weight_row<O>(j, l);
      a[j] = *reinterpret_cast<const i32x4*>(outs + n * STEP + 16 * ((k + q) ^ turn_of_out<O>(n)));
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = wave / WN * 16 * MI + 16 * i + l;
      b[i] = *reinterpret_cast<const i32x4*>(rows + r * STEP + 16 * ((k + q) ^ turn_of_row(r)));
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], b[i], sum[i][j], 0, 0, 0);
  }
}

// A tile's scales and biases in LDS.
template <class S>
struct alignas(16) Scales {
  float row[S::ROWS], out[S::OUTS], bias[S::OUTS];
};

// The results of the wavefront's part of a tile; whether all of it was there to write.
template <class O, class S, int WN, int MI>
__device__ __forceinline__ bool put_tile(const ProductArgs& p, int64_t m0, int n0, const Scales<S>& scales,
                                         const i32x4 (&sum)[MI][4]) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), q = lane >> 4, l = lane & 15;
  const int row = wave / WN * 16 * MI, out = wave % WN * 64;
  m0 += row;
  n0 += out;
  const bool whole = m0 + 16 * MI <= p.rows && n0 + 64 <= p.outputs;
  f32x4 b[4], bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = out + first_output<O>(j, q);
    b[j] = *reinterpret_cast<const f32x4*>(&scales.out[n]);
    bias[j] = p.bias ? *reinterpret_cast<const f32x4*>(&scales.bias[n]) : f32x4{};
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = m0 + 16 * i + l;
    const float a = scales.row[row + 16 * i + l];
    O* y = (O*)p.y + m * p.outputs + n0;
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = (float)sum[i][j][e] * (a * b[j][e]) + bias[j][e];
    if (whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(O) == 4) {
          put4(y + first_output<O>(j, q), v[j], 4);
        } else if (j % 2 == 0) {
          const u32x4 u{pack2(v[j][0], v[j][1]), pack2(v[j][2], v[j][3]), pack2(v[j + 1][0], v[j + 1][1]),
                        pack2(v[j + 1][2], v[j + 1][3])};
          __builtin_memcpy(y + first_output<O>(j, q), &u, 16);
        }
      }
    } else if (m < p.rows) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        put4(y + first_output<O>(j, q), v[j], p.outputs - n0 - first_output<O>(j, q));
    }
  }
  return whole;
}

// Operands go from memory into LDS without passing through registers, a step ahead of
// the products, also from one tile to the next: a workgroup walks its tiles as one
// row of steps.  A wavefront's loads and stores are done in the order of their issue,
// so that the first step of a tile, whose loads are older than the last tile's stores,
// need not wait for those.  Of 104 us the matrix units work 33 (8-bit products at
// their full rate).  The 24 outputs behind the last multiple of 256 of 3352 are 118 tiles
// of their own, and take the 1652 tiles from 5.99 rounds of the 256 CUs to 6.45, which is
// seven.  The rest is what loads, products and stores do not hide of each other: in an
// earlier form that took 132 us, 109 were left without the loads, 87 without the products
// and 86 without the stores.
template <class O, int WM, int WN, int MI>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_many(ProductArgs p) {
  using S = Shape<WM, WN, MI>;
  constexpr int DEPTH = 2;
  constexpr int STORES = MI * 4 * sizeof(O) / 4;  // of a whole tile's part, 16 bytes each
  // one object: between two the compiler waits for all loads into the one before it reads the other
  __shared__ struct {
    int8_t steps[DEPTH][S::BYTES];
    Scales<S> scales[DEPTH];
  } lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id();

  // The loads' place: a tile and an index.
  int load_tile = 0, load_k = 0;
  int64_t load_m0;
  int load_n0;
  bool left;
  // A load of a wavefront fills 1024 bytes of LDS, 8 rows: lane / 8 is the row, and
  // lane % 8 the place of the piece that it asks for.
  uint32_t row_at[S::ROW_LOADS], out_at[S::OUT_LOADS], out_part[S::OUT_LOADS];
  const int8_t *q, *weight;
  auto begin = [&] {
    int row_tile, out_tile;
    left = tile_of(p, load_tile, &row_tile, &out_tile);
    if (!left) return;
    load_m0 = (int64_t)row_tile * S::ROWS;
    load_n0 = out_tile * S::OUTS;
    q = p.q + load_m0 * p.pitch;
    weight = p.weight + (int64_t)load_n0 * p.inputs;
#pragma unroll
    for (int j = 0; j < S::ROW_LOADS; ++j) {
      const int r = (S::WAVES * j + wave) * 8 + (lane >> 3);
      const uint32_t last = (uint32_t)min((int64_t)r, p.rows - 1 - load_m0);
      row_at[j] = last * (uint32_t)p.pitch + 16 * ((lane & 7) ^ turn_of_row(r));
    }
#pragma unroll
    for (int j = 0; j < S::OUT_LOADS; ++j) {
      const int r = (S::WAVES * j + wave) * 8 + (lane >> 3);
      out_part[j] = 16 * ((lane & 7) ^ turn_of_out<O>(r));
      out_at[j] = (uint32_t)min(r, p.outputs - 1 - load_n0) * (uint32_t)p.inputs;
    }
  };
  auto load = [&](int8_t* to) {
    if (load_k == 0) {
      Scales<S>& s = lds.scales[load_tile % DEPTH];
#pragma unroll
      for (int i = 64 * wave; i < S::ROWS; i += S::THREADS)
        load_lds<4>(p.row_scale + load_m0 + min((int64_t)(i + lane), p.rows - 1 - load_m0), s.row + i);
#pragma unroll
      for (int i = 64 * wave; i < S::OUTS; i += S::THREADS) {
        const int64_t n = load_n0 + min(i + lane, p.outputs - 1 - load_n0);
        load_lds<4>(p.scale + n, s.out + i);
        if (p.bias) load_lds<4>(p.bias + n, s.bias + i);
      }
    }
#pragma unroll
    for (int j = 0; j < S::ROW_LOADS; ++j) load_lds<16>(q + load_k + row_at[j], to + (S::WAVES * j + wave) * 1024);
#pragma unroll
    for (int j = 0; j < S::OUT_LOADS; ++j) {
      // where q is zero, any bytes of the table do
      const uint32_t k = load_k + out_part[j];
      load_lds<16>(weight + out_at[j] + (k < (uint32_t)p.inputs ? k : 0),
                   to + S::ROWS * STEP + (S::WAVES * j + wave) * 1024);
    }
    load_k += STEP;
    if (load_k >= p.inputs) {
      load_k = 0;
      ++load_tile;
      begin();
    }
  };
  begin();
  if (!left) return;
  load(lds.steps[0]);
  int at = 0;
  bool stored = false;  // a whole tile's stores are younger than the loads of the step that begins
  for (int tile = 0;; ++tile) {
    int row_tile, out_tile;
    if (!tile_of(p, tile, &row_tile, &out_tile)) return;
    i32x4 sum[MI][4];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i][j] = i32x4{};
    for (int k = 0; k < p.inputs; k += STEP) {
      if (stored) wait_memory<STORES>();
      else wait_memory<0>();
      stored = false;
      barrier();  // all wavefronts' loads of this step have landed, and none reads the step before it any more
      if (left) load(lds.steps[at ^ 1]);
      multiply<O, S, WN, MI>(lds.steps[at], sum);
      at ^= 1;
    }
    stored = put_tile<O, S, WN, MI>(p, (int64_t)row_tile * S::ROWS, out_tile * S::OUTS, lds.scales[tile % DEPTH],
                                    sum);
  }
}

// The same for weights that are not aligned to 16 bytes, through registers.  With the
// rows' rounding, in bfloat16: 30011 rows of 333 inputs and 1280 outputs take 73 us (of
// 320 inputs, aligned, 45), of 1001 inputs and 643 outputs 83 (1008: 70).
template <class O>
__global__ __launch_bounds__(256) void k_many_narrow(ProductArgs p) {
  using S = Shape<2, 2, 4>;
  constexpr int MI = 4, PIECES = S::ROWS / 32;  // of 16 bytes, of a thread
  __shared__ alignas(16) int8_t lds[S::BYTES];
  __shared__ Scales<S> scales;
  int row_tile, out_tile;
  if (!tile_of(p, 0, &row_tile, &out_tile)) return;
  const int64_t m0 = (int64_t)row_tile * S::ROWS;
  const int n0 = out_tile * S::OUTS;
  if (threadIdx.x < S::ROWS) {
    scales.row[threadIdx.x] = p.row_scale[m0 + min((int64_t)threadIdx.x, p.rows - 1 - m0)];
  } else {
    const int i = threadIdx.x - S::ROWS, n = n0 + min(i, p.outputs - 1 - n0);
    scales.out[i] = p.scale[n];
    scales.bias[i] = p.bias ? p.bias[n] : 0.0f;
  }
  i32x4 sum[MI][4];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = i32x4{};
  const int part = threadIdx.x & 7, r = threadIdx.x >> 3;
  i32x4 x[PIECES], w[PIECES];
  auto load = [&](int k) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      x[j] = *reinterpret_cast<const i32x4*>(p.q + min(m0 + r + 32 * j, p.rows - 1) * p.pitch + k + 16 * part);
      w[j] = weight16<false>(p.weight + (int64_t)min(n0 + r + 32 * j, p.outputs - 1) * p.inputs, k + 16 * part,
                             p.inputs);
    }
  };
  load(0);
  for (int k = 0; k < p.inputs; k += STEP) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int at = r + 32 * j;
      *reinterpret_cast<i32x4*>(lds + at * STEP + 16 * (part ^ turn_of_row(at))) = x[j];
      *reinterpret_cast<i32x4*>(lds + (S::ROWS + at) * STEP + 16 * (part ^ turn_of_out<O>(at))) = w[j];
    }
    __syncthreads();
    if (k + STEP < p.inputs) load(k + STEP);
    multiply<O, S, 2, MI>(lds, sum);
  }
  put_tile<O, S, 2, MI>(p, m0, n0, scales, sum);
}

int64_t tiles_of(int64_t rows, int64_t outputs, int tile) {
  return ((rows + tile - 1) / tile) * ((outputs + tile - 1) / tile);
}

// In us, here and with rows rounded by a launch of their own, kernels alone: 768 inputs
// and 3352 outputs 4.6 and 6.1 for one row, 6.2 and 6.6 for 8, 8.5 and 6.7 for 16; 50280
// outputs 10.2 and 13.3 for one, 11.7 and 13.1 for 8, 15.0 and 13.3 for 16; 1536 inputs
// and 768 outputs 9.4 and 8.6 for 8.  One after another from Python, where a launch and a
// workspace more are 4 us: 8.7 and 13.1 for 16 rows of 768 inputs and 3352 outputs, 14.7
// and 13.1 of 50280 outputs, 12.8 and 13.5 of 1536 inputs and 768 outputs.
bool is_fewest(const Int8& p) {
  return rows_at_once(p.inputs) > 1 && p.rows <= (p.inputs <= 768 && p.outputs <= 16384 ? FEWEST : 8);
}

}  // namespace

void quantize_rows(const Quantize& z, int8_t* values, float* scale, hipStream_t stream) {
  quantize(z, values, z.channels, scale, stream);
}

size_t int8_workspace(const Int8& p) {
  return is_fewest(p) ? 0 : (size_t)p.rows * (pitch_of(p.inputs) + sizeof(float));
}

void int8_linear(const Int8& p, void* y, void* workspace, hipStream_t stream) {
  if (!p.rows) return;
  ProductArgs a{};
  a.pitch = pitch_of(p.inputs);
  a.rows = p.rows;
  a.weight = p.weight;
  a.scale = p.scale;
  a.bias = p.bias;
  a.inputs = p.inputs;
  a.outputs = p.outputs;
  a.y = y;
  const bool wide = p.inputs % 16 == 0 && reinterpret_cast<uintptr_t>(p.weight) % 16 == 0;
  auto by_type = [&](auto&& f) {
    if (p.dtype == BF16) f(bf16{});
    else f(float{});
  };
  if (is_fewest(p)) {
    by_type([&](auto zero) {
      using O = decltype(zero);
      by_shape(p.inputs, [&](auto w, auto per, auto) {
        if constexpr (w() == 1) {
          const uint32_t grid = (uint32_t)((p.outputs + 63) / 64);
          auto go = [&](auto each) {
            const O* x = (const O*)p.x.p;
            if (wide) k_fewest<O, per(), each(), true><<<grid, 256, 0, stream>>>(a, x, p.x.row);
            else k_fewest<O, per(), each(), false><<<grid, 256, 0, stream>>>(a, x, p.x.row);
          };
          if (p.rows <= 4) go(std::integral_constant<int, 1>{});
          else if (p.rows <= 8) go(std::integral_constant<int, 2>{});
          else go(std::integral_constant<int, 4>{});
        }
      });
    });
    hip_check(hipGetLastError(), "8-bit product");
    return;
  }
  int8_t* q = (int8_t*)workspace;
  float* row_scale = (float*)(q + p.rows * a.pitch);
  quantize({p.dtype, p.rows, p.inputs, p.x}, q, a.pitch, row_scale, stream);
  a.q = q;
  a.row_scale = row_scale;
  // Tiles that few CUs would have are cut finer.  128 rows of 768 inputs and 3352
  // outputs (27 tiles) take 10.4 us here and 11.4 in tiles, 192 (54 tiles) 12.4 and 11.4.
  if (tiles_of(p.rows, p.outputs, 128) < 32) {
    by_type([&](auto zero) {
      using O = decltype(zero);
      auto go = [&](auto mt) {
        a.row_tiles = (int)((p.rows + 16 * mt() - 1) / (16 * mt()));
        const uint32_t grid = (uint32_t)((int64_t)a.row_tiles * ((p.outputs + 15) / 16));
        if (wide) k_few<O, mt(), true><<<grid, 256, 0, stream>>>(a);
        else k_few<O, mt(), false><<<grid, 256, 0, stream>>>(a);
      };
      if (p.rows <= 16) go(std::integral_constant<int, 1>{});
      else if (p.rows <= 32) go(std::integral_constant<int, 2>{});
      else go(std::integral_constant<int, 4>{});
    });
  } else {
    // workgroups: as many as there are tiles, but no more than run at once
    auto tiles = [&](int rows, int outs, int at_once) {
      a.row_tiles = (int)((p.rows + rows - 1) / rows);
      a.out_tiles = (p.outputs + outs - 1) / outs;
      const int64_t share = ((int64_t)a.row_tiles * a.out_tiles + 7) / 8;
      return (uint32_t)(8 * std::min<int64_t>(share, at_once / 8));
    };
    by_type([&](auto zero) {
      using O = decltype(zero);
      // Large tiles as soon as every CU has one.  With the rows' rounding, of 768 inputs and
      // 3352 outputs: 2048 rows 22.2 us and 16.8 in small ones, 4096 26.3 and 26.1, 8192 41.4
      // and 40.3, 30011 122 and 125; of 8192 inputs and outputs 8192 rows 492 and 587.
      if (!wide) k_many_narrow<O><<<tiles(128, 128, 1 << 30), 256, 0, stream>>>(a);
      else if (tiles_of(p.rows, p.outputs, 256) >= 256) k_many<O, 2, 4, 8><<<tiles(256, 256, 256), 512, 0, stream>>>(a);
      else k_many<O, 2, 2, 4><<<tiles(128, 128, 512), 256, 0, stream>>>(a);
    });
  }
  hip_check(hipGetLastError(), "8-bit product");
}

}  // namespace fhe::clear
