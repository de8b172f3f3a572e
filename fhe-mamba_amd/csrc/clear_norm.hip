// Root mean square norms fused with what stands before them in a layer, and
// their gradients:
//   v = x, x silu(z) or h + s u;   r = (mean v^2 + eps)^(-1/2);   n = v r w
//   g = dn w,   dv = r (g - v r (r mean(g v))) (+ the gradient of h + s u itself)
//   dx = dv silu(z),  dz = dv x silu'(z);   dh = dv,  du = s dv
//   dw = sum over rows of dn v r,   ds = sum over rows of dv u
// A row is held in registers by one wavefront, four or sixteen, so that each
// input is read once, and v and r are computed again in the gradient instead of
// being kept.  Bound by memory: 30011 rows of 1536 channels with a gate in bfloat16
// take 45 us (6.2 TB/s, part of it from the last-level cache), the residual and norm
// of 8192 rows of 768 15 us, their gradient 25.  The sums over rows stay in registers
// over the rows that a wavefront walks, and a second kernel adds what the workgroups
// leave, in a fixed order (4.5 us).
//   The sixteen of a wide row have 128 registers each, which do not hold all: gradients
// of more than 8192 channels and most results of more than 16384 keep a part of the row in
// scratch memory.  Of 2^26 elements with a gate in bfloat16 the gradient takes 0.25 ms in
// rows of 8192, 0.95 of 8193, 0.15 of 16384, 1.8 of 16385 and 0.53 of 32768 (its bytes:
// 0.15), the results 0.07, 0.16, 0.08, 0.31 and 0.09.
#pragma clang fp contract(fast)
#include <algorithm>

#include "clear.hpp"
#include "clear_rows.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

enum Mode { PLAIN, GATED, ADDED, SUMMED };  // v: a, a silu(b), a + scale b, a itself but with ADDED's gradients

struct NormArgs {
  const void *a, *b;        // x or h; z or u
  int64_t a_row, b_row;     // elements between rows
  const float *scale, *weight;
  void *sum, *y;            // forward; contiguous
  const void *dy, *dsum;    // backward
  int64_t dy_row, dsum_row;
  void *da, *db;            // contiguous
  float* parts;             // [1 or 2][workgroups][all channels]: of the weight's gradient, of the scale's
  int64_t rows;
  int channels, all;        // of a group; of a row
  float eps;
};

// 1 / (1 + e^-v) of a gate in T.  The product -v log2 e rounded to 32 bits would be up to
// 2^-18 off at v = -80, and a closed gate as much of itself; so what is missing from it goes
// in as a factor.  For 16 bits that is one instruction: eight bits of v times sixteen of
// log2 e are exact, and the rest of log2 e times v is 2^-11 or less, its square nothing.
// 2^x and the reciprocal are the hardware's, good to a unit.
template <class T>
__device__ __forceinline__ float sigmoid(float v) {
  constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;
  float x, factor;
  if constexpr (sizeof(T) == 2) {
    constexpr float HIGH = 47274.0f / 32768.0f, LOW = (float)((LOG2E - (double)HIGH) * LN2);
    x = v * -HIGH;
    factor = __builtin_fmaf(v, -LOW, 1.0f);
  } else {
    constexpr float HIGH = (float)LOG2E, LOW = (float)((LOG2E - (double)HIGH) * LN2);
    v = __builtin_amdgcn_fmed3f(v, -128.0f, 128.0f);  // 0 or 1 beyond
    x = v * -HIGH;
    factor = __builtin_fmaf(v, -LOW, __builtin_fmaf(__builtin_fmaf(v, -HIGH, -x), (float)LN2, 1.0f));
  }
  return __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_amdgcn_exp2f(x), factor, 1.0f));
}

// The sums of W wavefronts' lanes; `lds` is free again after the next call's barrier.
template <int W, int COUNT>
__device__ __forceinline__ void row_sums(float (&s)[COUNT], float (*lds)[2][COUNT], int turn) {
#pragma unroll
  for (int i = 0; i < COUNT; ++i) s[i] = wave_sum(s[i]);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) lds[wave][turn][i] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      s[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) s[i] += lds[w][turn][i];
    }
  }
}

// W wavefronts a row, PER pieces of four channels a lane.  blockIdx.y is the group.
template <class A, class O, int MODE, int W, int PER, int COVER>
__global__ __launch_bounds__(threads_of(W)) void k_norm(NormArgs p) {
  using B = std::conditional_t<MODE == ADDED, O, A>;
  constexpr int LANES = 64 * W, ROWS = threads_of(W) / LANES;
  __shared__ float lds[W][2][1];
  const int lane = threadIdx.x % LANES;
  const int64_t first = (int64_t)blockIdx.y * p.channels;
  const float mean = 1.0f / (float)p.channels;
  Piece<COVER> piece[PER];
  f32x4 w[PER], scale[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    piece[k] = Piece<COVER>((k * LANES + lane) * 4, p.channels);
    w[k] = piece[k].get(p.weight + first);
    if constexpr (MODE == ADDED) scale[k] = p.scale ? piece[k].get(p.scale + first) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row < p.rows;
       row += (int64_t)gridDim.x * ROWS) {
    const A* a = (const A*)p.a + row * p.a_row + first;
    const B* b = (const B*)p.b + (MODE == PLAIN ? 0 : row * p.b_row + first);
    Raw4<A> raw_a[PER];
    Raw4<B> raw_b[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      raw_a[k] = piece[k].raw(a);
      if constexpr (MODE != PLAIN) raw_b[k] = piece[k].raw(b);
    }
    // All on their way: left to itself the compiler may widen each before the next is asked
    // for (a call of 30011 rows of 1536 with a gate in bfloat16: 72 us for 51).  Where
    // several wavefronts have a row and the last pieces are moved it does not, and its own
    // order is better (2^25 elements in rows of 2048: 43 us for 45; of 16384, not moved, 38
    // for 32).
    if constexpr (W == 1 || COVER == WHOLE) __builtin_amdgcn_sched_barrier(0);
    f32x4 v[PER], other[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      v[k] = widen(raw_a[k]);
      if constexpr (MODE != PLAIN) other[k] = widen(raw_b[k]);
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if constexpr (MODE == ADDED) {
        v[k] += scale[k] * other[k];
        piece[k].put((A*)p.sum + row * p.all + first, v[k]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (MODE == GATED) v[k][i] *= other[k][i] * sigmoid<B>(other[k][i]);
        s[0] += piece[k].mine(i, v[k][i] * v[k][i]);
      }
    }
    row_sums<W>(s, lds, turn ^= 1);
    const float r = rsqrtf(s[0] * mean + p.eps);
#pragma unroll
    for (int k = 0; k < PER; ++k) piece[k].put((O*)p.y + row * p.all + first, v[k] * r * w[k]);
  }
}

// Either gradient may be absent, which is looked at within the loop: 16-bit pieces of dy are
// waited for one by one for that, and those of dsum are asked for behind the reduction.
template <class A, class O, int MODE, int W, int PER, int COVER>
__global__ __launch_bounds__(threads_of(W)) void k_norm_back(NormArgs p) {
  using B = std::conditional_t<MODE == ADDED || MODE == SUMMED, O, A>;
  constexpr int LANES = 64 * W, ROWS = threads_of(W) / LANES;
  __shared__ float lds[W][2][2];
  __shared__ float totals[W == 1 ? ROWS - 1 : 1][W == 1 ? PER * 256 : 1];
  const int lane = threadIdx.x % LANES;
  const int64_t first = (int64_t)blockIdx.y * p.channels;
  const float mean = 1.0f / (float)p.channels;
  Piece<COVER> piece[PER];
  f32x4 w[PER], scale[PER], dw[PER], ds[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    piece[k] = Piece<COVER>((k * LANES + lane) * 4, p.channels);
    w[k] = piece[k].get(p.weight + first);
    if constexpr (MODE == ADDED) scale[k] = p.scale ? piece[k].get(p.scale + first) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
    dw[k] = ds[k] = f32x4{};
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row < p.rows;
       row += (int64_t)gridDim.x * ROWS) {
    const A* a = (const A*)p.a + row * p.a_row + first;
    const B* b = (const B*)p.b + (MODE == GATED || MODE == ADDED ? row * p.b_row + first : 0);
    const O* dy = (const O*)p.dy + row * p.dy_row + first;
    f32x4 v[PER], other[PER], g[PER], act[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      v[k] = piece[k].get(a);
      if constexpr (MODE == GATED || MODE == ADDED) other[k] = piece[k].get(b);
      g[k] = p.dy ? piece[k].get(dy) : f32x4{};
    }
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if constexpr (MODE == ADDED) v[k] += scale[k] * other[k];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float t = v[k][i];
        if constexpr (MODE == GATED) {
          act[k][i] = other[k][i] * sigmoid<B>(other[k][i]);
          t *= act[k][i];
        }
        s[0] += piece[k].mine(i, t * t);
        s[1] += piece[k].mine(i, t * g[k][i] * w[k][i]);
      }
    }
    row_sums<W>(s, lds, turn ^= 1);
    // v is made a unit before it is weighed: powers of r above the first leave 32 bits
    // for rows as small as 1e-13 or as large as 1e14
    const float r = rsqrtf(s[0] * mean + p.eps), back = r * (s[1] * mean);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int64_t at = row * p.all + first;
      f32x4 unit = v[k];
      if constexpr (MODE == GATED) unit *= act[k];
      unit *= r;
      f32x4 d = r * (g[k] * w[k] - unit * back);
      dw[k] += g[k] * unit;
      if constexpr (MODE == PLAIN) {
        piece[k].put((A*)p.da + at, d);
      } else if constexpr (MODE == GATED) {
        piece[k].put((A*)p.da + at, d * act[k]);
        f32x4 dz;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sig = sigmoid<B>(other[k][i]);
          dz[i] = d[i] * v[k][i] * (sig + act[k][i] * (1.0f - sig));
        }
        piece[k].put((A*)p.db + at, dz);
      } else {
        if (p.dsum) d += piece[k].get((const A*)p.dsum + row * p.dsum_row + first);
        if (p.da) piece[k].put((A*)p.da + at, d);
        if constexpr (MODE == ADDED) {
          ds[k] += d * other[k];
          d *= scale[k];
        }
        if (p.db) piece[k].put((B*)p.db + at, d);
      }
    }
  }
  // what the workgroup's rows add up to
  auto total = [&](f32x4(&t)[PER], float* out) {
    out += (int64_t)blockIdx.x * p.all + first;
    if constexpr (W == 1) {
      const int wave = threadIdx.x >> 6;
      __syncthreads();
      if (wave) {
#pragma unroll
        for (int k = 0; k < PER; ++k) *reinterpret_cast<f32x4*>(&totals[wave - 1][(k * 64 + lane) * 4]) = t[k];
      }
      __syncthreads();
      if (wave) return;
#pragma unroll
      for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int o = 0; o < ROWS - 1; ++o) t[k] += *reinterpret_cast<const f32x4*>(&totals[o][(k * 64 + lane) * 4]);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) piece[k].put(out, t[k]);
  };
  total(dw, p.parts);
  if constexpr (MODE == ADDED) {
    if (p.scale) total(ds, p.parts + (int64_t)gridDim.x * p.all);
  }
}

// out[c] = the sum over workgroups of parts[.][c]; blockIdx.y: of which of the outputs.
constexpr int SUM_COLUMNS = 16;
__global__ __launch_bounds__(1024) void k_norm_sum(const float* parts, int count, int all, float* out0, float* out1) {
  constexpr int LANES = 1024 / SUM_COLUMNS;
  __shared__ float lds[LANES][SUM_COLUMNS + 1];
  const int at = threadIdx.x % SUM_COLUMNS, lane = threadIdx.x / SUM_COLUMNS;
  const int c = blockIdx.x * SUM_COLUMNS + at;
  parts += (int64_t)blockIdx.y * count * all;
  float s = 0.0f;
  if (c < all) {
#pragma unroll 8
    for (int i = lane; i < count; i += LANES) s += parts[(int64_t)i * all + c];
  }
  lds[lane][at] = s;
#pragma unroll
  for (int half = LANES / 2; half; half /= 2) {
    __syncthreads();
    if (lane < half) lds[lane][at] = s += lds[lane + half][at];
  }
  float* out = blockIdx.y ? out1 : out0;
  if (!lane && c < all && out) out[c] = s;
}

template <class F>
void by_type(uint32_t dtype, uint32_t out, F&& f) {
  if (dtype == F32 && out == F32) f(float{}, float{});
  else if (dtype == F32) f(float{}, bf16{});
  else f(bf16{}, bf16{});
}

int forward_grid(int64_t rows, int channels) {
  const int at = rows_at_once(channels);
  return (int)std::min<int64_t>((rows + at - 1) / at, 1 << 16);
}

// Workgroups of the gradient: two a CU.  More leave more sums to add, fewer do not
// fill the chip: forward and gradient of 4096 rows of 1536 in bfloat16 take 30.7 us
// with 256, 27.7 with 512 and 30.8 with 1024; of 8192 rows of 768 31.2, 26.3 and 25.8.
int backward_grid(int64_t rows, int channels) {
  const int at = rows_at_once(channels);
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + at - 1) / at, 512));
}

template <int MODE>
void forward(const NormArgs& p, uint32_t dtype, uint32_t out, int groups, hipStream_t stream) {
  if (!p.rows) return;
  const dim3 grid(forward_grid(p.rows, p.channels), groups);
  by_type(dtype, out, [&](auto a, auto o) {
    by_shape(p.channels, [&](auto w, auto per, auto cover) {
      k_norm<decltype(a), decltype(o), MODE, w(), per(), cover()><<<grid, threads_of(w()), 0, stream>>>(p);
    });
  });
  hip_check(hipGetLastError(), "norm");
}

template <int MODE>
void backward(const NormArgs& p, uint32_t dtype, uint32_t out, int groups, float* dweight, float* dscale,
              hipStream_t stream) {
  const int count = backward_grid(p.rows, p.channels);
  by_type(dtype, out, [&](auto a, auto o) {
    by_shape(p.channels, [&](auto w, auto per, auto cover) {
      k_norm_back<decltype(a), decltype(o), MODE, w(), per(), cover()>
          <<<dim3(count, groups), threads_of(w()), 0, stream>>>(p);
    });
  });
  hip_check(hipGetLastError(), "norm gradient");
  const dim3 sums((p.all + SUM_COLUMNS - 1) / SUM_COLUMNS, p.scale ? 2 : 1);
  k_norm_sum<<<sums, 1024, 0, stream>>>(p.parts, count, p.all, dweight, dscale);
  hip_check(hipGetLastError(), "norm gradient sums");
}

NormArgs args_of(const Norm& n) {
  NormArgs p{};
  p.a = n.x.p;
  p.a_row = n.x.row;
  p.b = n.gate.p;
  p.b_row = n.gate.row;
  p.weight = n.weight;
  p.rows = n.rows;
  p.all = n.channels;
  p.channels = n.channels / n.groups;
  p.eps = n.eps;
  return p;
}

NormArgs args_of(const AddNorm& n) {
  NormArgs p{};
  p.a = n.hidden.p;
  p.a_row = n.hidden.row;
  p.b = n.update.p;
  p.b_row = n.update.row;
  p.scale = n.scale;
  p.weight = n.weight;
  p.rows = n.rows;
  p.all = p.channels = n.channels;
  p.eps = n.eps;
  return p;
}

}  // namespace

size_t norm_workspace(const Norm& n) {
  return (size_t)backward_grid(n.rows, n.channels / n.groups) * n.channels * sizeof(float);
}

void norm(const Norm& n, void* y, hipStream_t stream) {
  NormArgs p = args_of(n);
  p.y = y;
  if (n.gate.p) forward<GATED>(p, n.dtype, n.out_dtype, n.groups, stream);
  else forward<PLAIN>(p, n.dtype, n.out_dtype, n.groups, stream);
}

void norm_backward(const Norm& n, const NormGrads& g, void* workspace, hipStream_t stream) {
  NormArgs p = args_of(n);
  p.dy = g.dy.p;
  p.dy_row = g.dy.row;
  p.da = g.dx;
  p.db = g.dgate;
  p.parts = (float*)workspace;
  if (n.gate.p) backward<GATED>(p, n.dtype, n.out_dtype, n.groups, g.dweight, nullptr, stream);
  else backward<PLAIN>(p, n.dtype, n.out_dtype, n.groups, g.dweight, nullptr, stream);
}

size_t add_norm_workspace(const AddNorm& n) {
  return (size_t)backward_grid(n.rows, n.channels) * n.channels * sizeof(float) * (n.scale ? 2 : 1);
}

void add_norm(const AddNorm& n, void* sum, void* y, hipStream_t stream) {
  NormArgs p = args_of(n);
  p.sum = sum;
  p.y = y;
  forward<ADDED>(p, n.dtype, n.out_dtype, 1, stream);
}

void add_norm_backward(const AddNorm& n, const AddNormGrads& g, void* workspace, hipStream_t stream) {
  NormArgs p = args_of(n);
  p.dy = g.dy.p;
  p.dy_row = g.dy.row;
  p.dsum = g.dsum.p;
  p.dsum_row = g.dsum.row;
  p.da = g.dhidden;
  p.db = g.dupdate;
  p.parts = (float*)workspace;
  // The sum as the forward call left it is one read for two, where it is whole (32
  // bits) and the update's values are not needed for the scale's gradient.
  if (g.sum && n.dtype == F32 && !n.scale) {
    p.a = g.sum;
    p.a_row = n.channels;
    backward<SUMMED>(p, n.dtype, n.out_dtype, 1, g.dweight, nullptr, stream);
  } else {
    backward<ADDED>(p, n.dtype, n.out_dtype, 1, g.dweight, g.dscale, stream);
  }
}

}  // namespace fhe::clear
