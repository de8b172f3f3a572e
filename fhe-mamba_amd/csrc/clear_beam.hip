// A step of a beam search: the best continuations of each request's beams, and
// the beams' states behind them.
//
//   total_bt = score_b + (l_bt - m_b) - log(sum_t e^(l_bt - m_b))
//
// for every token t of a live beam; a finished beam goes on with the end token
// alone, at its score; a beam of score -inf with none.  The `width` largest of a
// request's totals, the lower beam and then the lower token first among equals.
// A beam's best tokens are those of its logits, so each row's are found as the
// likeliest tokens are, and beams times width candidates remain of a request.
// Exponentials, sums and totals are of 64 bits: which of two near totals of different
// beams is larger should depend neither on 32 bits' rounding nor on how a row was cut.
// Rows are cut by columns whatever their alignment, so that equal beams have equal
// totals.  Four beams of 50280 tokens take 7 + 8 + 3 us, the chains of three launches;
// 256 beams in 16 bits with a third of them masked 22 + 8 + 5, the first bound by its
// vector instructions, the exponentials among them.
#pragma clang fp contract(fast)
#include <algorithm>

#include "clear.hpp"
#include "clear_logits.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

constexpr int MAX_SPLITS = 64;  // workgroups of a row

struct Sum {
  float m;  // the largest logit; NaN if there is one
  double s;
};

struct BeamArgs {
  Beam b;
  BeamOut o;
  int splits, tiles;   // workgroups of a row; tiles of each
  int64_t all_tiles;   // of a row
  int list;            // candidates of a beam
  Sum* sums;           // [rows][splits]
  uint64_t* keys;      // [rows][all_tiles][SETS]
  double* total;       // [rows][list]
  int* token;
};

// e^d for d <= 0, to 2^-45 of it, the library's function in half of its instructions: 2^n 2^f
// with n the integer nearest to d log2 e and 2^f from the polynomial that meets it at the ten
// Chebyshev nodes of [-1/2, 1/2].  Below -700, and for -inf, as at -700, which is nothing
// beside the largest term's 1.
__device__ __forceinline__ double exp_low(double d) {
  constexpr double LOG2_E = 1.4426950408889634, INTEGER = 0x1.8p52;
  constexpr double C[10] = {0x1.000000000003dp+0,  0x1.62e42fefa39f7p-1,  0x1.ebfbdff8149f2p-3,  0x1.c6b08d7044119p-5,
                            0x1.3b2ab72b175eep-7,  0x1.5d87fe908f88ap-10, 0x1.43088e257f341p-13, 0x1.ffcb76789860fp-17,
                            0x1.63ef969a64d3cp-20, 0x1.b6571de2f2351p-24};
  d = fmax(d, -700.0);
  const double s = __builtin_fma(d, LOG2_E, INTEGER), f = __builtin_fma(d, LOG2_E, INTEGER - s);
  double p = C[9];
#pragma unroll
  for (int i = 8; i >= 0; --i) p = __builtin_fma(p, f, C[i]);
  // n lies in the low bits of s, and goes to the exponent
  return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + (__builtin_bit_cast(uint64_t, s) << 52));
}

__device__ __forceinline__ double raise(float m, float most, double s) {
  return s == 0.0 ? 0.0 : s * exp((double)m - (double)most);
}

__device__ __forceinline__ float max_nan(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

// Of a wavefront's lanes.
__device__ __forceinline__ Sum wave_join(float m, double s) {
  float most = m;
#pragma unroll
  for (int d = 32; d; d /= 2) most = max_nan(most, __shfl_xor(most, d));
  s = raise(m, most, s);
#pragma unroll
  for (int d = 32; d; d /= 2) s += __shfl_xor(s, d);
  return {most, s};
}

// Whether the beam's logits take part.
__device__ __forceinline__ bool is_read(const Beam& b, int64_t row) {
  return !(b.finished && b.finished[row]) && b.scores[row] != -INFINITY;
}

template <class T>
__global__ __launch_bounds__(THREADS) void k_beam_parts(BeamArgs a) {
  __shared__ Sum waves[THREADS / 64];
  const int64_t row_i = blockIdx.x / a.splits;
  if (!is_read(a.b, row_i)) return;
  const int split = blockIdx.x % a.splits;
  const T* row = (const T*)a.b.logits + row_i * a.b.row_stride;
  const int64_t start = (int64_t)split * a.tiles * TILE;
  float m = -INFINITY;
  double s = 0.0;
  Sixteen<T> x;
  x.template read<false>(row, start, a.b.vocab);
  for (int t = 0; t < a.tiles; ++t) {
    const int64_t base = start + (int64_t)t * TILE;
    if (base >= a.b.vocab) break;
    float v[16];
    x.widen(v);
    if (t + 1 < a.tiles) x.template read<false>(row, base + TILE, a.b.vocab);  // waited for in its branches
    float most = m;
    double sum = 0.0;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      most = fmaxf(most, v[j]);
      nan |= v[j] != v[j];
    }
    if (nan) most = NAN;
    if (most != -INFINITY) {
#pragma unroll
      for (int j = 0; j < 16; ++j) sum += exp_low((double)v[j] - (double)most);
      s = raise(m, most, s) + sum;
      m = max_nan(m, most);
    }
    const uint64_t key = set_key<T>(v, base, a.b.vocab);
    const int64_t tile = row_i * a.all_tiles + (int64_t)split * a.tiles + t;
    if (threadIdx.x % 4 == 0) a.keys[tile * SETS + threadIdx.x / 4] = key;
  }
  Sum st = wave_join(m, s);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x < 64) {
    const bool some = threadIdx.x < THREADS / 64;
    st = wave_join(some ? waves[threadIdx.x].m : -INFINITY, some ? waves[threadIdx.x].s : 0.0);
    if (threadIdx.x == 0) a.sums[row_i * a.splits + split] = st;
  }
}

// A workgroup a beam: its candidates, best first.
template <class T>
__global__ __launch_bounds__(THREADS) void k_beam_rows(BeamArgs a) {
  __shared__ TopLds lds;
  __shared__ Sum all;
  const int64_t row_i = blockIdx.x;
  const int i = threadIdx.x;
  double* total = a.total + row_i * a.list;
  int* token = a.token + row_i * a.list;
  const float score = a.b.scores[row_i];
  if (!is_read(a.b, row_i)) {
    if (i >= a.list) return;
    const bool finished = score != -INFINITY;  // else a beam without candidates, finished or not
    // behind the end token the others in order, which are not allowed
    const int end = finished ? (int)a.b.end : -1;
    total[i] = finished && i == 0 ? (double)score : -INFINITY;
    token[i] = !finished ? i : i == 0 ? end : i - 1 + (i - 1 >= end);
    return;
  }
  const T* row = (const T*)a.b.logits + row_i * a.b.row_stride;
  if (i < 64) {
    const bool some = i < a.splits;
    const Sum* sums = a.sums + row_i * a.splits;
    const Sum st = wave_join(some ? sums[i].m : -INFINITY, some ? sums[i].s : 0.0);
    if (i == 0) all = st;
  }
  best_of_row(row, a.b.vocab, 0, a.keys + row_i * a.all_tiles * SETS, a.list, lds);
  if (i >= a.list) return;
  const uint64_t k = lds.best[i];
  const float l = key_value(k);
  double t = l == -INFINITY ? -INFINITY : (((double)l - (double)all.m) - log(all.s)) + (double)score;
  // NaN or +inf among the logits or for a score is no candidate's order: all of the beam's are NaN
  const bool sound = all.m < INFINITY && score < INFINITY;
  token[i] = sound ? (int)key_index(k) : i;
  total[i] = sound ? t : NAN;
}

// A finished beam's score may be -inf or NaN too; totals as numbers that order as
// they do, NaN above all.
__device__ __forceinline__ uint64_t order64(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 1ull << 63);
}

// A workgroup a request.
__global__ __launch_bounds__(THREADS) void k_beam_pick(BeamArgs a) {
  __shared__ uint64_t key[MAX_TOP * MAX_TOP];
  const int count = (int)a.b.beams * a.list, width = a.b.width;
  const double* total = a.total + (int64_t)blockIdx.x * count;
  const int* token = a.token + (int64_t)blockIdx.x * count;
  for (int i = threadIdx.x; i < count; i += THREADS) key[i] = order64(total[i]);
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += THREADS) {
    const uint64_t mine = key[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) rank += key[j] > mine || (key[j] == mine && j < i);
    if (rank >= width) continue;
    const int64_t at = (int64_t)blockIdx.x * width + rank;
    a.o.score[at] = (float)total[i];
    a.o.parent[at] = i / a.list;
    a.o.token[at] = token[i];
  }
}

// ----------------------------------------------------------------- states
// A thread has one piece of all the beams' rows of a request: it reads those that
// move and then writes them, so that rows may change places without a copy, and a
// beam that goes on where it lies costs nothing.  Bound by memory: 256 beams' states of
// two layers, 0.8 MB each, take 125 us (5.7 TB/s) in searches of eight, four beams' of 24
// layers 22 us in one launch.  With more than eight beams the 16-byte pieces pass through
// scratch memory, one load at a time: 3.2 TB/s in searches of 16, 2.5 of 32.
constexpr int MAX_MOVED = 64;               // tensors of a launch
constexpr uint32_t MAX_BLOCKS = 1u << 22;  // as many has a row of 2^30 bytes in the narrowest pieces

struct MoveArgs {
  char* state[MAX_MOVED];
  int64_t row[MAX_MOVED];     // pieces of a row
  uint32_t first[MAX_MOVED];  // workgroups before this tensor's
  int count;
  int beams, cache;
  const int *parent, *slots;
};

template <class V, int BEAMS>
__global__ __launch_bounds__(256) void k_move(MoveArgs a) {
  int t = 0;
  while (t + 1 < a.count && blockIdx.x >= a.first[t + 1]) ++t;
  const int64_t row = a.row[t], piece = (int64_t)(blockIdx.x - a.first[t]) * 256 + threadIdx.x;
  if (piece >= row) return;
  V* state = (V*)a.state[t] + piece;
  const int* parent = a.parent + (int64_t)blockIdx.y * a.beams;
  const int* slots = a.slots ? a.slots + (int64_t)blockIdx.y * a.beams : nullptr;
  auto slot_of = [&](int beam) {
    const int64_t s = slots ? (int64_t)slots[beam] : (int64_t)blockIdx.y * a.beams + beam;
    return s >= 0 && s < a.cache ? s : -1;
  };
  V v[BEAMS];
  uint32_t moved = 0;
#pragma unroll
  for (int j = 0; j < BEAMS; ++j) {
    if (j >= a.beams) break;
    const int from = parent[j];
    if (from < 0 || from >= a.beams || from == j) continue;
    const int64_t source = slot_of(from);
    if (source < 0 || slot_of(j) < 0) continue;
    v[j] = state[source * row];
    moved |= 1u << j;
  }
#pragma unroll
  for (int j = 0; j < BEAMS; ++j)
    if (moved >> j & 1) state[slot_of(j) * row] = v[j];
}

int splits_of(int64_t rows, int64_t vocab) {
  const int64_t want = std::max<int64_t>(1, 4096 / rows);
  return (int)std::min<int64_t>({tiles_of(vocab), want, MAX_SPLITS});
}

size_t line(size_t bytes) { return (bytes + 255) / 256 * 256; }

int list_of(const Beam& b) { return (int)std::min<int64_t>(b.width, b.vocab); }

}  // namespace

size_t beam_workspace(const Beam& b) {
  const size_t rows = (size_t)b.requests * b.beams;
  return line(rows * tiles_of(b.vocab) * SETS * sizeof(uint64_t)) +
         line(rows * splits_of((int64_t)rows, b.vocab) * sizeof(Sum)) + rows * list_of(b) * (sizeof(double) + 4);
}

void beam_select(const Beam& b, const BeamOut& o, void* workspace, hipStream_t stream) {
  const int64_t rows = (int64_t)b.requests * b.beams;
  BeamArgs a{b, o, splits_of(rows, b.vocab), 0, tiles_of(b.vocab), list_of(b), nullptr, nullptr, nullptr, nullptr};
  a.tiles = (int)((a.all_tiles + a.splits - 1) / a.splits);
  char* w = (char*)workspace;
  a.keys = (uint64_t*)w;
  w += line((size_t)rows * a.all_tiles * SETS * sizeof(uint64_t));
  a.sums = (Sum*)w;
  w += line((size_t)rows * a.splits * sizeof(Sum));
  a.total = (double*)w;
  a.token = (int*)(a.total + rows * a.list);
  auto run = [&](auto zero) {
    using T = decltype(zero);
    k_beam_parts<T><<<(uint32_t)(rows * a.splits), THREADS, 0, stream>>>(a);
    hip_check(hipGetLastError(), "beam statistics");
    k_beam_rows<T><<<(uint32_t)rows, THREADS, 0, stream>>>(a);
    hip_check(hipGetLastError(), "beam candidates");
  };
  if (b.dtype == BF16) run(bf16{});
  else run(float{});
  k_beam_pick<<<b.requests, THREADS, 0, stream>>>(a);
  hip_check(hipGetLastError(), "beam choice");
}

void reorder_states(const Moved* states, int count, int requests, int beams, int cache, const int* parent,
                    const int* slots, hipStream_t stream) {
  // widest pieces that a tensor's rows divide into
  for (int size : {16, 4, 2, 1}) {
    MoveArgs a{};
    a.beams = beams;
    a.cache = cache;
    a.parent = parent;
    a.slots = slots;
    uint32_t blocks = 0;
    auto launch = [&] {
      if (!a.count) return;
      auto go = [&](auto zero) {
        using V = decltype(zero);
        const dim3 grid(blocks, requests);
        if (beams <= 4) k_move<V, 4><<<grid, 256, 0, stream>>>(a);
        else if (beams <= 8) k_move<V, 8><<<grid, 256, 0, stream>>>(a);
        else if (beams <= 16) k_move<V, 16><<<grid, 256, 0, stream>>>(a);
        else k_move<V, 32><<<grid, 256, 0, stream>>>(a);
      };
      if (size == 16) go(u32x4{});
      else if (size == 4) go(uint32_t{});
      else if (size == 2) go(uint16_t{});
      else go(uint8_t{});
      hip_check(hipGetLastError(), "states of the beams");
      a.count = 0;
      blocks = 0;
    };
    for (int i = 0; i < count; ++i) {
      const Moved& m = states[i];
      auto fits = [&](int s) { return m.row_bytes % s == 0 && reinterpret_cast<uintptr_t>(m.state) % s == 0; };
      int widest = 1;
      for (int s : {2, 4, 16})
        if (fits(s)) widest = s;
      if (widest != size || !m.row_bytes) continue;
      a.state[a.count] = (char*)m.state;
      a.row[a.count] = m.row_bytes / size;
      a.first[a.count] = blocks;
      blocks += (uint32_t)((m.row_bytes / size + 255) / 256);
      if (++a.count == MAX_MOVED || blocks >= MAX_BLOCKS) launch();
    }
    launch();
  }
}

}  // namespace fhe::clear
