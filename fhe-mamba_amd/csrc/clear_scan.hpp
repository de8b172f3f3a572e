// Shared by the scan's kernels: their arguments, the table of segments, the
// gates of a chunk.
#pragma once

#include "clear.hpp"
#include "clear_tile.hpp"
#include "context.hpp"

namespace fhe::clear {

constexpr int CHUNK = 64, TILES = CHUNK / 16;  // tokens of a chunk, its tiles
constexpr int COLS = 32;                       // head channels of a wavefront
constexpr int WAVES = 4;                       // wavefronts of a workgroup

// Consecutive tokens of one sequence.  `live` is 0 for tokens outside of every
// sequence, whose results are zeros; such an item has no sequence.
struct Item {
  int seq, start, count, live;
};

struct SweepArgs {
  int heads, head_dim, states, groups;
  int col_tiles;        // wavefronts a head: ceil(head_dim / COLS)
  int blocks;           // workgroups a group
  int64_t tokens;       // per sequence (0: packed)
  int64_t all_tokens;
  const Item* table;    // null: item i is segment i % segments of sequence i / segments
  int segments, length;
  Strided key, query, value, other, write, decay;
  bool wide_key, wide_query, wide_value, wide_other, wide_out;  // 16-byte accesses
  const float* d;
  const float* state_in;  // null: zeros
  float* state_out;
  bool by_item;           // states are indexed by item, not by sequence
  void* out;
  float *dwrite_part, *gate_part, *dd_part, *decay_out;
};

__device__ __forceinline__ Item find_item(const SweepArgs& a, int i) {
  if (a.table) return a.table[i];
  const int seq = i / a.segments, start = i % a.segments * a.length;
  return {seq, start, (int)min((int64_t)a.length, a.tokens - start), 1};
}

// Element offset of an item's first token in a strided tensor, and that
// token's place among all tokens.
__device__ __forceinline__ int64_t item_at(const SweepArgs& a, const Strided& t, const Item& it) {
  return (a.table ? 0 : it.seq * t.seq) + it.start * t.tok;
}
__device__ __forceinline__ int64_t item_token(const SweepArgs& a, const Item& it) {
  return (a.table ? 0 : it.seq * a.tokens) + it.start;
}

// 2^d, of a 64-bit difference of sums of logarithms: such differences lose
// nothing to the length of the sums.
__device__ __forceinline__ float exp2d(double d) { return __builtin_amdgcn_exp2f((float)d); }

// The decays of one chunk and head.  G_t is the sum of the base-2 logarithms of
// the decays up to token t; E_i is G at the end of tile i.  A token reaches a
// later one through the end of its own tile and the start of the other's, so
// that every factor is a decay over tokens between them: none grows where its
// product does not.  Forward, source s reaches target t >= s; in reverse the
// targets are the earlier ones.
struct Gates {
  double g[CHUNK], e[TILES];
  float src[CHUNK], dst[CHUNK], w[CHUNK];
  float cross[TILES][TILES];  // [i][j], i > j: start of tile i from the end of tile j
  float src_out[TILES];       // from a source's tile to the state behind the chunk
  float dst_in[TILES];        // from the state before the chunk to a target's tile
  float total;
  float pad[3];
};

// Fills `t` for tokens [first, first + n) (n <= CHUNK; the rest decay by
// nothing and write nothing).  One wavefront, a lane a token.
template <bool REV>
__device__ __forceinline__ void make_gates(Gates& t, const float* write, int64_t write_tok,
                                           const float* decay, int64_t decay_tok, int n) {
  const int lane = lane_id();
  float g = 0.0f, w = 0.0f;
  if (lane < n) {
    g = decay[lane * decay_tok];
    w = write[lane * write_tok];
  }
  // A decay of exp(-1e4) is 0 in 32 bits as exp(-inf) is, and its sums are finite.
  double sum = (double)(g < -1e4f ? -1e4f : g) * 1.4426950408889634;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
  }
  t.g[lane] = sum;
  t.w[lane] = w;
  if ((lane & 15) == 15) t.e[lane >> 4] = sum;
  wave_sync();
  const int tile = lane >> 4;
  const double start = tile ? t.e[tile - 1] : 0.0, end = t.e[tile], all = t.e[TILES - 1];
  const float in = exp2d(sum - start), out = exp2d(end - sum);
  t.src[lane] = REV ? in : out * w;
  t.dst[lane] = REV ? out : in;
  if (lane < TILES * TILES) {
    const int i = lane / TILES, j = lane % TILES;
    t.cross[i][j] = i > j ? exp2d(t.e[i - 1] - t.e[j]) : 0.0f;
  } else if (lane < TILES * TILES + TILES) {
    const int i = lane - TILES * TILES;
    const float first = exp2d(i ? t.e[i - 1] : 0.0), last = exp2d(all - t.e[i]);
    t.src_out[i] = REV ? first : last;
    t.dst_in[i] = REV ? last : first;
  } else if (lane == TILES * TILES + TILES) {
    t.total = exp2d(all);
  }
  wave_sync();
}

// A tile of products, rows the sources 16 j + 4 q + r and columns the targets
// 16 i + l, times their decays and the sources' weights; zeros where the
// target does not see the source.
template <bool REV>
__device__ __forceinline__ f32x4 decayed(const Gates& t, f32x4 s, int i, int j) {
  const int q = lane_id() >> 4, l = lane_id() & 15;
  if (i != j) {
    const float m = t.dst[16 * i + l] * (REV ? t.cross[j][i] : t.cross[i][j]);
    const f32x4 v = *reinterpret_cast<const f32x4*>(&t.src[16 * j + 4 * q]);
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] *= m * v[r];
    return s;
  }
  const double gt = t.g[16 * i + l];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int k = 4 * q + r;
    const double gs = t.g[16 * i + k];
    const float f = REV ? exp2d(gs - gt) : exp2d(gt - gs) * t.w[16 * i + k];
    s[r] = (REV ? k >= l : k <= l) ? s[r] * f : 0.0f;
  }
  return s;
}

// The factors from the sources of tiles 2 m and 2 m + 1 to the state behind the
// chunk, in the order of a fragment.
__device__ __forceinline__ f32x8 to_state(const Gates& t, int m) {
  const int q = lane_id() >> 4;
  f32x4 a = *reinterpret_cast<const f32x4*>(&t.src[32 * m + 4 * q]);
  f32x4 b = *reinterpret_cast<const f32x4*>(&t.src[32 * m + 16 + 4 * q]);
  const float fa = t.src_out[2 * m], fb = t.src_out[2 * m + 1];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    a[r] *= fa;
    b[r] *= fb;
  }
  return join(a, b);
}

// Copies tokens [0, n) of `width` contiguous elements into rows of an LDS tile
// of 64 rows and PITCH elements, `span` of them filled: zeros past the width and
// the count.  `threads` threads, this one the `thread`-th.
template <class T, int PITCH>
__device__ __forceinline__ void stage(T* tile, const T* src, int64_t tok, int n, int width,
                                      int span, bool wide, int thread, int threads) {
  constexpr int VEC = Num<T>::VEC;
  const int per = span / VEC;
  for (int i = thread; i < CHUNK * per; i += threads) {
    const int row = i / per, col = i % per * VEC;
    const u32x4 v = load16(src + row * tok + col, row < n ? width - col : 0, wide);
    *reinterpret_cast<u32x4*>(tile + row * PITCH + col) = v;
  }
}

// Sum over the sixteen lanes of one lane group, in each of them.
__device__ __forceinline__ float sum16(float v) {
#define FHE_ROW_ROR(n) \
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + n, 0xf, 0xf, false))
  FHE_ROW_ROR(8);
  FHE_ROW_ROR(4);
  FHE_ROW_ROR(2);
  FHE_ROW_ROR(1);
#undef FHE_ROW_ROR
  return v;
}
// Sum over the four lane groups, in each lane.
__device__ __forceinline__ float sum_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

template <class T, int NB>
struct Pitch {
  static constexpr int KEY = 32 * NB + Num<T>::PAD, VALUE = COLS + Num<T>::PAD;
};

inline uint32_t workgroups(const SweepArgs& a, int items) {
  const int64_t n = (int64_t)items * a.groups * a.blocks;
  if (n > INT32_MAX) throw ArgError("too many tokens and heads for one call");
  return (uint32_t)n;
}

// Launches of the sweeps, by type and state size (clear_scan_value.hip,
// clear_scan_query.hip).
void launch_value_sweep(uint32_t dtype, const SweepArgs& a, int items, bool rev, hipStream_t s);
void launch_state_sweep(uint32_t dtype, const SweepArgs& a, int items, bool rev, hipStream_t s);
void launch_query_sweep(uint32_t dtype, const SweepArgs& a, int items, bool rev, hipStream_t s);

}  // namespace fhe::clear
