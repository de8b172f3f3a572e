// Shared by the scan's kernels: their arguments, the table of segments, the
// gates of a chunk.
#pragma once

#include "clear.hpp"
#include "clear_tile.hpp"
#include "context.hpp"

namespace fhe::clear {

constexpr int CHUNK = 64, TILES = CHUNK / 16;  // tokens of a chunk, its tiles
constexpr int WAVES = 4;                       // wavefronts of a workgroup
constexpr int VALUE_COLS = 32;                 // head channels of a value sweep's wavefront
// Tokens over which the gates' gradients are one running sum, at most.  Of longer
// segments the gradient sweeps keep the states at every WINDOW tokens: their marks.
constexpr int WINDOW = 256;

// What crosses a place between two tokens of a head: the sum of the products of the
// adjoint and the state there, and that of their squares, by which the sum's rounding
// errors go.
struct Crossing {
  double sum, squares;
};

// Consecutive tokens of one sequence.  `live` is 0 for tokens outside of every
// sequence, whose results are zeros; such an item has no sequence.
struct Item {
  int seq, start, count, live;
};

struct SweepArgs {
  int heads, head_dim, states, groups;
  int cols;             // head channels of a wavefront: 32 or 64
  int col_tiles;        // wavefronts a head: ceil(head_dim / cols)
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
  float* marks;           // the gradients: states at multiples of WINDOW tokens inside of items, or null
  // the reverse sweep of x: the states at segments' ends, where those are cut, and what
  // crosses there
  int windows;            // of a segment
  const int* first;       // each sequence's first item where packed
  const float *end_states, *last_states, *initial;
  Crossing* crossings;    // [item][its beginning, its marks, its end][head][wavefronts a head]

  // an item's number among its sequence's, and how many those are
  __device__ __forceinline__ int number(int item, int seq) const {
    return table ? item - first[seq] : item % segments;
  }
  __device__ __forceinline__ int items_of(int seq) const { return table ? first[seq + 1] - first[seq] : segments; }
  __device__ __forceinline__ Crossing* crossing(int item, int edge, int head) const {
    return crossings + (((int64_t)item * (windows + 1) + edge) * heads + head) * col_tiles;
  }
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

// The number of the mark at token `at` of an item, a multiple of WINDOW inside of it.  By
// the tokens before it: two marks are WINDOW tokens apart or more, so no number comes twice.
__device__ __forceinline__ int64_t mark_of(int64_t token0, int at) { return (token0 + at) / WINDOW; }

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
  double g[CHUNK];
  float src[CHUNK], w[CHUNK];
  float steps[26];
  double ends[TILES + 1];  // of the tiles, after 0

  // start of tile i from the end of tile j < i
  __device__ __forceinline__ float cross(int i, int j) const { return steps[4 * i + j]; }
  // a tile's start from the chunk's, the chunk's end from that of the tile
  __device__ __forceinline__ float first(int i) const { return steps[16 + i]; }
  __device__ __forceinline__ float last(int i) const { return steps[20 + i]; }
  __device__ __forceinline__ float total() const { return steps[24]; }
  // to token `tok` of tile i from its tile's end on the sources' side
  template <bool REV>
  __device__ __forceinline__ float inside(int i, int tok) const {
    return exp2d(REV ? ends[i + 1] - g[tok] : g[tok] - ends[i]);
  }
  // from the state before the chunk to that end of tile i
  template <bool REV>
  __device__ __forceinline__ float into(int i) const {
    return REV ? last(i) : first(i);
  }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sums over the lanes up to each, without LDS.
__device__ __forceinline__ double wave_scan(double v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8: within sixteen lanes
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // row_bcast 15: of lanes 0 and 32 up to the next sixteen
  return dpp_add<0x143, 0xc>(v);  // row_bcast 31
}

__device__ __forceinline__ double read_lane(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Fills `t` from one token's gates in each lane (tokens that are not there decay
// by nothing and write nothing).
template <bool REV>
__device__ __forceinline__ void make_gates(Gates& t, float g, float w) {
  const int lane = lane_id(), tile = lane >> 4;
  // A decay of exp(-1e4) is 0 in 32 bits as exp(-inf) is, and its sums are finite.
  const double sum = wave_scan((double)(g < -1e4f ? -1e4f : g) * 1.4426950408889634);
  // the sum at the end of each tile, 0 before the first
  const double e0 = read_lane(sum, 15), e1 = read_lane(sum, 31), e2 = read_lane(sum, 47), e3 = read_lane(sum, 63);
  auto before = [&](int i) { return i == 0 ? 0.0 : i == 1 ? e0 : i == 2 ? e1 : i == 3 ? e2 : e3; };
  t.g[lane] = sum;
  t.w[lane] = w;
  t.src[lane] = REV ? exp2d(sum - before(tile)) : exp2d(before(tile + 1) - sum) * w;
  // lanes 0 .. 15: start of tile i from the end of tile j; 16 .. 19: start of
  // tile i from the chunk's; 20 .. 23: the chunk's end from that of tile i; 24: all
  const int i = lane < 16 ? lane >> 2 : lane & 3, j = lane & 3;
  const double to = lane < 20 ? before(i) : e3;
  const double from = lane < 16 ? before(j + 1) : lane < 20 || lane >= 24 ? 0.0 : before(i + 1);
  const float f = exp2d(to - from);
  if (lane < 25) t.steps[lane] = f;
  if (lane <= TILES) t.ends[lane] = before(lane);
  wave_sync();
}

// A tile of products, rows the sources 16 j + 4 q + r and columns the targets
// 16 i + l, times their decays and the sources' weights; zeros where the
// target does not see the source.
// `inside`: Gates::inside of the lane's target.
template <bool REV>
__device__ __forceinline__ f32x4 decayed(const Gates& t, f32x4 s, int i, int j, float inside) {
  const int q = lane_id() >> 4, l = lane_id() & 15;
  if (i != j) {
    const float m = inside * (REV ? t.cross(j, i) : t.cross(i, j));
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
template <bool REV>
__device__ __forceinline__ f32x8 to_state(const Gates& t, int m) {
  const int q = lane_id() >> 4;
  f32x4 a = *reinterpret_cast<const f32x4*>(&t.src[32 * m + 4 * q]);
  f32x4 b = *reinterpret_cast<const f32x4*>(&t.src[32 * m + 16 + 4 * q]);
  const float fa = REV ? t.first(2 * m) : t.last(2 * m), fb = REV ? t.first(2 * m + 1) : t.last(2 * m + 1);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    a[r] *= fa;
    b[r] *= fb;
  }
  return join(a, b);
}

// Tokens [0, n) of `width` contiguous elements on their way into the rows of an LDS
// tile of 64 rows and SPAN columns: zeros past the width and the count.  THREADS
// threads; loading and storing are apart so that a chunk's loads are all in flight
// at once.
//
// FULL: every row has SPAN elements and is wide, and there is a row 0.
template <class T, int SPAN, int THREADS, bool FULL>
struct Stage {
  static constexpr int VEC = Num<T>::VEC, PER = SPAN / VEC, PIECES = CHUNK * PER / THREADS;
  static_assert(CHUNK * PER % THREADS == 0);
  u32x4 v[PIECES];

  __device__ __forceinline__ void load(const T* src, int64_t tok, int n, int width, bool wide, int thread) {
    const int row = thread / PER, col = thread % PER * VEC;
    constexpr int STEP = THREADS / PER;
    if constexpr (FULL) {
      // no branches: rows past the last are that one again, and then zeros.  A
      // chunk's offsets take 32 bits (is_full).
      const uint32_t pitch = (uint32_t)(tok * sizeof(T));
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const uint32_t at = (uint32_t)max(min(row + k * STEP, n - 1), 0) * pitch + col * (uint32_t)sizeof(T);
        v[k] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(src) + at);
      }
      if (n < CHUNK) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
          if (row + k * STEP >= n) v[k] = u32x4{0, 0, 0, 0};
      }
    } else {
      const T* p = src + row * tok + col;
#pragma unroll
      for (int k = 0; k < PIECES; ++k) v[k] = load16(p + k * STEP * tok, row + k * STEP < n ? width - col : 0, wide);
    }
  }
  __device__ __forceinline__ void store(T* tile, int thread) const {
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
      *reinterpret_cast<u32x4*>(tile + Tile<T, SPAN>::at(thread / PER + k * (THREADS / PER), thread % PER)) = v[k];
  }
};

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
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
  return v;
}
// Sum over the four lane groups, in each lane.
__device__ __forceinline__ float sum_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Workgroups are dealt to the eight dies in turn: each die takes a run of
// consecutive numbers, so that those which share keys and queries share an L2.
__device__ __forceinline__ uint32_t deal(uint32_t b, uint32_t n) {
  return b < n / 8 * 8 ? b % 8 * (n / 8) + b / 8 : b;
}

// What every sweep derives from its workgroup and wavefront.
struct Place {
  Item it;
  int item, block, group, wave, head, p0, width;
  bool active;        // whether the wavefront has channels
  int64_t token0;     // of all tokens
  int64_t state_at;   // of its head in the states
  int64_t part;       // its row in per-wavefront results

  // `id`: the workgroup's number among its sweep's
  __device__ __forceinline__ Place(const SweepArgs& a, uint32_t id) {
    item = (int)(id / (uint32_t)(a.groups * a.blocks));
    block = (int)(id % (uint32_t)(a.groups * a.blocks));
    it = find_item(a, item);
    group = block / a.blocks;
    block %= a.blocks;
    const int per_group = a.heads / a.groups;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // one for all lanes: in scalar registers
    const int unit = block * WAVES + wave;
    active = unit < per_group * a.col_tiles;
    head = group * per_group + (active ? unit / a.col_tiles : 0);
    p0 = active ? unit % a.col_tiles * a.cols : 0;
    width = active ? min(a.cols, a.head_dim - p0) : 0;
    token0 = item_token(a, it);
    state_at = ((int64_t)(a.by_item ? item : it.seq) * a.heads + head) * a.head_dim * a.states;
    part = (int64_t)head * a.col_tiles + p0 / a.cols;
  }
  // of its head in the marks
  __device__ __forceinline__ int64_t mark_at(const SweepArgs& a, int token) const {
    return (mark_of(token0, token) * a.heads + head) * a.head_dim * a.states;
  }
};

// Whether a sweep's rows are all of whole 16-byte pieces and fill its tiles.
inline bool is_full(const SweepArgs& a, int nb) {
  for (const Strided& t : {a.key, a.query, a.value, a.other})
    if (t.tok >= (1 << 24)) return false;
  for (const float* p : {a.state_in, (const float*)a.state_out, a.initial})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return a.head_dim % a.cols == 0 && a.states == 32 * nb && a.wide_key && a.wide_query && a.wide_value &&
         a.wide_other && a.wide_out;
}

inline uint32_t workgroups(const SweepArgs& a, int items) {
  const int64_t n = (int64_t)items * a.groups * a.blocks;
  if (n > INT32_MAX) throw ArgError("too many tokens and heads for one call");
  return (uint32_t)n;
}

constexpr size_t LDS_BYTES = 160 * 1024;
inline void allow_lds(const void* kernel, size_t bytes) {
  hip_check(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "LDS of a sweep");
}

// f(an element, the 32-state blocks that hold the states)
template <class F>
void by_shape(uint32_t dtype, int states, F&& f) {
  auto by_size = [&](auto zero) {
    if (states <= 32) f(zero, std::integral_constant<int, 1>{});
    else if (states <= 64) f(zero, std::integral_constant<int, 2>{});
    else f(zero, std::integral_constant<int, 4>{});
  };
  if (dtype == BF16) by_size(bf16{});
  else by_size(float{});
}

// clear_scan_forward.hip and clear_scan_backward.hip
void launch_forward(uint32_t dtype, const SweepArgs& a, int items, hipStream_t s);
void launch_states(uint32_t dtype, const SweepArgs& a, const SweepArgs* reverse, int items, hipStream_t s);
void launch_backward(uint32_t dtype, const SweepArgs& c, const SweepArgs& b, const SweepArgs& x, int items,
                     hipStream_t s);

}  // namespace fhe::clear
