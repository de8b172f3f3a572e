// The selective scan over whole sequences and its gradients.
//
//   h_t = exp(g_t) h_{t-1} + w_t x_t B_t^T,   y_t = h_t C_t + D x_t
//
// In chunks of 64 tokens everything is a matrix product: the pairs of a chunk
// (C B^T under a triangle of decays) with its x, the state before it with C,
// and the state that it adds.  A wavefront keeps the state of 32 channels in
// registers and walks its segment's chunks, so that x, B and C are read once
// and y is written once.  A segment is a whole sequence where there are enough
// of them to fill the chip; else a first sweep makes the state that each
// segment adds, and a small kernel carries them along the sequence.
//
// Backwards the adjoint state A_t = exp(g_{t+1}) A_{t+1} + dy_t C_t^T is the
// same recurrence in reversed time with B and C, x and dy in each other's
// place, so the same sweeps give V_t = A_t B_t (dx = w V + D dy, dw = x . V),
// dB and dC.  With M_ts the part of the loss in source s and target t,
// dg_r is the sum of M over t >= r > s.  At a place where both states are known it is
// <A, h>, and from one token to the next it changes by what enters less what leaves;
// terms with s = t are in neither.  Those are rounded to 32 bits and may be far
// larger than what is left of them, so the running sums start again every 256 tokens
// (WINDOW) at the latest, whatever the segments' length, and a token takes the sum
// from that end of the window from where less was added up.  Less by the terms'
// squares, as independent roundings add up: the gradient of log_decay at 10 heads of
// 48, 40 states and 1777 tokens in 32 bits is 2.2e-7 off so, by the terms' sizes 2.8e-7,
// always from the end 2.2e-7 and, with two texts of 3000 tokens, 3.4e-7 for 2.5e-7.
//
// 24 heads of 64 x 128 in 16 bits: a prompt of 1000 tokens takes 13.9 us for the
// segments' states, 11.6 for carrying them and 12.5 for the results; 30011 packed
// tokens 62 + 23 + 148; 4 x 2048 tokens 26 + 9 + 48, and their gradients 35 + 16 +
// 192 and 15 for the last sums.  In 32 bits 1000 tokens take 16 + 11 + 33, 4 x 2048
// tokens 52 + 9 + 190 and their gradients 79 + 16 + 513 + 18.  32 x 2048 tokens stay
// whole: 328 us in 16 bits, their gradients 1453, 76 for the marks' products and 95 for
// the sums.
// The sweeps read and write a fifth of what memory would pass in that time, and no
// unit is full either: of a CU's 252 thousand cycles in the results of 30011 tokens
// the vector units work 119 (splits into 16-bit pieces, decays, pairs) and the matrix
// units 79.  What is left are the waits of a wavefront's chain of products, which the
// two wavefronts a SIMD that the states' registers leave do not cover.
#pragma clang fp contract(fast)
#include "clear_scan.hpp"

#include <algorithm>

#include "context.hpp"

namespace fhe::clear {
namespace {

// ---- segments of packed sequences ----
// first[s]: sequence s's first item, first[seqs] the end.  Offsets are taken as
// a partition whatever they hold: clamped to the tokens and made to rise.  The
// tokens before the first and after the last sequence are items without one;
// entries past the last item are empty.
__global__ __launch_bounds__(64) void k_items(const int* offsets, int seqs, int tokens, int length,
                                              bool keep_empty, int items, Item* table, int* first) {
  const int lane = lane_id();
  const int start0 = min(max(offsets[0], 0), tokens);
  int last = start0, count = 0;  // of the sequences so far: where they end, their items
  for (int s0 = 0; s0 < seqs; s0 += 64) {
    const int s = s0 + lane;
    int end = s < seqs ? min(max(offsets[s + 1], last), tokens) : last;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(end, d);
      if (lane >= d) end = max(end, up);
    }
    int begin = __shfl_up(end, 1);
    if (lane == 0) begin = last;
    int mine = 0;
    if (s < seqs) mine = max(keep_empty ? 1 : 0, (int)(((int64_t)end - begin + length - 1) / length));
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    if (s < seqs) {
      first[s] = count + sum - mine;
      for (int k = 0; k < mine; ++k)
        table[count + sum - mine + k] = {s, begin + k * length, min(length, end - begin - k * length), 1};
    }
    last = __shfl(end, 63);
    count += __shfl(sum, 63);
  }
  if (lane == 0) first[seqs] = count;
  // outside of the sequences
  const int head = (int)(((int64_t)start0 + length - 1) / length);
  const int tail = (int)(((int64_t)tokens - last + length - 1) / length);
  for (int k = lane; k < items - count; k += 64) {
    Item it = {-1, 0, 0, 0};
    if (k < head) it = {-1, k * length, min(length, start0 - k * length), 0};
    else if (k < head + tail)
      it = {-1, last + (k - head) * length, min(length, tokens - last - (k - head) * length), 0};
    table[count + k] = it;
  }
}

// ---- states carried from segment to segment ----
// In: the state that each item adds.  Out: the state before it (behind it in
// reverse), and the sequence's last.  A thread an element; eight items are read
// at a time, since only the sums depend on each other.
struct Join {
  float* states;
  const float* initial;
  float* last;
};

template <int VEC>
__global__ __launch_bounds__(256) void k_join(Join forward, Join reverse, const float* decay, const int* first,
                                              int segments, int size, int per_head, int heads) {
  typedef float Vec __attribute__((ext_vector_type(VEC)));
  const int e = (blockIdx.x * 256 + threadIdx.x) * VEC, seq = blockIdx.y;
  if (e >= size) return;
  const bool rev = blockIdx.z;
  const Join j = rev ? reverse : forward;
  const int head = e / per_head;
  const int from = first ? first[seq] : seq * segments;
  const int count = first ? first[seq + 1] - from : segments;
  auto at = [&](float* p, int64_t row) { return reinterpret_cast<Vec*>(p + row * size + e); };
  Vec run = j.initial ? *reinterpret_cast<const Vec*>(j.initial + (int64_t)seq * size + e) : Vec(0.0f);
  for (int i0 = 0; i0 < count; i0 += 8) {
    Vec add[8];
    float keep[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = min(i0 + u, count - 1), item = from + (rev ? count - 1 - i : i);
      add[u] = *at(j.states, item);
      keep[u] = decay[(int64_t)item * heads + head];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < count) {
        *at(j.states, from + (rev ? count - 1 - i0 - u : i0 + u)) = run;
        run = run * keep[u] + add[u];
      }
  }
  if (j.last) *at(j.last, seq) = run;
}

// ---- the ends of the gradients ----
// Four elements of a query gradient from its workgroups' parts.
template <class T>
__device__ __forceinline__ void sum_parts(const float* parts, int count, int64_t size, T* out, int64_t i) {
  if (i >= size) return;
  if (size % 4 == 0) {
    f32x4 sum = *reinterpret_cast<const f32x4*>(parts + i);
    for (int p = 1; p < count; ++p) sum += *reinterpret_cast<const f32x4*>(parts + p * size + i);
#pragma unroll
    for (int r = 0; r < 4; ++r) out[i + r] = (T)sum[r];
    return;
  }
  for (int64_t k = i; k < min(i + 4, size); ++k) {
    float sum = parts[k];
    for (int p = 1; p < count; ++p) sum += parts[p * size + k];
    out[k] = (T)sum;
  }
}

// What crosses the marks, and the ends of sequences that are not cut: the products of
// the adjoint and the state that the sweeps left there.  A wavefront a head, four
// heads a workgroup; it takes both states' bandwidth.
struct Marks {
  const float *adjoints, *states;  // the marks
  const float *dfinal, *last;      // null where sequences are cut or nothing enters at their end
};
__global__ __launch_bounds__(256) void k_cross(SweepArgs a, Marks m) {
  const int across = (a.heads + 3) / 4;
  const int edge = 1 + (int)(blockIdx.x / across) % a.windows, item_i = (int)(blockIdx.x / across) / a.windows;
  const int head = (int)(blockIdx.x % across) * 4 + (threadIdx.x >> 6), lane = lane_id();
  const Item it = find_item(a, item_i);
  if (!it.live || head >= a.heads) return;
  const int64_t size = (int64_t)a.head_dim * a.states, all = size * a.heads;
  const float *A, *h;
  if (edge < a.windows) {
    if (edge * WINDOW >= it.count) return;
    const int64_t mark = mark_of(item_token(a, it), edge * WINDOW);
    A = m.adjoints + mark * all;
    h = m.states + mark * all;
  } else {
    if (!m.dfinal) return;
    A = m.dfinal + it.seq * all;
    h = m.last + it.seq * all;
  }
  A += head * size;
  h += head * size;
  double sum = 0.0;
  float squares = 0.0f;
  auto add = [&](float x, float y) {
    sum += (double)x * y;
    squares += x * y * (x * y);
  };
  if (size % 4 == 0 && reinterpret_cast<uintptr_t>(A) % 16 == 0) {
#pragma unroll 8
    for (int64_t e = 4 * lane; e < size; e += 256) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(A + e), y = *reinterpret_cast<const f32x4*>(h + e);
#pragma unroll
      for (int r = 0; r < 4; ++r) add(x[r], y[r]);
    }
  } else {
    for (int64_t e = lane; e < size; e += 64) add(A[e], h[e]);
  }
  const Crossing c{wave_sum(sum), wave_sum((double)squares)};
  for (int p = lane; p < a.col_tiles; p += 64) a.crossing(item_i, edge, head)[p] = p ? Crossing{0.0, 0.0} : c;
}

constexpr int FINISH_THREADS = 256, FINISH_HEADS = FINISH_THREADS / 64, FINISH_STEPS = 4;

// What is left when the sweeps are done: the first workgroups, which take longest,
// make the gates' gradients of an item and four heads each, the next the gradient
// of D of four heads each, then `sums` sum the parts of dC and as many those of dB.
struct Finish {
  int64_t size;  // of dB and dC
  int parts, items, entering_tiles, group;
  bool ends;      // whether something crosses a sequence's end
  uint32_t sums;  // workgroups of one of the two
  const float *parts_c, *parts_b;
  void *dc, *db;
  const float *entering, *leaving;
  float *dwrite, *ddecay, *dd;
};

// A value of each lane, in the lanes' reverse order.
__device__ __forceinline__ double turned(double v) { return __shfl(v, 63 - lane_id()); }

// Gradients of write and log_decay of four heads, a wavefront each, and of a
// window of up to WINDOW tokens: the first summed over the head's channels, the
// second the running sums from the window's end backwards and from its beginning.  A
// window lies in an item that is longer, or it is up to `group` items of one sequence,
// done by the workgroup of the last of them.  What crosses its ends is known.  The
// results of 64 tokens go through LDS, so that a token's heads are written together.
__device__ __forceinline__ void gate_grads(const SweepArgs& a, const Finish& f, int item_i, int window, int head0,
                                           float (&tile)[2][64 * FINISH_STEPS][FINISH_HEADS + 1]) {
  static_assert(64 * FINISH_STEPS == WINDOW);
  const Item it = find_item(a, item_i);
  const int from = window * WINDOW;
  if (it.count <= from) return;
  const bool inside = it.count - from > WINDOW;  // its end is a mark
  const int end = inside ? from + WINDOW : it.count;  // in the item
  int count = end - from, before = 0;  // `before` items of the window come before this one
  bool is_first = true;
  if (a.by_item && it.live) {
    const int number = a.number(item_i, it.seq);
    before = number % f.group;
    is_first = number == before;
    if (number != a.items_of(it.seq) - 1 && before != f.group - 1) return;
    count += before * a.length;
  }
  const int lane = lane_id(), wave = threadIdx.x >> 6, head = min(head0 + wave, a.heads - 1);
  const int64_t token0 = item_token(a, it) + end - count;
  // what crosses before the window's first token and behind its last
  Crossing ahead{0.0, 0.0}, behind{0.0, 0.0};
  auto crossing = [&](int item, int edge) {
    Crossing c{0.0, 0.0};
    for (int p = 0; p < a.col_tiles; ++p) {
      const Crossing x = a.crossing(item, edge, head)[p];
      c.sum += x.sum;
      c.squares += x.squares;
    }
    return c;
  };
  if (it.live) {
    if (inside) behind = crossing(item_i, window + 1);
    else if (f.ends) behind = crossing(item_i, a.windows);
    if (from) ahead = crossing(item_i, window);
    else if (!is_first) ahead = crossing(item_i - before - 1, a.windows);
    else if (a.initial) ahead = crossing(item_i - before, 0);
  }
  // what enters at a token less what leaves, and the parts' squares
  double v[FINISH_STEPS] = {}, m[FINISH_STEPS] = {};
  float dw[FINISH_STEPS] = {};
  const int t0 = count - 1 - lane;  // the last token first, then those 64 before it
  for (int p = 0; p < a.col_tiles; ++p) {
    const int64_t at = ((int64_t)head * a.col_tiles + p) * a.all_tokens + token0 + t0;
#pragma unroll
    for (int u = 0; u < FINISH_STEPS; ++u)
      if (t0 >= 64 * u) {
        const double g = f.leaving[at - 64 * u];
        v[u] += g;
        m[u] += g * g;
        dw[u] += a.dwrite_part[at - 64 * u];
      }
  }
  for (int p = 0; p < f.entering_tiles; ++p) {
    const int64_t at = ((int64_t)head * f.entering_tiles + p) * a.all_tokens + token0 + t0;
#pragma unroll
    for (int u = 0; u < FINISH_STEPS; ++u)
      if (t0 >= 64 * u) {
        const double g = f.entering[at - 64 * u];
        v[u] += g;
        m[u] += g * g;
      }
  }
  // from the window's beginning: without the token itself, since what crosses there is
  // the gradient at the first one
  double fv[FINISH_STEPS], fm[FINISH_STEPS];
#pragma unroll
  for (int u = FINISH_STEPS - 1; u >= 0; --u) {
    const double mine = turned(v[u]), its = turned(m[u]);
    const double sum = wave_scan(mine), squares = wave_scan(its);
    fv[u] = turned(ahead.sum - (sum - mine));
    fm[u] = turned(ahead.squares + (squares - its));
    ahead.sum -= read_lane(sum, 63);
    ahead.squares += read_lane(squares, 63);
  }
#pragma unroll
  for (int u = 0; u < FINISH_STEPS; ++u) {
    const double sum = behind.sum + wave_scan(v[u]), squares = behind.squares + wave_scan(m[u]);
    tile[0][64 * u + lane][wave] = dw[u];
    // where one of the two is not finite, the other
    tile[1][64 * u + lane][wave] = (float)(squares <= fm[u] || fm[u] != fm[u] ? sum : fv[u]);
    behind.sum = read_lane(sum, 63);
    behind.squares = read_lane(squares, 63);
  }
  __syncthreads();
  const int col = threadIdx.x % FINISH_HEADS;
#pragma unroll
  for (int u = 0; u < FINISH_STEPS; ++u) {
    const int row = 64 * u + threadIdx.x / FINISH_HEADS;
    if (row < count && head0 + col < a.heads) {
      const int64_t at = (token0 + count - 1 - row) * a.heads + head0 + col;
      f.dwrite[at] = tile[0][row][col];
      f.ddecay[at] = tile[1][row][col];
    }
  }
}

__device__ __forceinline__ void skip_grad(const SweepArgs& a, const Finish& f, int head0) {
  const int head = head0 + (threadIdx.x >> 6);
  if (head >= a.heads) return;
  double v = 0.0;
  for (int i = lane_id(); i < f.items; i += 64) {
    const Item it = find_item(a, i);
    if (!it.live) continue;
    for (int p = 0; p < a.col_tiles; ++p) v += a.dd_part[((int64_t)i * a.heads + head) * a.col_tiles + p];
  }
  v = wave_sum(v);
  if (lane_id() == 0) f.dd[head] = (float)v;
}

template <class T>
__global__ __launch_bounds__(FINISH_THREADS, 8) void k_finish(SweepArgs a, Finish f) {
  __shared__ float tile[2][64 * FINISH_STEPS][FINISH_HEADS + 1];
  uint32_t block = blockIdx.x;
  const uint32_t across = (a.heads + FINISH_HEADS - 1) / FINISH_HEADS, gates = (uint32_t)f.items * a.windows * across;
  if (block < gates) {
    const uint32_t window = block / across;
    gate_grads(a, f, (int)(window / a.windows), (int)(window % a.windows), (int)(block % across) * FINISH_HEADS, tile);
    return;
  }
  block -= gates;
  if (f.dd) {
    if (block < across) {
      skip_grad(a, f, (int)block * FINISH_HEADS);
      return;
    }
    block -= across;
  }
  const bool is_b = block >= f.sums;
  const int64_t i = ((int64_t)(is_b ? block - f.sums : block) * FINISH_THREADS + threadIdx.x) * 4;
  sum_parts<T>(is_b ? f.parts_b : f.parts_c, f.parts, f.size, (T*)(is_b ? f.db : f.dc), i);
}

// ---- plan ----
// How a sweep cuts heads into wavefronts and workgroups.
struct Cut {
  int cols, col_tiles, blocks;
  Cut() = default;
  Cut(const Scan& s, int cols_) : cols(cols_) {
    col_tiles = (s.head_dim + cols - 1) / cols;
    blocks = (s.heads / s.groups * col_tiles + WAVES - 1) / WAVES;
  }
};

struct Plan {
  Cut value, query;
  int length, segments, items;
  int windows;  // of an item
  bool by_item;
  // workspace, in bytes
  size_t table, first, decays, states, adjoints, last, dwrite, gate_out, gate_in, dd, parts_c, parts_b, crossings,
      mark_states, mark_adjoints, total;
};

// Tokens of a segment: of all numbers of chunks the one whose estimated time is
// least.  Workgroups run in rounds of two a CU, a round as long as a segment; a
// chunk of a round takes about 14 us in the sweeps for the states and the results
// together, and a segment's states are written once and read and written once
// more, at 6.6 TB/s.  A whole sequence's state stays in registers.  The times are
// those of 24 heads of 64 x 128 in 16 bits and are taken for every type and size:
// 32-bit products are slower and few states quicker, and other lengths than these may
// be best there.  Packed sequences' lengths are not known on the host, so a batch of
// them is planned as one, and is cut also where each would fit a segment.  us of the
// launches forward, at lengths of 4 / 6 / 8 / 12 / 16 chunks of 30011 packed tokens of
// 24 heads of 64 x 128: 269 / 258 / 256 / 301 / 267; at 2 / 4 / 5 chunks of 4 x 2048:
// 89 / 84 / 92, and their gradients 281 / 265 / 268.
int segment_length(int64_t all, int64_t longest, int seqs, int64_t per_item, size_t state, bool packed) {
  const int64_t slots = 2 * 256, most = std::max<int64_t>(1, (longest + CHUNK - 1) / CHUNK);
  double best = 0;
  int64_t length = most;
  for (int64_t chunks = 1; chunks <= most; chunks += 1 + chunks / 16) {
    // ragged sequences end inside a segment each
    const int64_t items = packed ? (all + chunks * CHUNK - 1) / (chunks * CHUNK) + seqs
                                 : seqs * ((most + chunks - 1) / chunks);
    const int64_t rounds = (items * per_item + slots - 1) / slots;
    const double us = 14.0 * rounds * chunks + items * (3.0 * state / 6.6e6);
    if (chunks == 1 || us < best) {
      best = us;
      length = chunks;
    }
  }
  const double whole = 10.0 * most * ((seqs * per_item + slots - 1) / slots);
  if (whole <= best) length = most;
  return (int)std::min<int64_t>(length * CHUNK, std::max<int64_t>(longest, 1));
}

Plan make_plan(const Scan& s, bool backward) {
  Plan p{};
  const bool packed = s.offsets != nullptr;
  p.value = Cut(s, VALUE_COLS);
  // 64 channels take all of a head's registers there are, and halve the sums
  // over wavefronts and the parts: both sweeps by themselves, with their sums, took
  // 146 us at 4 x 2048 tokens of 24 heads of 64, with 32 channels 183
  p.query = Cut(s, s.head_dim <= 32 ? 32 : 64);
  const int64_t all = s.all_tokens();
  const size_t state = (size_t)s.heads * s.head_dim * s.states * 4;
  p.length = segment_length(all, s.tokens, s.seqs, (int64_t)p.value.blocks * s.groups, state, packed);
  p.segments = packed ? 0 : std::max<int>(1, (int)((s.tokens + p.length - 1) / p.length));
  p.by_item = p.length < s.tokens;
  p.items = packed ? (int)(s.tokens / p.length) + s.seqs + 2 : s.seqs * p.segments;
  p.windows = (p.length + WINDOW - 1) / WINDOW;
  const size_t rows = (size_t)s.heads * p.value.col_tiles;
  auto take = [&](size_t bytes) {
    const size_t at = p.total;
    p.total += (bytes + 255) / 256 * 256;
    return at;
  };
  if (packed) {
    p.table = take(sizeof(Item) * p.items);
    p.first = take(4 * ((size_t)s.seqs + 1));
  }
  if (p.by_item) {
    p.decays = take((size_t)p.items * s.heads * 4);
    p.states = take(p.items * state);
  }
  if (backward) {
    if (p.by_item) p.adjoints = take(p.items * state);
    p.last = take(s.seqs * state);
    p.dwrite = take(rows * all * 4);
    p.gate_out = take(rows * all * 4);
    p.gate_in = take((size_t)s.heads * p.query.col_tiles * all * 4);
    p.dd = take(rows * p.items * 4);
    p.parts_c = take((size_t)p.query.blocks * all * s.groups * s.states * 4);
    p.parts_b = take((size_t)p.query.blocks * all * s.groups * s.states * 4);
    p.crossings = take(rows * p.items * (p.windows + 1) * sizeof(Crossing));
    if (p.windows > 1) {
      p.mark_states = take((all / WINDOW + 1) * state);
      p.mark_adjoints = take((all / WINDOW + 1) * state);
    }
  }
  return p;
}

// Whether every row of 16-byte pieces starts at a multiple of 16 bytes.
bool is_wide(const Strided& t, int vec, bool packed) {
  return reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && (packed || t.seq % vec == 0) && t.tok % vec == 0 &&
         t.head % vec == 0;
}

struct Sweep {
  const Scan& s;
  const Plan& p;
  char* ws;
  SweepArgs a{};

  Sweep(const Scan& s_, const Plan& p_, char* ws_) : s(s_), p(p_), ws(ws_) {
    a.heads = s.heads;
    a.head_dim = s.head_dim;
    a.states = s.states;
    a.groups = s.groups;
    a.tokens = s.offsets ? 0 : s.tokens;
    a.all_tokens = s.all_tokens();
    a.table = s.offsets ? at<const Item>(p.table) : nullptr;
    a.segments = p.segments;
    a.length = p.length;
    a.write = s.write;
    a.decay = s.decay;
    a.by_item = p.by_item;
  }
  template <class T>
  T* at(size_t offset) const {
    return reinterpret_cast<T*>(ws + offset);
  }
  int elem() const { return s.dtype == BF16 ? 2 : 4; }
  bool wide(const Strided& t) const { return is_wide(t, 16 / elem(), s.offsets != nullptr); }
  SweepArgs with(const Cut& cut, const Strided& key, const Strided& query, const Strided& value,
                 const Strided& other) const {
    SweepArgs b = a;
    b.cols = cut.cols;
    b.col_tiles = cut.col_tiles;
    b.blocks = cut.blocks;
    b.key = key;
    b.query = query;
    b.value = value;
    b.other = other;
    b.wide_key = wide(key);
    b.wide_query = wide(query);
    b.wide_value = wide(value);
    b.wide_other = wide(other);
    return b;
  }
  const int* first() const { return s.offsets ? at<const int>(p.first) : nullptr; }

  void make_items(hipStream_t stream) const {
    if (!s.offsets) return;
    k_items<<<1, 64, 0, stream>>>(s.offsets, s.seqs, (int)s.tokens, p.length, !p.by_item, p.items,
                                   at<Item>(p.table), at<int>(p.first));
    hip_check(hipGetLastError(), "scan segments");
  }
  // The states before each segment, and each sequence's last; with `reverse` also
  // the adjoint's behind each.
  SweepArgs state_args(const Strided& key, const Strided& value, size_t states) const {
    SweepArgs b = with(p.value, key, key, value, value);
    b.wide_out = true;
    b.state_out = at<float>(states);
    b.decay_out = at<float>(p.decays);
    return b;
  }
  void carry(float* last, const ScanGrads* g, hipStream_t stream) const {
    const SweepArgs f = state_args(s.b, s.x, p.states);
    SweepArgs r{};
    if (g) r = state_args(s.c, g->dy, p.adjoints);
    launch_states(s.dtype, f, g ? &r : nullptr, p.items, stream);
    const int size = s.heads * s.head_dim * s.states;
    const Join forward{at<float>(p.states), s.initial, last};
    const Join reverse = g ? Join{at<float>(p.adjoints), g->dfinal, g->dinitial} : Join{};
    // four elements of one head a thread where all rows are of whole fours
    bool wide = s.head_dim * s.states % 4 == 0;
    for (const void* q : {(const void*)forward.initial, (const void*)forward.last, (const void*)reverse.initial,
                          (const void*)reverse.last})
      wide = wide && reinterpret_cast<uintptr_t>(q) % 16 == 0;
    const int vec = wide ? 4 : 1;
    auto* kernel = wide ? &k_join<4> : &k_join<1>;
    kernel<<<dim3((size / vec + 255) / 256, s.seqs, g ? 2 : 1), 256, 0, stream>>>(
        forward, reverse, at<float>(p.decays), first(), p.segments, size, s.head_dim * s.states, s.heads);
    hip_check(hipGetLastError(), "scan state join");
  }
};

}  // namespace

size_t scan_workspace(const Scan& s, bool backward) { return make_plan(s, backward).total; }

void scan(const Scan& s, void* y, float* final_state, void* workspace, hipStream_t stream) {
  const Plan p = make_plan(s, false);
  const Sweep sweep(s, p, (char*)workspace);
  sweep.make_items(stream);
  if (p.by_item) sweep.carry(final_state, nullptr, stream);
  SweepArgs a = sweep.with(p.value, s.b, s.c, s.x, s.x);
  a.wide_out = s.head_dim % 4 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  a.d = s.d;
  a.state_in = p.by_item ? sweep.at<float>(p.states) : s.initial;
  a.state_out = p.by_item ? nullptr : final_state;
  a.out = y;
  launch_forward(s.dtype, a, p.items, stream);
}

void scan_backward(const Scan& s, const ScanGrads& g, void* workspace, hipStream_t stream) {
  const Plan p = make_plan(s, true);
  const Sweep sweep(s, p, (char*)workspace);
  sweep.make_items(stream);
  if (p.by_item) sweep.carry(sweep.at<float>(p.last), &g, stream);
  const float* states = p.by_item ? sweep.at<float>(p.states) : s.initial;
  const float* adjoints = p.by_item ? sweep.at<float>(p.adjoints) : g.dfinal;

  SweepArgs x = sweep.with(p.value, s.c, s.b, g.dy, s.x);
  x.wide_out = s.head_dim % 4 == 0 && reinterpret_cast<uintptr_t>(g.dx) % 16 == 0;
  x.d = s.d;
  x.state_in = adjoints;
  x.state_out = p.by_item ? nullptr : g.dinitial;
  x.out = g.dx;
  x.dwrite_part = sweep.at<float>(p.dwrite);
  x.gate_part = sweep.at<float>(p.gate_out);
  x.dd_part = sweep.at<float>(p.dd);
  x.windows = p.windows;
  x.first = sweep.first();
  x.end_states = states;
  x.last_states = sweep.at<float>(p.last);
  x.initial = s.initial;
  x.crossings = sweep.at<Crossing>(p.crossings);
  if (p.windows > 1) x.marks = sweep.at<float>(p.mark_adjoints);

  SweepArgs c = sweep.with(p.query, s.b, s.c, s.x, g.dy);
  c.state_in = states;
  c.state_out = p.by_item || !g.dfinal ? nullptr : sweep.at<float>(p.last);
  c.out = sweep.at<float>(p.parts_c);
  c.wide_out = s.states % 4 == 0;
  c.gate_part = sweep.at<float>(p.gate_in);
  if (p.windows > 1) c.marks = sweep.at<float>(p.mark_states);

  SweepArgs b = sweep.with(p.query, s.c, s.b, g.dy, s.x);
  b.state_in = adjoints;
  b.out = sweep.at<float>(p.parts_b);
  b.wide_out = s.states % 4 == 0;
  const int64_t across = (s.heads + FINISH_HEADS - 1) / FINISH_HEADS, windows = (int64_t)p.items * p.windows;
  const int64_t sums = (s.all_tokens() * s.groups * s.states + 4 * FINISH_THREADS - 1) / (4 * FINISH_THREADS);
  const int64_t grid = 2 * sums + windows * across + (g.dd ? across : 0);
  if (grid > INT32_MAX) throw ArgError("too many tokens and heads for one call");
  launch_backward(s.dtype, c, b, x, p.items, stream);
  const bool ends = !p.by_item && g.dfinal;
  if (x.marks || ends) {
    k_cross<<<(uint32_t)(windows * across), 256, 0, stream>>>(
        x, Marks{x.marks, c.marks, ends ? g.dfinal : nullptr, sweep.at<float>(p.last)});
    hip_check(hipGetLastError(), "scan crossings");
  }

  Finish f{};
  f.size = s.all_tokens() * s.groups * s.states;
  f.parts = p.query.blocks;
  f.items = p.items;
  f.entering_tiles = p.query.col_tiles;
  f.ends = p.by_item || g.dfinal;
  f.sums = (uint32_t)sums;
  f.group = std::max(1, WINDOW / p.length);
  f.parts_c = (const float*)c.out;
  f.parts_b = (const float*)b.out;
  f.dc = g.dc;
  f.db = g.db;
  f.entering = c.gate_part;
  f.leaving = x.gate_part;
  f.dwrite = g.dwrite;
  f.ddecay = g.ddecay;
  f.dd = g.dd;
  if (s.dtype == BF16) k_finish<bf16><<<(uint32_t)grid, FINISH_THREADS, 0, stream>>>(x, f);
  else k_finish<float><<<(uint32_t)grid, FINISH_THREADS, 0, stream>>>(x, f);
  hip_check(hipGetLastError(), "scan gradients");
}

}  // namespace fhe::clear
