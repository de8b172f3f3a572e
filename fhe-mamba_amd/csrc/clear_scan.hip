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
// dg_r is the sum of M over t >= r > s: what crosses the segment's end,
// <A, h> there, plus the sums over t >= r of what enters at t less what leaves.
// Terms with s = t are in neither, and the sums restart in every segment.
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

__global__ __launch_bounds__(256) void k_join(Join forward, Join reverse, const float* decay, const int* first,
                                              int segments, int size, int per_head, int heads) {
  const int e = blockIdx.x * 256 + threadIdx.x, seq = blockIdx.y;
  if (e >= size) return;
  const bool rev = blockIdx.z;
  const Join j = rev ? reverse : forward;
  const int head = e / per_head;
  const int from = first ? first[seq] : seq * segments;
  const int count = first ? first[seq + 1] - from : segments;
  float run = j.initial ? j.initial[(int64_t)seq * size + e] : 0.0f;
  for (int i0 = 0; i0 < count; i0 += 8) {
    float add[8], keep[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = min(i0 + u, count - 1), item = from + (rev ? count - 1 - i : i);
      add[u] = j.states[(int64_t)item * size + e];
      keep[u] = decay[(int64_t)item * heads + head];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < count) {
        const int item = from + (rev ? count - 1 - i0 - u : i0 + u);
        j.states[(int64_t)item * size + e] = run;
        run = run * keep[u] + add[u];
      }
  }
  if (j.last) j.last[(int64_t)seq * size + e] = run;
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

__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
  for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// What is left when the sweeps are done: workgroups [0, 2 sums) sum the parts of
// dC and then of dB, the next the gates' gradients of an item and head each, the
// last the gradient of D a head each.
struct Finish {
  int64_t size;  // of dB and dC
  int parts, items, entering_tiles;
  uint32_t sums;  // workgroups of one of the two
  const float *parts_c, *parts_b;
  void *dc, *db;
  const int* first;
  const float *entering, *leaving, *adjoint, *states, *last;
  float *dwrite, *ddecay, *dd;
};

// Gradients of write and log_decay of one item and head: the first summed over
// the head's channels, the second from the segment's end backwards.
__device__ __forceinline__ void gate_grads(const SweepArgs& a, const Finish& f, int item_i, int head,
                                           double* scratch) {
  const Item it = find_item(a, item_i);
  if (it.count <= 0) return;
  const int64_t token0 = item_token(a, it);
  const int64_t size = (int64_t)a.head_dim * a.states, all = size * a.heads;
  double carry = 0.0;
  if (f.adjoint && it.live) {
    const float* A = f.adjoint + (a.by_item ? item_i : it.seq) * all + head * size;
    const bool more = a.by_item && (a.table ? item_i + 1 < f.first[it.seq + 1] : (item_i + 1) % a.segments != 0);
    const float* h = (more ? f.states + (item_i + 1) * all : f.last + it.seq * all) + head * size;
    for (int64_t e = threadIdx.x; e < size; e += 256) carry += (double)A[e] * h[e];
    carry = block_sum(carry, scratch);
  }
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  for (int end = it.count; end > 0; end -= 256) {
    const int t = end - 1 - (int)threadIdx.x;  // the last token first
    double v = 0.0;
    if (t >= 0) {
      float dw = 0.0f;
      for (int p = 0; p < a.col_tiles; ++p) {
        const int64_t at = ((int64_t)head * a.col_tiles + p) * a.all_tokens + token0 + t;
        v += (double)f.leaving[at];
        dw += a.dwrite_part[at];
      }
      for (int p = 0; p < f.entering_tiles; ++p)
        v += (double)f.entering[((int64_t)head * f.entering_tiles + p) * a.all_tokens + token0 + t];
      f.dwrite[(token0 + t) * a.heads + head] = dw;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double up = __shfl_up(v, d);
      if (lane >= d) v += up;
    }
    __syncthreads();
    if (lane == 63) scratch[wave] = v;
    __syncthreads();
    double before = carry;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += scratch[w];
      carry += scratch[w];
    }
    if (t >= 0) f.ddecay[(token0 + t) * a.heads + head] = (float)(before + v);
  }
}

__device__ __forceinline__ void skip_grad(const SweepArgs& a, const Finish& f, int head, double* scratch) {
  double v = 0.0;
  for (int i = threadIdx.x; i < f.items; i += 256) {
    const Item it = find_item(a, i);
    if (!it.live) continue;
    for (int p = 0; p < a.col_tiles; ++p) v += a.dd_part[((int64_t)i * a.heads + head) * a.col_tiles + p];
  }
  v = block_sum(v, scratch);
  if (threadIdx.x == 0) f.dd[head] = (float)v;
}

template <class T>
__global__ __launch_bounds__(256) void k_finish(SweepArgs a, Finish f) {
  __shared__ double scratch[4];
  uint32_t block = blockIdx.x;
  if (block < 2 * f.sums) {
    const bool is_b = block >= f.sums;
    const int64_t i = ((int64_t)(is_b ? block - f.sums : block) * 256 + threadIdx.x) * 4;
    sum_parts<T>(is_b ? f.parts_b : f.parts_c, f.parts, f.size, (T*)(is_b ? f.db : f.dc), i);
    return;
  }
  block -= 2 * f.sums;
  const uint32_t gates = (uint32_t)f.items * a.heads;
  if (block < gates) gate_grads(a, f, (int)(block / a.heads), (int)(block % a.heads), scratch);
  else skip_grad(a, f, (int)(block - gates), scratch);
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
  bool by_item;
  // workspace, in bytes
  size_t table, first, decays, states, adjoints, last, dwrite, gate_out, gate_in, dd, parts_c, parts_b, total;
};

// Tokens of a segment: a whole sequence where the sequences alone fill half of
// the chip's places for workgroups (two a CU), else as many chunks as leave
// about three workgroups a CU: lengths are whole chunks and sequences ragged, and
// with fewer the last round is half empty.  Each segment's states are written
// and read twice, which holds the number down.  us of all launches, two / three /
// four a CU: 30011 packed tokens of 24 heads 314 / 265 / 265, the gradients of
// 4 x 2048 349 / 313 / 314.
int segment_length(int64_t all, int64_t longest, int seqs, int64_t per_item, bool packed) {
  constexpr int64_t WANT = 768, ENOUGH = 256;
  if (!packed && seqs * per_item >= ENOUGH) return (int)std::max<int64_t>(longest, 1);
  const int64_t items = std::max<int64_t>(1, WANT / per_item);
  const int64_t chunks = (all + CHUNK - 1) / CHUNK;
  const int64_t len = std::max<int64_t>(1, (chunks + items - 1) / items) * CHUNK;
  return (int)std::min<int64_t>(len, std::max<int64_t>(longest, 1));
}

Plan make_plan(const Scan& s, bool backward) {
  Plan p{};
  const bool packed = s.offsets != nullptr;
  p.value = Cut(s, VALUE_COLS);
  // 64 channels take all of a head's registers there are, and halve the sums
  // over wavefronts and the parts: 146 us for both sweeps and their sums at
  // 4 x 2048 tokens of 24 heads of 64, 32 channels 183
  p.query = Cut(s, s.head_dim <= 32 ? 32 : 64);
  const int64_t all = s.all_tokens();
  p.length = segment_length(all, s.tokens, s.seqs, (int64_t)p.value.blocks * s.groups, packed);
  p.segments = packed ? 0 : std::max<int>(1, (int)((s.tokens + p.length - 1) / p.length));
  p.by_item = p.length < s.tokens;
  p.items = packed ? (int)(s.tokens / p.length) + s.seqs + 2 : s.seqs * p.segments;
  const size_t state = (size_t)s.heads * s.head_dim * s.states * 4;
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
    k_join<<<dim3((size + 255) / 256, s.seqs, g ? 2 : 1), 256, 0, stream>>>(
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

  SweepArgs c = sweep.with(p.query, s.b, s.c, s.x, g.dy);
  c.state_in = states;
  c.state_out = p.by_item || !g.dfinal ? nullptr : sweep.at<float>(p.last);
  c.out = sweep.at<float>(p.parts_c);
  c.wide_out = s.states % 4 == 0;
  c.gate_part = sweep.at<float>(p.gate_in);

  SweepArgs b = sweep.with(p.query, s.c, s.b, g.dy, s.x);
  b.state_in = adjoints;
  b.out = sweep.at<float>(p.parts_b);
  b.wide_out = s.states % 4 == 0;
  launch_backward(s.dtype, c, b, x, p.items, stream);

  Finish f{};
  f.size = s.all_tokens() * s.groups * s.states;
  f.parts = p.query.blocks;
  f.items = p.items;
  f.entering_tiles = p.query.col_tiles;
  f.sums = (uint32_t)((f.size + 1023) / 1024);
  f.parts_c = (const float*)c.out;
  f.parts_b = (const float*)b.out;
  f.dc = g.dc;
  f.db = g.db;
  f.first = sweep.first();
  f.entering = c.gate_part;
  f.leaving = x.gate_part;
  f.adjoint = adjoints;
  f.states = states;
  f.last = sweep.at<float>(p.last);
  f.dwrite = g.dwrite;
  f.ddecay = g.ddecay;
  f.dd = g.dd;
  const int64_t grid = 2 * (int64_t)f.sums + (int64_t)p.items * s.heads + (g.dd ? s.heads : 0);
  if (grid > INT32_MAX) throw ArgError("too many tokens and heads for one call");
  if (s.dtype == BF16) k_finish<bf16><<<(uint32_t)grid, 256, 0, stream>>>(x, f);
  else k_finish<float><<<(uint32_t)grid, 256, 0, stream>>>(x, f);
  hip_check(hipGetLastError(), "scan gradients");
}

}  // namespace fhe::clear
