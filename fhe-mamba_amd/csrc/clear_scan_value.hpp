// Sweeps over the chunks of a segment with the state in registers: the scan's
// results, and the state that a segment leaves.
#pragma once

#include "clear_scan.hpp"

#pragma clang fp contract(fast)
namespace fhe::clear {
namespace {

template <class T, int NB, int PT, bool VALUES>
struct ValueLds {
  using Key = Tile<T, 32 * NB>;
  using Value = Tile<T, 16 * PT>;
  // 16-byte rows: a tile that a kernel does not have must not shift the others
  alignas(16) T key[CHUNK * Key::PITCH];
  alignas(16) T query[VALUES ? CHUNK * Key::PITCH : 1];
  alignas(16) T value[WAVES][CHUNK * Value::PITCH];
  alignas(16) Gates gates[WAVES];
};

// Adds a chunk to a wavefront's state [states][channels]:
// h <- total h + sum_s key_s (factor_s value_s).
template <class T, int NB, int PT, bool REV>
__device__ __forceinline__ void add_chunk(f32x4 (&h)[2 * NB][PT], const T* key, const T* value, const Gates& t,
                                          int n) {
  using N = Num<T>;
  const float total = t.total();
#pragma unroll
  for (int nt = 0; nt < 2 * NB; ++nt)
#pragma unroll
    for (int p = 0; p < PT; ++p) h[nt][p] *= total;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (32 * m >= n) break;
    const f32x8 f = to_state<REV>(t, m);
    Split<T, N::FULL> s[PT];
#pragma unroll
    for (int p = 0; p < PT; ++p)
      s[p] = split<T, N::FULL>(widen(Tile<T, 16 * PT>::cols(value, 32 * m, 16 * p)) * f);
#pragma unroll
    for (int nt = 0; nt < 2 * NB; ++nt) {
      if (REV && nt % 2 == 0) step_end();
      const auto k = Tile<T, 32 * NB>::cols(key, 32 * m, 16 * nt);
#pragma unroll
      for (int p = 0; p < PT; ++p) h[nt][p] = mma<T, N::FULL>(k, s[p], h[nt][p]);
    }
  }
}

// State tiles (rows 4 q + r the states, column l the channel) to and from
// [head_dim][states].
template <int NB, int PT, bool FULL>
__device__ __forceinline__ void state_io(f32x4 (&h)[2 * NB][PT], const float* from, float* to, int p0,
                                         int head_dim, int states, int lane) {
  const int q = lane >> 4, l = lane & 15;
  const bool wide = FULL || (states % 4 == 0 && reinterpret_cast<uintptr_t>(to ? to : from) % 16 == 0);
#pragma unroll
  for (int p = 0; p < PT; ++p) {
    const int row = p0 + 16 * p + l;
    if (!FULL && row >= head_dim) continue;
#pragma unroll
    for (int nt = 0; nt < 2 * NB; ++nt) {
      const int n = 16 * nt + 4 * q;
      const int64_t at = (int64_t)row * states + n;
      const int left = FULL ? 4 : states - n;
      if (to) store4(to + at, h[nt][p], left, wide);
      else h[nt][p] = load4(from + at, left, wide);
    }
  }
}

// The products of a state's tiles and those of another at `with`.
template <int NB, int PT, bool FULL>
__device__ __forceinline__ Crossing state_dot(const f32x4 (&h)[2 * NB][PT], const float* with, int p0, int head_dim,
                                              int states, int lane) {
  const int q = lane >> 4, l = lane & 15;
  const bool wide = FULL || (states % 4 == 0 && reinterpret_cast<uintptr_t>(with) % 16 == 0);
  double sum = 0.0;
  float squares = 0.0f;
#pragma unroll
  for (int p = 0; p < PT; ++p) {
    const int row = p0 + 16 * p + l;
    if (!FULL && row >= head_dim) continue;
#pragma unroll
    for (int nt = 0; nt < 2 * NB; ++nt) {
      const int n = 16 * nt + 4 * q;
      const f32x4 o = load4(with + (int64_t)row * states + n, FULL ? 4 : states - n, wide);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sum += (double)h[nt][p][r] * o[r];
        squares += h[nt][p][r] * o[r] * (h[nt][p][r] * o[r]);
      }
    }
  }
  return {wave_sum(sum), wave_sum((double)squares)};
}

// In reverse a wavefront holds all the registers there are, and step_end() keeps the
// scheduler from asking for many more: at 128 states the gradients' kernel spills 36 in
// 16 bits and 146 in 32, without step_end() 76 and 269.
//
// y (or, in reverse, the gradient of x) of a segment, 16 PT channels of one head
// a wavefront, four wavefronts of one group on shared keys and queries.
template <class T, int NB, int PT, bool REV, bool VALUES, bool FULL>
__device__ __forceinline__ void value_sweep(const SweepArgs& a, char* lds_raw, uint32_t id) {
  using N = Num<T>;
  using Frag = typename N::Frag;
  using Lds = ValueLds<T, NB, PT, VALUES>;
  // in reverse the results end in the gates' gradients too
  constexpr int PIECES = REV ? N::FULL : N::FAIR;
  using Key = typename Lds::Key;
  using Value = typename Lds::Value;
  Lds& lds = *reinterpret_cast<Lds*>(lds_raw);

  const Place at(a, id);
  const Item it = at.it;
  if (it.count <= 0 && it.seq < 0) return;
  const int lane = lane_id(), q = lane >> 4, l = lane & 15;
  const T* key = (const T*)a.key.p + item_at(a, a.key, it) + at.group * a.key.head;
  const T* query = VALUES ? (const T*)a.query.p + item_at(a, a.query, it) + at.group * a.query.head : nullptr;
  const T* value = (const T*)a.value.p + item_at(a, a.value, it) + at.head * a.value.head + at.p0;
  const T* other =
      VALUES && REV ? (const T*)a.other.p + item_at(a, a.other, it) + at.head * a.other.head + at.p0 : nullptr;
  const float* write = (const float*)a.write.p + item_at(a, a.write, it) + at.head * a.write.head;
  const float* decay = (const float*)a.decay.p + item_at(a, a.decay, it) + at.head * a.decay.head;
  T* out = VALUES ? (T*)a.out + (at.token0 * a.heads + at.head) * a.head_dim + at.p0 : nullptr;
  const int64_t out_tok = (int64_t)a.heads * a.head_dim;
  const uint32_t out_at = (uint32_t)(l * out_tok + 4 * q) * (uint32_t)sizeof(T);  // a lane's place in 16 rows
  float* dwrite = VALUES && REV ? a.dwrite_part + at.part * a.all_tokens + at.token0 : nullptr;
  float* gate_grad = VALUES && REV ? a.gate_part + at.part * a.all_tokens + at.token0 : nullptr;
  const int width = FULL ? 16 * PT : at.width;
  const float skip = VALUES && a.d && at.active ? a.d[at.head] : 0.0f;

  f32x4 h[2 * NB][PT] = {};
  if (VALUES && a.state_in && at.active && it.live)
    state_io<NB, PT, FULL>(h, a.state_in + at.state_at, nullptr, at.p0, a.head_dim, a.states, lane);

  T* vt = lds.value[at.wave];
  Gates& t = lds.gates[at.wave];
  float dd = 0.0f;
  double log_total = 0.0;
  const int chunks = (it.count + CHUNK - 1) / CHUNK;
  for (int c = 0; c < chunks || (VALUES && REV); ++c) {
    if constexpr (VALUES && REV) {
      // what crosses a cut segment's end and a sequence's beginning, whose states are known
      if (at.active && it.live && (c == 0 || c == chunks)) {
        const float* with = nullptr;
        const int number = a.by_item ? a.number(at.item, it.seq) : 0;
        const int64_t all = (int64_t)a.heads * a.head_dim * a.states;
        if (c == chunks) with = number == 0 && a.initial ? a.initial + it.seq * all : nullptr;
        else if (a.by_item && number == a.items_of(it.seq) - 1) with = a.last_states + it.seq * all;
        else if (a.by_item) with = a.end_states + (at.item + 1) * all;
        if (with) {
          step_end();
          const Crossing x = state_dot<NB, PT, FULL>(h, with + (int64_t)at.head * a.head_dim * a.states, at.p0,
                                                     a.head_dim, a.states, lane_here());
          if (lane == 0) a.crossing(at.item, c == chunks ? 0 : a.windows, at.head)[at.p0 / a.cols] = x;
          step_end();
        }
      }
      if (c == chunks) break;
    }
    const int first = (REV ? chunks - 1 - c : c) * CHUNK;
    const int n = min(CHUNK, it.count - first), live = it.live ? n : 0;
    {
      Stage<T, 32 * NB, 64 * WAVES, FULL> sk, sq;
      Stage<T, 16 * PT, 64, FULL> sv;
      float g = 0.0f, w = 0.0f;
      if (at.active && lane < live) {
        g = decay[(int64_t)(first + lane) * a.decay.tok];
        w = write[(int64_t)(first + lane) * a.write.tok];
      }
      sk.load(key + first * a.key.tok, a.key.tok, live, a.states, a.wide_key, threadIdx.x);
      if constexpr (VALUES)
        sq.load(query + first * a.query.tok, a.query.tok, live, a.states, a.wide_query, threadIdx.x);
      sv.load(value + first * a.value.tok, a.value.tok, live, at.width, a.wide_value, lane);
      __syncthreads();
      if (at.active) make_gates<REV>(t, g, w);
      sk.store(lds.key, threadIdx.x);
      if constexpr (VALUES) sq.store(lds.query, threadIdx.x);
      sv.store(vt, lane);
      __syncthreads();
    }
    if (!at.active) continue;

    if constexpr (VALUES) {
      // what the state before the chunk gives: rows 4 q + r the channels, columns
      // l the tokens, so that a lane has four neighbouring channels of its token
      f32x4 y[TILES][PT] = {};
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        Split<T, PIECES> state[PT];
#pragma unroll
        for (int p = 0; p < PT; ++p) state[p] = split<T, PIECES>(join(h[2 * k][p], h[2 * k + 1][p]));
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const Frag qf = Key::rows(lds.query, 16 * i, 32 * k);
#pragma unroll
          for (int p = 0; p < PT; ++p) y[i][p] = mma<T, PIECES>(state[p], qf, y[i][p]);
        }
      }
      f32x4 row_sum[REV ? TILES : 1] = {};
      float gate[REV ? TILES : 1] = {};
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        if (16 * i >= n) break;
        if constexpr (REV) step_end();
        const int tok = 16 * i + l;
        const float inside = t.template inside<REV>(i, tok), in = inside * t.template into<REV>(i), w = t.w[tok];
        Frag of[REV ? PT / 2 : 1];
        if constexpr (REV) {
#pragma unroll
          for (int k = 0; k < PT / 2; ++k)
            of[k] = row_frag<T, FULL>(other + (int64_t)(first + 16 * i) * a.other.tok + 32 * k, a.other.tok,
                                      live - 16 * i, width - 32 * k, a.wide_other);
        }
#pragma unroll
        for (int p = 0; p < PT; ++p) {
          y[i][p] *= in;
          if constexpr (REV) {
            const f32x4 x = half_of(of[p / 2], p % 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) gate[i] -= w * (y[i][p][r] * x[r]);
          }
        }
        // and the tokens of the chunk
        if constexpr (REV) step_end();
        Frag qf[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) qf[k] = Key::rows(lds.query, 16 * i, 32 * k);
        f32x4 pairs[TILES] = {};
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
          if (REV ? j < i : j > i) continue;
          if constexpr (REV) step_end();
          f32x4 s = {};
#pragma unroll
          for (int k = 0; k < NB; ++k) s = N::mma(Key::rows(lds.key, 16 * j, 32 * k), qf[k], s);
          pairs[j] = decayed<REV>(t, s, i, j, inside);
          if constexpr (REV) {  // the pairs' own parts of the loss, off the diagonal
            f32x4 z = {};
#pragma unroll
            for (int k = 0; k < PT / 2; ++k) z = N::mma(Value::rows(vt, 16 * j, 32 * k), of[k], z);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float m = i == j && 4 * q + r == l ? 0.0f : pairs[j][r] * z[r] * w;
              row_sum[j][r] += m;
              gate[i] -= m;
            }
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if (REV ? 2 * m + 1 < i : 2 * m > i) continue;
          const auto s = split<T, PIECES>(join(pairs[2 * m], pairs[2 * m + 1]));
#pragma unroll
          for (int p = 0; p < PT; ++p)
            y[i][p] = mma<T, PIECES>(Value::cols(vt, 32 * m, 16 * p), s, y[i][p]);
        }
        if constexpr (REV) step_end();
        Frag vf[PT / 2];
#pragma unroll
        for (int k = 0; k < PT / 2; ++k) vf[k] = Value::rows(vt, 16 * i, 32 * k);
        float against = 0.0f;
#pragma unroll
        for (int p = 0; p < PT; ++p) {
          const f32x4 mine = half_of(vf[p / 2], p % 2);
          if constexpr (REV) {
            const f32x4 x = half_of(of[p / 2], p % 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              against += y[i][p][r] * x[r];
              dd += mine[r] * x[r];
              y[i][p][r] *= w;
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) y[i][p][r] += skip * mine[r];
        }
        if constexpr (REV) against = sum_groups(against);
        if (tok < n) {
          T* rows = out + (int64_t)(first + 16 * i) * out_tok;
          T* to = FULL ? reinterpret_cast<T*>(reinterpret_cast<char*>(rows) + out_at) : rows + l * out_tok + 4 * q;
#pragma unroll
          for (int p = 0; p < PT; ++p) store4(to + 16 * p, y[i][p], width - 16 * p - 4 * q, FULL || a.wide_out);
          if constexpr (REV) {
            if (q == 0) (dwrite + first + 16 * i)[l] = against;
          }
        }
      }
      if constexpr (REV) {
        wave_sync();  // the sums of logarithms are read for the last time: their place is free
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float sum = sum16(row_sum[i][r]);
            if (l == 0) t.g[16 * i + 4 * q + r] = sum;
          }
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const float sum = sum_groups(gate[i]) + (float)t.g[16 * i + l];
          if (q == 0 && 16 * i + l < n) (gate_grad + first + 16 * i)[l] = sum;
        }
      }
    } else {
      log_total += t.ends[TILES];
    }
    add_chunk<T, NB, PT, REV>(h, lds.key, vt, t, n);
    // the adjoint behind the tokens before the chunk, where the gates' gradients start again
    if constexpr (VALUES && REV) {
      if (a.marks && first % WINDOW == 0 && first > 0 && it.live)
        state_io<NB, PT, FULL>(h, nullptr, a.marks + at.mark_at(a, first), at.p0, a.head_dim, a.states, lane_here());
    }
  }
  if (!at.active) return;
  if (a.state_out && (a.by_item || it.live))
    state_io<NB, PT, FULL>(h, nullptr, a.state_out + at.state_at, at.p0, a.head_dim, a.states, lane);
  if constexpr (!VALUES) {
    if (lane == 0 && at.p0 == 0) a.decay_out[(int64_t)at.item * a.heads + at.head] = exp2d(log_total);
  }
  if constexpr (VALUES && REV) {
    dd = sum_groups(sum16(dd));
    if (lane == 0) a.dd_part[(int64_t)at.item * a.heads * a.col_tiles + at.part] = dd;
  }
}

}  // namespace
}  // namespace fhe::clear
