// Sweeps that give the gradients of the scan's queries: forward those of C, and
// in reverse, where keys and queries change places, those of B.
#pragma once

#include "clear_scan.hpp"

#pragma clang fp contract(fast)
namespace fhe::clear {
namespace {

template <class T, int NB, int PT>
struct QueryLds {
  using Key = Tile<T, 32 * NB>;
  using Value = Tile<T, 16 * PT>;
  static constexpr int ROUND = NB < 2 ? 2 * NB : 4;  // tiles of states summed over the wavefronts at a time
  static constexpr int SUM = 16 * ROUND + 4;
  alignas(16) T key[CHUNK * Key::PITCH];
  alignas(16) T value[WAVES][CHUNK * Value::PITCH];
  alignas(16) float sum[WAVES][16 * SUM];
  alignas(16) Gates gates[WAVES];
};

// State tiles (rows 4 q + r the channel, column l the state) from and to
// [head_dim][states].
template <int NB, int PT>
__device__ __forceinline__ void channel_state_io(f32x4 (&h)[PT][2 * NB], const float* from, float* to, int p0,
                                         int head_dim, int states, int lane) {
  const int q = lane >> 4, l = lane & 15;
#pragma unroll
  for (int p = 0; p < PT; ++p)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = p0 + 16 * p + 4 * q + r;
#pragma unroll
      for (int nt = 0; nt < 2 * NB; ++nt) {
        const int n = 16 * nt + l;
        if (row < head_dim && n < states) {
          if (to) to[(int64_t)row * states + n] = h[p][nt][r];
          else h[p][nt][r] = from[(int64_t)row * states + n];
        }
      }
    }
}

// Target t's gradient from 16 PT channels of one head,
//   in_t sum_p other[t][p] h[p] + sum_s decay(t, s) (other_t . value_s) key_s,
// summed over a workgroup's wavefronts and written for each workgroup of a
// group; forward also the part of the gates' gradient that the state before the
// chunk has in it.
template <class T, int NB, int PT, bool REV, bool FULL>
__device__ __forceinline__ void query_sweep(const SweepArgs& a, char* lds_raw, uint32_t id) {
  using N = Num<T>;
  using Frag = typename N::Frag;
  using Lds = QueryLds<T, NB, PT>;
  // forward the state's part ends in the gates' gradients too
  constexpr int STATE = REV ? N::FAIR : N::FULL, PAIRS = N::FAIR;
  using Key = typename Lds::Key;
  using Value = typename Lds::Value;
  Lds& lds = *reinterpret_cast<Lds*>(lds_raw);

  const Place at(a, id);
  const Item it = at.it;
  if (it.count <= 0 && it.seq < 0) return;
  const int lane = lane_id(), q = lane >> 4, l = lane & 15;
  const T* key = (const T*)a.key.p + item_at(a, a.key, it) + at.group * a.key.head;
  const T* query = REV ? nullptr : (const T*)a.query.p + item_at(a, a.query, it) + at.group * a.query.head;
  const T* value = (const T*)a.value.p + item_at(a, a.value, it) + at.head * a.value.head + at.p0;
  const T* other = (const T*)a.other.p + item_at(a, a.other, it) + at.head * a.other.head + at.p0;
  const float* write = (const float*)a.write.p + item_at(a, a.write, it) + at.head * a.write.head;
  const float* decay = (const float*)a.decay.p + item_at(a, a.decay, it) + at.head * a.decay.head;
  float* out =
      (float*)a.out + (((int64_t)at.block * a.all_tokens + at.token0) * a.groups + at.group) * a.states;
  const int64_t out_tok = (int64_t)a.groups * a.states;
  float* gate_grad = REV ? nullptr : a.gate_part + at.part * a.all_tokens + at.token0;

  f32x4 h[PT][2 * NB] = {};
  if (a.state_in && at.active && it.live)
    channel_state_io<NB, PT>(h, a.state_in + at.state_at, nullptr, at.p0, a.head_dim, a.states, lane);

  T* vt = lds.value[at.wave];
  Gates& t = lds.gates[at.wave];
  const int chunks = (it.count + CHUNK - 1) / CHUNK;
  for (int c = 0; c < chunks; ++c) {
    const int first = (REV ? chunks - 1 - c : c) * CHUNK;
    const int n = min(CHUNK, it.count - first), live = it.live ? n : 0;
    {
      Stage<T, 32 * NB, 64 * WAVES, FULL> sk;
      Stage<T, 16 * PT, 64, FULL> sv;
      float g = 0.0f, w = 0.0f;
      if (at.active && lane < live) {
        g = decay[(int64_t)(first + lane) * a.decay.tok];
        w = write[(int64_t)(first + lane) * a.write.tok];
      }
      sk.load(key + first * a.key.tok, a.key.tok, live, a.states, a.wide_key, threadIdx.x);
      sv.load(value + first * a.value.tok, a.value.tok, live, at.width, a.wide_value, lane);
      __syncthreads();
      if (at.active) make_gates<REV>(t, g, w);
      sk.store(lds.key, threadIdx.x);
      sv.store(vt, lane);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      if (16 * i >= n) break;
      step_end();
      const int tok = 16 * i + l;
      f32x4 got[2 * NB] = {};
      if (at.active) {
        Frag of[PT / 2];
#pragma unroll
        for (int k = 0; k < PT / 2; ++k)
          of[k] = row_frag<T, FULL>(other + (int64_t)(first + 16 * i) * a.other.tok + 32 * k, a.other.tok,
                                    live - 16 * i, at.width - 32 * k, a.wide_other);
        const float inside = t.template inside<REV>(i, tok), in = inside * t.template into<REV>(i);
#pragma unroll
        for (int nt = 0; nt < 2 * NB; ++nt) {
#pragma unroll
          for (int k = 0; k < PT / 2; ++k)
            got[nt] = mma<T, STATE>(split<T, STATE>(join(h[2 * k][nt], h[2 * k + 1][nt])), of[k], got[nt]);
          got[nt] *= in;
        }
        if constexpr (!REV) {
          float sum = 0.0f;
#pragma unroll
          for (int k = 0; k < NB; ++k) {
            const Frag qf = row_frag<T, FULL>(query + (int64_t)(first + 16 * i) * a.query.tok + 32 * k, a.query.tok,
                                              live - 16 * i, a.states - 32 * k, a.wide_query);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const f32x4 v = half_of(qf, half);
#pragma unroll
              for (int r = 0; r < 4; ++r) sum += got[2 * k + half][r] * v[r];
            }
          }
          sum = sum_groups(sum);
          if (q == 0 && tok < n) (gate_grad + first + 16 * i)[l] = sum;
        }
        f32x4 pairs[TILES] = {};
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
          if (REV ? j < i : j > i) continue;
          f32x4 z = {};
#pragma unroll
          for (int k = 0; k < PT / 2; ++k) z = N::mma(Value::rows(vt, 16 * j, 32 * k), of[k], z);
          pairs[j] = decayed<REV>(t, z, i, j, inside);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if (REV ? 2 * m + 1 < i : 2 * m > i) continue;
          const auto s = split<T, PAIRS>(join(pairs[2 * m], pairs[2 * m + 1]));
#pragma unroll
          for (int nt = 0; nt < 2 * NB; ++nt)
            got[nt] = mma<T, PAIRS>(Key::cols(lds.key, 32 * m, 16 * nt), s, got[nt]);
        }
        if constexpr (REV) {
          const float w = t.w[tok];
#pragma unroll
          for (int nt = 0; nt < 2 * NB; ++nt) got[nt] *= w;
        }
      }
#pragma unroll
      for (int n0 = 0; n0 < 2 * NB; n0 += Lds::ROUND) {
#pragma unroll
        for (int nt = 0; nt < Lds::ROUND; ++nt)
          *reinterpret_cast<f32x4*>(&lds.sum[at.wave][l * Lds::SUM + 16 * nt + 4 * q]) = got[n0 + nt];
        __syncthreads();
        const int row = threadIdx.x / (4 * Lds::ROUND), col = threadIdx.x % (4 * Lds::ROUND) * 4;
        if (row < 16 && 16 * i + row < n) {
          f32x4 sum = {};
#pragma unroll
          for (int w = 0; w < WAVES; ++w) sum += *reinterpret_cast<const f32x4*>(&lds.sum[w][row * Lds::SUM + col]);
          const int at_n = 16 * n0 + col;
          store4(out + (first + 16 * i + row) * out_tok + at_n, sum, (FULL ? 32 * NB : a.states) - at_n,
                 FULL || a.wide_out);
        }
        __syncthreads();
      }
    }
    if (!at.active) continue;
    // h <- total h + sum_s (factor_s value_s) key_s
    const float total = t.total();
#pragma unroll
    for (int p = 0; p < PT; ++p)
#pragma unroll
      for (int nt = 0; nt < 2 * NB; ++nt) h[p][nt] *= total;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (32 * m >= n) break;
      const f32x8 f = to_state<REV>(t, m);
#pragma unroll
      for (int p2 = 0; p2 < PT; p2 += 2) {
        step_end();
        Split<T, N::FULL> s[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const Frag v = Value::cols(vt, 32 * m, 16 * (p2 + p));
          s[p] = split<T, N::FULL>(widen(v) * f);
        }
#pragma unroll
        for (int nt = 0; nt < 2 * NB; ++nt) {
          const auto k = Key::cols(lds.key, 32 * m, 16 * nt);
#pragma unroll
          for (int p = 0; p < 2; ++p) h[p2 + p][nt] = mma<T, N::FULL>(s[p], k, h[p2 + p][nt]);
        }
      }
    }
    // the state behind the chunk, where the gates' gradients start again
    if constexpr (!REV) {
      const int end = first + CHUNK;
      if (a.marks && end % WINDOW == 0 && end < it.count && it.live)
        channel_state_io<NB, PT>(h, nullptr, a.marks + at.mark_at(a, end), at.p0, a.head_dim, a.states,
                                 lane_here());
    }
  }
  if (a.state_out && at.active && it.live)
    channel_state_io<NB, PT>(h, nullptr, a.state_out + at.state_at, at.p0, a.head_dim, a.states, lane);
}

}  // namespace
}  // namespace fhe::clear
