// Sweeps over the chunks of a segment with the state in registers: the scan's
// results, and the state that a segment leaves.
#pragma clang fp contract(fast)
#include "clear_scan.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

template <class T, int NB, bool REV, bool VALUES>
struct ValueLds {
  // 16-byte rows: a tile that a kernel does not have must not shift the others
  alignas(16) T key[CHUNK * Pitch<T, NB>::KEY];
  alignas(16) T query[VALUES ? CHUNK * Pitch<T, NB>::KEY : 1];
  alignas(16) T value[WAVES][CHUNK * Pitch<T, NB>::VALUE];
  alignas(16) T other[VALUES && REV ? WAVES : 1][VALUES && REV ? CHUNK * Pitch<T, NB>::VALUE : 1];
  alignas(16) Gates gates[WAVES];
};

// Adds a chunk to a wavefront's state [states][32 channels]:
// h <- total h + sum_s key_s (factor_s value_s).
template <class T, int NB>
__device__ __forceinline__ void add_chunk(f32x4 (&h)[2 * NB][2], const T* key, const Gates& t,
                                          const typename Num<T>::Frag (&v)[2][2], int n) {
  using N = Num<T>;
  const float total = t.total;
#pragma unroll
  for (int nt = 0; nt < 2 * NB; ++nt)
#pragma unroll
    for (int p = 0; p < 2; ++p) h[nt][p] *= total;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (32 * m >= n) break;
    const f32x8 f = to_state(t, m);
    Split<T, N::FINE> s[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      f32x8 x;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (float)v[m][p][j] * f[j];
      s[p] = split<T, N::FINE>(x);
    }
#pragma unroll
    for (int nt = 0; nt < 2 * NB; ++nt) {
      const auto k = N::cols(key + 32 * m * Pitch<T, NB>::KEY + 16 * nt, Pitch<T, NB>::KEY);
#pragma unroll
      for (int p = 0; p < 2; ++p) h[nt][p] = mma<T, N::FINE>(k, s[p], h[nt][p]);
    }
  }
}

// State tiles (rows 4 q + r the states, column l the channel) to and from
// [head_dim][states].
template <int NB>
__device__ __forceinline__ void state_io(f32x4 (&h)[2 * NB][2], const float* from, float* to, int p0,
                                         int head_dim, int states) {
  const int q = lane_id() >> 4, l = lane_id() & 15;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = p0 + 16 * p + l;
#pragma unroll
    for (int nt = 0; nt < 2 * NB; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = 16 * nt + 4 * q + r;
        if (row < head_dim && n < states) {
          if (to) to[(int64_t)row * states + n] = h[nt][p][r];
          else h[nt][p][r] = from[(int64_t)row * states + n];
        }
      }
  }
}

// y (or, in reverse, the gradient of x) of a segment, 32 channels of one head a
// wavefront, four wavefronts of one group on shared keys and queries.
template <class T, int NB, bool REV, bool VALUES>
__global__ __launch_bounds__(64 * WAVES, VALUES && REV ? 1 : 2) void k_value_sweep(SweepArgs a) {
  using N = Num<T>;
  using Frag = typename N::Frag;
  using Lds = ValueLds<T, NB, REV, VALUES>;
  constexpr int KP = Pitch<T, NB>::KEY, VP = Pitch<T, NB>::VALUE;
  extern __shared__ __align__(16) char lds_raw[];
  Lds& lds = *reinterpret_cast<Lds*>(lds_raw);

  const int item_i = blockIdx.x / (a.groups * a.blocks);
  const int block = blockIdx.x % (a.groups * a.blocks);
  const Item it = find_item(a, item_i);
  if (it.count <= 0 && it.seq < 0) return;
  const int group = block / a.blocks, per_group = a.heads / a.groups;
  const int wave = threadIdx.x >> 6, lane = lane_id(), q = lane >> 4, l = lane & 15;
  const int unit = block % a.blocks * WAVES + wave;
  const bool active = unit < per_group * a.col_tiles;
  const int head = group * per_group + (active ? unit / a.col_tiles : 0);
  const int p0 = active ? unit % a.col_tiles * COLS : 0;
  const int width = active ? min(COLS, a.head_dim - p0) : 0;
  const int64_t part = (int64_t)head * a.col_tiles + p0 / COLS;  // row of the per-unit results
  const int64_t token0 = item_token(a, it);
  const int64_t state_at =
      ((int64_t)(a.by_item ? item_i : it.seq) * a.heads + head) * a.head_dim * a.states;

  const T* key = (const T*)a.key.p + item_at(a, a.key, it) + group * a.key.head;
  const T* query = VALUES ? (const T*)a.query.p + item_at(a, a.query, it) + group * a.query.head : nullptr;
  const T* value = (const T*)a.value.p + item_at(a, a.value, it) + head * a.value.head + p0;
  const T* other =
      VALUES && REV ? (const T*)a.other.p + item_at(a, a.other, it) + head * a.other.head + p0 : nullptr;
  const float* write = (const float*)a.write.p + item_at(a, a.write, it) + head * a.write.head;
  const float* decay = (const float*)a.decay.p + item_at(a, a.decay, it) + head * a.decay.head;
  T* out = VALUES ? (T*)a.out + (token0 * a.heads + head) * a.head_dim + p0 : nullptr;
  const int64_t out_tok = (int64_t)a.heads * a.head_dim;
  const float skip = VALUES && a.d && active ? a.d[head] : 0.0f;

  f32x4 h[2 * NB][2] = {};
  const bool seeded = VALUES && a.state_in && active && it.live;
  if (seeded) state_io<NB>(h, a.state_in + state_at, nullptr, p0, a.head_dim, a.states);

  T* vt = lds.value[wave];
  T* ot = lds.other[VALUES && REV ? wave : 0];
  Gates& t = lds.gates[wave];
  float dd = 0.0f;
  double log_total = 0.0;
  const int chunks = (it.count + CHUNK - 1) / CHUNK;
  for (int c = 0; c < chunks; ++c) {
    const int first = (REV ? chunks - 1 - c : c) * CHUNK;
    const int n = min(CHUNK, it.count - first), live = it.live ? n : 0;
    __syncthreads();
    stage<T, KP>(lds.key, key + first * a.key.tok, a.key.tok, live, a.states, 32 * NB, a.wide_key,
                 threadIdx.x, 64 * WAVES);
    if constexpr (VALUES)
      stage<T, KP>(lds.query, query + first * a.query.tok, a.query.tok, live, a.states, 32 * NB,
                   a.wide_query, threadIdx.x, 64 * WAVES);
    if (active) {
      stage<T, VP>(vt, value + first * a.value.tok, a.value.tok, live, width, COLS, a.wide_value,
                   lane, 64);
      if constexpr (VALUES && REV)
        stage<T, VP>(ot, other + first * a.other.tok, a.other.tok, live, width, COLS, a.wide_other,
                     lane, 64);
      make_gates<REV>(t, write + first * a.write.tok, a.write.tok, decay + first * a.decay.tok,
                      a.decay.tok, live);
    }
    __syncthreads();
    if (!active) continue;

    Frag v[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int p = 0; p < 2; ++p) v[m][p] = N::cols(vt + 32 * m * VP + 16 * p, VP);

    if constexpr (VALUES) {
      Split<T, N::FAIR> state[NB][2];
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int p = 0; p < 2; ++p) state[k][p] = split<T, N::FAIR>(join(h[2 * k][p], h[2 * k + 1][p]));
      float row_sum[TILES][4] = {}, col_sum[TILES] = {};
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        if (16 * i >= n) break;
        Frag qf[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) qf[k] = N::rows(lds.query + 16 * i * KP + 32 * k, KP);
        // what the state before the chunk gives
        f32x4 y[2] = {};
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int p = 0; p < 2; ++p) y[p] = mma<T, N::FAIR>(qf[k], state[k][p], y[p]);
        f32x4 din = *reinterpret_cast<const f32x4*>(&t.dst[16 * i + 4 * q]);
#pragma unroll
        for (int r = 0; r < 4; ++r) din[r] *= t.dst_in[i];
        f32x4 from_state = {};
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          y[p] *= din;
          if constexpr (REV) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              from_state[r] += y[p][r] * (float)ot[(16 * i + 4 * q + r) * VP + 16 * p + l];
          }
        }
        // and the tokens of the chunk
        f32x4 pairs[TILES] = {};
        Frag of;
        if constexpr (REV) of = N::rows(ot + 16 * i * VP, VP);
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
          if (REV ? j < i : j > i) continue;
          f32x4 s = {};
#pragma unroll
          for (int k = 0; k < NB; ++k)
            s = N::mma(N::rows(lds.key + 16 * j * KP + 32 * k, KP), qf[k], s);
          pairs[j] = decayed<REV>(t, s, i, j);
          if constexpr (REV) {  // the pairs' own parts of the loss, off the diagonal
            f32x4 z = {};
            z = N::mma(N::rows(vt + 16 * j * VP, VP), of, z);
            const float w = t.w[16 * i + l];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float m = i == j && 4 * q + r == l ? 0.0f : pairs[j][r] * z[r] * w;
              row_sum[j][r] += m;
              col_sum[i] += m;
            }
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if (REV ? 2 * m + 1 < i : 2 * m > i) continue;
          const auto s = split<T, N::FAIR>(join(pairs[2 * m], pairs[2 * m + 1]));
#pragma unroll
          for (int p = 0; p < 2; ++p) y[p] = mma<T, N::FAIR>(s, v[m][p], y[p]);
        }
        f32x4 against = {};
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = (16 * i + 4 * q + r) * VP + 16 * p + l;
            const float mine = (float)vt[at];
            float got = y[p][r];
            if constexpr (REV) {
              const float x = (float)ot[at];
              against[r] += got * x;
              dd += mine * x;
              got *= t.w[16 * i + 4 * q + r];
            }
            vt[at] = (T)(got + skip * mine);
          }
        if constexpr (REV) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = first + 16 * i + 4 * q + r;
            const float dw = sum16(against[r]), k = sum16(from_state[r]);
            if (l == 0 && 16 * i + 4 * q + r < n) {
              a.dwrite_part[part * a.all_tokens + token0 + at] = dw;
              // kept until the row sums are whole; the same lane adds them
              t.g[16 * i + 4 * q + r] = -(double)(t.w[16 * i + 4 * q + r] * k);
            }
          }
        }
      }
      if constexpr (REV) {
        wave_sync();
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const float cs = sum_groups(col_sum[i]);
          f32x4 rs;
#pragma unroll
          for (int r = 0; r < 4; ++r) rs[r] = sum16(row_sum[i][r]);
          if (l == 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) t.g[16 * i + 4 * q + r] += rs[r];
          }
          wave_sync();
          if (q == 0 && 16 * i + l < n)
            a.gate_part[part * a.all_tokens + token0 + first + 16 * i + l] =
                (float)(t.g[16 * i + l] - cs);
        }
      }
      wave_sync();
      for (int i = lane; i < CHUNK * (COLS / N::VEC); i += 64) {
        const int row = i / (COLS / N::VEC), col = i % (COLS / N::VEC) * N::VEC;
        if (row < n)
          store16(out + (first + row) * out_tok + col,
                  *reinterpret_cast<const u32x4*>(vt + row * VP + col), width - col, a.wide_out);
      }
    } else {
      log_total += t.e[TILES - 1];
    }
    add_chunk<T, NB>(h, lds.key, t, v, n);
  }
  if (!active) return;
  if (a.state_out && (a.by_item || it.live))
    state_io<NB>(h, nullptr, a.state_out + state_at, p0, a.head_dim, a.states);
  if constexpr (!VALUES) {
    if (lane == 0 && p0 == 0) a.decay_out[(int64_t)item_i * a.heads + head] = exp2d(log_total);
  }
  if constexpr (VALUES && REV) {
    dd = sum_groups(sum16(dd));
    if (lane == 0) a.dd_part[(int64_t)item_i * a.heads * a.col_tiles + part] = dd;
  }
}

template <class T, int NB, bool REV, bool VALUES>
void launch(const SweepArgs& a, int items, hipStream_t s) {
  constexpr size_t bytes = sizeof(ValueLds<T, NB, REV, VALUES>);
  static_assert(bytes <= 160 * 1024);
  auto* kernel = &k_value_sweep<T, NB, REV, VALUES>;
  hip_check(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
            "scan sweep");
  kernel<<<workgroups(a, items), 64 * WAVES, bytes, s>>>(a);
  hip_check(hipGetLastError(), "scan sweep");
}

template <bool VALUES>
void dispatch(uint32_t dtype, const SweepArgs& a, int items, bool rev, hipStream_t s) {
  auto by_size = [&](auto zero, auto reverse) {
    using T = decltype(zero);
    constexpr bool R = decltype(reverse)::value;
    if (a.states <= 32) launch<T, 1, R, VALUES>(a, items, s);
    else if (a.states <= 64) launch<T, 2, R, VALUES>(a, items, s);
    else launch<T, 4, R, VALUES>(a, items, s);
  };
  auto by_type = [&](auto reverse) {
    if (dtype == BF16) by_size(bf16{}, reverse);
    else by_size(float{}, reverse);
  };
  if (rev) by_type(std::true_type{});
  else by_type(std::false_type{});
}

}  // namespace

void launch_value_sweep(uint32_t dtype, const SweepArgs& a, int items, bool rev, hipStream_t s) {
  dispatch<true>(dtype, a, items, rev, s);
}
void launch_state_sweep(uint32_t dtype, const SweepArgs& a, int items, bool rev, hipStream_t s) {
  dispatch<false>(dtype, a, items, rev, s);
}

}  // namespace fhe::clear
