// Sweeps that give the gradients of the scan's queries: forward those of C, and
// in reverse, where keys and queries change places, those of B.
#pragma clang fp contract(fast)
#include "clear_scan.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

template <class T, int NB>
struct QueryLds {
  static constexpr int SUM = 32 * NB + 4;
  alignas(16) T key[CHUNK * Pitch<T, NB>::KEY];
  alignas(16) T value[WAVES][CHUNK * Pitch<T, NB>::VALUE];
  alignas(16) T other[WAVES][CHUNK * Pitch<T, NB>::VALUE];
  alignas(16) float sum[WAVES][16 * SUM];
  alignas(16) Gates gates[WAVES];
};

// State tiles (rows 4 q + r the channel, column l the state) from and to
// [head_dim][states].
template <int NB>
__device__ __forceinline__ void state_io(f32x4 (&h)[2][2 * NB], const float* from, float* to, int p0,
                                         int head_dim, int states) {
  const int q = lane_id() >> 4, l = lane_id() & 15;
#pragma unroll
  for (int p = 0; p < 2; ++p)
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

// Target t's gradient from 32 channels of one head,
//   in_t sum_p other[t][p] h[p] + sum_s decay(t, s) (other_t . value_s) key_s,
// summed over a workgroup's wavefronts and written for each workgroup of a
// group; forward also the part of the gates' gradient that the state before the
// chunk has in it.
template <class T, int NB, bool REV>
__global__ __launch_bounds__(64 * WAVES, 1) void k_query_sweep(SweepArgs a) {
  using N = Num<T>;
  using Frag = typename N::Frag;
  using Lds = QueryLds<T, NB>;
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
  const int64_t part = (int64_t)head * a.col_tiles + p0 / COLS;
  const int64_t token0 = item_token(a, it);
  const int64_t state_at =
      ((int64_t)(a.by_item ? item_i : it.seq) * a.heads + head) * a.head_dim * a.states;

  const T* key = (const T*)a.key.p + item_at(a, a.key, it) + group * a.key.head;
  const T* query = REV ? nullptr : (const T*)a.query.p + item_at(a, a.query, it) + group * a.query.head;
  const T* value = (const T*)a.value.p + item_at(a, a.value, it) + head * a.value.head + p0;
  const T* other = (const T*)a.other.p + item_at(a, a.other, it) + head * a.other.head + p0;
  const float* write = (const float*)a.write.p + item_at(a, a.write, it) + head * a.write.head;
  const float* decay = (const float*)a.decay.p + item_at(a, a.decay, it) + head * a.decay.head;
  float* out = (float*)a.out +
               (((int64_t)(block % a.blocks) * a.all_tokens + token0) * a.groups + group) * a.states;
  const int64_t out_tok = (int64_t)a.groups * a.states;

  f32x4 h[2][2 * NB] = {};
  if (a.state_in && active && it.live)
    state_io<NB>(h, a.state_in + state_at, nullptr, p0, a.head_dim, a.states);

  T* vt = lds.value[wave];
  T* ot = lds.other[wave];
  Gates& t = lds.gates[wave];
  const int chunks = (it.count + CHUNK - 1) / CHUNK;
  for (int c = 0; c < chunks; ++c) {
    const int first = (REV ? chunks - 1 - c : c) * CHUNK;
    const int n = min(CHUNK, it.count - first), live = it.live ? n : 0;
    __syncthreads();
    stage<T, KP>(lds.key, key + first * a.key.tok, a.key.tok, live, a.states, 32 * NB, a.wide_key,
                 threadIdx.x, 64 * WAVES);
    if (active) {
      stage<T, VP>(vt, value + first * a.value.tok, a.value.tok, live, width, COLS, a.wide_value,
                   lane, 64);
      stage<T, VP>(ot, other + first * a.other.tok, a.other.tok, live, width, COLS, a.wide_other,
                   lane, 64);
      make_gates<REV>(t, write + first * a.write.tok, a.write.tok, decay + first * a.decay.tok,
                      a.decay.tok, live);
    }
    __syncthreads();

    Split<T, N::FAIR> state[2 * NB];
#pragma unroll
    for (int nt = 0; nt < 2 * NB; ++nt) state[nt] = split<T, N::FAIR>(join(h[0][nt], h[1][nt]));
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      if (16 * i >= n) break;
      f32x4 got[2 * NB] = {};
      if (active) {
        const Frag of = N::rows(ot + 16 * i * VP, VP);
        const float in = t.dst[16 * i + l] * t.dst_in[i];
#pragma unroll
        for (int nt = 0; nt < 2 * NB; ++nt) {
          got[nt] = mma<T, N::FAIR>(state[nt], of, got[nt]);
          got[nt] *= in;
        }
        if constexpr (!REV) {
          float sum = 0.0f;
          if (16 * i + l < live) {
            const T* row = query + (first + 16 * i + l) * a.query.tok + 4 * q;
#pragma unroll
            for (int nt = 0; nt < 2 * NB; ++nt)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (16 * nt + 4 * q + r < a.states) sum += got[nt][r] * (float)row[16 * nt + r];
          }
          sum = sum_groups(sum);
          if (q == 0 && 16 * i + l < n) a.gate_part[part * a.all_tokens + token0 + first + 16 * i + l] = sum;
        }
        f32x4 pairs[TILES] = {};
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
          if (REV ? j < i : j > i) continue;
          f32x4 z = {};
          z = N::mma(N::rows(vt + 16 * j * VP, VP), of, z);
          pairs[j] = decayed<REV>(t, z, i, j);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if (REV ? 2 * m + 1 < i : 2 * m > i) continue;
          const auto s = split<T, N::FAIR>(join(pairs[2 * m], pairs[2 * m + 1]));
#pragma unroll
          for (int nt = 0; nt < 2 * NB; ++nt)
            got[nt] = mma<T, N::FAIR>(N::cols(lds.key + 32 * m * KP + 16 * nt, KP), s, got[nt]);
        }
        if constexpr (REV) {
          const float w = t.w[16 * i + l];
#pragma unroll
          for (int nt = 0; nt < 2 * NB; ++nt) got[nt] *= w;
        }
      }
#pragma unroll
      for (int nt = 0; nt < 2 * NB; ++nt)
        *reinterpret_cast<f32x4*>(&lds.sum[wave][l * Lds::SUM + 16 * nt + 4 * q]) = got[nt];
      __syncthreads();
      for (int e = threadIdx.x; e < 16 * 32 * NB; e += 64 * WAVES) {
        const int row = e / (32 * NB), col = e % (32 * NB);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += lds.sum[w][row * Lds::SUM + col];
        if (16 * i + row < n && col < a.states) out[(first + 16 * i + row) * out_tok + col] = sum;
      }
      __syncthreads();
    }
    if (!active) continue;
    // h <- total h + sum_s (factor_s value_s) key_s
    const float total = t.total;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int nt = 0; nt < 2 * NB; ++nt) h[p][nt] *= total;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (32 * m >= n) break;
      const f32x8 f = to_state(t, m);
      Split<T, N::FINE> s[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const Frag v = N::cols(vt + 32 * m * VP + 16 * p, VP);
        f32x8 x;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)v[j] * f[j];
        s[p] = split<T, N::FINE>(x);
      }
#pragma unroll
      for (int nt = 0; nt < 2 * NB; ++nt) {
        const auto k = N::cols(lds.key + 32 * m * KP + 16 * nt, KP);
#pragma unroll
        for (int p = 0; p < 2; ++p) h[p][nt] = mma<T, N::FINE>(s[p], k, h[p][nt]);
      }
    }
  }
  if (a.state_out && active && it.live)
    state_io<NB>(h, nullptr, a.state_out + state_at, p0, a.head_dim, a.states);
}

template <class T, int NB, bool REV>
void launch(const SweepArgs& a, int items, hipStream_t s) {
  constexpr size_t bytes = sizeof(QueryLds<T, NB>);
  static_assert(bytes <= 160 * 1024);
  auto* kernel = &k_query_sweep<T, NB, REV>;
  hip_check(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
            "scan gradient sweep");
  kernel<<<workgroups(a, items), 64 * WAVES, bytes, s>>>(a);
  hip_check(hipGetLastError(), "scan gradient sweep");
}

template <bool REV>
void dispatch(uint32_t dtype, const SweepArgs& a, int items, hipStream_t s) {
  auto by_size = [&](auto zero) {
    using T = decltype(zero);
    if (a.states <= 32) launch<T, 1, REV>(a, items, s);
    else if (a.states <= 64) launch<T, 2, REV>(a, items, s);
    else launch<T, 4, REV>(a, items, s);
  };
  if (dtype == BF16) by_size(bf16{});
  else by_size(float{});
}

}  // namespace

void launch_query_sweep(uint32_t dtype, const SweepArgs& a, int items, bool rev, hipStream_t s) {
  if (rev) dispatch<true>(dtype, a, items, s);
  else dispatch<false>(dtype, a, items, s);
}

}  // namespace fhe::clear
