// The causal convolution of each channel, its gradients and its single-token
// form:  y_t = act(bias + sum_k weight_k x_{t - taps + 1 + k}).
//
// Bound by memory: a thread keeps the window of its channels in registers and
// walks a run of tokens, loads ahead, so that an input is read once and, at the
// start of a run, taps - 1 times more, which the caches answer.  Two channels a
// thread: a wavefront's loads are whole lines either way, and more wavefronts
// cover more of a load's wait than wider ones.
// Before a sequence's first token the window holds its initial state, oldest
// first, or zeros.
#pragma clang fp contract(fast)
#include "clear.hpp"
#include "clear_tile.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

// Tokens of a run, loads ahead and channels of a thread.  30011 tokens of 1792
// channels in 16 bits: 47.6 us (the copy's rate) with these; with 8 channels and
// 4 loads ahead 67, with 4 and 8 50, with 2 and runs of 32 or 64 45 and 48.
// 8192 tokens: 16.6 us, with runs of 32 or 64 18.3 and 22.  A single token of
// 1792 channels: 3.7 us, with 8 channels a thread 5.6.
constexpr int RUN = 16, AHEAD = 8, NARROW = 2;
// A backward workgroup: BACK_RUNS runs of BACK_PIECES pieces of the channels,
// whose weights' gradients it sums before it writes them.  8192 tokens of 1792
// channels in 16 bits: 33 us; runs of 8 or 32 37 and 40; pieces of 2 channels 41;
// four loads ahead 42, for a thread's weights, their gradients, its window and
// its inputs' fill its registers.
constexpr int RUN_BACK = 16, BACK_PIECES = 32, BACK_RUNS = 8, WIDE = 4;

struct ConvArgs {
  Conv c;
  void* y;
  void* final_state;
  // backward
  Strided dy;
  const void* dfinal;
  void* dx;
  void* dinitial;
  float* parts;    // [workgroups' runs][taps + 1][channels]
  int run, runs;   // tokens of a run; runs of all tokens (packed) or of one sequence
  int pieces;      // ceil(channels / elements of a thread)
};

// The sequence of a token: [begin, end) in the token's own numbering (all
// tokens where packed, the sequence's otherwise).  seq < 0: of none.
struct Span {
  int seq, begin, end;
};

// The last sequence that begins at or before token t and is not empty, if t is
// in it.  Offsets are read as a rising partition clamped to the tokens.
__device__ __forceinline__ Span find_span(const Conv& c, int t) {
  int lo = 0, hi = c.seqs;  // offsets[lo] <= t < offsets[hi], where they rise
  if (t < c.offsets[0] || t >= c.offsets[c.seqs]) {
    // outside: up to the first sequence, or to the end
    const int first = c.offsets[0];
    return {-1, 0, t < first ? min(first, (int)c.tokens) : (int)c.tokens};
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (c.offsets[mid] <= t) lo = mid;
    else hi = mid;
  }
  return {lo, max(c.offsets[lo], 0), max(t + 1, min(c.offsets[lo + 1], (int)c.tokens))};
}

template <class T, int VEC>
struct Piece {
  float v[VEC];
};

// A thread's channels as they lie in memory.
template <class T, int VEC>
struct Raw {
  union {
    uint32_t w __attribute__((ext_vector_type(VEC * sizeof(T) < 4 ? 1 : VEC * sizeof(T) / 4)));
    T e[VEC];
  };
  __device__ __forceinline__ operator Piece<T, VEC>() const {
    Piece<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = (float)e[i];
    return r;
  }
};

// Elements [0, count) of them at p; zeros past the count.
template <class T, int VEC>
__device__ __forceinline__ Raw<T, VEC> read(const T* p, int count) {
  Raw<T, VEC> r;
  if (VEC > 1 && count >= VEC) {
    r.w = *reinterpret_cast<const decltype(r.w)*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.e[i] = VEC == 1 || i < count ? p[i] : (T)0.0f;
  }
  return r;
}
template <class T, int VEC>
__device__ __forceinline__ void write(T* p, const Piece<T, VEC>& v, int count) {
  Raw<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.e[i] = (T)v.v[i];
  if (VEC > 1 && count >= VEC) {
    *reinterpret_cast<decltype(r.w)*>(p) = r.w;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (VEC == 1 || i < count) p[i] = r.e[i];
  }
}

// Weights [channels][taps] of a thread's channels, in the last `taps` of KT
// places.  The places before them take no part: their inputs, which may be
// anything, are not multiplied.
template <int VEC, int KT>
__device__ __forceinline__ void read_weights(const float* weight, const float* bias, int c0, int count,
                                             int taps, float (&w)[KT][VEC], float (&b)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) b[i] = bias && i < count ? bias[c0 + i] : 0.0f;
  if (KT == 4 && taps == 4 && reinterpret_cast<uintptr_t>(weight) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float4 v = i < count ? reinterpret_cast<const float4*>(weight)[c0 + i] : float4{};
      w[0][i] = v.x;
      w[1][i] = v.y;
      w[2][i] = v.z;
      w[3][i] = v.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const int at = k - (KT - taps);
      w[k][i] = at >= 0 && i < count ? weight[(int64_t)(c0 + i) * taps + at] : 0.0f;
    }
  }
}

// v += the taps of a window.
template <class T, int VEC, int KT>
__device__ __forceinline__ void add_taps(float (&v)[VEC], const float (&w)[KT][VEC],
                                         const Piece<T, VEC>* window, int taps) {
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    if (k < KT - taps) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] += w[k][i] * window[k].v[i];
  }
}

// From the hardware's 2^x and reciprocal, each good to about a unit in the last
// place: with the exact functions the arithmetic takes twice as long as the
// memory.
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}

// The input at position t of a sequence (in its numbering, begin its first
// token): its tokens, before them its initial state, before that nothing.
template <class T, int VEC>
__device__ __forceinline__ Piece<T, VEC> input_at(const Conv& c, const T* x, const Span& s, int t, int c0,
                                                  int count) {
  Piece<T, VEC> zero = {};
  if (t >= s.begin) return read<T, VEC>(x + t * c.x.tok + c0, count);
  const int row = t - s.begin + c.taps - 1;
  if (!c.initial || row < 0) return zero;
  return read<T, VEC>((const T*)c.initial + ((int64_t)s.seq * (c.taps - 1) + row) * c.channels + c0, count);
}

// Blocks of the last rows write the final states: the last taps - 1 inputs of
// each sequence.
template <class T, int VEC>
__device__ void final_states(const ConvArgs& a, int index, int c0, int count) {
  const Conv& c = a.c;
  const int seq = index / (c.taps - 1), row = index % (c.taps - 1);
  Span s{seq, 0, (int)c.tokens};
  const T* x = (const T*)c.x.p;
  if (c.offsets) {
    s.begin = min(max(c.offsets[seq], 0), (int)c.tokens);
    s.end = max(s.begin, min(c.offsets[seq + 1], (int)c.tokens));
  } else {
    x += seq * c.x.seq;
  }
  const Piece<T, VEC> p = input_at<T, VEC>(c, x, s, s.end - (c.taps - 1) + row, c0, count);
  write<T, VEC>((T*)a.final_state + (int64_t)index * c.channels + c0, p, count);
}

// Grid: x the pieces of the channels, y the runs (of each sequence), then the
// rows of the final states.
template <class T, int VEC, int KT>
__global__ __launch_bounds__(256) void k_conv(ConvArgs a) {
  const Conv& c = a.c;
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int piece = (int)(at % a.pieces);
  const int64_t job = at / a.pieces;
  const int c0 = piece * VEC, count = min(VEC, c.channels - c0);
  const int64_t jobs = c.offsets ? a.runs : (int64_t)a.runs * c.seqs;
  if (job >= jobs) {
    const int64_t row = job - jobs;
    if (a.final_state && row < (int64_t)c.seqs * (c.taps - 1)) final_states<T, VEC>(a, (int)row, c0, count);
    return;
  }
  float w[KT][VEC], b[VEC];
  read_weights<VEC, KT>(c.weight, c.bias, c0, count, c.taps, w, b);
  const int seq = c.offsets ? 0 : (int)(job / a.runs);
  const int t0 = (int)(c.offsets ? job : job % a.runs) * a.run, t1 = min(t0 + a.run, (int)c.tokens);
  const T* x = (const T*)c.x.p + (c.offsets ? 0 : seq * c.x.seq);
  T* y = (T*)a.y + (c.offsets ? 0 : (int64_t)seq * c.tokens * c.channels) + c0;

  Piece<T, VEC> window[KT - 1 + AHEAD];  // the inputs from KT - 1 before token t
  int t = t0;
  while (t < t1) {
    const Span s = c.offsets ? find_span(c, t) : Span{seq, 0, (int)c.tokens};
    const int end = min(s.end, t1);
    if (s.seq < 0) {
      for (; t < end; ++t) write<T, VEC>(y + (int64_t)t * c.channels, {}, count);
      continue;
    }
#pragma unroll
    for (int k = 0; k < KT - 1; ++k) window[k] = input_at<T, VEC>(c, x, s, t - (KT - 1) + k, c0, count);
    for (; t < end; t += AHEAD) {
      Raw<T, VEC> in[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        in[u] = read<T, VEC>(x + min(t + u, end - 1) * c.x.tok + c0, count);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) window[KT - 1 + u] = in[u];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        Piece<T, VEC> out;
#pragma unroll
        for (int i = 0; i < VEC; ++i) out.v[i] = b[i];
        add_taps<T, VEC, KT>(out.v, w, window + u, c.taps);
        if (c.silu) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) out.v[i] *= sigmoid(out.v[i]);
        }
        if (t + u < end) write<T, VEC>(y + (int64_t)(t + u) * c.channels, out, count);
      }
#pragma unroll
      for (int k = 0; k < KT - 1; ++k) window[k] = window[k + AHEAD];
    }
    t = end;
  }
}

// A run's gradients.  d_t = dy_t act'(pre_t) feeds the inputs t - taps + 1 .. t;
// a run owns the inputs at its tokens (and the initial state of a sequence that
// begins in it) and so walks taps - 1 tokens further, whose d it makes again,
// and sums the weights' gradients over its own tokens.
template <class T, int VEC, int KT>
__device__ __forceinline__ void conv_back_run(const ConvArgs& a, int64_t job, int c0, int count,
                                              float (&dw)[KT][VEC], float (&db)[VEC]) {
  const Conv& c = a.c;
  const int keep = c.taps - 1;
  float w[KT][VEC], b[VEC];
  read_weights<VEC, KT>(c.weight, c.bias, c0, count, c.taps, w, b);
  const int seq = c.offsets ? 0 : (int)(job / a.runs);
  const int t0 = (int)(c.offsets ? job : job % a.runs) * a.run, t1 = min(t0 + a.run, (int)c.tokens);
  const T* x = (const T*)c.x.p + (c.offsets ? 0 : seq * c.x.seq);
  const T* dy = (const T*)a.dy.p + (c.offsets ? 0 : seq * a.dy.seq) + c0;
  T* dx = (T*)a.dx + (c.offsets ? 0 : (int64_t)seq * c.tokens * c.channels) + c0;

  int t = t0;
  while (t < t1) {
    const Span s = c.offsets ? find_span(c, t) : Span{seq, 0, (int)c.tokens};
    if (s.seq < 0) {
      const int end = min(s.end, t1);
      for (; t < end; ++t) write<T, VEC>(dx + (int64_t)t * c.channels, {}, count);
      continue;
    }
    const int own = min(s.end, t1), last = min(s.end, t1 + keep);
    const bool starts = t == s.begin;
    Piece<T, VEC> window[KT], grad[KT] = {};  // inputs and their gradients, t - KT + 1 .. t
#pragma unroll
    for (int k = 0; k < KT - 1; ++k) window[k] = input_at<T, VEC>(c, x, s, t - (KT - 1) + k, c0, count);
    // The gradient of the input at position p is whole.
    auto emit = [&](int p, Piece<T, VEC> g) {
      if (p < s.begin ? !starts || p < s.begin - keep : p < t0 || p >= own) return;
      if (a.dfinal && p >= s.end - keep) {
        const int64_t row = (int64_t)s.seq * keep + p - (s.end - keep);
        const Piece<T, VEC> f = read<T, VEC>((const T*)a.dfinal + row * c.channels + c0, count);
#pragma unroll
        for (int i = 0; i < VEC; ++i) g.v[i] += f.v[i];
      }
      if (p >= s.begin) {
        write<T, VEC>(dx + (int64_t)p * c.channels, g, count);
      } else if (a.dinitial) {
        const int64_t row = (int64_t)s.seq * keep + p - (s.begin - keep);
        write<T, VEC>((T*)a.dinitial + row * c.channels + c0, g, count);
      }
    };
    for (; t < last; ++t) {
      window[KT - 1] = read<T, VEC>(x + t * c.x.tok + c0, count);
      Piece<T, VEC> d = read<T, VEC>(dy + t * a.dy.tok, count);
      if (c.silu) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = b[i];
        add_taps<T, VEC, KT>(v, w, window, c.taps);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float g = sigmoid(v[i]);
          d.v[i] *= g * (1.0f + v[i] * (1.0f - g));
        }
      }
      grad[KT - 1] = {};
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        if (k < KT - c.taps) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          grad[k].v[i] += d.v[i] * w[k][i];
          if (t < own) dw[k][i] += d.v[i] * window[k].v[i];
        }
      }
      if (t < own) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) db[i] += d.v[i];
      }
      emit(t - (KT - 1), grad[0]);
#pragma unroll
      for (int k = 0; k < KT - 1; ++k) {
        window[k] = window[k + 1];
        grad[k] = grad[k + 1];
      }
    }
    // what is left of the run's own inputs has all its taps; at the sequence's
    // end nothing more reaches its last inputs
#pragma unroll
    for (int k = 0; k < KT - 1; ++k) emit(last - (KT - 1) + k, grad[k]);
    t = own;
  }
}

// The gradients of the initial states of empty sequences, which no run visits.
template <class T>
__global__ __launch_bounds__(256) void k_conv_empty(ConvArgs a) {
  const Conv& c = a.c;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, size = (int64_t)(c.taps - 1) * c.channels;
  const int seq = (int)(at / size);
  if (seq >= c.seqs) return;
  int begin = 0, end = (int)c.tokens;
  if (c.offsets) {
    begin = min(max(c.offsets[seq], 0), (int)c.tokens);
    end = min(c.offsets[seq + 1], (int)c.tokens);
  }
  if (end <= begin) ((T*)a.dinitial)[at] = a.dfinal ? ((const T*)a.dfinal)[at] : (T)0.0f;
}

template <class T, int VEC, int KT>
__global__ __launch_bounds__(256) void k_conv_back(ConvArgs a) {
  const Conv& c = a.c;
  const int lane = threadIdx.x % BACK_PIECES, line = threadIdx.x / BACK_PIECES;
  const int c0 = (blockIdx.y * BACK_PIECES + lane) * VEC, count = min(VEC, c.channels - c0);
  const int64_t job = (int64_t)blockIdx.x * BACK_RUNS + line;
  const int64_t jobs = c.offsets ? a.runs : (int64_t)a.runs * c.seqs;
  float dw[KT][VEC] = {}, db[VEC] = {};
  if (count > 0 && job < jobs) conv_back_run<T, VEC, KT>(a, job, c0, count, dw, db);
  // the workgroup's runs, in order
  __shared__ float sums[BACK_RUNS][BACK_PIECES * VEC + 1];
#pragma unroll
  for (int k = 0; k <= KT; ++k) {
    const int tap = k - (KT - c.taps);
    if (tap < 0) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[line][lane * VEC + i] = k < KT ? dw[k < KT ? k : 0][i] : db[i];
    __syncthreads();
    for (int e = threadIdx.x; e < BACK_PIECES * VEC; e += 256) {
      const int ch = blockIdx.y * BACK_PIECES * VEC + e;
      float sum = sums[0][e];
#pragma unroll
      for (int r = 1; r < BACK_RUNS; ++r) sum += sums[r][e];
      if (ch < c.channels) a.parts[((int64_t)blockIdx.x * (c.taps + 1) + tap) * c.channels + ch] = sum;
    }
    __syncthreads();
  }
}
// Sums the workgroups' parts: 64 channels a workgroup, each of its sixteen
// wavefronts every sixteenth part.
__global__ __launch_bounds__(1024) void k_conv_sum(const float* parts, int64_t count, int channels, int taps,
                                                   float* dweight, float* dbias) {
  __shared__ float sums[16][64];
  const int ch = blockIdx.x * 64 + (threadIdx.x & 63), k = blockIdx.y, wave = threadIdx.x >> 6;
  float sum = 0.0f;
  if (ch < channels) {
#pragma unroll 4
    for (int64_t r = wave; r < count; r += 16) sum += parts[(r * (taps + 1) + k) * channels + ch];
  }
  sums[wave][threadIdx.x & 63] = sum;
  __syncthreads();
  if (wave || ch >= channels) return;
  for (int w = 1; w < 16; ++w) sum += sums[w][threadIdx.x & 63];
  if (k < taps) dweight[(int64_t)ch * taps + k] = sum;
  else if (dbias) dbias[ch] = sum;
}

template <class T, int VEC, int KT>
__global__ __launch_bounds__(256) void k_conv_step(ConvStep c, T* y, int pieces) {
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int request = (int)(at / pieces), c0 = (int)(at % pieces) * VEC, count = min(VEC, c.channels - c0);
  if (request >= c.requests) return;
  const int slot = c.slots ? c.slots[request] : request;
  T* out = y + (int64_t)request * c.channels + c0;
  if (slot < 0 || slot >= c.cache) {
    write<T, VEC>(out, {}, count);
    return;
  }
  float w[KT][VEC], b[VEC];
  read_weights<VEC, KT>(c.weight, c.bias, c0, count, c.taps, w, b);
  T* state = (T*)c.state + (int64_t)slot * (c.taps - 1) * c.channels + c0;
  Piece<T, VEC> window[KT], r;
#pragma unroll
  for (int k = 0; k < KT - 1; ++k) {
    const int row = k - (KT - c.taps);
    window[k] = row >= 0 ? read<T, VEC>(state + (int64_t)row * c.channels, count) : Piece<T, VEC>{};
  }
  window[KT - 1] = read<T, VEC>((const T*)c.x.p + request * c.x.tok + c0, count);
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.v[i] = b[i];
  add_taps<T, VEC, KT>(r.v, w, window, c.taps);
  if (c.silu) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] *= sigmoid(r.v[i]);
  }
  write<T, VEC>(out, r, count);
#pragma unroll
  for (int k = 0; k < KT - 1; ++k) {
    const int row = k - (KT - c.taps);
    if (row >= 0) write<T, VEC>(state + (int64_t)row * c.channels, window[k + 1], count);
  }
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// f(type, most elements of a thread, places of the window) for a launch.  Pieces
// of more than one need the channels to be a multiple of 16 bytes and every row
// aligned.
template <class F>
void dispatch(uint32_t dtype, bool wide, int taps, F&& f) {
  auto by_taps = [&](auto zero, auto vec) {
    if (taps <= 4) f(zero, vec, std::integral_constant<int, 4>{});
    else f(zero, vec, std::integral_constant<int, 8>{});
  };
  if (dtype == BF16) {
    if (wide) by_taps(bf16{}, std::integral_constant<int, 8>{});
    else by_taps(bf16{}, std::integral_constant<int, 1>{});
  } else {
    if (wide) by_taps(float{}, std::integral_constant<int, 4>{});
    else by_taps(float{}, std::integral_constant<int, 1>{});
  }
}

int vec_of(uint32_t dtype) { return dtype == BF16 ? 8 : 4; }
bool wide_rows(const Strided& t, uint32_t dtype, bool packed) {
  const int vec = vec_of(dtype);
  return aligned(t.p) && t.tok % vec == 0 && (packed || t.seq % vec == 0);
}

int64_t jobs_of(const Conv& c, int run) {
  const int64_t runs = (c.tokens + run - 1) / run;
  return c.offsets ? runs : runs * c.seqs;
}

int64_t parts_of(const Conv& c) { return (jobs_of(c, RUN_BACK) + BACK_RUNS - 1) / BACK_RUNS; }

uint32_t grid_of(int64_t threads) { return (uint32_t)((threads + 255) / 256); }

}  // namespace

size_t conv_workspace(const Conv& c) {
  return (size_t)parts_of(c) * (c.taps + 1) * c.channels * sizeof(float);
}

void conv(const Conv& c, void* y, void* final_state, hipStream_t stream) {
  ConvArgs a{};
  a.c = c;
  a.y = y;
  a.final_state = final_state;
  a.run = RUN;
  a.runs = (int)((c.tokens + RUN - 1) / RUN);
  const bool wide = c.channels % vec_of(c.dtype) == 0 && wide_rows(c.x, c.dtype, c.offsets) && aligned(y) &&
                    aligned(final_state) && aligned(c.initial);
  dispatch(c.dtype, wide, c.taps, [&](auto zero, auto vec, auto kt) {
    using T = decltype(zero);
    constexpr int VEC = vec() > NARROW ? NARROW : vec();
    a.pieces = (c.channels + VEC - 1) / VEC;
    const int64_t rows = jobs_of(c, RUN) + (final_state ? (int64_t)c.seqs * (c.taps - 1) : 0);
    if (!rows) return;
    k_conv<T, VEC, kt()><<<grid_of(rows * a.pieces), 256, 0, stream>>>(a);
  });
  hip_check(hipGetLastError(), "convolution");
}

void conv_backward(const Conv& c, const ConvGrads& g, void* workspace, hipStream_t stream) {
  ConvArgs a{};
  a.c = c;
  a.dy = g.dy;
  a.dfinal = g.dfinal;
  a.dx = g.dx;
  a.dinitial = g.dinitial;
  a.parts = (float*)workspace;
  a.run = RUN_BACK;
  a.runs = (int)((c.tokens + RUN_BACK - 1) / RUN_BACK);
  const bool wide = c.channels % vec_of(c.dtype) == 0 && wide_rows(c.x, c.dtype, c.offsets) &&
                    wide_rows(g.dy, c.dtype, c.offsets) && aligned(g.dx) && aligned(c.initial) &&
                    aligned(g.dfinal) && aligned(g.dinitial);
  const int64_t parts = parts_of(c);
  dispatch(c.dtype, wide, c.taps, [&](auto zero, auto vec, auto kt) {
    using T = decltype(zero);
    if (parts) {
      constexpr int VEC = vec() > WIDE ? WIDE : vec();
      const dim3 grid((uint32_t)parts, (c.channels + BACK_PIECES * VEC - 1) / (BACK_PIECES * VEC));
      k_conv_back<T, VEC, kt()><<<grid, BACK_PIECES * BACK_RUNS, 0, stream>>>(a);
    }
    if (g.dinitial && (c.offsets || !c.tokens))
      k_conv_empty<T><<<grid_of((int64_t)c.seqs * (c.taps - 1) * c.channels), 256, 0, stream>>>(a);
  });
  hip_check(hipGetLastError(), "convolution gradient");
  k_conv_sum<<<dim3((c.channels + 63) / 64, c.taps + 1), 1024, 0, stream>>>(a.parts, parts, c.channels, c.taps,
                                                                           g.dweight, g.dbias);
  hip_check(hipGetLastError(), "convolution gradient sums");
}

void conv_step(const ConvStep& c, void* y, hipStream_t stream) {
  const bool wide = c.channels % vec_of(c.dtype) == 0 && aligned(c.x.p) && c.x.tok % vec_of(c.dtype) == 0 &&
                    aligned(y) && aligned(c.state);
  dispatch(c.dtype, wide, c.taps, [&](auto zero, auto vec, auto kt) {
    using T = decltype(zero);
    constexpr int VEC = vec() > NARROW ? NARROW : vec();
    const int pieces = (c.channels + VEC - 1) / VEC;
    k_conv_step<T, VEC, kt()><<<grid_of((int64_t)c.requests * pieces), 256, 0, stream>>>(c, (T*)y, pieces);
  });
  hip_check(hipGetLastError(), "convolution step");
}

}  // namespace fhe::clear
