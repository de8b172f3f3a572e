// Operators that run Mamba-2 in the clear, on the caller's device memory and
// stream.  They allocate nothing and never wait for the GPU; the caller checks
// nothing that these do not check again (clear_capi.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace fhe::clear {

enum : uint32_t { F32 = 0, BF16 = 1 };

// A tensor [sequence][token][head or group][contiguous], strides in elements.
struct Strided {
  const void* p;
  int64_t seq, tok, head;
};

struct Scan {
  uint32_t dtype;
  int seqs, heads, head_dim, states, groups;
  int64_t tokens;      // of each sequence, or of all where `offsets` is set
  const int* offsets;  // [seqs + 1] on the device, or null
  Strided x, b, c, write, decay;
  const float *d, *initial;

  int64_t all_tokens() const { return offsets ? tokens : tokens * seqs; }
};

struct ScanGrads {
  Strided dy;
  const float* dfinal;
  void* dx;
  float *dwrite, *ddecay;
  void *db, *dc;
  float *dd, *dinitial;
};

size_t scan_workspace(const Scan& s, bool backward);
void scan(const Scan& s, void* y, float* final_state, void* workspace, hipStream_t stream);
void scan_backward(const Scan& s, const ScanGrads& g, void* workspace, hipStream_t stream);

// One token of each request; `slots` names its row of the cache (null: the
// request's own number), rows outside of it are padding.  Strided::seq unused:
// tok is the request's stride.
struct Step {
  uint32_t dtype;
  int requests, cache, heads, head_dim, states, groups;
  const int* slots;
  Strided x, b, c, write, decay;
  const float* d;
  float* state;  // [cache][heads][head_dim][states]
};
void step(const Step& s, void* y, hipStream_t stream);

struct Conv {
  uint32_t dtype;
  int seqs, channels, taps;
  int64_t tokens;
  const int* offsets;
  Strided x;               // head unused
  const float *weight, *bias;  // [channels][taps], [channels] or null
  const void* initial;     // [seqs][taps - 1][channels] or null
  bool silu;

  int64_t all_tokens() const { return offsets ? tokens : tokens * seqs; }
};
struct ConvGrads {
  Strided dy;
  const void* dfinal;  // as initial, or null
  void* dx;
  float *dweight, *dbias;
  void* dinitial;
};
size_t conv_workspace(const Conv& c);
void conv(const Conv& c, void* y, void* final_state, hipStream_t stream);
void conv_backward(const Conv& c, const ConvGrads& g, void* workspace, hipStream_t stream);

struct ConvStep {
  uint32_t dtype;
  int requests, cache, channels, taps;
  const int* slots;
  Strided x;
  const float *weight, *bias;
  void* state;  // [cache][taps - 1][channels]
  bool silu;
};
void conv_step(const ConvStep& c, void* y, hipStream_t stream);

struct Logprob {
  uint32_t dtype;
  int64_t rows, vocab, row_stride;
  int top;
  const void* logits;
  const int64_t* targets;
};
struct LogprobOut {
  float *logprob, *entropy, *peak, *log_sum;  // [rows]
  float* top_logprob;              // [rows][top]
  int* top_index;
};
size_t logprob_workspace(const Logprob& l);
void logprob(const Logprob& l, const LogprobOut& o, void* workspace, hipStream_t stream);
// dlogits [rows][vocab] from what the forward call gave; either gradient may be null
void logprob_backward(const Logprob& l, const float* peak, const float* log_sum, const float* entropy,
                      const float* dlogprob, const float* dentropy, void* dlogits, hipStream_t stream);

constexpr int MAX_STATES = 128, MAX_TAPS = 8, MAX_TOP = 32;

}  // namespace fhe::clear
