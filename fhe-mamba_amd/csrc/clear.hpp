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

// Rows of contiguous elements, `row` elements apart.
struct Rows {
  const void* p;
  int64_t row;
};

struct Norm {
  uint32_t dtype, out_dtype;  // of x and the gate; of y
  int64_t rows;
  int channels, groups;  // of a row
  float eps;
  Rows x, gate;  // gate.p may be null
  const float* weight;
};
struct NormGrads {
  Rows dy;
  void *dx, *dgate;
  float* dweight;
};
size_t norm_workspace(const Norm& n);
void norm(const Norm& n, void* y, hipStream_t stream);
void norm_backward(const Norm& n, const NormGrads& g, void* workspace, hipStream_t stream);

struct AddNorm {
  uint32_t dtype, out_dtype;  // of hidden and the sum; of the update and y
  int64_t rows;
  int channels;
  float eps;
  Rows hidden, update;
  const float *scale, *weight;  // scale may be null
};
struct AddNormGrads {
  Rows dy, dsum;    // either may be null
  const void* sum;  // as the forward call left it, or null
  void *dhidden, *dupdate;
  float *dscale, *dweight;
};
size_t add_norm_workspace(const AddNorm& n);
void add_norm(const AddNorm& n, void* sum, void* y, hipStream_t stream);
void add_norm_backward(const AddNorm& n, const AddNormGrads& g, void* workspace, hipStream_t stream);

struct Quantize {
  uint32_t dtype;
  int64_t rows;
  int channels;
  Rows x;
};
// values [rows][channels], scale [rows]
void quantize_rows(const Quantize& z, int8_t* values, float* scale, hipStream_t stream);

struct Int8 {
  uint32_t dtype;
  int64_t rows;
  int inputs, outputs;
  Rows x;
  const int8_t* weight;  // [outputs][inputs]
  const float *scale, *bias;  // [outputs]; bias may be null
};
size_t int8_workspace(const Int8& p);
void int8_linear(const Int8& p, void* y, void* workspace, hipStream_t stream);

struct Embed {
  uint32_t dtype;
  int64_t tokens, vocab;
  int channels;
  const void* weight;
  int64_t weight_row;
  const int64_t* ids;
  float scale;
};
size_t embed_workspace(const Embed& e);
void embed(const Embed& e, void* y, hipStream_t stream);
void embed_backward(const Embed& e, const Rows& dy, void* dweight, void* workspace, hipStream_t stream);

struct Beam {
  uint32_t dtype;
  int requests, beams, width;
  int64_t vocab, row_stride, end;
  const void* logits;       // [requests * beams][vocab]
  const float* scores;      // [requests][beams]
  const uint8_t* finished;  // or null
};
struct BeamOut {
  float* score;  // [requests][width]
  int *parent, *token;
};
size_t beam_workspace(const Beam& b);
void beam_select(const Beam& b, const BeamOut& o, void* workspace, hipStream_t stream);

struct Moved {
  void* state;  // [cache][row_bytes]
  int64_t row_bytes;
};
// state[slot of beam j] <- state[slot of beam parent[j]] in place, for each request
void reorder_states(const Moved* states, int count, int requests, int beams, int cache, const int* parent,
                    const int* slots, hipStream_t stream);

constexpr int MAX_STATES = 128, MAX_TAPS = 8, MAX_TOP = 32;

}  // namespace fhe::clear
