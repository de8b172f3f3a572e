// extern "C" boundary of the operators in the clear (include/fhecore.h):
// validation of everything that the host can see, and their descriptors as the
// kernels take them.
#include <algorithm>
#include <cstdint>
#include <functional>
#include <vector>

#include "clear.hpp"
#include "status.hpp"

namespace {

using fhe::guard;
using fhe::need;
namespace clear = fhe::clear;

constexpr int64_t MAX_TOKENS = INT32_MAX, MAX_SEQS = 65535;

size_t elem(uint32_t dtype) {
  need(dtype == FHE_F32 || dtype == FHE_BF16, "dtype must be FHE_F32 or FHE_BF16");
  return dtype == FHE_BF16 ? 2 : 4;
}

void aligned(const void* p, size_t to, const char* msg) {
  need(reinterpret_cast<uintptr_t>(p) % to == 0, msg);
}

clear::Strided strided(const fhe_strided& t, size_t size) {
  need(t.data, "null input");
  aligned(t.data, size, "an input is not aligned to its type");
  for (int64_t s : t.stride) need(s >= 0, "strides must not be negative");
  return {t.data, t.stride[0], t.stride[1], t.stride[2]};
}

void check_workspace(const void* workspace, size_t bytes, size_t wanted) {
  need(bytes >= wanted, "the workspace is too small");
  need(workspace || !wanted, "null workspace");
  aligned(workspace, 256, "the workspace must be 256-byte aligned");
}

clear::Scan to_scan(const fhe_scan_args* a) {
  need(a, "null argument");
  const size_t size = elem(a->dtype);
  need(a->seqs >= 1 && a->seqs <= MAX_SEQS, "seqs must be 1 .. 65535");
  need(a->heads >= 1 && a->heads <= 4096 && a->groups >= 1 && a->heads % a->groups == 0,
       "heads must be 1 .. 4096 and a multiple of groups");
  need(a->head_dim >= 1 && a->head_dim <= 1024, "head_dim must be 1 .. 1024");
  need(a->states >= 1 && a->states <= FHE_MAX_STATES, "states must be 1 .. 128");
  need(a->tokens >= 0 && a->tokens <= MAX_TOKENS - 64, "tokens must be below 2^31");
  clear::Scan s{};
  s.dtype = a->dtype;
  s.seqs = (int)a->seqs;
  s.heads = (int)a->heads;
  s.head_dim = (int)a->head_dim;
  s.states = (int)a->states;
  s.groups = (int)a->groups;
  s.tokens = a->tokens;
  s.offsets = a->offsets;
  aligned(a->offsets, 4, "offsets are not aligned");
  aligned(a->d, 4, "d is not aligned");
  aligned(a->initial, 4, "initial is not aligned");
  s.d = a->d;
  s.initial = a->initial;
  if (s.all_tokens()) {
    s.x = strided(a->x, size);
    s.b = strided(a->b, size);
    s.c = strided(a->c, size);
    s.write = strided(a->write, 4);
    s.decay = strided(a->log_decay, 4);
  }
  return s;
}

clear::Conv to_conv(const fhe_conv_args* a) {
  need(a, "null argument");
  const size_t size = elem(a->dtype);
  need(a->seqs >= 1 && a->seqs <= MAX_SEQS, "seqs must be 1 .. 65535");
  need(a->channels >= 1 && a->channels <= (1u << 20), "channels must be 1 .. 2^20");
  need(a->taps >= 2 && a->taps <= FHE_MAX_TAPS, "taps must be 2 .. 8");
  need(a->tokens >= 0 && a->tokens <= MAX_TOKENS - 64, "tokens must be below 2^31");
  need(a->weight, "null weight");
  aligned(a->weight, 4, "weight is not aligned");
  aligned(a->bias, 4, "bias is not aligned");
  aligned(a->offsets, 4, "offsets are not aligned");
  aligned(a->initial, size, "initial is not aligned");
  clear::Conv c{};
  c.dtype = a->dtype;
  c.seqs = (int)a->seqs;
  c.channels = (int)a->channels;
  c.taps = (int)a->taps;
  c.tokens = a->tokens;
  c.offsets = a->offsets;
  if (c.all_tokens()) c.x = strided(a->x, size);
  c.weight = a->weight;
  c.bias = a->bias;
  c.initial = a->initial;
  c.silu = a->silu != 0;
  return c;
}

clear::Logprob to_logprob(const fhe_logprob_args* a) {
  need(a, "null argument");
  const size_t size = elem(a->dtype);
  need(a->rows >= 1 && a->rows <= (1 << 22), "rows must be 1 .. 2^22");
  need(a->vocab >= 1 && a->vocab <= (1 << 24), "vocab must be 1 .. 2^24");
  need(a->rows * (a->vocab / 4096 + 2) <= INT32_MAX, "too many logits for one call");
  need(a->row_stride >= a->vocab || a->rows == 1, "row_stride must be vocab or more");
  need(a->top <= FHE_MAX_TOP && a->top <= a->vocab, "top must be at most 32 and at most vocab");
  need(a->logits, "null logits");
  aligned(a->logits, size, "logits are not aligned to their type");
  aligned(a->targets, 8, "targets are not aligned");
  return {a->dtype, a->rows, a->vocab, a->row_stride, (int)a->top, a->logits, a->targets};
}

clear::Rows rows_at(const fhe_rows& r, size_t size) {
  need(r.data, "null input");
  aligned(r.data, size, "an input is not aligned to its type");
  need(r.stride >= 0, "strides must not be negative");
  return {r.data, r.stride};
}

int channels_of(int64_t channels, int64_t most, const char* msg) {
  need(channels >= 1 && channels <= most, msg);
  return (int)channels;
}

int64_t rows_of(int64_t rows) {
  need(rows >= 0 && rows <= INT32_MAX, "rows must be 0 .. 2^31 - 1");
  return rows;
}

void check_eps(float eps) { need(eps >= 0.0f && eps <= 3.4e38f, "eps must be 0 or more and finite"); }

void check_out(uint32_t dtype, uint32_t out) {
  elem(out);
  need(out == dtype || out == FHE_BF16, "out_dtype must be dtype or FHE_BF16");
}

clear::Norm to_norm(const fhe_norm_args* a) {
  need(a, "null argument");
  const size_t size = elem(a->dtype);
  check_out(a->dtype, a->out_dtype);
  check_eps(a->eps);
  clear::Norm n{};
  n.dtype = a->dtype;
  n.out_dtype = a->out_dtype;
  n.rows = rows_of(a->rows);
  n.channels = channels_of(a->channels, 1 << 20, "channels must be 1 .. 2^20");
  need(a->groups >= 1 && a->groups <= MAX_SEQS && a->channels % a->groups == 0,
       "channels must be a multiple of groups, which are at most 65535");
  n.groups = (int)a->groups;
  need(n.channels / n.groups <= FHE_MAX_ROW, "a group has at most 32768 channels");
  n.eps = a->eps;
  if (n.rows) {
    n.x = rows_at(a->x, size);
    if (a->gate.data) n.gate = rows_at(a->gate, size);
  } else {
    n.gate.p = a->gate.data;
  }
  need(a->weight, "null weight");
  aligned(a->weight, 4, "weight is not aligned");
  n.weight = a->weight;
  return n;
}

clear::AddNorm to_add_norm(const fhe_add_norm_args* a, bool read) {
  need(a, "null argument");
  elem(a->dtype);
  check_out(a->dtype, a->out_dtype);
  check_eps(a->eps);
  clear::AddNorm n{};
  n.dtype = a->dtype;
  n.out_dtype = a->out_dtype;
  n.rows = rows_of(a->rows);
  n.channels = channels_of(a->channels, FHE_MAX_ROW, "channels must be 1 .. 32768");
  n.eps = a->eps;
  if (n.rows && read) {
    n.hidden = rows_at(a->hidden, elem(a->dtype));
    n.update = rows_at(a->update, elem(a->out_dtype));
  }
  need(a->weight, "null weight");
  aligned(a->weight, 4, "weight is not aligned");
  aligned(a->scale, 4, "scale is not aligned");
  n.scale = a->scale;
  n.weight = a->weight;
  return n;
}

clear::Int8 to_int8(const fhe_int8_args* a) {
  need(a, "null argument");
  const size_t size = elem(a->dtype);
  clear::Int8 p{};
  p.dtype = a->dtype;
  p.rows = rows_of(a->rows);
  p.inputs = channels_of(a->inputs, FHE_MAX_ROW, "inputs must be 1 .. 32768");
  p.outputs = channels_of(a->outputs, 1 << 24, "outputs must be 1 .. 2^24");
  // Below this the largest products, of 128 x 128 tiles or more, have fewer than 2^24 workgroups
  // or tiles to number; a result has fewer than 2^34 elements.
  need((p.rows + 63) / 64 * ((a->outputs + 15) / 16) < (1 << 24), "too many outputs for one call");
  if (p.rows) p.x = rows_at(a->x, size);
  need(a->weight && a->scale, "null weight or scale");
  aligned(a->scale, 4, "scale is not aligned");
  aligned(a->bias, 4, "bias is not aligned");
  p.weight = a->weight;
  p.scale = a->scale;
  p.bias = a->bias;
  return p;
}

clear::Embed to_embed(const fhe_embed_args* a, bool read) {
  need(a, "null argument");
  const size_t size = elem(a->dtype);
  clear::Embed e{};
  e.dtype = a->dtype;
  need(a->tokens >= 0 && a->tokens <= (1 << 28), "tokens must be 0 .. 2^28");
  need(a->vocab >= 1 && a->vocab <= (1 << 24), "vocab must be 1 .. 2^24");
  e.tokens = a->tokens;
  e.vocab = a->vocab;
  e.channels = channels_of(a->channels, 1 << 20, "channels must be 1 .. 2^20");
  if (read) {
    const clear::Rows w = rows_at(a->weight, size);
    e.weight = w.p;
    e.weight_row = w.row;
  }
  need(a->ids || !a->tokens, "null ids");
  aligned(a->ids, 8, "ids are not aligned");
  e.ids = a->ids;
  e.scale = a->scale;
  return e;
}

clear::Beam to_beam(const fhe_beam_args* a) {
  need(a, "null argument");
  const size_t size = elem(a->dtype);
  need(a->requests >= 1 && a->requests <= MAX_SEQS, "requests must be 1 .. 65535");
  need(a->beams >= 1 && a->beams <= FHE_MAX_TOP, "beams must be 1 .. 32");
  need(a->vocab >= 1 && a->vocab <= (1 << 24), "vocab must be 1 .. 2^24");
  need(a->width >= 1 && a->width <= FHE_MAX_TOP && a->width <= a->beams * a->vocab,
       "width must be 1 .. 32 and at most beams * vocab");
  const int64_t rows = (int64_t)a->requests * a->beams;
  need(rows * (a->vocab / 4096 + 2) < (1 << 24), "too many logits for one call");
  need(a->row_stride >= a->vocab || rows == 1, "row_stride must be vocab or more");
  need(a->logits && a->scores, "null logits or scores");
  aligned(a->logits, size, "logits are not aligned to their type");
  aligned(a->scores, 4, "scores are not aligned");
  need(!a->finished || (a->end >= 0 && a->end < a->vocab), "end must be a token where beams may be finished");
  return {a->dtype, (int)a->requests, (int)a->beams, (int)a->width, a->vocab, a->row_stride, a->end,
          a->logits, a->scores, a->finished};
}

}  // namespace

extern "C" {

int fhe_ssm_scan_workspace(const fhe_scan_args* args, int backward, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::scan_workspace(to_scan(args), backward != 0);
  });
}

int fhe_ssm_scan(const fhe_scan_args* args, void* y, float* final_state, void* workspace, size_t bytes,
                 void* hip_stream) {
  return guard([&] {
    const clear::Scan s = to_scan(args);
    need(y || !s.all_tokens(), "null output");
    aligned(y, elem(s.dtype), "y is not aligned to its type");
    aligned(final_state, 4, "final_state is not aligned");
    check_workspace(workspace, bytes, clear::scan_workspace(s, false));
    clear::scan(s, y, final_state, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_ssm_scan_backward(const fhe_scan_args* args, const fhe_scan_grads* grads, void* workspace,
                          size_t bytes, void* hip_stream) {
  return guard([&] {
    const clear::Scan s = to_scan(args);
    need(grads, "null argument");
    clear::ScanGrads g{};
    if (s.all_tokens()) {
      g.dy = strided(grads->dy, elem(s.dtype));
      need(grads->dx && grads->dwrite && grads->dlog_decay && grads->db && grads->dc, "null output");
    }
    for (const void* p : {grads->dx, grads->db, grads->dc})
      aligned(p, elem(s.dtype), "a gradient is not aligned to its type");
    for (const float* p : {grads->dfinal, (const float*)grads->dwrite, (const float*)grads->dlog_decay,
                           (const float*)grads->dd, (const float*)grads->dinitial})
      aligned(p, 4, "a gradient is not aligned to its type");
    g.dfinal = grads->dfinal;
    g.dx = grads->dx;
    g.dwrite = grads->dwrite;
    g.ddecay = grads->dlog_decay;
    g.db = grads->db;
    g.dc = grads->dc;
    g.dd = grads->dd;
    g.dinitial = grads->dinitial;
    check_workspace(workspace, bytes, clear::scan_workspace(s, true));
    clear::scan_backward(s, g, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_ssm_step(const fhe_ssm_step_args* a, void* y, void* hip_stream) {
  return guard([&] {
    need(a && y, "null argument");
    const size_t size = elem(a->dtype);
    need(a->requests >= 1 && a->requests <= MAX_SEQS, "requests must be 1 .. 65535");
    need(a->cache >= 1 && a->cache <= INT32_MAX, "cache must be 1 .. 2^31 - 1");
    need(a->slots || a->requests <= a->cache, "more requests than rows of the state");
    need(a->heads >= 1 && a->heads <= 4096 && a->groups >= 1 && a->heads % a->groups == 0,
         "heads must be 1 .. 4096 and a multiple of groups");
    need(a->head_dim >= 1 && a->head_dim <= 1024, "head_dim must be 1 .. 1024");
    need(a->states >= 1 && a->states <= FHE_MAX_STATES, "states must be 1 .. 128");
    need(a->state, "null state");
    aligned(a->state, 4, "state is not aligned");
    aligned(a->slots, 4, "slots are not aligned");
    aligned(a->d, 4, "d is not aligned");
    aligned(y, size, "y is not aligned to its type");
    const clear::Step s{a->dtype, (int)a->requests, (int)a->cache, (int)a->heads, (int)a->head_dim,
                        (int)a->states, (int)a->groups, a->slots, strided(a->x, size), strided(a->b, size),
                        strided(a->c, size), strided(a->write, 4), strided(a->log_decay, 4), a->d, a->state};
    clear::step(s, y, (hipStream_t)hip_stream);
  });
}

int fhe_causal_conv(const fhe_conv_args* args, void* y, void* final_state, void* hip_stream) {
  return guard([&] {
    const clear::Conv c = to_conv(args);
    need(y || !c.all_tokens(), "null output");
    aligned(y, elem(c.dtype), "y is not aligned to its type");
    aligned(final_state, elem(c.dtype), "final_state is not aligned to its type");
    clear::conv(c, y, final_state, (hipStream_t)hip_stream);
  });
}

int fhe_causal_conv_workspace(const fhe_conv_args* args, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::conv_workspace(to_conv(args));
  });
}

int fhe_causal_conv_backward(const fhe_conv_args* args, const fhe_conv_grads* grads, void* workspace,
                             size_t bytes, void* hip_stream) {
  return guard([&] {
    const clear::Conv c = to_conv(args);
    need(grads && grads->dweight, "null output");
    clear::ConvGrads g{};
    if (c.all_tokens()) {
      g.dy = strided(grads->dy, elem(c.dtype));
      need(grads->dx, "null output");
    }
    for (const void* p : {(const void*)grads->dx, grads->dfinal, (const void*)grads->dinitial})
      aligned(p, elem(c.dtype), "a gradient is not aligned to its type");
    aligned(grads->dweight, 4, "dweight is not aligned");
    aligned(grads->dbias, 4, "dbias is not aligned");
    g.dfinal = grads->dfinal;
    g.dx = grads->dx;
    g.dweight = grads->dweight;
    g.dbias = grads->dbias;
    g.dinitial = grads->dinitial;
    check_workspace(workspace, bytes, clear::conv_workspace(c));
    clear::conv_backward(c, g, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_causal_conv_step(const fhe_conv_step_args* a, void* y, void* hip_stream) {
  return guard([&] {
    need(a && y, "null argument");
    const size_t size = elem(a->dtype);
    need(a->requests >= 1 && a->requests <= (1u << 20), "requests must be 1 .. 2^20");
    need(a->cache >= 1 && a->cache <= INT32_MAX, "cache must be 1 .. 2^31 - 1");
    need(a->slots || a->requests <= a->cache, "more requests than rows of the state");
    need(a->channels >= 1 && a->channels <= (1u << 20), "channels must be 1 .. 2^20");
    need(a->taps >= 2 && a->taps <= FHE_MAX_TAPS, "taps must be 2 .. 8");
    need(a->weight && a->state, "null weight or state");
    aligned(a->weight, 4, "weight is not aligned");
    aligned(a->bias, 4, "bias is not aligned");
    aligned(a->slots, 4, "slots are not aligned");
    aligned(a->state, size, "state is not aligned to its type");
    aligned(y, size, "y is not aligned to its type");
    const clear::ConvStep c{a->dtype, (int)a->requests, (int)a->cache, (int)a->channels, (int)a->taps,
                            a->slots, strided(a->x, size), a->weight, a->bias, a->state, a->silu != 0};
    clear::conv_step(c, y, (hipStream_t)hip_stream);
  });
}

int fhe_token_logprobs_workspace(const fhe_logprob_args* args, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::logprob_workspace(to_logprob(args));
  });
}

int fhe_token_logprobs(const fhe_logprob_args* args, const fhe_logprob_out* out, void* workspace,
                       size_t bytes, void* hip_stream) {
  return guard([&] {
    const clear::Logprob l = to_logprob(args);
    need(out && out->logprob && out->entropy && out->peak && out->log_sum, "null output");
    need(!l.top || (out->top_logprob && out->top_index), "null output");
    for (const void* p : {(const void*)out->logprob, (const void*)out->entropy, (const void*)out->peak,
                          (const void*)out->log_sum, (const void*)out->top_logprob, (const void*)out->top_index})
      aligned(p, 4, "an output is not aligned to its type");
    check_workspace(workspace, bytes, clear::logprob_workspace(l));
    clear::logprob(l, {out->logprob, out->entropy, out->peak, out->log_sum, out->top_logprob, out->top_index},
                   workspace, (hipStream_t)hip_stream);
  });
}

int fhe_token_logprobs_backward(const fhe_logprob_args* args, const float* peak, const float* log_sum,
                                const float* entropy, const float* dlogprob, const float* dentropy,
                                void* dlogits, void* hip_stream) {
  return guard([&] {
    const clear::Logprob l = to_logprob(args);
    need(peak && log_sum && entropy && dlogits, "null argument");
    need(l.targets || !dlogprob, "a gradient of log probabilities without targets");
    for (const float* p : {peak, log_sum, entropy, dlogprob, dentropy})
      aligned(p, 4, "an input is not aligned to its type");
    aligned(dlogits, elem(l.dtype), "dlogits is not aligned to its type");
    clear::logprob_backward(l, peak, log_sum, entropy, dlogprob, dentropy, dlogits,
                            (hipStream_t)hip_stream);
  });
}

int fhe_rms_norm(const fhe_norm_args* args, void* y, void* hip_stream) {
  return guard([&] {
    const clear::Norm n = to_norm(args);
    need(y || !n.rows, "null output");
    aligned(y, elem(n.out_dtype), "y is not aligned to its type");
    clear::norm(n, y, (hipStream_t)hip_stream);
  });
}

int fhe_rms_norm_workspace(const fhe_norm_args* args, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::norm_workspace(to_norm(args));
  });
}

int fhe_rms_norm_backward(const fhe_norm_args* args, const fhe_norm_grads* grads, void* workspace, size_t bytes,
                          void* hip_stream) {
  return guard([&] {
    const clear::Norm n = to_norm(args);
    need(grads && grads->dweight, "null output");
    clear::NormGrads g{};
    if (n.rows) {
      g.dy = rows_at(grads->dy, elem(n.out_dtype));
      need(grads->dx && (grads->dgate || !n.gate.p), "null output");
    }
    aligned(grads->dx, elem(n.dtype), "a gradient is not aligned to its type");
    aligned(grads->dgate, elem(n.dtype), "a gradient is not aligned to its type");
    aligned(grads->dweight, 4, "dweight is not aligned");
    g.dx = grads->dx;
    g.dgate = grads->dgate;
    g.dweight = grads->dweight;
    check_workspace(workspace, bytes, clear::norm_workspace(n));
    clear::norm_backward(n, g, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_add_norm(const fhe_add_norm_args* args, void* sum, void* y, void* hip_stream) {
  return guard([&] {
    const clear::AddNorm n = to_add_norm(args, true);
    need((sum && y) || !n.rows, "null output");
    aligned(sum, elem(n.dtype), "sum is not aligned to its type");
    aligned(y, elem(n.out_dtype), "y is not aligned to its type");
    clear::add_norm(n, sum, y, (hipStream_t)hip_stream);
  });
}

int fhe_add_norm_workspace(const fhe_add_norm_args* args, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::add_norm_workspace(to_add_norm(args, false));
  });
}

int fhe_add_norm_backward(const fhe_add_norm_args* args, const fhe_add_norm_grads* grads, void* workspace,
                          size_t bytes, void* hip_stream) {
  return guard([&] {
    need(args && grads && grads->dweight, "null output");
    need(!grads->dscale || args->scale, "a gradient of a scale that is not there");
    const bool whole = grads->sum && args->dtype == FHE_F32 && !args->scale;  // as add_norm_backward
    const clear::AddNorm n = to_add_norm(args, !whole);
    clear::AddNormGrads g{};
    if (n.rows) {
      if (grads->dy.data) g.dy = rows_at(grads->dy, elem(n.out_dtype));
      if (grads->dsum.data) g.dsum = rows_at(grads->dsum, elem(n.dtype));
    }
    aligned(grads->sum, elem(n.dtype), "sum is not aligned to its type");
    aligned(grads->dhidden, elem(n.dtype), "a gradient is not aligned to its type");
    aligned(grads->dupdate, elem(n.out_dtype), "a gradient is not aligned to its type");
    aligned(grads->dscale, 4, "dscale is not aligned");
    aligned(grads->dweight, 4, "dweight is not aligned");
    g.sum = grads->sum;
    g.dhidden = grads->dhidden;
    g.dupdate = grads->dupdate;
    g.dscale = grads->dscale;
    g.dweight = grads->dweight;
    check_workspace(workspace, bytes, clear::add_norm_workspace(n));
    clear::add_norm_backward(n, g, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_quantize_rows(const fhe_quantize_args* a, int8_t* values, float* scale, void* hip_stream) {
  return guard([&] {
    need(a, "null argument");
    const size_t size = elem(a->dtype);
    clear::Quantize z{};
    z.dtype = a->dtype;
    z.rows = rows_of(a->rows);
    z.channels = channels_of(a->channels, FHE_MAX_ROW, "channels must be 1 .. 32768");
    if (z.rows) {
      z.x = rows_at(a->x, size);
      need(values && scale, "null output");
    }
    aligned(scale, 4, "scale is not aligned");
    clear::quantize_rows(z, values, scale, (hipStream_t)hip_stream);
  });
}

int fhe_int8_linear_workspace(const fhe_int8_args* args, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::int8_workspace(to_int8(args));
  });
}

int fhe_int8_linear(const fhe_int8_args* args, void* y, void* workspace, size_t bytes, void* hip_stream) {
  return guard([&] {
    const clear::Int8 p = to_int8(args);
    need(y || !p.rows, "null output");
    aligned(y, elem(p.dtype), "y is not aligned to its type");
    check_workspace(workspace, bytes, clear::int8_workspace(p));
    clear::int8_linear(p, y, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_embed(const fhe_embed_args* args, void* y, void* hip_stream) {
  return guard([&] {
    const clear::Embed e = to_embed(args, true);
    need(y || !e.tokens, "null output");
    aligned(y, elem(e.dtype), "y is not aligned to its type");
    clear::embed(e, y, (hipStream_t)hip_stream);
  });
}

int fhe_embed_workspace(const fhe_embed_args* args, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::embed_workspace(to_embed(args, false));
  });
}

int fhe_embed_backward(const fhe_embed_args* args, const fhe_rows* dy, void* dweight, void* workspace, size_t bytes,
                       void* hip_stream) {
  return guard([&] {
    const clear::Embed e = to_embed(args, false);
    need(dy && dweight, "null argument");
    clear::Rows d{};
    if (e.tokens) d = rows_at(*dy, elem(e.dtype));
    aligned(dweight, elem(e.dtype), "dweight is not aligned to its type");
    check_workspace(workspace, bytes, clear::embed_workspace(e));
    clear::embed_backward(e, d, dweight, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_beam_select_workspace(const fhe_beam_args* args, size_t* bytes) {
  return guard([&] {
    need(bytes, "null argument");
    *bytes = clear::beam_workspace(to_beam(args));
  });
}

int fhe_beam_select(const fhe_beam_args* args, const fhe_beam_out* out, void* workspace, size_t bytes,
                    void* hip_stream) {
  return guard([&] {
    const clear::Beam b = to_beam(args);
    need(out && out->score && out->parent && out->token, "null output");
    for (const void* p : {(const void*)out->score, (const void*)out->parent, (const void*)out->token})
      aligned(p, 4, "an output is not aligned to its type");
    check_workspace(workspace, bytes, clear::beam_workspace(b));
    clear::beam_select(b, {out->score, out->parent, out->token}, workspace, (hipStream_t)hip_stream);
  });
}

int fhe_reorder_states(const fhe_state_rows* states, uint32_t count, uint32_t requests, uint32_t beams,
                       uint32_t cache, const int32_t* parent, const int32_t* slots, void* hip_stream) {
  return guard([&] {
    need(states && parent, "null argument");
    need(count >= 1 && count <= 65536, "count must be 1 .. 65536");
    need(requests >= 1 && requests <= MAX_SEQS, "requests must be 1 .. 65535");
    need(beams >= 1 && beams <= FHE_MAX_TOP, "beams must be 1 .. 32");
    need(cache >= 1 && cache <= INT32_MAX, "cache must be 1 .. 2^31 - 1");
    need(slots || (int64_t)requests * beams <= cache, "more beams than rows of the states");
    aligned(parent, 4, "parent is not aligned");
    aligned(slots, 4, "slots are not aligned");
    std::vector<clear::Moved> moved;
    for (uint32_t i = 0; i < count; ++i) {
      need(states[i].data || !states[i].row_bytes, "null state");
      need(states[i].row_bytes >= 0 && states[i].row_bytes <= (1 << 30), "row_bytes must be 0 .. 2^30");
      moved.push_back({states[i].data, states[i].row_bytes});
    }
    // two threads would move the same bytes
    std::vector<clear::Moved> by_place = moved;
    std::sort(by_place.begin(), by_place.end(), [](auto& a, auto& b) { return std::less<>()(a.state, b.state); });
    const char* end = nullptr;
    for (const clear::Moved& m : by_place) {
      if (!m.row_bytes) continue;
      need(!std::less<>()((const char*)m.state, end), "two of the states share memory");
      end = (const char*)m.state + m.row_bytes * cache;
    }
    clear::reorder_states(moved.data(), (int)count, (int)requests, (int)beams, (int)cache, parent, slots,
                          (hipStream_t)hip_stream);
  });
}

}  // extern "C"
