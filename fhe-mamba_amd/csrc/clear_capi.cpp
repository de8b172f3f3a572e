// extern "C" boundary of the operators in the clear (include/fhecore.h):
// validation of everything that the host can see, and their descriptors as the
// kernels take them.
#include <cstdint>

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

}  // extern "C"
