// The three sweeps of the scan's gradients in one launch: those of C forward,
// those of B and of x in reverse.  None needs another's results, and together
// they leave fewer places of the chip empty than one after the other: 192 us at
// 4 x 2048 tokens of 24 heads of 64 x 128 in 16 bits, apart about 75 for x and 140
// for the two others.
#include "clear_scan_query.hpp"
#include "clear_scan_value.hpp"

#pragma clang fp contract(fast)
namespace fhe::clear {
namespace {

extern __shared__ __align__(16) char lds_raw[];

template <class T, int NB, int PT, bool FULL>
__global__ __launch_bounds__(64 * WAVES, 2) void k_backward(SweepArgs c, SweepArgs b, SweepArgs x, uint32_t queries) {
  // the longest first
  const uint32_t id = blockIdx.x;
  if (id < queries) query_sweep<T, NB, PT, false, FULL>(c, lds_raw, deal(id, queries));
  else if (id < 2 * queries) query_sweep<T, NB, PT, true, FULL>(b, lds_raw, deal(id - queries, queries));
  else
    value_sweep<T, NB, VALUE_COLS / 16, true, true, FULL>(x, lds_raw,
                                                          deal(id - 2 * queries, gridDim.x - 2 * queries));
}

template <class T, int NB, int PT>
void launch(const SweepArgs& c, const SweepArgs& b, const SweepArgs& x, int items, hipStream_t s) {
  constexpr size_t bytes = std::max(sizeof(QueryLds<T, NB, PT>), sizeof(ValueLds<T, NB, VALUE_COLS / 16, true>));
  static_assert(bytes <= LDS_BYTES);
  const bool full = is_full(c, NB) && is_full(b, NB) && is_full(x, NB);
  auto* kernel = full ? &k_backward<T, NB, PT, true> : &k_backward<T, NB, PT, false>;
  allow_lds((const void*)kernel, bytes);
  const uint32_t queries = workgroups(c, items), values = workgroups(x, items);
  if ((int64_t)2 * queries + values > INT32_MAX) throw ArgError("too many tokens and heads for one call");
  kernel<<<2 * queries + values, 64 * WAVES, bytes, s>>>(c, b, x, queries);
}

}  // namespace

void launch_backward(uint32_t dtype, const SweepArgs& c, const SweepArgs& b, const SweepArgs& x, int items,
                     hipStream_t s) {
  by_shape(dtype, c.states, [&](auto zero, auto blocks) {
    using T = decltype(zero);
    constexpr int NB = decltype(blocks)::value;
    if (c.cols == 32) launch<T, NB, 2>(c, b, x, items, s);
    else launch<T, NB, 4>(c, b, x, items, s);
  });
  hip_check(hipGetLastError(), "scan gradient sweeps");
}

}  // namespace fhe::clear
