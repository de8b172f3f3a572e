// The scan's forward sweep, and the sweeps that make the states of segments: of
// the recurrence, and for the gradients also of its adjoint, in one launch.
#include "clear_scan_value.hpp"

#pragma clang fp contract(fast)
namespace fhe::clear {
namespace {

extern __shared__ __align__(16) char lds_raw[];

template <class T, int NB, bool FULL>
__global__ __launch_bounds__(64 * WAVES, 2) void k_forward(SweepArgs a) {
  value_sweep<T, NB, VALUE_COLS / 16, false, true, FULL>(a, lds_raw, deal(blockIdx.x, gridDim.x));
}

template <class T, int NB, bool FULL>
__global__ __launch_bounds__(64 * WAVES, 2) void k_states(SweepArgs a, SweepArgs r) {
  const uint32_t id = deal(blockIdx.x, gridDim.x);
  if (blockIdx.y == 0) value_sweep<T, NB, VALUE_COLS / 16, false, false, FULL>(a, lds_raw, id);
  else value_sweep<T, NB, VALUE_COLS / 16, true, false, FULL>(r, lds_raw, id);
}

}  // namespace

void launch_forward(uint32_t dtype, const SweepArgs& a, int items, hipStream_t s) {
  by_shape(dtype, a.states, [&](auto zero, auto blocks) {
    using T = decltype(zero);
    constexpr int NB = decltype(blocks)::value;
    constexpr size_t bytes = sizeof(ValueLds<T, NB, VALUE_COLS / 16, true>);
    static_assert(bytes <= LDS_BYTES);
    auto* kernel = is_full(a, NB) ? &k_forward<T, NB, true> : &k_forward<T, NB, false>;
    allow_lds((const void*)kernel, bytes);
    kernel<<<workgroups(a, items), 64 * WAVES, bytes, s>>>(a);
  });
  hip_check(hipGetLastError(), "scan sweep");
}

void launch_states(uint32_t dtype, const SweepArgs& a, const SweepArgs* reverse, int items, hipStream_t s) {
  by_shape(dtype, a.states, [&](auto zero, auto blocks) {
    using T = decltype(zero);
    constexpr int NB = decltype(blocks)::value;
    constexpr size_t bytes = sizeof(ValueLds<T, NB, VALUE_COLS / 16, false>);
    static_assert(bytes <= LDS_BYTES);
    const bool full = is_full(a, NB) && (!reverse || is_full(*reverse, NB));
    auto* kernel = full ? &k_states<T, NB, true> : &k_states<T, NB, false>;
    allow_lds((const void*)kernel, bytes);
    kernel<<<dim3(workgroups(a, items), reverse ? 2 : 1), 64 * WAVES, bytes, s>>>(a, reverse ? *reverse : a);
  });
  hip_check(hipGetLastError(), "scan states");
}

}  // namespace fhe::clear
