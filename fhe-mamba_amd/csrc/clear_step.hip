// The scan's single-token form on a cache of states:
//   h <- exp(g) h + (w x) B^T,  y = h C + D x   for each request and head.
// A request reads and writes its states once (8 head_dim states bytes a head)
// and nothing else of size: bound by memory, and by the launch for a few.  24
// heads of 64 x 128: one request 4.0 us, the least a launch takes; 218 requests
// 56 us (6.2 TB/s) when their states are still in the last-level cache, about 80
// (4.3 TB/s) when they are not.
#pragma clang fp contract(fast)
#include "clear.hpp"
#include "clear_tile.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

struct StepArgs {
  Step s;
  void* y;
  int lanes_log;  // of the lanes of a state row
};

template <class T>
__device__ __forceinline__ float get(const void* p, int64_t i) {
  return (float)((const T*)p)[i];
}

// A row of the state (one channel) lies across 2^lanes_log lanes, VEC states
// each, PER times; a wavefront has 64 >> lanes_log rows at a time.
template <class T, int VEC, int PER>
__global__ __launch_bounds__(256) void k_step(StepArgs a) {
  const Step& s = a.s;
  const int head = blockIdx.y, request = blockIdx.z;
  const int lanes = 1 << a.lanes_log, lane = lane_id() & (lanes - 1);
  const int rows = 64 >> a.lanes_log;
  const int row0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * rows + (lane_id() >> a.lanes_log);
  const int step_rows = gridDim.x * 4 * rows;
  const int slot = s.slots ? s.slots[request] : request;
  T* y = (T*)a.y + ((int64_t)request * s.heads + head) * s.head_dim;
  if (slot < 0 || slot >= s.cache) {
    for (int p = row0; p < s.head_dim; p += step_rows)
      if (lane == 0) y[p] = (T)0.0f;
    return;
  }
  const int group = head / (s.heads / s.groups);
  const float decay = expf(((const float*)s.decay.p)[request * s.decay.tok + head * s.decay.head]);
  const float write = ((const float*)s.write.p)[request * s.write.tok + head * s.write.head];
  const float skip = s.d ? s.d[head] : 0.0f;
  const T* b = (const T*)s.b.p + request * s.b.tok + group * s.b.head;
  const T* c = (const T*)s.c.p + request * s.c.tok + group * s.c.head;
  const T* x = (const T*)s.x.p + request * s.x.tok + head * s.x.head;
  float* state = s.state + ((int64_t)slot * s.heads + head) * s.head_dim * s.states;

  float bv[PER][VEC], cv[PER][VEC];
#pragma unroll
  for (int k = 0; k < PER; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int n = (k * lanes + lane) * VEC + j;
      bv[k][j] = n < s.states ? (float)b[n] : 0.0f;
      cv[k][j] = n < s.states ? (float)c[n] : 0.0f;
    }
  for (int p = row0; p < s.head_dim; p += step_rows) {
    float* row = state + (int64_t)p * s.states;
    const float xv = (float)x[p], in = write * xv;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int n = (k * lanes + lane) * VEC;
      if (n >= s.states) continue;
      if constexpr (VEC == 4) {
        f32x4 h = *reinterpret_cast<const f32x4*>(row + n);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[j] = decay * h[j] + in * bv[k][j];
          sum += h[j] * cv[k][j];
        }
        *reinterpret_cast<f32x4*>(row + n) = h;
      } else {
        const float h = decay * row[n] + in * bv[k][0];
        sum += h * cv[k][0];
        row[n] = h;
      }
    }
    for (int d = lanes / 2; d; d /= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) y[p] = (T)(sum + skip * xv);
  }
}

template <class T>
void launch_step(const Step& s, void* y, hipStream_t stream) {
  StepArgs a{s, y, 0};
  const bool wide = s.states % 4 == 0 && reinterpret_cast<uintptr_t>(s.state) % 16 == 0;
  const int pieces = wide ? s.states / 4 : s.states;
  while (a.lanes_log < 6 && (1 << a.lanes_log) < pieces) ++a.lanes_log;
  const int rows = 4 * (64 >> a.lanes_log);  // of a workgroup, at a time
  const int most = (s.head_dim + rows - 1) / rows;
  // Few requests: as many workgroups as there are rows.  Many: a workgroup
  // walks up to eight groups of rows, so that B and C are read once for them.
  int split = most;
  while (split > 1 && (int64_t)split * s.heads * s.requests > 4096 && most / split < 8) split = (split + 1) / 2;
  const dim3 grid(split, s.heads, s.requests);
  if (wide) k_step<T, 4, 1><<<grid, 256, 0, stream>>>(a);
  else k_step<T, 1, 2><<<grid, 256, 0, stream>>>(a);
  hip_check(hipGetLastError(), "scan step");
}

}  // namespace

void step(const Step& s, void* y, hipStream_t stream) {
  if (s.dtype == BF16) launch_step<bf16>(s, y, stream);
  else launch_step<float>(s, y, stream);
}

}  // namespace fhe::clear
