// Embedding lookup and its gradient:
//   y_t = scale weight[id_t];   dweight[v] = scale sum over t with id_t = v of dy_t
// Bound by memory: the rows read, the rows written, and for the gradient, which
// is dense, the whole table: 30011 tokens of 768 channels in 32 bits take 24 us, the
// gradient of 8192 in a table of 50280 11 + 43 + 5 (3.7 TB/s of reads and writes in the
// second of its kernels).  The gradient adds each row's tokens in an order that the ids
// fix, so that equal inputs give equal bits; no atomic addition of floats.  It is the
// tokens' own order but for frequent rows, which are cut where pieces of the order of all
// tokens end, so that their bits depend on how many tokens of lower ids there are:
//   k_direct does all for few tokens; for more
//   k_sort   a workgroup for each 256 rows of the table reads all ids, counts those
//            of its rows and those before them, and writes its tokens in order of
//            (id, token).  The ids are few beside the table, so that each workgroup
//            can read all of them, and nothing waits for a sort's passes.
//   k_sums   a wavefront a row of the table adds the row's tokens, or writes zeros.
//            Rows of more than `piece` tokens are left out here; a workgroup each
//            `piece` tokens of the order adds what of it belongs to such rows.
//   k_join   adds the pieces of such rows.
#pragma clang fp contract(fast)
#include <algorithm>

#include "clear.hpp"
#include "clear_rows.hpp"
#include "context.hpp"

namespace fhe::clear {
namespace {

// ----------------------------------------------------------------- lookup
// A wavefront a token, 16 bytes a lane.
template <class T>
__global__ __launch_bounds__(256) void k_embed(Embed e, T* y) {
  constexpr int VEC = Num<T>::VEC;
  const int64_t step = (int64_t)gridDim.x * 4;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < e.tokens; t += step) {
    const int64_t id = e.ids[t];
    T* out = y + t * e.channels;
    if (id < 0 || id >= e.vocab) {  // padding, or no token at all
      const T fill = (T)(id < 0 ? 0.0f : NAN);
      for (int c = lane_id(); c < e.channels; c += 64) out[c] = fill;
      continue;
    }
    const T* row = (const T*)e.weight + id * e.weight_row;
    if (e.channels < VEC) {
      const int c = lane_id();
      if (c < e.channels) out[c] = (T)((float)row[c] * e.scale);
      continue;
    }
    for (int c = lane_id() * VEC; c < e.channels; c += 64 * VEC) {
      const int at = min(c, e.channels - VEC);  // the last piece over the end of the one before
      union {
        u32x4 w;
        T v[VEC];
      } u;
      __builtin_memcpy(&u.w, row + at, 16);
      if (e.scale != 1.0f) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) u.v[i] = (T)((float)u.v[i] * e.scale);
      }
      __builtin_memcpy(out + at, &u.w, 16);
    }
  }
}

// ----------------------------------------------------------------- order of the tokens
constexpr int SPAN = 256, SORT_WAVES = 16, AHEAD = 4;

struct Order {
  int* start;  // [vocab + 1]: where each row's tokens begin
  int *token, *row;  // [tokens]: in order
};

// Each wavefront has a stretch of the tokens and a count for each row of its own,
// so that their order is that of (row, wavefront, place in the stretch).
__global__ __launch_bounds__(64 * SORT_WAVES) void k_sort(const int64_t* ids, int64_t tokens, int64_t vocab, Order o) {
  __shared__ int counts[SORT_WAVES][SPAN];
  __shared__ int sums[SORT_WAVES], before[SORT_WAVES];
  const int wave = threadIdx.x >> 6, lane = lane_id();
  const int64_t lo = (int64_t)blockIdx.x * SPAN;
  const int rows = (int)(vocab - lo < SPAN ? vocab - lo : SPAN);
  for (int i = lane; i < SPAN; i += 64) counts[wave][i] = 0;
  wave_sync();
  const int64_t length = (tokens + 64 * SORT_WAVES - 1) / (64 * SORT_WAVES) * 64;
  const int64_t begin = wave * length, end = begin + length < tokens ? begin + length : tokens;
  // an id beyond all rows stands for no token
  auto load = [&](int64_t t) { return t < end ? ids[t] : (int64_t)-1; };
  int lower = 0;
  for (int64_t t = begin + lane; t < end + lane; t += 64 * AHEAD) {
    int64_t id[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) id[j] = load(t + 64 * j);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      lower += id[j] >= 0 && id[j] < lo;
      const int64_t at = id[j] - lo;
      if (at >= 0 && at < rows) atomicAdd(&counts[wave][at], 1);
    }
  }
#pragma unroll
  for (int d = 32; d; d /= 2) lower += __shfl_xor(lower, d);
  if (lane == 0) before[wave] = lower;
  __syncthreads();
  // where each wavefront's tokens of each row begin: thread i has row i
  int total = 0, base = 0;
  if (threadIdx.x < SPAN) {
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int n = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = total;
      total += n;
      base += before[w];
    }
    int upto = total;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int n = __shfl_up(upto, d);
      if (lane >= d) upto += n;
    }
    if (lane == 63) sums[wave] = upto;
    base += upto - total;
  }
  __syncthreads();
  if (threadIdx.x < SPAN) {
    for (int w = 0; w < wave; ++w) base += sums[w];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) counts[w][threadIdx.x] += base;
    if ((int)threadIdx.x < rows) {
      o.start[lo + threadIdx.x] = base;
      if (lo + threadIdx.x + 1 == vocab) o.start[vocab] = base + total;
    }
  }
  __syncthreads();
  for (int64_t t = begin + lane; t < end + lane; t += 64 * AHEAD) {
    int64_t id[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) id[j] = load(t + 64 * j);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t at = id[j] - lo;
      const bool mine = at >= 0 && at < rows;
      uint64_t same = __ballot(mine);
      if (!same) continue;
      const int key = mine ? (int)at : 0;
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {  // the lanes of the same row
        const uint64_t set = __ballot(key >> bit & 1);
        same &= key >> bit & 1 ? set : ~set;
      }
      if (mine) {
        const int rank = __popcll(same & ((1ull << lane) - 1)), place = counts[wave][key] + rank;
        o.token[place] = (int)(t + 64 * j);
        o.row[place] = (int)id[j];
      }
      wave_sync();
      if (mine && __popcll(same >> lane) == 1) counts[wave][key] += __popcll(same);
      wave_sync();
    }
  }
}

// ----------------------------------------------------------------- sums
struct SumArgs {
  const void* dy;
  int64_t dy_row;
  void* dweight;
  Order o;
  int64_t vocab, tokens;
  int channels, piece, pieces;
  float scale;
  float* parts;  // [pieces][2][channels]: of the row that began before the piece, of the one that begins in it
};

constexpr int COLUMNS = 4;  // pieces of 256 channels at a time
// Tokens whose rows are asked for together.  In 32 bits all of them are in flight; in 16
// the widening stands in the branch on the channel, and each 256 channels are waited for.
constexpr int LOADS = 4;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The sum of dy over `token[0 .. count)`, for the channels that `first` and up hold
// in this wavefront's lanes.  count and first are the same in all lanes.
template <class T, int COVER>
__device__ __forceinline__ void add_rows(const SumArgs& a, const int* token, int count, int first,
                                         f32x4 (&sum)[COLUMNS]) {
  const int lane = lane_id();
#pragma unroll
  for (int k = 0; k < COLUMNS; ++k) sum[k] = f32x4{};
  for (int base = 0; base < count; base += 64) {
    const int some = count - base < 64 ? count - base : 64;
    const int mine = lane < some ? token[base + lane] : 0;
    for (int i = 0; i < some; i += LOADS) {
      f32x4 v[LOADS][COLUMNS];
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        // past the last token the last one again, times nothing
        const int t = __builtin_amdgcn_readlane(mine, i + j < some ? i + j : some - 1);
        const T* row = (const T*)a.dy + (int64_t)t * a.dy_row;
#pragma unroll
        for (int k = 0; k < COLUMNS; ++k) {
          const int c = first + k * 256;
          v[j][k] = c < a.channels ? Piece<COVER>(c + 4 * lane, a.channels).get(row) : f32x4{};
        }
      }
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        if (i + j < some) {
#pragma unroll
          for (int k = 0; k < COLUMNS; ++k) sum[k] += v[j][k];
        }
    }
  }
}

template <class T, int COVER>
__global__ __launch_bounds__(256) void k_sums(SumArgs a) {
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  if ((int)blockIdx.x < a.pieces) {
    // a row of more than `piece` tokens covers a piece's end or its begin
    const int64_t begin = (int64_t)blockIdx.x * a.piece, all = a.o.start[a.vocab];
    if (begin >= all) return;
    const int64_t end = begin + a.piece < all ? begin + a.piece : all;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int row = a.o.row[side ? end - 1 : begin];
      const int from = a.o.start[row], to = a.o.start[row + 1];
      if (to - from <= a.piece || (side ? from < begin : from >= begin)) continue;
      const int64_t f = from > begin ? from : begin, t = to < end ? to : end;
      float* out = a.parts + ((int64_t)blockIdx.x * 2 + side) * a.channels;
      for (int c0 = wave * 256 * COLUMNS; c0 < a.channels; c0 += 4 * 256 * COLUMNS) {
        f32x4 sum[COLUMNS];
        add_rows<T, COVER>(a, a.o.token + f, uniform((int)(t - f)), c0, sum);
#pragma unroll
        for (int k = 0; k < COLUMNS; ++k) {
          const int c = c0 + k * 256;
          if (c < a.channels) Piece<COVER>(c + 4 * lane, a.channels).put(out, sum[k]);
        }
      }
    }
    return;
  }
  const int64_t row = ((int64_t)blockIdx.x - a.pieces) * 4 + wave;
  if (row >= a.vocab) return;
  const int from = uniform(a.o.start[row]), count = uniform(a.o.start[row + 1]) - from;
  if (count > a.piece) return;
  T* out = (T*)a.dweight + row * a.channels;
  for (int c0 = 0; c0 < a.channels; c0 += 256 * COLUMNS) {
    f32x4 sum[COLUMNS];
    add_rows<T, COVER>(a, a.o.token + from, count, c0, sum);
#pragma unroll
    for (int k = 0; k < COLUMNS; ++k) {
      const int c = c0 + k * 256;
      if (c < a.channels) Piece<COVER>(c + 4 * lane, a.channels).put(out, sum[k] * a.scale);
    }
  }
}

// Few tokens, in one launch and without a workspace: a wavefront a row looks through
// all of them for its own.  Lookup and gradient of 128 tokens take 25 us in a table of
// 50280 x 768 (31 by their order), 6 in one of 93 x 768 (11); of 128 tokens of one row
// 37 and 33, of 256 63 and 33.
constexpr int DIRECT = 128;

template <class T, int COVER>
__global__ __launch_bounds__(256) void k_direct(SumArgs a, const int64_t* ids) {
  __shared__ int rows[DIRECT], mine[4][DIRECT];
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  for (int t = threadIdx.x; t < DIRECT; t += 256) {
    const int64_t id = t < a.tokens ? ids[t] : -1;
    rows[t] = id >= 0 && id < a.vocab ? (int)id : -1;
  }
  __syncthreads();
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.vocab) return;
  int count = 0;
#pragma unroll
  for (int j = 0; j < DIRECT; j += 64) {
    const bool own = rows[j + lane] == (int)row;
    const uint64_t found = __ballot(own);
    if (own) mine[wave][count + __popcll(found & ((1ull << lane) - 1))] = j + lane;
    count += __popcll(found);
  }
  wave_sync();
  T* out = (T*)a.dweight + row * a.channels;
  for (int c0 = 0; c0 < a.channels; c0 += 256 * COLUMNS) {
    f32x4 sum[COLUMNS];
    add_rows<T, COVER>(a, mine[wave], uniform(count), c0, sum);
#pragma unroll
    for (int k = 0; k < COLUMNS; ++k) {
      const int c = c0 + k * 256;
      if (c < a.channels) Piece<COVER>(c + 4 * lane, a.channels).put(out, sum[k] * a.scale);
    }
  }
}

// A workgroup a piece: if a long row begins in it, the sum of that row's parts, every
// sixteenth of them in one of its wavefronts.
constexpr int JOIN_WAVES = 16;

template <class T>
__global__ __launch_bounds__(64 * JOIN_WAVES) void k_join(SumArgs a) {
  __shared__ f32x4 lds[JOIN_WAVES][64];
  const int64_t begin = (int64_t)blockIdx.x * a.piece, all = a.o.start[a.vocab];
  if (begin >= all) return;
  const int64_t end = begin + a.piece < all ? begin + a.piece : all;
  const int row = a.o.row[end - 1];
  const int from = a.o.start[row], to = a.o.start[row + 1];
  if (to - from <= a.piece || from < begin) return;
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const int64_t first = blockIdx.x, last = (to - 1) / a.piece;
  for (int c0 = 0; c0 < a.channels; c0 += 256) {
    const int c = c0 + 4 * lane, count = a.channels - c;
    f32x4 sum{};
    for (int64_t i = first + wave; i <= last; i += JOIN_WAVES)
      sum += get4(a.parts + (2 * i + (i == first)) * a.channels + (count > 0 ? c : 0), count);
    lds[wave][lane] = sum;
    __syncthreads();
    if (!wave) {
#pragma unroll
      for (int w = 1; w < JOIN_WAVES; ++w) sum += lds[w][lane];
      if (count > 0) put4((T*)a.dweight + (int64_t)row * a.channels + c, sum * a.scale, count);
    }
    __syncthreads();
  }
}

// Tokens of a piece: 32, but at most 1024 pieces.  Longer ones leave one wavefront
// more rows to add one after another: 8192 tokens of 768 channels, as frequent as in
// text, take 58 us with 32, 70 with 128.
int piece_of(int64_t tokens) { return (int)std::max<int64_t>(32, (tokens + 1023) / 1024); }
size_t line(size_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

void embed(const Embed& e, void* y, hipStream_t stream) {
  if (!e.tokens) return;
  const uint32_t grid = (uint32_t)std::min<int64_t>((e.tokens + 3) / 4, 1 << 16);
  if (e.dtype == BF16) k_embed<bf16><<<grid, 256, 0, stream>>>(e, (bf16*)y);
  else k_embed<float><<<grid, 256, 0, stream>>>(e, (float*)y);
  hip_check(hipGetLastError(), "embedding");
}

size_t embed_workspace(const Embed& e) {
  if (e.tokens <= DIRECT) return 0;
  const int piece = piece_of(e.tokens);
  const int64_t pieces = (e.tokens + piece - 1) / piece;
  return line(4 * ((size_t)e.vocab + 1)) + 2 * line(4 * (size_t)e.tokens) + (size_t)pieces * 2 * e.channels * 4;
}

void embed_backward(const Embed& e, const Rows& dy, void* dweight, void* workspace, hipStream_t stream) {
  SumArgs a{};
  a.dy = dy.p;
  a.dy_row = dy.row;
  a.dweight = dweight;
  a.vocab = e.vocab;
  a.tokens = e.tokens;
  a.channels = e.channels;
  a.scale = e.scale;
  // f(type, cover)
  auto by_cover = [&](auto&& f) {
    auto go = [&](auto zero) {
      if (e.channels % 256 == 0) f(zero, std::integral_constant<int, WHOLE>{});
      else if (e.channels >= 4) f(zero, std::integral_constant<int, MOVED>{});
      else f(zero, std::integral_constant<int, SHORT>{});
    };
    if (e.dtype == BF16) go(bf16{});
    else go(float{});
  };
  if (e.tokens <= DIRECT) {
    by_cover([&](auto zero, auto cover) {
      k_direct<decltype(zero), cover()><<<(uint32_t)((e.vocab + 3) / 4), 256, 0, stream>>>(a, e.ids);
    });
    hip_check(hipGetLastError(), "embedding gradient of few tokens");
    return;
  }
  char* w = (char*)workspace;
  a.o.start = (int*)w;
  w += line(4 * ((size_t)e.vocab + 1));
  a.o.token = (int*)w;
  w += line(4 * (size_t)e.tokens);
  a.o.row = (int*)w;
  a.parts = (float*)(w + line(4 * (size_t)e.tokens));
  a.piece = piece_of(e.tokens);
  a.pieces = (int)((e.tokens + a.piece - 1) / a.piece);
  k_sort<<<(uint32_t)((e.vocab + SPAN - 1) / SPAN), 64 * SORT_WAVES, 0, stream>>>(e.ids, e.tokens, e.vocab, a.o);
  hip_check(hipGetLastError(), "order of tokens");
  const uint32_t grid = (uint32_t)(a.pieces + (e.vocab + 3) / 4);
  by_cover([&](auto zero, auto cover) { k_sums<decltype(zero), cover()><<<grid, 256, 0, stream>>>(a); });
  hip_check(hipGetLastError(), "embedding gradient");
  if (e.dtype == BF16) k_join<bf16><<<a.pieces, 64 * JOIN_WAVES, 0, stream>>>(a);
  else k_join<float><<<a.pieces, 64 * JOIN_WAVES, 0, stream>>>(a);
  hip_check(hipGetLastError(), "embedding gradient of frequent tokens");
}

}  // namespace fhe::clear
