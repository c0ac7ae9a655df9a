// Moves of cached sequences: rows (sequences) of a cache's buffers copied within it or from another cache, all rows
// read before any is written, or emptied.
//
// A move is a pair (source row order[i], destination row rows[i]). A row's bytes are cut into spans; a workgroup takes
// one span of one buffer for EVERY move. Different spans never touch the same bytes, so the only order to keep is
// inside the workgroup: it loads a pass (the same columns of every moving row) into registers, waits, meets at a
// barrier and stores. So a permutation, a cycle or a row that is both read and written needs no second buffer and no
// ordering of the moves, and every byte crosses the memory bus once each way. All buffers of all layers go in one
// launch, their table in the kernel's arguments: a 40-layer cache has 56 to 64 of them.
#include <type_traits>

#include "common.h"

namespace dsv41 {

constexpr int kMoveThreads = 256;
constexpr int kMovePieces = 16;        // pieces of 16 bytes per thread and pass: 64 KB per workgroup
constexpr int kMoveBuffers = 64;       // buffers per launch (3 KB of kernel arguments)
constexpr int kMoveRows = 4096;        // most moves and most rows of a cache: one column of every row fits a pass
static_assert(kMoveRows <= kMoveThreads * kMovePieces, "a pass holds at least one piece of every move");

struct MoveArgs {
  const uint8_t* src[kMoveBuffers];
  uint8_t* dst[kMoveBuffers];
  int64_t src_stride[kMoveBuffers];    // bytes between the sequences of a buffer
  int64_t dst_stride[kMoveBuffers];
  int64_t bytes[kMoveBuffers];         // bytes of a sequence that move
  uint32_t first[kMoveBuffers];        // the buffer's first workgroup
  uint32_t fill[kMoveBuffers];         // what an emptied row holds, word by word
  const int32_t* order;
  const int32_t* rows;                 // null: move i goes to row i
  int buffers, moves, src_rows, dst_rows;
  int same;                            // source and destination are one cache: a row onto itself moves nothing
  int span;                            // bytes of a row per workgroup
};

// `bytes` bytes of one buffer for all n moves of the list, in pieces of W bytes (16, 4 or 1: what pointers, strides and
// length are multiples of). list[i]: source row (-1: emptied), destination row.
template <int W>
__device__ __forceinline__ void move_span(const uint8_t* src, uint8_t* dst, int64_t ss, int64_t ds, int bytes,
                                          uint32_t fill, const int2* list, int n) {
  using P = std::conditional_t<W == 16, uint4, std::conditional_t<W == 4, uint32_t, uint8_t>>;
  const int per = bytes / W;                                                  // pieces of one row
  const int cols = min(per, kMoveThreads * kMovePieces / n);                  // of each row in one pass, at least 1
  P none;
  if constexpr (W == 16) none = make_uint4(fill, fill, fill, fill);
  else none = (P)fill;
  for (int at = 0; at < per; at += cols) {
    const int w = min(cols, per - at), total = w * n;
    P v[kMovePieces];
    int64_t to[kMovePieces];
#pragma unroll
    for (int j = 0; j < kMovePieces; ++j) {
      const int p = threadIdx.x + j * kMoveThreads;
      if (p >= total) continue;
      const int i = p / w;
      const int64_t c = (int64_t)(at + p - i * w) * W;
      const int2 mv = list[i];
      to[j] = mv.y * ds + c;
      v[j] = mv.x < 0 ? none : *reinterpret_cast<const P*>(src + mv.x * ss + c);
    }
    // every load of the pass has returned before any wave stores
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMovePieces; ++j)
      if (threadIdx.x + j * kMoveThreads < total) *reinterpret_cast<P*>(dst + to[j]) = v[j];
  }
}

__global__ __launch_bounds__(kMoveThreads) void cache_move_kernel(MoveArgs a) {
  extern __shared__ int2 list[];                            // [moves], then the last move to each row [dst_rows]
  __shared__ int count;
  int* last = reinterpret_cast<int*>(list + a.moves);
  if (threadIdx.x == 0) count = 0;
  for (int i = threadIdx.x; i < a.dst_rows; i += kMoveThreads) last[i] = -1;
  __syncthreads();
  // the moves that do something: a destination outside the cache is none; of several to one row the last counts; a
  // row onto itself is left alone
  for (int i = threadIdx.x; i < a.moves; i += kMoveThreads) {
    const int d = a.rows ? a.rows[i] : i;
    if (d >= 0 && d < a.dst_rows) atomicMax(&last[d], i);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.moves; i += kMoveThreads) {
    const int d = a.rows ? a.rows[i] : i;
    int s = a.order[i];
    if (s < 0 || s >= a.src_rows) s = -1;
    if (d >= 0 && d < a.dst_rows && last[d] == i && !(a.same && s == d)) list[atomicAdd(&count, 1)] = make_int2(s, d);
  }
  __syncthreads();
  const int n = count;
  if (n == 0) return;
  int b = 0;
  while (b + 1 < a.buffers && a.first[b + 1] <= blockIdx.x) ++b;
  const int64_t at = (int64_t)(blockIdx.x - a.first[b]) * a.span;
  const int bytes = (int)min((int64_t)a.span, a.bytes[b] - at);
  const uint8_t* src = a.src[b] + at;
  uint8_t* dst = a.dst[b] + at;
  const int64_t ss = a.src_stride[b], ds = a.dst_stride[b];
  const uint64_t all = reinterpret_cast<uint64_t>(src) | reinterpret_cast<uint64_t>(dst) | (uint64_t)ss | (uint64_t)ds |
                       (uint64_t)bytes;
  if ((all & 15) == 0) move_span<16>(src, dst, ss, ds, bytes, a.fill[b], list, n);
  else if ((all & 3) == 0) move_span<4>(src, dst, ss, ds, bytes, a.fill[b], list, n);
  else move_span<1>(src, dst, ss, ds, bytes, a.fill[b], list, n);
}

}  // namespace dsv41

using namespace dsv41;

extern "C" int dsv41_cache_move(const void* const* src, void* const* dst, const int64_t* src_stride,
                                const int64_t* dst_stride, const int64_t* bytes, const uint32_t* fill, int32_t buffers,
                                const int32_t* order, const int32_t* rows, int32_t moves, int32_t src_rows,
                                int32_t dst_rows, int32_t same, hipStream_t stream) {
  const char* what = "dsv41_cache_move";
  DSV41_REQUIRE(buffers >= 0 && moves >= 0 && src_rows > 0 && dst_rows > 0, DSV41_E_ARG,
                "%s: buffers %d, moves %d, rows %d and %d", what, buffers, moves, src_rows, dst_rows);
  DSV41_REQUIRE(moves <= kMoveRows && dst_rows <= kMoveRows, DSV41_E_SHAPE, "%s: at most %d moves and rows, got %d and %d",
                what, kMoveRows, moves, dst_rows);
  if (buffers == 0 || moves == 0) return 0;
  DSV41_REQUIRE(src && dst && src_stride && dst_stride && bytes && fill && order, DSV41_E_ARG, "%s: null table", what);
  DSV41_REQUIRE(rows || moves <= dst_rows, DSV41_E_ARG, "%s: %d moves without rows into %d rows", what, moves, dst_rows);
  // a pass of the workgroup holds 64 KB of all moves: long spans where few rows move
  int span = kMoveThreads * kMovePieces * 16;
  while (span > 4096 && (int64_t)span * moves > kMoveThreads * kMovePieces * 16) span >>= 1;
  MoveArgs a;
  a.order = order;
  a.rows = rows;
  a.moves = moves;
  a.src_rows = src_rows;
  a.dst_rows = dst_rows;
  a.same = same;
  a.span = span;
  for (int i = 0; i < buffers;) {
    int64_t blocks = 0;
    a.buffers = 0;
    for (; i < buffers && a.buffers < kMoveBuffers; ++i) {
      DSV41_REQUIRE(bytes[i] >= 0, DSV41_E_ARG, "%s: buffer %d moves %lld bytes", what, i, (long long)bytes[i]);
      if (bytes[i] == 0) continue;
      DSV41_REQUIRE(src[i] && dst[i], DSV41_E_ARG, "%s: buffer %d is null", what, i);
      const int b = a.buffers++;
      a.src[b] = static_cast<const uint8_t*>(src[i]);
      a.dst[b] = static_cast<uint8_t*>(dst[i]);
      a.src_stride[b] = src_stride[i];
      a.dst_stride[b] = dst_stride[i];
      a.bytes[b] = bytes[i];
      a.fill[b] = fill[i];
      a.first[b] = (uint32_t)blocks;
      blocks += (bytes[i] + span - 1) / span;
      DSV41_REQUIRE(blocks < (1ll << 31), DSV41_E_ARG, "%s: too many bytes", what);
    }
    if (a.buffers == 0) continue;
    const size_t lds = (size_t)moves * sizeof(int2) + (size_t)dst_rows * sizeof(int);
    hipLaunchKernelGGL(cache_move_kernel, dim3((unsigned)blocks), dim3(kMoveThreads), lds, stream, a);
    const int rc = check_launch(what);
    if (rc) return rc;
  }
  return 0;
}
