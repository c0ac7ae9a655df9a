// Moves of cached sequences: rows (sequences) of a cache's buffers copied within it or from another cache, all rows
// read before any is written, or emptied.
//
// A move is a pair (source row order[i], destination row rows[i]). A row's bytes are cut into spans; a workgroup takes
// one span of one buffer for EVERY move. Different spans never touch the same bytes, so the only order to keep is
// inside the workgroup: it loads a pass (the same columns of every moving row) into registers, waits, meets at a
// barrier and stores. So a permutation, a cycle or a row that is both read and written needs no second buffer and no
// ordering of the moves, and every byte crosses the memory bus once each way. All buffers of all layers (56 to 64 of a
// 40-layer cache) go in one launch; one workgroup before it lists the moves that do something.
#include <type_traits>

#include "common.h"

namespace dsv41 {

constexpr int kMoveThreads = 256;
constexpr int kMoveWaves = kMoveThreads / 64;
constexpr int kMovePieces = 16;        // pieces of 16 bytes per thread and pass: 64 KB per workgroup
constexpr int kMoveBuffers = 64;       // buffers per plan launch (3 KB of kernel arguments)
constexpr int kMoveRows = 4096;        // most moves and most rows of a cache: one column of every row fits a pass
static_assert(kMoveRows <= kMoveThreads * kMovePieces, "a pass holds at least one piece of every move");
static_assert(kMoveBuffers <= kMoveThreads, "one thread per buffer of a plan launch");

// A buffer as the moves see it, in device memory.
struct MoveBuffer {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_stride, dst_stride;      // bytes between the sequences
  int64_t bytes;                       // bytes of a sequence that move
  uint32_t first;                      // the buffer's first workgroup
  uint32_t fill;                       // what an emptied row holds, word by word
};

// What the plan kernel leaves in the workspace: this, the buffers, then the moves that do something.
struct MovePlan {
  int32_t copies, emptied;
  int32_t pad[2];
};

// The plan kernel's arguments: up to 64 buffers by value. The table goes to device memory once, from one workgroup:
// arguments lie in host memory, and read by every workgroup of the moves they cost more than the moves (16 rows of
// 26 MB: 223 us against 100).
struct PlanArgs {
  MoveBuffer buffer[kMoveBuffers];
  MovePlan* plan;
  MoveBuffer* to;                      // this call's slice of the plan's buffers
  int2* list;                          // [moves]: copies from the front, emptied rows from the end
  const int32_t* order;
  const int32_t* rows;                 // null: move i goes to row i
  int buffers, moves, src_rows, dst_rows;
  int same;                            // source and destination are one cache: a row onto itself moves nothing
};

__global__ __launch_bounds__(kMoveThreads) void cache_plan_kernel(PlanArgs a) {
  extern __shared__ int last[];                             // the last move to each row [dst_rows]
  __shared__ int copies, emptied;
  for (int i = threadIdx.x; i < a.buffers; i += kMoveThreads) a.to[i] = a.buffer[i];
  if (a.moves == 0) return;                                 // a later slice of the buffers: the moves are listed
  if (threadIdx.x == 0) copies = emptied = 0;
  for (int i = threadIdx.x; i < a.dst_rows; i += kMoveThreads) last[i] = -1;
  __syncthreads();
  // a destination outside the cache is no move; of several to one row the last counts; a row onto itself is left alone
  for (int i = threadIdx.x; i < a.moves; i += kMoveThreads) {
    const int d = a.rows ? a.rows[i] : i;
    if (d >= 0 && d < a.dst_rows) atomicMax(&last[d], i);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.moves; i += kMoveThreads) {
    const int d = a.rows ? a.rows[i] : i, s = a.order[i];
    if (d < 0 || d >= a.dst_rows || last[d] != i) continue;
    if (s < 0 || s >= a.src_rows) a.list[a.moves - 1 - atomicAdd(&emptied, 1)] = make_int2(-1, d);
    else if (!(a.same && s == d)) a.list[atomicAdd(&copies, 1)] = make_int2(s, d);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.plan->copies = copies;
    a.plan->emptied = emptied;
  }
}

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// Moved rows are not read again soon: past the L2 (16 rows of 26 MB: 99 us against 110).
template <typename P>
__device__ __forceinline__ void put(P* p, P v) {
  if constexpr (sizeof(P) == 16) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// `bytes` bytes of one buffer for all n copies and m emptied rows of the list, in pieces of W bytes (16, 4 or 1: what
// pointers, strides and length are multiples of). list[i]: source row, destination row; gone[i]: emptied row.
//
// A wave's load takes 64 pieces: of one copy while there are at most 64 copies, of 2^s of them side by side beyond, so
// that one column of every copy always fits a pass. No load stands behind a branch (lanes past the end read the span's
// first piece again), so all 16 of a thread are in flight at once: with a wait behind each, 16 rows of 26 MB took 205 us.
template <int W>
__device__ __forceinline__ void move_span(const uint8_t* src, uint8_t* dst, int64_t ss, int64_t ds, int bytes,
                                          uint32_t fill, const int2* list, const int2* gone, int n, int m) {
  using P = std::conditional_t<W == 16, u32x4, std::conditional_t<W == 4, uint32_t, uint8_t>>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n > 0) {
    int s = 0;
    while (64 << s < n) ++s;
    const int groups = (n + (1 << s) - 1) >> s;             // wave loads for one column chunk of every copy
    const int width = 64 * W >> s;                          // bytes of a column chunk
    const int cols = kMoveWaves * kMovePieces / groups;     // chunks of a pass
    const int sub = lane >> (6 - s), col = (lane & ((64 >> s) - 1)) * W;
    const int c0 = wave / groups, g0 = wave - c0 * groups;  // the wave's first chunk and load, and the step to its next
    const int dc = kMoveWaves / groups, dg = kMoveWaves - dc * groups;
    for (int at = 0; at < bytes; at += cols * width) {
      P v[kMovePieces];
      int c = c0, g = g0;
      auto step = [&]() {
        c += dc;
        g += dg;
        if (g >= groups) {
          g -= groups;
          ++c;
        }
      };
#pragma unroll
      for (int j = 0; j < kMovePieces; ++j, step()) {
        const int i = (g << s) + sub, off = at + c * width + col;
        const bool live = c < cols && i < n && off < bytes;
        v[j] = *reinterpret_cast<const P*>(src + list[live ? i : 0].x * ss + (live ? off : 0));
      }
      // every load of the pass has returned before any wave stores
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      c = c0;
      g = g0;
      asm volatile("" : "+s"(c), "+s"(g));                  // counted again, not kept: 16 places are too many registers
#pragma unroll
      for (int j = 0; j < kMovePieces; ++j, step()) {
        const int i = (g << s) + sub, off = at + c * width + col;
        if (c < cols && i < n && off < bytes) put(reinterpret_cast<P*>(dst + list[i].y * ds + off), v[j]);
      }
    }
  }
  // behind the last pass's barrier: a row that was read may be emptied
  P none;
  if constexpr (W == 16) none = u32x4{fill, fill, fill, fill};
  else if constexpr (W == 4) none = fill;
  else none = (P)(fill >> 8 * (threadIdx.x & 3));           // byte by byte: spans and steps are whole words
  for (int i = 0; i < m; ++i)
    for (int off = threadIdx.x * W; off < bytes; off += kMoveThreads * W)
      put(reinterpret_cast<P*>(dst + gone[i].y * ds + off), none);
}

__global__ __launch_bounds__(kMoveThreads) void cache_move_kernel(const MovePlan* plan, const MoveBuffer* table,
                                                                  const int2* moved, int buffers, int moves, int span) {
  extern __shared__ int2 list[];                            // [moves]
  const int n = plan->copies, m = plan->emptied;
  if (n + m == 0) return;
  for (int i = threadIdx.x; i < n; i += kMoveThreads) list[i] = moved[i];
  for (int i = moves - m + threadIdx.x; i < moves; i += kMoveThreads) list[i] = moved[i];
  // this workgroup's buffer: the last one that starts at or before it
  const int lane = threadIdx.x & 63;
  int b = -1;
  for (int i = 0; i < buffers; i += 64)
    b += __popcll(__ballot(i + lane < buffers && table[min(i + lane, buffers - 1)].first <= blockIdx.x));
  const MoveBuffer t = table[b];
  const int64_t at = (int64_t)(blockIdx.x - t.first) * span;
  const int bytes = (int)min((int64_t)span, t.bytes - at);
  const uint8_t* src = t.src + at;
  uint8_t* dst = t.dst + at;
  const uint64_t all = reinterpret_cast<uint64_t>(src) | reinterpret_cast<uint64_t>(dst) | (uint64_t)t.src_stride |
                       (uint64_t)t.dst_stride | (uint64_t)bytes;
  const int2* gone = list + moves - m;
  __syncthreads();
  if ((all & 15) == 0) move_span<16>(src, dst, t.src_stride, t.dst_stride, bytes, t.fill, list, gone, n, m);
  else if ((all & 3) == 0) move_span<4>(src, dst, t.src_stride, t.dst_stride, bytes, t.fill, list, gone, n, m);
  else move_span<1>(src, dst, t.src_stride, t.dst_stride, bytes, t.fill, list, gone, n, m);
}

}  // namespace dsv41

using namespace dsv41;

extern "C" size_t dsv41_cache_move_workspace_bytes(int32_t buffers, int32_t moves) {
  if (buffers <= 0 || moves <= 0) return 0;
  return sizeof(MovePlan) + (size_t)buffers * sizeof(MoveBuffer) + (size_t)moves * sizeof(int2);
}

extern "C" int dsv41_cache_move(const void* const* src, void* const* dst, const int64_t* src_stride,
                                const int64_t* dst_stride, const int64_t* bytes, const uint32_t* fill, int32_t buffers,
                                const int32_t* order, const int32_t* rows, int32_t moves, int32_t src_rows,
                                int32_t dst_rows, int32_t same, void* workspace, size_t workspace_bytes,
                                hipStream_t stream) {
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
  int64_t blocks = 0;
  int live = 0;
  for (int i = 0; i < buffers; ++i) {
    DSV41_REQUIRE(bytes[i] >= 0, DSV41_E_ARG, "%s: buffer %d moves %lld bytes", what, i, (long long)bytes[i]);
    DSV41_REQUIRE(bytes[i] == 0 || (src[i] && dst[i]), DSV41_E_ARG, "%s: buffer %d is null", what, i);
    DSV41_REQUIRE(dst_rows == 1 || dst_stride[i] >= bytes[i], DSV41_E_ARG, "%s: buffer %d: rows of %lld bytes, %lld apart",
                  what, i, (long long)bytes[i], (long long)dst_stride[i]);
    live += bytes[i] > 0;
    blocks += (bytes[i] + span - 1) / span;
    DSV41_REQUIRE(blocks < (1 << 24), DSV41_E_ARG, "%s: too many bytes", what);   // a grid holds fewer than 2^32 threads
  }
  if (live == 0) return 0;
  const size_t need = dsv41_cache_move_workspace_bytes(buffers, moves);
  DSV41_REQUIRE(workspace && workspace_bytes >= need && aligned16(workspace), DSV41_E_WORKSPACE,
                "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  PlanArgs a;
  a.plan = static_cast<MovePlan*>(workspace);
  MoveBuffer* table = reinterpret_cast<MoveBuffer*>(a.plan + 1);
  a.list = reinterpret_cast<int2*>(table + buffers);
  a.order = order;
  a.rows = rows;
  a.src_rows = src_rows;
  a.dst_rows = dst_rows;
  a.same = same;
  uint32_t first = 0;
  int done = 0;
  for (int i = 0; i < buffers;) {
    a.buffers = 0;
    a.to = table + done;
    a.moves = done == 0 ? moves : 0;
    for (; i < buffers && a.buffers < kMoveBuffers; ++i) {
      if (bytes[i] == 0) continue;
      a.buffer[a.buffers++] = MoveBuffer{static_cast<const uint8_t*>(src[i]), static_cast<uint8_t*>(dst[i]), src_stride[i],
                                         dst_stride[i], bytes[i], first, fill[i]};
      first += (uint32_t)((bytes[i] + span - 1) / span);
    }
    if (a.buffers == 0) break;
    done += a.buffers;
    hipLaunchKernelGGL(cache_plan_kernel, dim3(1), dim3(kMoveThreads), (size_t)dst_rows * sizeof(int), stream, a);
  }
  hipLaunchKernelGGL(cache_move_kernel, dim3((unsigned)blocks), dim3(kMoveThreads), (size_t)moves * sizeof(int2), stream,
                     a.plan, table, a.list, done, moves, span);
  return check_launch(what);
}
