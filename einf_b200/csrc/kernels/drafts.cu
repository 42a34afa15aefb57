// After the step that verified a draft: the longest path of the tree that the model agrees with, and the keys and
// values of its nodes moved to where the cache goes on.  Both are a few kilobytes and bound by the latency of their
// loads: each is one launch for all requests (and, for the move, all layers).  In captured graphs: paths of 64 trees of
// 64 nodes 2.7 us, of one tree of 8 2.0 us; the rows of 32 paths of 6 nodes in all layers' caches 3.9 us, of one of three 2.9 us.
#include "common.cuh"

namespace einf {

constexpr int kWalkNodes = 1024;      // nodes whose children lie in shared memory

// A call's arguments, as the caller packs them.
struct WalkParams {
  const int* tokens;       // [rows]: a node's token
  const int* targets;      // [rows]: the model's token behind that node
  const int* parents;      // [rows]: index within the request, before the node's own; others hang on nothing
  const int* q_start;      // [requests + 1]
  int* path;               // [requests, depth]: the kept nodes, -1 behind the last
  int* answer;             // [requests, depth]: the tokens that the step answers, -1 behind the last
  int* counts;             // [requests]
  int rows, requests, depth, more;
};
static_assert(sizeof(WalkParams) == 7 * 8 + 4 * 4, "as packed");

// A warp per request.  Every node that agrees with its parent's target reports to that parent, which keeps the lowest
// (an integer minimum: no order of arrival shows); the walk from the root then is a chain of reads of shared memory.
__global__ void __launch_bounds__(32) accept_drafts_kernel(WalkParams p) {
  __shared__ int child[kWalkNodes];
  __shared__ int walked[kWalkNodes];
  // No early launch of the dependents: where a path is its root alone this is the last kernel of a step, and the next step's read
  // the step's keys and values before their own wait.
  pdl_wait();
  const int request = blockIdx.x, lane = threadIdx.x;
  const int first = max(0, min(p.q_start[request], p.rows)), nodes = max(0, min(p.q_start[request + 1], p.rows) - first);
  const int *tokens = p.tokens + first, *targets = p.targets + first, *parents = p.parents + first;
  int* path = p.path + (size_t)request * p.depth;
  int* answer = p.answer + (size_t)request * p.depth;
  int count = 0;
  if (nodes <= kWalkNodes) {
    for (int k = lane; k < nodes; k += 32) child[k] = nodes;
    __syncwarp();
    for (int k = lane; k < nodes; k += 32) {
      const int up = parents[k];
      if (up >= 0 && up < k && tokens[k] == targets[up]) atomicMin(child + up, k);
    }
    __syncwarp();
    for (int node = 0; node < nodes && count < p.depth; node = child[node]) {
      if (lane == 0) walked[count] = node;
      ++count;
    }
    __syncwarp();
    for (int i = lane; i < count; i += 32) {
      path[i] = walked[i];
      answer[i] = targets[walked[i]];
    }
  } else {
    for (int node = 0; node < nodes && count < p.depth;) {
      const int target = targets[node];
      if (lane == 0) {
        path[count] = node;
        answer[count] = target;
      }
      ++count;
      int next = nodes;
      for (int k0 = node + 1; k0 < nodes && next == nodes; k0 += 32) {
        const int k = k0 + lane;
        const uint32_t found = __ballot_sync(0xffffffffu, k < nodes && parents[k] == node && tokens[k] == target);
        if (found) next = k0 + __ffs(found) - 1;
      }
      node = next;
    }
  }
  for (int i = count + lane; i < p.depth; i += 32) path[i] = answer[i] = -1;
  if (lane == 0) p.counts[request] = count;
}

constexpr int kMoveTensors = 192;     // tensors of one launch: their table travels with the launch
constexpr int kMoveThreads = 128;
constexpr int kMoveSteps = 64;        // steps of a path whose places lie in shared memory at a time
constexpr int kMoveAhead = 8;         // rows that a thread has in flight

struct MoveTensor {
  void* base;              // [pages, kv_heads, page_size, row_units units]
  int first_column;        // of the launch's columns
  int row_units;
};
// A call's arguments, as the caller packs them.
struct MoveCall {
  const int* block_table;  // [requests, table_width]
  const int* cached_lens;
  const int* path;         // [requests, depth]
  const int* counts;
  int* status;
  int requests, depth, table_width, more;
};
static_assert(sizeof(MoveCall) == 5 * 8 + 4 * 4, "as packed");
struct MoveParams {
  MoveTensor tensors[kMoveTensors];
  MoveCall call;
  int count, columns, page_size, num_pages;
};

// A column is one unit (16 bytes where all rows allow it) of one head's row in one tensor; a thread takes a column and
// moves it from place cached + path[i] to cached + i for i = 1, 2, ...  A path only rises, so path[i] >= i: no place is
// read after it was written as long as a thread reads in order, a few rows ahead of its stores.
template <typename Unit>
__global__ void __launch_bounds__(kMoveThreads) move_accepted_kernel(const __grid_constant__ MoveParams p) {
  __shared__ long long from[kMoveSteps], to[kMoveSteps];     // places: the page in the high half, the row in the low one
  // No early launch of the dependents: the rows are those of cached tokens from here on, which the attention of later steps reads
  // before its own wait.
  pdl_wait();
  const int request = blockIdx.x;
  const int count = max(0, min(p.call.counts[request], p.call.depth)), cached = p.call.cached_lens[request];
  const int* path = p.call.path + (size_t)request * p.call.depth;
  const int* table = p.call.block_table + (size_t)request * p.call.table_width;
  const int column = blockIdx.y * kMoveThreads + threadIdx.x;
  Unit* base = nullptr;
  int head = 0, unit = 0, row_units = 0, heads = 1;
  if (column < p.columns) {
    int low = 0, high = p.count - 1;
    while (low < high) {
      const int middle = (low + high + 1) >> 1;
      if (p.tensors[middle].first_column <= column) low = middle;
      else high = middle - 1;
    }
    const int next = low + 1 < p.count ? p.tensors[low + 1].first_column : p.columns;
    base = static_cast<Unit*>(p.tensors[low].base);
    row_units = p.tensors[low].row_units;
    heads = (next - p.tensors[low].first_column) / row_units;
    head = (column - p.tensors[low].first_column) / row_units;
    unit = (column - p.tensors[low].first_column) % row_units;
  }
  auto place = [&](int at) -> long long {     // page and row of a place, or -1
    if (at < 0 || at / p.page_size >= p.call.table_width) {
      atomicOr(p.call.status, kStatusBadPage);
      return -1;
    }
    const int page = table[at / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      atomicOr(p.call.status, kStatusBadPage);
      return -1;
    }
    return (long long)page << 32 | (unsigned)(at % p.page_size);
  };
  for (int i0 = 1; i0 < count; i0 += kMoveSteps) {
    __syncthreads();
    for (int i = i0 + threadIdx.x; i < min(count, i0 + kMoveSteps); i += kMoveThreads) {
      const int step = path[i];
      long long a = -1, b = -1;
      if (step < i || step <= path[i - 1]) atomicOr(p.call.status, kStatusBadIndex);
      else if (step != i) a = place(cached + step), b = place(cached + i);
      from[i - i0] = b < 0 ? -1 : a;
      to[i - i0] = b;
    }
    __syncthreads();
    if (!base) continue;
    const int steps = min(count - i0, kMoveSteps);
    for (int s0 = 0; s0 < steps; s0 += kMoveAhead) {
      Unit held[kMoveAhead];
      auto row = [&](long long at) {
        return base + (((at >> 32) * heads + head) * p.page_size + (long long)(at & 0xffffffff)) * row_units + unit;
      };
#pragma unroll
      for (int s = 0; s < kMoveAhead; ++s)
        if (s0 + s < steps && from[s0 + s] >= 0) held[s] = *row(from[s0 + s]);
#pragma unroll
      for (int s = 0; s < kMoveAhead; ++s)
        if (s0 + s < steps && from[s0 + s] >= 0) *row(to[s0 + s]) = held[s];
    }
  }
}

}  // namespace einf

using namespace einf;

// call: a WalkParams, on the host.
extern "C" int einf_accept_drafts(const char* call, cudaStream_t stream) {
  const WalkParams& p = *reinterpret_cast<const WalkParams*>(call);
  if (p.requests == 0) return 0;
  if (p.depth < 1) return (int)cudaErrorInvalidValue;
  return (int)launch_pdl(accept_drafts_kernel, dim3(p.requests), dim3(32), 0, stream, p);
}

// tensors: how many, bytes of a unit (2, 4, 8 or 16), page size, pages, then each tensor's address, heads and units of a
// row; call: a MoveCall.  Both on the host.
extern "C" int einf_move_accepted(const long long* tensors, const char* call, cudaStream_t stream) {
  const MoveCall& c = *reinterpret_cast<const MoveCall*>(call);
  const long long count = tensors[0], unit = tensors[1];
  if (c.requests == 0 || count == 0 || c.depth < 2) return 0;
  if (count < 0 || count > kMoveTensors || tensors[2] < 1) return (int)cudaErrorInvalidValue;
  MoveParams p;
  p.call = c;
  p.count = (int)count;
  p.columns = 0;
  p.page_size = (int)tensors[2];
  p.num_pages = (int)tensors[3];
  for (int t = 0; t < count; ++t) {
    const long long* tensor = tensors + 4 + 3 * t;
    p.tensors[t] = {reinterpret_cast<void*>(tensor[0]), p.columns, (int)tensor[2]};
    p.columns += (int)(tensor[1] * tensor[2]);
  }
  const dim3 grid(c.requests, (p.columns + kMoveThreads - 1) / kMoveThreads);
  if (grid.y > 65535) return (int)cudaErrorInvalidValue;
  switch (unit) {
    case 16: return (int)launch_pdl(move_accepted_kernel<uint4>, grid, dim3(kMoveThreads), 0, stream, p);
    case 8: return (int)launch_pdl(move_accepted_kernel<uint2>, grid, dim3(kMoveThreads), 0, stream, p);
    case 4: return (int)launch_pdl(move_accepted_kernel<uint32_t>, grid, dim3(kMoveThreads), 0, stream, p);
    case 2: return (int)launch_pdl(move_accepted_kernel<uint16_t>, grid, dim3(kMoveThreads), 0, stream, p);
    default: return (int)cudaErrorInvalidValue;
  }
}
