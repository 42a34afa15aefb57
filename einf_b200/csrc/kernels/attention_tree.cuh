// What the attention kernels over drafted trees share: how a launch's work is cut, which keys a node sees, how
// the shares of a row that several CTAs worked on are put together.
//
// A request brings n nodes (packed rows q_start[r] .. of the queries) behind `cached` tokens.  The keys of its nodes lie in
// its pages at places cached .. cached + n - 1.  Node i sees every cached key (with a window of W: those less
// than W positions before its own) and node k where bit k of its mask is set (and the same window).
//
// The rows of a unit are those of some nodes x the query heads that share one key/value head, so that a tile of keys is
// read once for all of them; with trees of 8 to 64 nodes that is what makes the work more than a read of the cache.  A
// launch's work is the list of all (unit, key tile) pairs in the order of requests, and CTA b takes an equal piece of that
// list: one long context spreads over the whole device, a batch of unequal ones leaves no CTA behind, and at
// most the first and the last unit of a piece are shared with other CTAs.  Those go to scratch memory
// as (sums, reference, sum of weights), and a second launch puts them together in the order of the keys.
#pragma once

#include "common.cuh"

namespace einf {

struct TreeParams {
  const void* q;             // [tokens, heads, D]
  const void* k_cache;       // [pages, kv_heads, page_size, D]
  const void* v_cache;
  const int* block_table;    // [requests, table_width]
  const int* q_start;        // [requests + 1]
  const int* cached_lens;    // [requests]
  const uint32_t* mask;      // [tokens, 2 * words]: bit k of a row's words is node k of its request
  const int* positions;      // [tokens], read with a window alone
  void* out;                 // [tokens, heads, D]
  float* part_o;             // [2 * ctas][rows of a unit][padded D]
  float2* part_ml;           // [2 * ctas][rows of a unit]: reference (exponent of 2) and sum
  int4* notes;               // [ctas], see tree_note
  int* status;
  int requests, tokens, heads, kv_heads, size, page_size, num_pages, table_width, words, window;
  float scale, softcap;
  int unit_heads;            // query heads of a unit: all of a key/value head, or a block of them
  int unit_nodes;            // at most that many nodes
  int unit_rows;             // rows of a share in scratch memory
  int padded;                // elements of a share's row
  int tile_keys, min_chunk, ctas;
};

inline TreeParams tree_params(const void* q, const void* k_cache, const void* v_cache, const int* block_table, const int* q_start,
                              const int* cached_lens, const void* mask, const int* positions, void* out, float* part_o,
                              float* part_ml, int* notes, int requests, int tokens, int heads, int kv_heads, int size, int page_size,
                              int num_pages, int table_width, int words, int window, float scale, float softcap, int ctas,
                              int min_chunk, int* status) {
  TreeParams p = {};
  p.q = q;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.block_table = block_table;
  p.q_start = q_start;
  p.cached_lens = cached_lens;
  p.mask = static_cast<const uint32_t*>(mask);
  p.positions = positions;
  p.out = out;
  p.part_o = part_o;
  p.part_ml = reinterpret_cast<float2*>(part_ml);
  p.notes = reinterpret_cast<int4*>(notes);
  p.status = status;
  p.requests = requests;
  p.tokens = tokens;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.size = size;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.table_width = table_width;
  p.words = words;
  p.window = window;
  p.scale = scale;
  p.softcap = softcap;
  p.ctas = ctas;
  p.min_chunk = min_chunk;
  return p;
}

// One request's figures, out of step inputs that are held to what memory there is.
struct TreeRequest {
  int first, nodes, cached, begin, units, tiles, node_blocks;
};

__device__ __forceinline__ TreeRequest tree_request(const TreeParams& p, int r) {
  TreeRequest t;
  t.first = max(0, min(p.q_start[r], p.tokens));
  t.nodes = max(0, min(p.q_start[r + 1], p.tokens) - t.first);
  const long long room = (long long)p.table_width * p.page_size - t.nodes;
  t.cached = p.cached_lens[r];
  if (t.nodes > 0 && (t.cached < 0 || t.cached > room)) {     // places that the block table does not have
    atomicOr(p.status, kStatusBadPage);
    t.cached = (int)max(0ll, min((long long)t.cached, room));
    if (room < 0) t.nodes = 0;
  }
  // no node stands before its request's cached tokens, so none sees a key before this one
  t.begin = p.window > 0 ? max(0, t.cached - p.window + 1) / p.page_size * p.page_size : 0;
  t.node_blocks = (t.nodes + p.unit_nodes - 1) / p.unit_nodes;
  const int group = p.heads / p.kv_heads;
  t.units = t.node_blocks * p.kv_heads * ((group + p.unit_heads - 1) / p.unit_heads);
  t.tiles = (t.cached + t.nodes - t.begin + p.tile_keys - 1) / p.tile_keys;
  return t;
}

// A unit's rows: row i is node first_node + i / heads, head first_head + i % heads.
struct TreeUnit {
  int kv_head, first_head, heads, first_node, nodes;
};

__device__ __forceinline__ TreeUnit tree_unit(const TreeParams& p, const TreeRequest& t, int unit) {
  TreeUnit u;
  const int group = p.heads / p.kv_heads;
  const int head_blocks = (group + p.unit_heads - 1) / p.unit_heads;
  const int pair = unit / t.node_blocks, block = unit - pair * t.node_blocks;
  u.kv_head = pair / head_blocks;
  const int head_block = pair - u.kv_head * head_blocks;
  u.first_head = u.kv_head * group + head_block * p.unit_heads;
  u.heads = min(p.unit_heads, group - head_block * p.unit_heads);
  const int each = (t.nodes + t.node_blocks - 1) / t.node_blocks;     // blocks of one size
  u.first_node = min(t.nodes, block * each);
  u.nodes = min(each, t.nodes - u.first_node);
  return u;
}

// Every warp works out the cut by itself: all (unit, tile) pairs of the launch, and a CTA's share of them.
__device__ __forceinline__ long long tree_pairs(const TreeParams& p) {
  long long sum = 0;
  for (int r0 = 0; r0 < p.requests; r0 += 32) {
    const int r = r0 + (threadIdx.x & 31);
    long long mine = 0;
    if (r < p.requests) {
      const TreeRequest t = tree_request(p, r);
      mine = (long long)t.units * t.tiles;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    sum += mine;
  }
  return sum;
}

// The pieces of a CTA's share, one unit after the other.
struct TreeWalk {
  int request, unit;         // where the walk stands
  int tile_begin, tile_end;  // tiles of that unit that are this CTA's
  bool whole;                // no other CTA has tiles of this unit
  int share;                 // where its results go otherwise
  TreeRequest t;
  long long left;            // pairs of the share that come after this piece
  int pieces, chunk;
};

__device__ __forceinline__ void tree_piece(const TreeParams& p, TreeWalk* w, int tile_begin, long long available) {
  w->tile_begin = tile_begin;
  w->tile_end = (int)min((long long)w->t.tiles, tile_begin + available);
  w->left = available - (w->tile_end - tile_begin);
  w->whole = tile_begin == 0 && w->tile_end == w->t.tiles;
  w->share = 2 * blockIdx.x + (w->pieces > 0 ? 1 : 0);
  ++w->pieces;
}
// False where the CTA has nothing to do.
__device__ __forceinline__ bool tree_first(const TreeParams& p, TreeWalk* w) {
  const long long pairs = tree_pairs(p);
  const long long chunk = max((long long)p.min_chunk, (pairs + p.ctas - 1) / p.ctas);
  const long long begin = chunk * blockIdx.x;
  if (begin >= pairs) return false;
  const int lane = threadIdx.x & 31;
  long long before = 0;
  w->pieces = 0;
  w->chunk = (int)chunk;
  for (int r0 = 0; r0 < p.requests; r0 += 32) {
    const int r = r0 + lane;
    long long mine = 0;
    if (r < p.requests) {
      const TreeRequest t = tree_request(p, r);
      mine = (long long)t.units * t.tiles;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t after = __ballot_sync(0xffffffffu, before + upto > begin);
    if (after) {
      const int at = __ffs(after) - 1;
      const long long start = before + __shfl_sync(0xffffffffu, upto - mine, at);
      w->request = r0 + at;
      w->t = tree_request(p, w->request);
      w->unit = (int)((begin - start) / w->t.tiles);
      tree_piece(p, w, (int)((begin - start) - (long long)w->unit * w->t.tiles), min(chunk, pairs - begin));
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}
__device__ __forceinline__ bool tree_next(const TreeParams& p, TreeWalk* w) {
  if (w->left <= 0) return false;
  if (++w->unit >= w->t.units) {
    w->unit = 0;
    do {
      if (++w->request >= p.requests) return false;
      w->t = tree_request(p, w->request);
    } while (w->t.units == 0);
  }
  tree_piece(p, w, 0, w->left);
  return true;
}

// 32 bits of a node's mask from bit `from` on (which may lie before the first), none beyond `nodes`.
__device__ __forceinline__ uint32_t tree_mask_bits(const TreeParams& p, int token, int from, int nodes) {
  const uint32_t* row = p.mask + (size_t)token * 2 * p.words;
  const int limit = min(nodes, 64 * p.words);
  if (from >= limit || from <= -32) return 0u;
  const int word = from >> 5, shift = from & 31;
  const uint32_t low = word >= 0 ? row[word] : 0u;
  const uint32_t high = shift && word + 1 < 2 * p.words ? row[word + 1] : 0u;
  uint32_t bits = __funnelshift_r(low, high, shift);
  if (limit - from < 32) bits &= (1u << (limit - from)) - 1u;
  return bits;
}
// Which of the 32 keys from place `key` on the node sees that stands at `token` (its window ends at `lowest`).
__device__ __forceinline__ uint32_t tree_visible(const TreeParams& p, const TreeRequest& t, int token, int lowest, int position,
                                                 int key) {
  uint32_t seen = 0u;
  const int hi = t.cached - key;                      // cached keys are bits below this
  if (hi > 0) {
    seen = hi >= 32 ? 0xffffffffu : (1u << hi) - 1u;
    const int lo = lowest - key;
    if (lo >= 32) seen = 0u;
    else if (lo > 0) seen &= ~((1u << lo) - 1u);
  }
  if (hi < 32) {
    uint32_t bits = tree_mask_bits(p, token, -hi, t.nodes);
    if (p.window > 0)
      for (uint32_t rest = bits; rest; rest &= rest - 1) {
        const int bit = __ffs(rest) - 1;
        if ((long long)position - max(p.positions[t.first + bit - hi], t.cached) >= p.window) bits &= ~(1u << bit);
      }
    seen |= bits;
  }
  return seen;
}
__device__ __forceinline__ int tree_position(const TreeParams& p, const TreeRequest& t, int token) {
  return p.window > 0 ? max(p.positions[token], t.cached) : 0;
}
__device__ __forceinline__ int tree_lowest(const TreeParams& p, int position) {
  return p.window > 0 ? max(0, position - p.window + 1) : 0;
}

constexpr int kTreeMergeWarps = 8;
constexpr int kTreeMergeBlocks = 16;       // CTAs that take one unit's rows in turn

// What the second launch has to know of a CTA's share: the unit of its first piece, where that piece begins, the length of
// a share.  (x = -1: nothing to put together here.)
__device__ __forceinline__ void tree_note(const TreeParams& p, const TreeWalk& w, bool any) {
  if (threadIdx.x == 0)
    p.notes[blockIdx.x] = any && w.tile_begin > 0 ? make_int4(w.request, w.unit, w.tile_begin, w.chunk) : make_int4(-1, 0, 0, 0);
}

// Rows whose keys several CTAs had: o = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c over the shares in the order of
// their keys.  The CTAs (blockIdx.x) stand for the places where a share ends and the next begins; the first of
// those inside a unit puts that unit together.  A warp per row.
template <typename T>
__global__ void __launch_bounds__(32 * kTreeMergeWarps) tree_merge_kernel(TreeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int4 note = p.notes[blockIdx.x + 1];
  const int chunk = note.w;
  if (note.x < 0 || note.z > chunk) return;              // no unit is cut here, or it was cut before
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const TreeRequest t = tree_request(p, note.x);
  const TreeUnit u = tree_unit(p, t, note.y);
  const int first = blockIdx.x, last = first + (t.tiles - note.z + chunk - 1) / chunk;
  const int second = note.z < chunk ? 1 : 0;             // the unit was not the first piece of its first CTA
  for (int row = blockIdx.y * kTreeMergeWarps + warp; row < u.nodes * u.heads; row += gridDim.y * kTreeMergeWarps) {
    auto share = [&](int c) { return (size_t)(2 * c + (c == first ? second : 0)) * p.unit_rows + row; };
    float m = -INFINITY, l = 0.f;
    for (int c0 = first; c0 <= last; c0 += 32) {
      const float2 ml = c0 + lane <= last ? __ldcg(p.part_ml + share(c0 + lane)) : make_float2(-INFINITY, 0.f);
      const float top = fmaxf(m, warp_max(ml.x));
      // a sum that is not a number stays one, whatever the reference beside it
      const float here = ml.y == 0.f ? 0.f : ml.y * (ml.x == -INFINITY ? 0.f : exp2f(ml.x - top));
      l = (l == 0.f ? 0.f : l * (m == -INFINITY ? 0.f : exp2f(m - top))) + warp_sum(here);
      m = top;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t at = ((size_t)(t.first + u.first_node + row / u.heads) * p.heads + u.first_head + row % u.heads) * p.size;
    T* out = static_cast<T*>(p.out) + at;
    for (int d0 = 0; d0 < p.size; d0 += 128) {
      const int d = d0 + 4 * lane;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (d < p.padded)
#pragma unroll 4
        for (int c = first; c <= last; ++c) {
          const float mc = __ldcg(&p.part_ml[share(c)].x);
          if (mc == -INFINITY) continue;
          const float f = exp2f(mc - m);
          const float4 o = __ldcg(reinterpret_cast<const float4*>(p.part_o + share(c) * p.padded + d));
          sum.x += o.x * f;
          sum.y += o.y * f;
          sum.z += o.z * f;
          sum.w += o.w * f;
        }
      const float v[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < p.size) out[d + e] = from_float<T>(v[e]);
    }
  }
}

template <typename T>
inline int tree_merge(const TreeParams& p, cudaStream_t stream) {
  if (p.ctas < 2) return 0;
  return (int)launch_pdl(tree_merge_kernel<T>, dim3((unsigned)p.ctas - 1, kTreeMergeBlocks), dim3(32 * kTreeMergeWarps), 0, stream, p);
}

}  // namespace einf
