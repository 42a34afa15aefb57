// What the attention kernels over drafted trees share: how a launch's work is cut, which keys a node sees, how
// the shares of a row that several CTAs worked on are put together.
//
// A request brings n nodes (packed rows q_start[r] .. of the queries) behind `cached` tokens.  The keys of its nodes lie in
// its pages at places cached .. cached + n - 1.  Node i sees every cached key (with a window of W: those less
// than W positions before its own) and node k where bit k of its mask is set (and the same window).
//
// The rows of a unit are those of some nodes x the query heads that share one key/value head, so that a tile of keys is
// read once for all of them; with trees of 8 to 64 nodes that is what makes the work more than a read of the cache.  A
// worker is a CTA or, where every unit has a worker, a thread-block cluster.  A launch's work is cut over its workers in one of three ways:
//   whole    a unit to a worker (a cluster shares its key tiles out among its CTAs), nothing is put together afterwards
//   aligned  no more units than workers: a unit is cut into pieces of `chunk` key tiles, a piece to a worker
//   list     more units than workers: worker w takes an equal piece of the list of all (unit, key tile) pairs, in the order
//            of requests, so that a batch of unequal contexts leaves no worker behind; at most the first and the last
//            unit of a piece are shared with other workers
// The first is the caller's choice, who says how many workers there are; between the others the kernel chooses, who
// knows the lengths.  Shares of a unit go to scratch memory as (sums, reference, sum of weights), and a second
// launch puts them together in the order of the keys.
#pragma once

#include "tcgen05.cuh"

namespace einf {

// What the second launch has to know where a worker's first piece goes on with a unit that began with another worker.
struct __align__(16) TreeNote {
  int places;                // workers less one that have the unit; 0: nothing to put together here
  int place;                 // which of them this one is, from 0
  int second;                // the unit was not the first piece of its first worker
  int token;                 // the unit's first token, its nodes, heads and first head
  int nodes, heads, first_head, more;
};

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
  float* part_o;             // [2 * workers][rows of a unit / 32][padded D / 4][32][4]
  float2* part_ml;           // [2 * workers][rows of a unit]: reference (exponent of 2) and sum
  TreeNote* notes;           // [workers]
  int* status;
  int requests, tokens, heads, kv_heads, size, page_size, num_pages, table_width, words, window;
  float scale, softcap;
  int unit_heads;            // query heads of a unit: all of a key/value head, or a block of them
  int unit_nodes;            // at most that many nodes
  int unit_rows;             // rows of a share in scratch memory, a multiple of 32
  int padded;                // elements of a share's row
  int tile_shift;            // a tile is 1 << tile_shift keys
  int group, head_blocks;    // query heads of a key/value head, and blocks of them
  int min_chunk, workers, cluster, whole;
};

// The arguments of a launcher, as the caller packs them.
struct TreeCall {
  const void *q, *k_cache, *v_cache;
  const int *block_table, *q_start, *cached_lens;
  const uint32_t* mask;
  const int* positions;
  void* out;
  int* status;
  float* part_o;
  float2* part_ml;
  TreeNote* notes;
  int requests, tokens, heads, kv_heads, size, page_size, num_pages, table_width, words, window, dtype, workers, cluster, whole, min_chunk;
  float scale, softcap;
};
static_assert(sizeof(TreeCall) == 13 * 8 + 17 * 4 + 4, "as packed");

inline bool tree_call_fits(const TreeCall& c) {
  return c.workers >= 1 && c.cluster >= 1 && c.min_chunk >= 1 && c.kv_heads >= 1 && c.heads % c.kv_heads == 0 && c.size >= 1 && c.page_size >= 1 && c.words >= 1 &&
         (c.window <= 0 || c.positions);
}
inline TreeParams tree_params(const TreeCall& c) {
  TreeParams p = {};
  p.q = c.q;
  p.k_cache = c.k_cache;
  p.v_cache = c.v_cache;
  p.block_table = c.block_table;
  p.q_start = c.q_start;
  p.cached_lens = c.cached_lens;
  p.mask = c.mask;
  p.positions = c.positions;
  p.out = c.out;
  p.part_o = c.part_o;
  p.part_ml = c.part_ml;
  p.notes = c.notes;
  p.status = c.status;
  p.requests = c.requests;
  p.tokens = c.tokens;
  p.heads = c.heads;
  p.kv_heads = c.kv_heads;
  p.size = c.size;
  p.page_size = c.page_size;
  p.num_pages = c.num_pages;
  p.table_width = c.table_width;
  p.words = c.words;
  p.window = c.window;
  p.scale = c.scale;
  p.softcap = c.softcap;
  p.workers = c.workers;
  p.cluster = c.cluster;
  p.whole = c.whole;
  p.min_chunk = c.min_chunk;
  return p;
}

// a / b for a >= 0, b > 0 and a quotient below 2^20.  (The compiler's own takes three times the instructions, and in kernels of a few
// microseconds an instruction that a launch comes to for the first time costs more to fetch than to run.)
__device__ __forceinline__ int divide(int a, int b) {
  int q = (int)__fdividef((float)a, (float)b);
  const int rest = a - q * b;
  q += rest >= b ? 1 : 0;
  return q - (rest < 0 ? 1 : 0);
}

// One request's figures, out of step inputs that are held to what memory there is.
struct TreeRequest {
  int first, nodes, cached, begin, units, tiles, node_blocks;
};

__device__ __forceinline__ TreeRequest tree_request(const TreeParams& p, int r) {
  TreeRequest t;
  t.first = max(0, min(p.q_start[r], p.tokens));
  t.nodes = max(0, min(p.q_start[r + 1], p.tokens) - t.first);
  const long long room = min((long long)p.table_width * p.page_size, 1ll << 27) - t.nodes;      // (2^27: see divide)
  t.cached = p.cached_lens[r];
  if (t.nodes > 0 && (t.cached < 0 || t.cached > room)) {     // places that the block table does not have
    atomicOr(p.status, kStatusBadPage);
    t.cached = (int)max(0ll, min((long long)t.cached, room));
    if (room < 0) t.nodes = 0;
  }
  // no node stands before its request's cached tokens, so none sees a key before this one
  t.begin = p.window > 0 ? max(0, t.cached - p.window + 1) / p.page_size * p.page_size : 0;
  t.node_blocks = divide(t.nodes + p.unit_nodes - 1, p.unit_nodes);
  t.units = t.node_blocks * p.kv_heads * p.head_blocks;
  t.tiles = (t.cached + t.nodes - t.begin + (1 << p.tile_shift) - 1) >> p.tile_shift;
  return t;
}

// A unit's rows: row i is node first_node + i / heads, head first_head + i % heads.
struct TreeUnit {
  int kv_head, first_head, heads, first_node, nodes;
};

__device__ __forceinline__ TreeUnit tree_unit(const TreeParams& p, const TreeRequest& t, int unit) {
  TreeUnit u;
  const int pair = divide(unit, t.node_blocks), block = unit - pair * t.node_blocks;
  u.kv_head = p.head_blocks == 1 ? pair : divide(pair, p.head_blocks);
  const int head_block = pair - u.kv_head * p.head_blocks;
  u.first_head = u.kv_head * p.group + head_block * p.unit_heads;
  u.heads = min(p.unit_heads, p.group - head_block * p.unit_heads);
  const int each = divide(t.nodes + t.node_blocks - 1, t.node_blocks);     // blocks of one size
  u.first_node = min(t.nodes, block * each);
  u.nodes = min(each, t.nodes - u.first_node);
  return u;
}

// The pieces of a worker, one unit after the other.
struct TreeWalk {
  int request, unit;         // where the walk stands
  int tile_begin, tile_end;  // key tiles of that unit that are this worker's
  bool whole;                // no other worker has tiles of this unit
  int share;                 // where its results go otherwise
  TreeRequest t;
  int left;                  // what comes after this piece: pairs of the list, or units
  int pieces, chunk;
  bool list;
};

// A launch's units (nodes and heads that the caller holds to this many, unless trees overlap) and its pairs of a unit and a key
// tile, so that places in the list are 32-bit.  (Pairs are not bounded by memory: all units of a key/value head read the same
// keys, and requests may share pages.)
constexpr int kTreeMostUnits = 1 << 20, kTreeMostPairs = 1 << 30;

__device__ __forceinline__ int warp_add(int v) { return __reduce_add_sync(0xffffffffu, v); }
// Of 64-bit numbers below 2^52, in two sums that 32 bits hold.
__device__ __forceinline__ long long warp_add(long long v) {
  const unsigned low = __reduce_add_sync(0xffffffffu, (unsigned)v & 0x3ffffffu);
  return ((long long)__reduce_add_sync(0xffffffffu, (unsigned)(v >> 26)) << 26) + low;
}
__device__ __forceinline__ void tree_piece(const TreeParams& p, int worker, TreeWalk* w, int tile_begin, int available) {
  w->tile_begin = tile_begin;
  w->tile_end = min(w->t.tiles, tile_begin + available);
  w->left = available - (w->tile_end - tile_begin);
  w->whole = tile_begin == 0 && w->tile_end == w->t.tiles;
  w->share = 2 * worker + (w->pieces > 0 ? 1 : 0);
  ++w->pieces;
}
// The first piece of a worker; every warp works it out by itself.  False where there is nothing to do, or more than a launch
// takes: then the status word is set, and no worker has a piece.
__device__ __forceinline__ bool tree_first(const TreeParams& p, int worker, TreeWalk* w) {
  const int lane = threadIdx.x & 31;
  TreeRequest mine = {};
  if (lane < p.requests) mine = tree_request(p, lane);
  const bool few = p.requests <= 32;
  auto request = [&](int r) {                    // lane's request of the 32 from r - lane on
    if (few) return mine;
    TreeRequest none = {};
    return r < p.requests ? tree_request(p, r) : none;
  };
  auto total = [&](auto weight) {
    if (few) return warp_add(weight(mine));
    auto sum = weight(TreeRequest{});
    for (int r0 = 0; r0 < p.requests; r0 += 32) sum += warp_add(weight(request(r0 + lane)));
    return sum;
  };
  auto too_many = [&] {
    if (lane == 0) atomicOr(p.status, kStatusBadIndex);
    return false;
  };
  const long long all_units = total([](const TreeRequest& t) { return (long long)t.units; });
  if (all_units > kTreeMostUnits) return too_many();
  const int units = (int)all_units;
  int chunk = 1, begin, end;
  w->list = false;
  if (p.whole) {
    chunk = 0x7fffffff;
    const int each = divide(units + p.workers - 1, p.workers);
    begin = worker * each;
    end = min(units, begin + each);
  } else {
    const long long all_pairs = total([](const TreeRequest& t) { return (long long)t.units * t.tiles; });
    if (all_pairs > kTreeMostPairs) return too_many();
    const int pairs = (int)all_pairs;
    chunk = max(p.min_chunk, (pairs + p.workers - 1) / p.workers);
    if (units > p.workers) {
      w->list = true;
      begin = worker * chunk;
      end = min(pairs, begin + chunk);
    } else {
      int pieces;
#pragma unroll 1
      while ((pieces = total([&](const TreeRequest& t) { return t.units * divide(t.tiles + chunk - 1, chunk); })) > p.workers)
        chunk = max(chunk + 1, (int)__fdividef((float)chunk * pieces, (float)p.workers));
      begin = worker;
      end = min(pieces, begin + 1);
    }
  }
  w->pieces = 0;
  w->chunk = chunk;
  if (begin >= end) return false;
  int before = 0;
  for (int r0 = 0; r0 < p.requests; r0 += 32) {
    const TreeRequest t = request(r0 + lane);
    const int each = w->list ? t.tiles : p.whole ? 1 : divide(t.tiles + chunk - 1, chunk);      // of a unit
    const int here = t.units * each;
    int upto = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t after = __ballot_sync(0xffffffffu, before + upto > begin);
    if (after) {
      const int at = __ffs(after) - 1;
      const int skip = begin - before - __shfl_sync(0xffffffffu, upto - here, at), unit_each = __shfl_sync(0xffffffffu, each, at);
      w->request = r0 + at;
      w->t.first = __shfl_sync(0xffffffffu, t.first, at);
      w->t.nodes = __shfl_sync(0xffffffffu, t.nodes, at);
      w->t.cached = __shfl_sync(0xffffffffu, t.cached, at);
      w->t.begin = __shfl_sync(0xffffffffu, t.begin, at);
      w->t.units = __shfl_sync(0xffffffffu, t.units, at);
      w->t.tiles = __shfl_sync(0xffffffffu, t.tiles, at);
      w->t.node_blocks = __shfl_sync(0xffffffffu, t.node_blocks, at);
      w->unit = divide(skip, unit_each);
      const int part = skip - w->unit * unit_each;
      if (w->list) {
        tree_piece(p, worker, w, part, end - begin);
      } else if (p.whole) {
        tree_piece(p, worker, w, 0, w->t.tiles);
        w->left = end - begin - 1;
      } else {
        tree_piece(p, worker, w, part * chunk, min(chunk, w->t.tiles - part * chunk));
      }
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}
__device__ __forceinline__ bool tree_next(const TreeParams& p, int worker, TreeWalk* w) {
  if (w->left <= 0) return false;
  if (++w->unit >= w->t.units) {
    w->unit = 0;
    do {
      if (++w->request >= p.requests) return false;
      w->t = tree_request(p, w->request);
    } while (w->t.units == 0);
  }
  if (w->list) {
    tree_piece(p, worker, w, 0, w->left);
  } else {
    const int left = w->left;
    tree_piece(p, worker, w, 0, w->t.tiles);
    w->left = left - 1;
  }
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

// Where four elements of a row of a share lie.
__device__ __forceinline__ float* tree_share(const TreeParams& p, int share, int row, int d) {
  return p.part_o + ((((size_t)share * (p.unit_rows >> 5) + (row >> 5)) * (p.padded >> 2) + (d >> 2)) * 32 + (row & 31)) * 4;
}

__device__ __forceinline__ void tree_note(const TreeParams& p, int worker, const TreeWalk& w, bool any) {
  if (!p.notes) return;
  TreeNote n = {};
  if (any && w.tile_begin > 0) {
    const TreeUnit u = tree_unit(p, w.t, w.unit);
    n.place = divide(w.tile_begin - 1, w.chunk);
    n.places = n.place + divide(w.t.tiles - w.tile_begin + w.chunk - 1, w.chunk);
    n.second = w.tile_begin - n.place * w.chunk < w.chunk ? 1 : 0;
    n.token = w.t.first + u.first_node;
    n.nodes = u.nodes;
    n.heads = u.heads;
    n.first_head = u.first_head;
  }
  p.notes[worker] = n;
}

// A row's reference m and sum of weights l: where m is -inf, l is 0 for a row that saw no key, 1 for one whose scores were all -inf (its
// softmax is no number), and no number for one that saw a score that is none.  What two shares of a row's keys come to:
__device__ __forceinline__ float tree_sums(float m_a, float l_a, float factor_a, float m_b, float l_b, float factor_b) {
  if (m_a == -INFINITY && m_b == -INFINITY) return l_a + l_b;
  return (l_a == 0.f ? 0.f : l_a * factor_a) + (l_b == 0.f ? 0.f : l_b * factor_b);
}
// What a row's sums are multiplied by in the end.
__device__ __forceinline__ float tree_inverse(float m, float l) {
  return l == 0.f ? 0.f : m == -INFINITY ? NAN : 1.f / l;
}

constexpr int kTreeMergeWarps = 4;
constexpr int kTreeMergeShares = 4;        // shares that a warp has in flight

// Rows whose keys several workers had: o = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c over the shares in the order of
// their keys.  blockIdx.x stands for the place where a worker's list ends and the next one's begins; the places inside one
// unit share its work out: an item is 32 rows, one a lane, and eight elements of each, which lie as 2 x 512 bytes in a
// share.  Loops stay rolled: the kernel runs for a few microseconds, and its instructions come at the pace of their first fetch.
// What bounds it is the latency of loads that follow one another: with the shares of an item split among a CTA's four
// warps where there are CTAs for that, 38 shares of 256 rows x 128 (17 MB, out of the L2) took 5.5 us instead of 9.5, 9 of 96
// x 128 3.8 instead of 4.3.  (Eight warps, or eight shares of a warp in flight, were no faster where it matters: 37.2 us for 38.0
// of the former's two launches, 18.7 for 17.1 of the latter's.)
template <typename T>
__global__ void __launch_bounds__(32 * kTreeMergeWarps) tree_merge_kernel(TreeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const TreeNote n = p.notes[blockIdx.x + 1];
  if (n.places == 0) return;                             // no unit is cut here
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = blockIdx.x - n.place, rows = n.nodes * n.heads, groups = p.padded >> 2;
  // With a CTA for every item (a unit in many pieces) an item's shares are split among the CTA's warps, else a warp has an item.
  const int pairs = (groups + 1) >> 1, items = ((rows + 31) >> 5) * pairs;
  const bool together = n.places * (int)gridDim.y >= items;
  const int item0 = together ? blockIdx.y * n.places + n.place : (blockIdx.y * kTreeMergeWarps + warp) * n.places + n.place;
  __shared__ float left[kTreeMergeWarps - 1][10][32];      // what a warp has of the item: reference, sum, eight sums of values
  for (int item = item0; item < items; item += n.places * gridDim.y * kTreeMergeWarps) {
    const int row_block = divide(item, pairs), row = row_block * 32 + lane, group = 2 * (item - row_block * pairs);
    const float2* ml = p.part_ml + min(row, rows - 1);
    const float4* sums = reinterpret_cast<const float4*>(p.part_o) + ((size_t)row_block * groups + group) * 32 + lane;
    const size_t share_rows = (size_t)p.unit_rows, share_sums = (size_t)(p.unit_rows >> 5) * groups * 32;
    const bool two = group + 1 < groups;
    float m = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 1
    for (int c0 = together ? warp * kTreeMergeShares : 0; c0 <= n.places; c0 += together ? kTreeMergeWarps * kTreeMergeShares : kTreeMergeShares) {
      float2 v[kTreeMergeShares];
      float4 x[kTreeMergeShares], y[kTreeMergeShares];
      // all of these in flight at once; what lies beyond the last share is the last one again
#pragma unroll
      for (int i = 0; i < kTreeMergeShares; ++i) {
        const int c = min(c0 + i, n.places);
        const size_t share = 2 * (first + c) + (c == 0 ? n.second : 0);
        v[i] = __ldcg(ml + share * share_rows);
        x[i] = __ldcg(sums + share * share_sums);
        y[i] = __ldcg(sums + share * share_sums + (two ? 32 : 0));
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < kTreeMergeShares; ++i) top = fmaxf(top, v[i].x);
      const float keep = m == -INFINITY ? 0.f : fast_exp2(m - top);
      m = top;
      // a sum of weights that is not a number stays one, whatever the reference beside it
      l = l == 0.f ? 0.f : top == -INFINITY ? l : l * keep;
      a.x *= keep, a.y *= keep, a.z *= keep, a.w *= keep;
      b.x *= keep, b.y *= keep, b.z *= keep, b.w *= keep;
#pragma unroll
      for (int i = 0; i < kTreeMergeShares; ++i) {
        const float f = v[i].x == -INFINITY || c0 + i > n.places ? 0.f : fast_exp2(v[i].x - top);
        l += v[i].y == 0.f || c0 + i > n.places ? 0.f : top == -INFINITY ? v[i].y : v[i].y * f;
        if (f == 0.f) continue;                          // a share without a reference has nothing in its sums
        a.x = fmaf(x[i].x, f, a.x), a.y = fmaf(x[i].y, f, a.y), a.z = fmaf(x[i].z, f, a.z), a.w = fmaf(x[i].w, f, a.w);
        b.x = fmaf(y[i].x, f, b.x), b.y = fmaf(y[i].y, f, b.y), b.z = fmaf(y[i].z, f, b.z), b.w = fmaf(y[i].w, f, b.w);
      }
    }
    if (together) {
      if (warp) {
        float(*mine)[32] = left[warp - 1];
        mine[0][lane] = m, mine[1][lane] = l;
        mine[2][lane] = a.x, mine[3][lane] = a.y, mine[4][lane] = a.z, mine[5][lane] = a.w;
        mine[6][lane] = b.x, mine[7][lane] = b.y, mine[8][lane] = b.z, mine[9][lane] = b.w;
      }
      __syncthreads();      // once at most in a CTA: it has one item then
      if (warp) return;
#pragma unroll 1
      for (int o = 0; o < kTreeMergeWarps - 1; ++o) {
        const float(*x)[32] = left[o];
        const float top = fmaxf(m, x[0][lane]), keep = m == -INFINITY ? 0.f : fast_exp2(m - top);
        const float f = x[0][lane] == -INFINITY ? 0.f : fast_exp2(x[0][lane] - top);
        l = tree_sums(m, l, keep, x[0][lane], x[1][lane], f);
        m = top;
        // a share without a reference has nothing in its sums
        a.x = fmaf(x[2][lane], f, a.x * keep), a.y = fmaf(x[3][lane], f, a.y * keep);
        a.z = fmaf(x[4][lane], f, a.z * keep), a.w = fmaf(x[5][lane], f, a.w * keep);
        b.x = fmaf(x[6][lane], f, b.x * keep), b.y = fmaf(x[7][lane], f, b.y * keep);
        b.z = fmaf(x[8][lane], f, b.z * keep), b.w = fmaf(x[9][lane], f, b.w * keep);
      }
    }
    if (row >= rows) continue;
    const float inv = tree_inverse(m, l);
    const int node = divide(row, n.heads), d = 4 * group;
    T* out = static_cast<T*>(p.out) + ((size_t)(n.token + node) * p.heads + n.first_head + row - node * n.heads) * p.size + d;
    const float v[8] = {a.x * inv, a.y * inv, a.z * inv, a.w * inv, b.x * inv, b.y * inv, b.z * inv, b.w * inv};
    if (p.size % 8 == 0 && ((uintptr_t)out & 15) == 0) {
      // sixteen bytes at a time (element by element, rows apart, these stores took most of the kernel's time)
      __align__(16) T narrow[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) narrow[e] = from_float<T>(v[e]);
#pragma unroll
      for (int e = 0; e < (int)(8 * sizeof(T) / 16); ++e) reinterpret_cast<uint4*>(out)[e] = reinterpret_cast<const uint4*>(narrow)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d + e < p.size) out[e] = from_float<T>(v[e]);
    }
  }
}

template <typename T>
inline int tree_merge(const TreeParams& p, cudaStream_t stream) {
  if (p.workers < 2 || p.whole) return 0;
  // two items a warp where a unit is cut once
  const int items = p.unit_rows / 32 * ((p.padded + 7) / 8);
  return (int)launch_pdl(tree_merge_kernel<T>, dim3((unsigned)p.workers - 1, (unsigned)(items + 2 * kTreeMergeWarps - 1) / (2 * kTreeMergeWarps)),
                         dim3(32 * kTreeMergeWarps), 0, stream, p);
}

}  // namespace einf
