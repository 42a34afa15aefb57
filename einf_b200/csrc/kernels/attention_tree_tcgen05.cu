// Attention of drafted trees over the paged cache on the fifth-generation tensor cores, for bfloat16 heads of 64 and 128
// and pages of 8 to 128 tokens.  What is computed and how a launch is cut into shares: attention_tree.cuh.
//
// A unit is up to two tiles of 128 rows (nodes x the query heads that share a key/value head) over the keys of
// one request, 128 at a time.  The CTA has two slots, each a tile of rows with its own issuing warp, tensor memory and
// two softmax warpgroups, one for either half of a tile's keys.  The slots take turns: while one's threads are at their
// exponentials the other's products have the tensor core.  A unit of two tiles gives each slot one of them, and every
// tile of keys in shared memory serves both; a unit of one tile gives both slots the same rows and every second tile of keys, and
// they are put together at the end.  (Scores half a tile at a time, the other half's in the making meanwhile, were no faster:
// 247 us against 221 below; twice the instructions for the scores, which the issuing warps were slower to come by than the
// tensor core to carry out.)
//
// What bounds it: with many rows a slot's way from one score product to the next, 3,900 cycles for 256 rows x 128 keys x 128 of a head,
// of which the slots' products take 2,050 of the tensor core and their exponentials 2,050 of their unit: the two hardly overlap.  With
// few rows the launch's start (2.5 us until the lengths are known, 3 until the first scores are) and the second launch.  Measured in
// captured graphs with 28 query and 4 key/value heads of 128: 32 requests of up to 8,192 keys and 64 nodes 220 to 230 us, which is
// 0.6 PFLOP/s of the products that count (265 to 271 after seconds without a pause, at the power limit and 1.42 GHz); one of 32,768
// keys and 32 nodes 35.6 us, 1.9 TB/s; 8 of 4,096 and 64 52 us, 29 with a window of 1,024 and 180 with a cap.  With 12 and 2 heads, 8
// requests of up to 4,096 keys and 16 nodes: 17.4 us.  With 14 and 2 of 64, one of 1,024 keys and 8 nodes: 10.9 us.
//
//   warps 0, 1    K and V producers: TMA-load the pages that the block table names into rings of tiles
//   warps 2, 3    issue a slot's products: S = Q K^T into tensor memory, then O += P V with P from there, half by half
//   warps 4-19    softmax: thread r of a warpgroup has row r of the slot's tile and 64 of a tile's 128 keys
//
// The two warpgroups of a slot agree on nothing while they run: a row's reference is the maximum of its first tile,
// and stays.  What that leaves to be done comes out at the end of a piece: a row with a sum of
// weights above 2^40 (scores far above the reference; an overflow is such a sum too), or one that saw keys and has less
// than 2^-40, sends the piece through again, once for the rows' maxima and once against those.  So sums hold values of up to 2^86
// times their weights, and down to 2^-86 nothing of them is lost.
//
// Tiles with keys that some row does not see (the drafted ones, a window) run with masks of 64 bits a thread.  There a
// value that is not finite must not meet a weight of zero, so the V producer looks over such a tile and clears the
// elements it finds; if any of them is a key's, the rows that see it add them at the end of the piece, out of the cache.
#include "attention_tree.cuh"
#include "mma_sync.cuh"
#include "tcgen05.cuh"

namespace einf {

constexpr int kTile = 128;                     // rows of a slot, keys of a tile
constexpr int kSlice = kTile * 128;            // a [128 rows x 64] bfloat16 slice: 16 KB
constexpr int kTreeThreads = 640;
constexpr float kSumLimit = 1099511627776.f;   // 2^40
constexpr float kLowest = -3.40282347e38f;
constexpr int kHalf = kTile / 2;               // keys of a softmax thread
constexpr int kTmemColumns = 512;              // S: 2 x 128 columns, O: 2 x D

template <int D>
struct Layout {
  static constexpr int kBlocks = D / 64;                       // 64-wide slices of the head
  static constexpr int kTileBytes = kBlocks * kSlice;
  // even: where the slots take every second tile, a stage is always the same slot's, which has seen each of its phases
  static constexpr int kKStages = D == 64 ? 6 : 2;
  static constexpr int kVStages = D == 64 ? 4 : 2;
  static_assert(kKStages % 2 == 0 && kVStages % 2 == 0, "stages of one slot");
  static constexpr int kQ = 0;                                 // a tile of rows per slot
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kKStages * kTileBytes;
  static constexpr int kBars = kV + kVStages * kTileBytes;
  static constexpr int kNumBars = 10 + 3 * kKStages + 4 * kVStages;
  static constexpr int kFlags = kBars + 8 * kNumBars + 8;      // to be done again (four, in turn), values that are not finite (four)
  static constexpr int kXchg = kFlags + 32;                    // a float for every thread of the softmax warps
  // what the CTAs of a cluster exchange, in the place of the Q, K and V tiles: the sums of 256 rows (padded so that neither
  // threads with a row each nor warps with a row each meet a bank twice), then reference and sum of every row
  static constexpr int kPitch = D + 4;
  static constexpr int kSums = kQ;
  static constexpr int kSumsMl = kSums + 256 * kPitch * 4;
  static_assert(kSumsMl + 256 * 8 <= kBars, "the exchange needs the tiles");
  static constexpr int kBytes = kXchg + 4 * 128 * 4;
  static_assert(kBytes <= 227 * 1024, "shared memory of the tree attention kernel exceeds an SM");
  static_assert(2 * kBytes > 228 * 1024, "two CTAs on an SM would wait for each other's tensor memory");
  static_assert(kXchg % 8 == 0 && kFlags % 4 == 0, "alignment");
};

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// True in one lane of the warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(elected));
  return elected != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float4 ld_peer4(uint32_t local, uint32_t rank) {
  uint32_t peer;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(local), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_peer2(uint32_t local, uint32_t rank) {
  uint32_t peer;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(local), "r"(rank));
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer) : "memory");
  return v;
}
__device__ __forceinline__ void both_slots_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }
// A slot's warpgroup passes the turn on to the other slot's of the same keys, which takes it.
__device__ __forceinline__ void pass_turn(int id) { asm volatile("barrier.cta.arrive %0, 256;" ::"r"(10 + id) : "memory"); }
__device__ __forceinline__ void take_turn(int id) { asm volatile("barrier.cta.sync %0, 256;" ::"r"(10 + id) : "memory"); }
// The two warps of a slot with the same rows meet.
__device__ __forceinline__ void pair_sync(int pair) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(2 + pair) : "memory"); }

// 16 scores of a row to 2^(scale s - m): packed, and added to `sum`.  Packed they are bfloat16, up to 2^-8 off each, as the second
// product's operands have one type and the values are bfloat16; the sum takes them as they are, in 32 bits.  (Taken from the
// exponentials' unit, 16 a cycle, three of eight by a polynomial of the fourth degree made tree-sized launches 4 per cent slower: while
// a slot's threads are at this the other slot's products run, and it is the way from scores to weights, not the unit, that a tile waits for.)
__device__ __forceinline__ void exps(const float* v, uint32_t* packed, float2 scale2, float2 shift2, float2* sum) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 x = __ffma2_rn(make_float2(v[2 * i], v[2 * i + 1]), scale2, shift2);
    const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
    *sum = __fadd2_rn(*sum, e);
    packed[i] = pack_pair(e.x, e.y);
  }
}
// tmem_ld_wait32 of tcgen05.cuh for 16 columns.
__device__ __forceinline__ void tmem_ld_wait16(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                 "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// A cluster shares the key tiles of its piece out among its CTAs.
__device__ __forceinline__ void share_out(TreeWalk* w, int rank, int cluster) {
  const int each = divide(w->tile_end - w->tile_begin + cluster - 1, cluster);
  w->tile_begin = min(w->tile_end, w->tile_begin + rank * each);
  w->tile_end = min(w->tile_end, w->tile_begin + each);
}

// The shares of a unit's rows that the CTAs of a cluster left in their shared memory, put together: rank takes a run of rows.
template <int D>
__device__ __forceinline__ void merge_cluster(const TreeParams& p, const TreeWalk& w, const TreeUnit& u, uint32_t base, int rank) {
  using L = Layout<D>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = u.nodes * u.heads;
  const int each = divide(rows + p.cluster - 1, p.cluster), first = rank * each, last = min(rows, first + each);
#pragma unroll 1
  for (int row = first + warp; row < last; row += kTreeThreads / 32) {
    const float2 ml = lane < p.cluster ? ld_peer2(base + L::kSumsMl + row * 8, lane) : make_float2(-INFINITY, 0.f);
    const float m = warp_max(ml.x);
    const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - m);
    const float l = warp_sum(ml.y == 0.f ? 0.f : m == -INFINITY ? ml.y : ml.y * f);
    const uint32_t at = base + L::kSums + (row * L::kPitch + (4 * lane) % D) * 4;      // (D = 64: the upper lanes repeat the lower)
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < p.cluster; ++c) {
      const float fc = __shfl_sync(0xffffffffu, f, c);
      const float4 o = ld_peer4(at, c);
      if (fc == 0.f) continue;
      sum.x += o.x * fc;
      sum.y += o.y * fc;
      sum.z += o.z * fc;
      sum.w += o.w * fc;
    }
    if (4 * lane < D) {
      const float inv = tree_inverse(m, l);
      const int node = divide(row, u.heads);
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) +
          ((size_t)(w.t.first + u.first_node + node) * p.heads + u.first_head + row - node * u.heads) * D + 4 * lane;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_pair(sum.x * inv, sum.y * inv), pack_pair(sum.z * inv, sum.w * inv));
    }
    __syncwarp();
  }
}

// A softmax thread's row.
struct Row {
  bool live;
  int token, position, lowest;
  float m, l;               // the reference and the sum of weights
};

// What a slot has of a unit.
struct Slot {
  int first_node, rows, first_tile, step, tiles;   // tiles of the piece: first_tile, first_tile + step, ...
  bool pair;                                       // the unit has two tiles of rows, one a slot
};
__device__ __forceinline__ Slot slot_of(const TreeWalk& w, const TreeUnit& u, int g) {
  Slot s;
  const int most = divide(kTile, u.heads);
  s.pair = u.nodes > most;
  const int half = (u.nodes + 1) >> 1;
  s.first_node = s.pair && g ? half : 0;
  s.rows = (s.pair ? (g ? u.nodes - half : half) : u.nodes) * u.heads;
  s.step = s.pair ? 1 : 2;
  s.first_tile = w.tile_begin + (s.pair ? 0 : g);
  s.tiles = max(0, (w.tile_end - s.first_tile + s.step - 1) >> (s.pair ? 0 : 1));
  return s;
}

template <int D>
__global__ void __launch_bounds__(kTreeThreads, 1)
tree_attention_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap run_k,
                              const __grid_constant__ CUtensorMap run_v, const __grid_constant__ TreeParams p) {
  using L = Layout<D>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t base = saddr(smem_raw);
  if (base & 1023u) {      // the tiles need whole swizzle groups; the declaration asks for them
    if (threadIdx.x == 0) atomicOr(p.status, kStatusWaitExpired);
    return;
  }
  const uint32_t bars = base + L::kBars;
  auto q_full = [&](int g) { return bars + 8u * g; };
  auto s_full = [&](int g) { return bars + 8u * (2 + g); };
  auto p_full = [&](int g, int h) { return bars + 8u * (4 + 2 * g + h); };
  auto o_done = [&](int g) { return bars + 8u * (8 + g); };
  auto k_full = [&](int s) { return bars + 8u * (10 + s); };
  auto k_empty = [&](int g, int s) { return bars + 8u * (10 + (1 + g) * L::kKStages + s); };
  auto v_full = [&](int s) { return bars + 8u * (10 + 3 * L::kKStages + s); };
  auto v_checked = [&](int s) { return bars + 8u * (10 + 3 * L::kKStages + L::kVStages + s); };
  auto v_empty = [&](int g, int s) { return bars + 8u * (10 + 3 * L::kKStages + (2 + g) * L::kVStages + s); };
  const uint32_t tmem_holder = bars + 8 * L::kNumBars;
  volatile int* flags = reinterpret_cast<volatile int*>(smem_raw + L::kFlags);      // [4] to be done again, [4] values that are not finite
  float* xchg = reinterpret_cast<float*>(smem_raw + L::kXchg);              // [slot][half of the keys][row]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int g = 0; g < 2; ++g) {
      bar_init(q_full(g), 1);
      bar_init(s_full(g), 1);
      bar_init(p_full(g, 0), 128);
      bar_init(p_full(g, 1), 128);
      bar_init(o_done(g), 1);
      for (int s = 0; s < L::kKStages; ++s) bar_init(k_empty(g, s), 1);
      for (int s = 0; s < L::kVStages; ++s) bar_init(v_empty(g, s), 1);
    }
    for (int i = 0; i < 8; ++i) flags[i] = 0;
    for (int s = 0; s < L::kKStages; ++s) bar_init(k_full(s), 1);
    for (int s = 0; s < L::kVStages; ++s) {
      bar_init(v_full(s), 1);
      bar_init(v_checked(s), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_holder), "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(smem_raw + L::kBars + 8 * L::kNumBars);
  // the scores of half a tile of keys and, in the first 32 of their 64 columns, the probabilities
  auto tmem_s = [&](int g, int h) { return tmem_base + 128u * g + 64u * h; };
  auto tmem_o = [&](int g) { return tmem_base + 256u + (uint32_t)D * g; };
  pdl_launch_dependents();   // after the tensor-memory allocation, see common.cuh
  pdl_wait();

  const int cluster = p.cluster, worker = divide(blockIdx.x, cluster), rank = blockIdx.x - worker * cluster;
  TreeWalk w;
  bool any = tree_first(p, worker, &w);
  if (threadIdx.x == 0 && rank == 0) tree_note(p, worker, w, any);
  if (any && cluster > 1) share_out(&w, rank, cluster);
  // How a piece is gone through: as it comes, then, if that did not serve, for its rows' maxima and against them.
  enum { kAsItComes = 0, kForMaxima = 1, kAgainstMaxima = 2 };
  int way = kAsItComes, turn = 0, pieces = 0;
  // Every warp ends a passage through a piece here, when its products are complete, and learns whether it is the last.  (A flag is
  // cleared three turns after it was last looked at.)
  auto last_passage = [&]() {
    if (threadIdx.x == 0) {
      flags[(turn + 1) & 3] = 0;
      flags[4 + ((pieces + 1) & 3)] = 0;
    }
    __syncwarp();
    __syncthreads();
    const bool again = way == kForMaxima || (way == kAsItComes && flags[turn & 3] != 0);
    ++turn;
    way = again ? way + 1 : kAsItComes;
    return !again;
  };
  // And a piece here.  The CTAs of a cluster put their shares of it together: once they have all left them in shared
  // memory, and before any of them takes that for the next piece (or leaves).
  auto next_piece = [&]() {
    if (cluster > 1) {
      __syncwarp();
      cluster_barrier();
      merge_cluster<D>(p, w, tree_unit(p, w.t, w.unit), base, rank);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // TMA and the tensor core have the place next
      __syncwarp();
      cluster_barrier();
    }
    any = tree_next(p, worker, &w);
    if (any && cluster > 1) share_out(&w, rank, cluster);
    ++pieces;
  };

  if (warp < 2) {
    // ---- producers: warp 0 the K tiles, warp 1 the V tiles; lane j fetches page j of a tile ----
    const int stages = warp ? L::kVStages : L::kKStages;
    const CUtensorMap* map = warp ? &map_v : &map_k;
    const CUtensorMap* run_map = warp ? &run_v : &run_k;
    auto full_bar = [&](int s) { return warp ? v_full(s) : k_full(s); };
    auto empty_bar = [&](int g, int s) { return warp ? v_empty(g, s) : k_empty(g, s); };
    const int page_shift = __ffs(p.page_size) - 1, pages_per_tile = kTile >> page_shift;
    const uint32_t page_bytes = (uint32_t)p.page_size * 128u;
    // per stage and slot: whether the slot has a tile there to give back, and the parity it will give it back with
    uint32_t held[2] = {0u, 0u}, parity[2] = {0u, 0u};
    bool ok = true, bad = false;
    int stage = 0, round = 0;
    for (; any; next_piece()) {
      const TreeUnit u = tree_unit(p, w.t, w.unit);
      const bool pair = slot_of(w, u, 0).pair;
      const int* table = p.block_table + (size_t)w.request * p.table_width;
      const int keys_end = w.t.cached + w.t.nodes;
      auto pages_of = [&](int i) {
        return (min(kTile, keys_end - w.t.begin - i * kTile) + p.page_size - 1) >> page_shift;
      };
      auto read_page = [&](int i) {
        if (i >= w.tile_end || lane >= pages_of(i)) return 0;
        return table[((w.t.begin + i * kTile) >> page_shift) + lane];
      };
      do {
        // read two tiles ahead of their use
        int page = read_page(w.tile_begin), page_next = read_page(w.tile_begin + 1);
        for (int i = w.tile_begin; i < w.tile_end && ok; ++i) {
          const int page_after = read_page(i + 2);
          const int pages = pages_of(i);
          if (page < 0 || page >= p.num_pages) {
            bad = true;
            page = 0;   // keep the byte count right; the status word fails the step
          }
          const int page0 = __shfl_sync(0xffffffffu, page, 0);
          // pages that follow one another in the pool come as one box
          const bool run = pages_per_tile > 1 && pages == pages_per_tile && page0 + pages <= p.num_pages &&
                           __all_sync(0xffffffffu, lane >= pages || page == page0 + lane);
          const uint32_t bit = 1u << stage;
#pragma unroll
          for (int g = 0; g < 2; ++g)
            if (held[g] & bit) {
              ok = __all_sync(0xffffffffu, bar_wait(empty_bar(g, stage), (parity[g] >> stage) & 1u, p.status)) && ok;
              parity[g] ^= bit;
              held[g] &= ~bit;
            }
          if (!ok) break;
          if (pair) {
            held[0] |= bit;
            held[1] |= bit;
          } else {
            held[(i - w.tile_begin) & 1] |= bit;
          }
          const uint32_t full = full_bar(stage);
          if (lane == 0) bar_expect_tx(full, (uint32_t)pages * page_bytes * L::kBlocks);
          __syncwarp();
          const uint32_t offset = (warp ? L::kV : L::kK) + stage * L::kTileBytes;
          if (run) {
            if (lane < L::kBlocks) tma_4d(base + offset + lane * kSlice, run_map, lane * 64, 0, u.kv_head, page0, full);
          } else if (lane < pages) {
            const int row = (page * p.kv_heads + u.kv_head) * p.page_size;
#pragma unroll
            for (int db = 0; db < L::kBlocks; ++db)
              tma_2d(base + offset + db * kSlice + lane * page_bytes, map, db * 64, row, full);
          }
          if (warp) {
            if (p.window > 0 || w.t.begin + (i + 1) * kTile > w.t.cached) {
              // some row may not see some key of the tile: what is not finite is cleared
              ok = __all_sync(0xffffffffu, bar_wait(full, round & 1, p.status));
#pragma unroll 1
              for (int r0 = 0; r0 < kTile; r0 += 32) {
                const int r = r0 + lane;
                unsigned char* row = smem_raw + offset + (r >> 3) * 1024 + (r & 7) * 128;
                uint32_t found = 0u;
#pragma unroll
                for (int db = 0; db < L::kBlocks; ++db)
#pragma unroll
                  for (int c = 0; c < 8; ++c) {
                    const uint4 v = *reinterpret_cast<const uint4*>(row + db * kSlice + ((c ^ (r & 7)) << 4));
                    found |= not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w);
                  }
                if (found)
                  for (int c = 0; c < 32 * L::kBlocks; ++c) {
                    uint32_t* pair = reinterpret_cast<uint32_t*>(row + (c >> 5) * kSlice + ((c & 31) << 2));
                    *pair &= ~((not_finite(*pair) >> 15) * 0xffffu);
                  }
                if (found && w.t.begin + i * kTile + r < keys_end) flags[4 + (pieces & 3)] = 1;
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            __syncwarp();
            if (lane == 0) bar_arrive(v_checked(stage));
          }
          page = page_next;
          page_next = page_after;
          if (++stage == stages) {
            stage = 0;
            ++round;
          }
        }
      } while (!last_passage());
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(p.status, kStatusBadPage);
    // no copy is under way when the CTA leaves: lane j waits for the last one into stage j
    if (!ok && lane < stages && (lane < stage || round > 0)) bar_poll(full_bar(lane), (lane < stage ? round : round - 1) & 1);
  } else if (warp < 4) {
    // ---- a slot's products: the whole warp goes the way of the lane that issues, so that addresses stay in uniform registers ----
    const int g = warp - 2;
    // S: M = 128 rows, N = 128 keys, both K-major.  O: M = 128, N = D, P from tensor memory, V MN-major.
    constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kTile >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
    const uint64_t desc_q = desc_k_major(base + L::kQ + g * L::kTileBytes);
    auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, bar_wait_likely_done(bar, parity, p.status)) != 0; };
    bool ok = true;
    int queries = 0;               // loads of Q so far
    int done = 0;                  // this slot's tiles so far
    int before = 0;                // the CTA's tiles before this passage
    for (; any; next_piece()) {
      const TreeUnit u = tree_unit(p, w.t, w.unit);
      const Slot s = slot_of(w, u, g);
      if (s.tiles > 0 && ok) {
        if (elect_one()) {
          bar_expect_tx(q_full(g), (uint32_t)(p.unit_nodes / 2 * u.heads) * 128u * L::kBlocks);
          for (int db = 0; db < L::kBlocks; ++db)
            tma_3d(base + L::kQ + g * L::kTileBytes + db * kSlice, &map_q, db * 64, u.first_head, w.t.first + u.first_node + s.first_node,
                   q_full(g));
        }
        __syncwarp();
        ok = wait(q_full(g), queries & 1);
        ++queries;
      }
      do {
        const int first = before + s.first_tile - w.tile_begin;
        before += w.tile_end - w.tile_begin;
#pragma unroll 1
        for (int j = 0; j < s.tiles && ok; ++j, ++done) {
          const int c = first + j * s.step, k_stage = c % L::kKStages, v_stage = c % L::kVStages;
          ok = wait(k_full(k_stage), (c / L::kKStages) & 1);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (elect_one()) {
            const uint64_t desc_k = desc_k_major(base + L::kK + k_stage * L::kTileBytes);
#pragma unroll
            for (int db = 0; db < L::kBlocks; ++db)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_ss(tmem_s(g, 0), desc_advance(desc_q, db * kSlice + kk * 32), desc_advance(desc_k, db * kSlice + kk * 32), idesc_s,
                       (db > 0 || kk > 0) ? 1u : 0u);
            mma_commit(s_full(g));
            mma_commit(k_empty(g, k_stage));
          }
          __syncwarp();
          const uint32_t parity = (c / L::kVStages) & 1;
          ok = wait(v_full(v_stage), parity) && wait(v_checked(v_stage), parity);
          const uint64_t desc_v = desc_mn_major(base + L::kV + v_stage * L::kTileBytes, kSlice);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && wait(p_full(g, h), done & 1);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < kHalf / 16; ++ks)      // onto the zeros or sums that are there
                mma_ts(tmem_o(g), tmem_s(g, h) + ks * 8, desc_advance(desc_v, (h * kHalf + ks * 16) * 128), idesc_o, 1u);
              if (h) {
                mma_commit(o_done(g));
                mma_commit(v_empty(g, v_stage));
              }
            }
            __syncwarp();
          }
          // The scores' place holds the probabilities until the product has them; after the last, Q's place and the sums are
          // free too.
          ok = ok && wait(o_done(g), done & 1);
        }
      } while (!last_passage());
    }
  } else {
    // ---- softmax: thread r has row r of its slot, and the first or the second 64 of a tile's 128 keys ----
    const int g = (warp - 4) >> 3, part = (warp - 4) >> 2 & 1, r = (warp & 3) * 32 + lane, pair = g * 4 + (warp & 3);
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_row = tmem_s(g, part) + lane_addr, o_row = tmem_o(g) + lane_addr;
    float* my_xchg = xchg + (g * 2 + part) * 128 + r;
    const float* pair_xchg = xchg + (g * 2 + (part ^ 1)) * 128 + r;
    const ScoreScale sc = make_score_scale(p.scale, p.softcap);
    bool ok = true;
    int done = 0;                      // this slot's tiles so far
    for (; any; next_piece()) {
      const TreeUnit u = tree_unit(p, w.t, w.unit);
      const Slot s = slot_of(w, u, g);
      const int other_tiles = slot_of(w, u, g ^ 1).tiles;
      const bool turns = s.tiles > 1 || other_tiles > 1;
      const bool warp_live = (warp & 3) * 32 < s.rows;
      const int unit_row = s.first_node * u.heads + r;
      Row row;
      row.live = r < s.rows;
      const int node = divide(r, u.heads);
      row.token = w.t.first + u.first_node + (row.live ? s.first_node + node : 0);
      row.position = row.live ? tree_position(p, w.t, row.token) : 0;
      row.lowest = row.live ? tree_lowest(p, row.position) : 0;
      row.m = -INFINITY;
      // keys that every row of the warp sees, but for those from the drafted ones on
      const int all_from = p.window > 0 ? __reduce_max_sync(0xffffffffu, row.lowest) : 0;
      do {
        float best = -INFINITY;
        bool some = false;      // the row has seen a key
        row.l = 0.f;
        if (s.tiles > 0 && warp_live) {
          uint32_t zero[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) zero[c] = 0u;
#pragma unroll 1
          for (int c0 = part * (D / 2); c0 < (part + 1) * (D / 2); c0 += 16) tmem_st16(o_row + c0, zero);
          tmem_st_wait();
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          pair_sync(pair);      // the first product of either half finds all of the row's zeros
        }
#pragma unroll 1
        for (int j = 0; j < s.tiles; ++j, ++done) {      // `done` counts this slot's tiles
          // The turns: slot 1's exponentials wait for slot 0's of its tile, slot 0's for slot 1's of the one before.  Every turn
          // passed on is taken, whatever else went wrong, and none is passed on before the one it answers was taken.  Left to
          // themselves the slots fall into step and have their exponentials at the same time, 286 us against 221 for 32
          // requests of 8,192 keys and 64 nodes; turns from score product to score product, by the issuing warps, took 244; by
          // the barrier of the probabilities 224 (300 cycles until it is seen); passed on before they are all there 244 to
          // 306.  Where neither slot has a second tile there is nothing to gain: 11.0 us without, 12.2 with turns for one
          // request of 1,024 keys.
          if (turns && (g || (j > 0 && j <= other_tiles))) take_turn(2 * (g ^ 1) + part);
          if (ok) ok = __all_sync(0xffffffffu, bar_wait_likely_done(s_full(g), done & 1, p.status));
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (warp_live) {
            const int key0 = w.t.begin + (s.first_tile + j * s.step) * kTile + part * kHalf;
            const bool all_visible = key0 >= all_from && key0 + kHalf <= w.t.cached;
            uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
            if (!all_visible) {
#pragma unroll 1
              for (int c = 0; c < 2; ++c) {
                const uint32_t bits = row.live ? tree_visible(p, w.t, row.token, row.lowest, row.position, key0 + 32 * c) : 0u;
                if (c) seen[1] = bits;
                else seen[0] = bits;
              }
              __syncwarp();
            }
            some = some || (seen[0] | seen[1]) != 0u;
            // sixteen scores from column c0 on, -inf where the key is not seen
            auto scores = [&](int c0, float* v, bool masked) {
              tmem_ld16(s_row + c0, v);
              tmem_ld_wait16(v);
              if (masked) {
                const uint32_t bits = (c0 < 32 ? seen[0] : seen[1]) >> (c0 & 31);
#pragma unroll
                for (int c = 0; c < 16; ++c) v[c] = bits >> c & 1u ? v[c] : -INFINITY;
              }
            };
            if (way == kForMaxima || (way == kAsItComes && j == 0)) {
              float top = -INFINITY;
#pragma unroll 1
              for (int c0 = 0; c0 < kHalf; c0 += 16) {
                float v[16];
                scores(c0, v, !all_visible);
#pragma unroll
                for (int c = 0; c < 16; c += 4) top = max3(top, max3(v[c], v[c + 1], v[c + 2]), v[c + 3]);
              }
              // under a cap a score of -inf is one as any other, the lowest: no row that sees one is without a reference
              if (sc.tanh_in != 0.f && (seen[0] | seen[1])) top = fmaxf(top, kLowest);
              best = fmaxf(best, top);
              if (way == kAsItComes) {
                // The row's reference: the maximum of the tile (the scale is positive and the cap grows with the score: the
                // maximum and either commute); nothing where the row sees none of it.
                *my_xchg = best;
                pair_sync(pair);
                best = fmaxf(best, *pair_xchg);
                row.m = best == -INFINITY ? 0.f : score_log2(best, sc);
              }
            }
            const float2 scale2 = make_float2(sc.scale_log2, sc.scale_log2), shift2 = make_float2(-row.m, -row.m);
            float2 sum2 = make_float2(0.f, 0.f);
            if (all_visible && sc.tanh_in == 0.f && way != kForMaxima) {
#pragma unroll 1
              for (int c0 = 0; c0 < kHalf; c0 += 16) {
                float v[16];
                uint32_t packed[8];
                tmem_ld16(s_row + c0, v);
                tmem_ld_wait16(v);
                exps(v, packed, scale2, shift2, &sum2);
                tmem_st8(s_row + (c0 >> 1), packed);      // two keys to a column, over scores that were read
              }
            } else {
              if (way == kForMaxima) seen[0] = seen[1] = 0u;
#pragma unroll 1
              for (int c0 = 0; c0 < kHalf; c0 += 16) {
                float v[16];
                uint32_t packed[8];
                scores(c0, v, sc.tanh_in == 0.f);
                if (sc.tanh_in != 0.f) {
                  const uint32_t bits = (c0 < 32 ? seen[0] : seen[1]) >> (c0 & 31);
#pragma unroll
                  for (int c = 0; c < 16; ++c) v[c] = bits >> c & 1u ? __fdividef(capped(v[c], sc), sc.scale_log2) : -INFINITY;
                }
                exps(v, packed, scale2, shift2, &sum2);
                tmem_st8(s_row + (c0 >> 1), packed);
              }
            }
            row.l += sum2.x + sum2.y;
            tmem_st_wait();
          }
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          bar_arrive(p_full(g, part));
          if (turns && (g ? j + 1 < other_tiles : j < other_tiles)) pass_turn(2 * g + part);
        }
        if (ok && s.tiles > 0) {
          ok = __all_sync(0xffffffffu, bar_wait(o_done(g), (done - 1) & 1, p.status));
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        pair_sync(pair);      // both have read what the other left
        *my_xchg = way == kForMaxima ? best : row.l == 0.f && some ? -1.f : row.l;
        pair_sync(pair);
        if (way == kForMaxima) {
          best = fmaxf(best, *pair_xchg);
          row.m = best == -INFINITY ? 0.f : score_log2(best, sc);
        } else {
          const float a = *my_xchg, b = *pair_xchg;
          row.l = (a < 0.f ? 0.f : a) + (b < 0.f ? 0.f : b);
          if (row.l == 0.f && a + b < 0.f) row.l = -1.f;      // the row has seen keys, and scores of -inf alone
          if (way == kAsItComes && ok && row.live && !(row.l <= kSumLimit && (row.l * kSumLimit >= 1.f || !some)))
            flags[turn & 3] = 1;
        }
      } while (!last_passage());
      if (row.l <= 0.f) row.m = -INFINITY, row.l = -row.l;      // nothing to put together with others
      // The row's sums: this slot's alone, half of the head to a warp, or, where both slots had the same rows, both slots',
      // a quarter of the head to a warp.
      float m = row.m, l = row.l, mine = 1.f, other = 0.f;
      int d0 = part * (D / 2), d1 = d0 + D / 2;
      if (!s.pair) {
        *my_xchg = part ? l : m;
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        both_slots_sync();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float m_other = xchg[(g ^ 1) * 256 + r], l_other = xchg[(g ^ 1) * 256 + 128 + r];
        m = fmaxf(row.m, m_other);
        mine = row.m == -INFINITY ? 0.f : fast_exp2(row.m - m);
        other = m_other == -INFINITY ? 0.f : fast_exp2(m_other - m);
        l = tree_sums(row.m, l, mine, m_other, l_other, other);
        d0 = (g * 2 + part) * (D / 4);
        d1 = d0 + D / 4;
      }
      const bool write = row.live && ok, not_all_finite = flags[4 + (pieces & 3)] != 0;
      const float inv = tree_inverse(m, l);
      const uint32_t o_other = tmem_o(g ^ 1) + lane_addr;
      float* left = reinterpret_cast<float*>(smem_raw + L::kSums) + unit_row * L::kPitch;
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + ((size_t)row.token * p.heads + u.first_head + (row.live ? r - node * u.heads : 0)) * D;
      if (warp_live) {
#pragma unroll 1
        for (int c0 = d0; c0 < d1; c0 += 16) {
          float v[16], x[16];
          tmem_ld16(o_row + c0, v);
          if (!s.pair) {
            tmem_ld16(o_other + c0, x);
            tmem_ld_wait16(x);
          }
          tmem_ld_wait16(v);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            v[c] = mine == 0.f ? 0.f : v[c] * mine;
            if (!s.pair && other != 0.f) v[c] += x[c] * other;
          }
          if (not_all_finite && row.live) {
            // the values that were cleared, for the rows that see their keys, times a weight above zero
            const __nv_bfloat16* values = static_cast<const __nv_bfloat16*>(p.v_cache) + (size_t)u.kv_head * p.page_size * D + c0;
            const int keys_end = min(w.t.cached + w.t.nodes, w.t.begin + w.tile_end * kTile);
#pragma unroll 1
            for (int key0 = w.t.begin + w.tile_begin * kTile; key0 < keys_end; key0 += 32) {
              if (p.window == 0 && key0 + kTile <= w.t.cached) continue;      // its tile was not looked over
#pragma unroll 1
              for (uint32_t rest = tree_visible(p, w.t, row.token, row.lowest, row.position, key0); rest; rest &= rest - 1) {
                const int key = key0 + __ffs(rest) - 1, page = p.block_table[(size_t)w.request * p.table_width + key / p.page_size];
                if (page < 0 || page >= p.num_pages) continue;
                const __nv_bfloat16* value = values + ((size_t)page * p.kv_heads * p.page_size + key % p.page_size) * D;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const float x = __bfloat162float(value[e]);
                  if (!isfinite(x)) v[e] += x;
                }
              }
            }
          }
          __syncwarp();
          if (write && cluster == 1 && w.whole) {
#pragma unroll
            for (int d = 0; d < 16; d += 8)
              *reinterpret_cast<uint4*>(dst + c0 + d) =
                  make_uint4(pack_pair(v[d] * inv, v[d + 1] * inv), pack_pair(v[d + 2] * inv, v[d + 3] * inv),
                             pack_pair(v[d + 4] * inv, v[d + 5] * inv), pack_pair(v[d + 6] * inv, v[d + 7] * inv));
          } else if (write) {
            // a share: a cluster's, in shared memory, or a worker's
            float* to = cluster > 1 ? left + c0 : tree_share(p, w.share, unit_row, c0);
            const int step4 = cluster > 1 ? 4 : 128;
#pragma unroll
            for (int d = 0; d < 4; ++d)
              *reinterpret_cast<float4*>(to + d * step4) = make_float4(v[4 * d], v[4 * d + 1], v[4 * d + 2], v[4 * d + 3]);
          }
          __syncwarp();
        }
      }
      if (write && part == 0 && (s.pair || g == 0)) {
        if (cluster > 1) reinterpret_cast<float2*>(smem_raw + L::kSumsMl)[unit_row] = make_float2(m, l);
        else if (!w.whole) p.part_ml[(size_t)w.share * p.unit_rows + unit_row] = make_float2(m, l);
      }
      if (!s.pair) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        both_slots_sync();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemColumns) : "memory");
  }
}

// Queries [tokens, heads, D] as a three-dimensional map whose box is a slot's rows: `nodes` nodes of `group` heads, one 64-wide slice.
static int make_query_map(CUtensorMap* map, const void* base, int tokens, int heads, int size, int group, int nodes) {
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return (int)cudaErrorNotSupported;
  cuuint64_t dims[3] = {(cuuint64_t)size, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)size * 2, (cuuint64_t)heads * size * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)nodes};
  cuuint32_t element_strides[3] = {1, 1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, element_strides,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <int D>
int launch_tree(const TreeParams& p, cudaStream_t stream) {
  CUtensorMap map_q, map_k, map_v, run_k, run_v;
  const long long cache_rows = (long long)p.num_pages * p.kv_heads * p.page_size;
  int rc = make_query_map(&map_q, p.q, p.tokens, p.heads, D, p.unit_heads, kTile / p.unit_heads);
  if (!rc) rc = make_map(&map_k, p.k_cache, cache_rows, D, p.page_size);
  if (!rc) rc = make_map(&map_v, p.v_cache, cache_rows, D, p.page_size);
  if (!rc) rc = make_run_map(&run_k, p.k_cache, p.num_pages, p.kv_heads, p.page_size, D, kTile / p.page_size);
  if (!rc) rc = make_run_map(&run_v, p.v_cache, p.num_pages, p.kv_heads, p.page_size, D, kTile / p.page_size);
  if (rc) return rc;
  const auto kernel = tree_attention_tcgen05_kernel<D>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kBytes);
  if (e != cudaSuccess) return (int)e;
  e = launch_pdl_cluster(kernel, dim3(p.workers * p.cluster), dim3(kTreeThreads), Layout<D>::kBytes, p.cluster, stream, map_q, map_k, map_v, run_k, run_v, p);
  if (e != cudaSuccess) return (int)e;
  return tree_merge<__nv_bfloat16>(p, stream);
}

}  // namespace einf

using namespace einf;

// How many clusters of `cluster` CTAs the device holds at once; 0 on error.
extern "C" int einf_tree_attention_tcgen05_max_clusters(int cluster) {
  if (cluster < 1 || cluster > 8) return 0;
  const auto kernel = tree_attention_tcgen05_kernel<128>;      // the other takes as much of an SM: one CTA
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(cluster);
  config.blockDim = dim3(kTreeThreads);
  config.dynamicSmemBytes = Layout<128>::kBytes;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = cluster;
  attribute.val.clusterDim.y = 1;
  attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  int clusters = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<128>::kBytes) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return clusters;
}

// call: a TreeCall, on the host; a worker is a CTA or, where every unit has a worker, a cluster of up to 8.  part_o: [2 * workers][256][size] floats, part_ml:
// [2 * workers][256][2], notes: [workers][8]; none of them where every unit has one worker (whole).
extern "C" int einf_tree_attention_tcgen05(const char* call, cudaStream_t stream) {
  const TreeCall& c = *reinterpret_cast<const TreeCall*>(call);
  if (c.requests == 0 || c.tokens == 0) return 0;
  if (!tree_call_fits(c) || c.cluster > 8 || (c.cluster > 1 && !c.whole) || c.dtype != kBFloat16 || (c.size != 64 && c.size != 128) || c.heads / c.kv_heads > kTile ||
      c.page_size < 8 || c.page_size > 128 || (c.page_size & (c.page_size - 1)) ||
      ((uintptr_t)c.q | (uintptr_t)c.k_cache | (uintptr_t)c.v_cache | (uintptr_t)c.out) % 16)
    return (int)cudaErrorInvalidValue;
  TreeParams p = tree_params(c);
  p.unit_heads = c.heads / c.kv_heads;
  p.unit_nodes = 2 * (kTile / p.unit_heads);
  p.group = p.unit_heads;
  p.head_blocks = 1;
  p.unit_rows = 2 * kTile;
  p.padded = c.size;
  p.tile_shift = 7;
  static_assert(kTile == 128, "a tile of keys");
  return c.size == 64 ? launch_tree<64>(p, stream) : launch_tree<128>(p, stream);
}
