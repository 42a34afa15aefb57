// Attention of drafted trees over the paged cache on the fifth-generation tensor cores, for bfloat16 heads of 64 and 128
// and pages of 8 to 128 tokens.  What is computed and how a launch is cut into shares: attention_tree.cuh.
//
// A unit is up to two tiles of 128 rows (nodes x the query heads that share a key/value head) over the keys of
// one request, 128 at a time.  The CTA has two slots, each a tile of rows with its own issuing thread, tensor memory and
// softmax warpgroup; while one slot's scores are on their way through the exponentials' unit, the other's products
// have the tensor core.  A unit of two tiles gives each slot one of them, and every tile of keys in shared memory serves
// both; a unit of one tile gives both slots the same rows and every second tile of keys, and they are put
// together at the end.
//
//   warps 0, 1    K and V producers: TMA-load the pages that the block table names into rings of tiles
//   warps 2, 3    one lane each issues a slot's products: S = Q K^T into tensor memory, O += P V with P from there
//   warps 4-11    softmax, a warpgroup a slot: thread r has row r of the slot's tile
//
// Sums stay in tensor memory, scaled by a reference that is the maximum of the row's first tile and moves only when a
// later tile has a score 2^8 above it.  Thread r looks for its row's maximum first and then goes over the scores again: the
// probabilities take the place of scores that were read (head size 128, where tensor memory has no other) or a
// place of their own (64, where the next scores need not wait for the second product).
//
// Tiles with keys that some row does not see (the drafted ones, a window) run with masks of 128 bits a row.  There a
// value that is not finite must not meet a weight of zero, so the V producer looks over such a tile, clears the
// elements it finds and names their keys; the rows that do see such a key add them to their sums themselves.
#include <type_traits>

#include "attention_tree.cuh"
#include "mma_sync.cuh"
#include "tcgen05.cuh"

namespace einf {

constexpr int kTile = 128;                     // rows of a slot, keys of a tile
constexpr int kSlice = kTile * 128;            // a [128 rows x 64] bfloat16 slice: 16 KB
constexpr int kTreeThreads = 384;
constexpr float kMove = 8.f;                   // exponents above its reference at which a row moves it
constexpr int kTmemColumns = 512;

template <int D>
struct Layout {
  static constexpr int kBlocks = D / 64;                       // 64-wide slices of the head
  static constexpr int kTileBytes = kBlocks * kSlice;
  static constexpr bool kOwnP = D == 64;                       // P has tensor memory of its own
  static constexpr int kKStages = D == 64 ? 5 : 3;
  static constexpr int kVStages = D == 64 ? 5 : 2;
  static constexpr int kQ = 0;                                 // a tile of rows per slot
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kKStages * kTileBytes;
  static constexpr int kBars = kV + kVStages * kTileBytes;
  static constexpr int kNumBars = 10 + 3 * kKStages + 4 * kVStages;
  static constexpr int kBad = kBars + 8 * kNumBars + 16;       // per V stage: 128 bits, rows of the tile that were cleared
  static constexpr int kXchg = kBad + 16 * kVStages;           // reference and sum of every row, per slot
  static constexpr int kBytes = kXchg + 2 * 128 * 8;
  static_assert(kBytes <= 227 * 1024, "shared memory of the tree attention kernel exceeds an SM");
  static_assert(2 * kBytes > 228 * 1024, "two CTAs on an SM would wait for each other's tensor memory");
  static_assert(kXchg % 8 == 0 && kBad % 4 == 0, "alignment");
};

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void both_slots_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// What a slot has of a unit.
struct Slot {
  int first_node, rows, first_tile, step, tiles;   // tiles of the piece: first_tile, first_tile + step, ...
  bool pair;                                       // the unit has two tiles of rows, one a slot
};
__device__ __forceinline__ Slot slot_of(const TreeParams& p, const TreeWalk& w, const TreeUnit& u, int g) {
  Slot s;
  const int most = kTile / u.heads;
  s.pair = u.nodes > most;
  const int half = (u.nodes + 1) >> 1;
  s.first_node = s.pair && g ? half : 0;
  s.rows = (s.pair ? (g ? u.nodes - half : half) : u.nodes) * u.heads;
  s.step = s.pair ? 1 : 2;
  s.first_tile = w.tile_begin + (s.pair ? 0 : g);
  s.tiles = max(0, (w.tile_end - s.first_tile + s.step - 1) / s.step);
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
  auto p_full = [&](int g) { return bars + 8u * (4 + g); };
  auto o_done = [&](int g) { return bars + 8u * (6 + g); };
  auto s_free = [&](int g) { return bars + 8u * (8 + g); };
  auto k_full = [&](int s) { return bars + 8u * (10 + s); };
  auto k_empty = [&](int g, int s) { return bars + 8u * (10 + (1 + g) * L::kKStages + s); };
  auto v_full = [&](int s) { return bars + 8u * (10 + 3 * L::kKStages + s); };
  auto v_checked = [&](int s) { return bars + 8u * (10 + 3 * L::kKStages + L::kVStages + s); };
  auto v_empty = [&](int g, int s) { return bars + 8u * (10 + 3 * L::kKStages + (2 + g) * L::kVStages + s); };
  const uint32_t tmem_holder = bars + 8 * L::kNumBars;
  uint32_t* cleared = reinterpret_cast<uint32_t*>(smem_raw + L::kBad);      // [V stage][4]
  float2* xchg = reinterpret_cast<float2*>(smem_raw + L::kXchg);            // [slot][row]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int g = 0; g < 2; ++g) {
      bar_init(q_full(g), 1);
      bar_init(s_full(g), 1);
      bar_init(p_full(g), 128);
      bar_init(o_done(g), 1);
      bar_init(s_free(g), 128);
      for (int s = 0; s < L::kKStages; ++s) bar_init(k_empty(g, s), 1);
      for (int s = 0; s < L::kVStages; ++s) bar_init(v_empty(g, s), 1);
    }
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
  auto tmem_s = [&](int g) { return tmem_base + 128u * g; };
  auto tmem_o = [&](int g) { return tmem_base + 256u + (uint32_t)D * g; };
  auto tmem_p = [&](int g) { return L::kOwnP ? tmem_base + 384u + 64u * g : tmem_base + 128u * g; };
  pdl_launch_dependents();   // after the tensor-memory allocation, see common.cuh
  pdl_wait();

  TreeWalk w;
  bool any = tree_first(p, &w);
  tree_note(p, w, any);

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
    for (; any; any = tree_next(p, &w)) {
      const TreeUnit u = tree_unit(p, w.t, w.unit);
      const bool pair = slot_of(p, w, u, 0).pair;
      const int* table = p.block_table + (size_t)w.request * p.table_width;
      const int keys_end = w.t.cached + w.t.nodes;
      auto pages_of = [&](int i) {
        return (min(kTile, keys_end - w.t.begin - i * kTile) + p.page_size - 1) >> page_shift;
      };
      auto read_page = [&](int i) {
        if (i >= w.tile_end || lane >= pages_of(i)) return 0;
        return table[((w.t.begin + i * kTile) >> page_shift) + lane];
      };
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
            // some row may not see some key of the tile: rows that are not finite are cleared and named
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
              const uint32_t rows = __ballot_sync(0xffffffffu, found != 0u);
              if (lane == 0) cleared[stage * 4 + (r0 >> 5)] = rows;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          } else if (lane < 4) {
            cleared[stage * 4 + lane] = 0u;
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
      if (!ok) break;
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(p.status, kStatusBadPage);
  } else if (warp < 4) {
    // ---- a slot's products ----
    const int g = warp - 2;
    if (lane == 0) {
      // S: M = 128 rows, N = 128 keys, both K-major.  O: M = 128, N = D, P from tensor memory, V MN-major.
      const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kTile >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
      const uint64_t desc_q = desc_k_major(base + L::kQ + g * L::kTileBytes);
      bool ok = true;
      int queries = 0;               // loads of Q so far
      int done = 0;                  // this slot's tiles so far
      int before = 0;                // the CTA's tiles before this piece
      for (; any && ok; any = tree_next(p, &w)) {
        const TreeUnit u = tree_unit(p, w.t, w.unit);
        const Slot s = slot_of(p, w, u, g);
        const int first = before + s.first_tile - w.tile_begin;
        before += w.tile_end - w.tile_begin;
        if (s.tiles == 0) continue;
        bar_expect_tx(q_full(g), (uint32_t)(kTile / u.heads * u.heads) * 128u * L::kBlocks);
        for (int db = 0; db < L::kBlocks; ++db)
          tma_3d(base + L::kQ + g * L::kTileBytes + db * kSlice, &map_q, db * 64, u.first_head, w.t.first + u.first_node + s.first_node,
                 q_full(g));
        ok = bar_wait(q_full(g), queries & 1, p.status);
        ++queries;
        auto scores = [&](int j) {
          const int c = first + j * s.step, stage = c % L::kKStages;
          if (!bar_wait_likely_done(k_full(stage), (c / L::kKStages) & 1, p.status)) return false;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t desc_k = desc_k_major(base + L::kK + stage * L::kTileBytes);
#pragma unroll
          for (int db = 0; db < L::kBlocks; ++db)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(tmem_s(g), desc_advance(desc_q, db * kSlice + kk * 32), desc_advance(desc_k, db * kSlice + kk * 32), idesc_s,
                     (db > 0 || kk > 0) ? 1u : 0u);
          mma_commit(s_full(g));
          mma_commit(k_empty(g, stage));
          return true;
        };
        auto sums = [&](int j) {
          const int c = first + j * s.step, stage = c % L::kVStages;
          const uint32_t parity = (c / L::kVStages) & 1;
          if (!bar_wait_likely_done(v_full(stage), parity, p.status) || !bar_wait_likely_done(v_checked(stage), parity, p.status) ||
              !bar_wait(p_full(g), (done + j) & 1, p.status))
            return false;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t desc_v = desc_mn_major(base + L::kV + stage * L::kTileBytes, kSlice);
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)      // onto the zeros or sums that the softmax warps left
            mma_ts(tmem_o(g), tmem_p(g) + ks * 8, desc_advance(desc_v, ks * 16 * 128), idesc_o, 1u);
          mma_commit(o_done(g));
          mma_commit(v_empty(g, stage));
          return true;
        };
        if (L::kOwnP) {
          ok = ok && scores(0);
          for (int j = 0; j < s.tiles && ok; ++j) {
            if (j + 1 < s.tiles) ok = bar_wait(s_free(g), (done + j) & 1, p.status) && scores(j + 1);
            ok = ok && sums(j);
          }
          done += s.tiles;
          ok = ok && bar_wait(o_done(g), (done - 1) & 1, p.status);      // the queries' place is free again
        } else {
          for (int j = 0; j < s.tiles && ok; ++j)      // the scores' place holds the probabilities until the product has them
            ok = scores(j) && sums(j) && bar_wait(o_done(g), (done + j) & 1, p.status);
          done += s.tiles;
        }
      }
    }
  } else {
    // ---- softmax: thread r has row r of its slot ----
    const int g = warp >= 8 ? 1 : 0, r = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_row = tmem_s(g) + lane_addr, o_row = tmem_o(g) + lane_addr, p_row = tmem_p(g) + lane_addr;
    const ScoreScale sc = make_score_scale(p.scale, p.softcap);
    const bool has_cap = p.softcap > 0.f;
    bool ok = true;
    int done = 0, before = 0;
    for (; any; any = tree_next(p, &w)) {
      const TreeUnit u = tree_unit(p, w.t, w.unit);
      const Slot s = slot_of(p, w, u, g);
      const bool live = r < s.rows, warp_live = (warp & 3) * 32 < s.rows;
      const int row = s.first_node * u.heads + r;                  // of the unit
      const int token = w.t.first + u.first_node + (live ? s.first_node + r / u.heads : 0);
      const int position = live ? tree_position(p, w.t, token) : 0;
      const int lowest = live ? tree_lowest(p, position) : 0;
      const int first = before + s.first_tile - w.tile_begin;
      before += w.tile_end - w.tile_begin;
      float m_ref = -INFINITY, l_run = 0.f;
      if (s.tiles > 0 && warp_live) {
        float zero[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) zero[c] = 0.f;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) tmem_st32(o_row + c0, zero);
      }
      for (int j = 0; j < s.tiles; ++j, ++done) {
        if (ok) ok = __all_sync(0xffffffffu, bar_wait(s_full(g), done & 1, p.status));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (!warp_live || !ok) {
          if (L::kOwnP) bar_arrive(s_free(g));
          bar_arrive(p_full(g));
          continue;
        }
        const int tile = s.first_tile + j * s.step, key0 = w.t.begin + tile * kTile;
        const bool all_visible = __all_sync(0xffffffffu, !live || (key0 + kTile <= w.t.cached && key0 >= lowest));
        uint32_t seen[4];
        if (!all_visible) {
#pragma unroll
          for (int c = 0; c < 4; ++c) seen[c] = live ? tree_visible(p, w.t, token, lowest, position, key0 + 32 * c) : 0u;
          __syncwarp();
        }
        // The second product of this slot's previous tile is complete: with scores and probabilities in one place the scores
        // could not be there otherwise.
        auto wait_product = [&]() {
          if (L::kOwnP && j > 0) {
            ok = __all_sync(0xffffffffu, bar_wait_likely_done(o_done(g), (done - 1) & 1, p.status)) && ok;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
        };
        auto walk = [&](auto masked_tag) {
          constexpr bool kMasked = decltype(masked_tag)::value;
          auto mask = [&](float* v, uint32_t bits) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = bits >> c & 1u ? v[c] : -INFINITY;
          };
          float top = -INFINITY;
#pragma unroll 1
          for (int c0 = 0; c0 < kTile; c0 += 64) {
            float a[32], b[32];
            tmem_ld32(s_row + c0, a);
            tmem_ld32(s_row + c0 + 32, b);
            tmem_ld_wait();
            if (kMasked) {
              mask(a, c0 ? seen[2] : seen[0]);
              mask(b, c0 ? seen[3] : seen[1]);
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 32; ++c) m4[c & 3] = fmaxf(m4[c & 3], fmaxf(a[c], b[c]));
            top = fmaxf(top, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
          }
          top = top == -INFINITY ? -INFINITY : score_log2(top, sc);
          const bool move = live && top > (m_ref == -INFINITY ? -INFINITY : m_ref + kMove);
          wait_product();
          if (__any_sync(0xffffffffu, move)) {
            const float factor = !move ? 1.f : m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - top);
            if (j > 0) {
#pragma unroll 1
              for (int c0 = 0; c0 < D; c0 += 32) {
                float v[32];
                tmem_ld32(o_row + c0, v);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 32; ++c) v[c] *= factor;
                tmem_st32(o_row + c0, v);
              }
            }
            l_run = l_run == 0.f ? 0.f : l_run * factor;
            if (move) m_ref = top;
          }
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
          const float2 scale2 = make_float2(sc.scale_log2, sc.scale_log2), shift2 = make_float2(-m_use, -m_use);
          float2 sum2 = make_float2(0.f, 0.f);
          auto exps = [&](float* v, uint32_t bits, int c0) {
            if (kMasked) mask(v, bits);
            if (has_cap) {
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                const float x = kMasked && v[c] == -INFINITY ? -INFINITY : capped(v[c], sc) - m_use;
                v[c] = fast_exp2(x);
              }
            } else {
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                const float2 x = __ffma2_rn(make_float2(v[c], v[c + 1]), scale2, shift2);
                v[c] = fast_exp2(x.x);
                v[c + 1] = fast_exp2(x.y);
              }
            }
            uint32_t packed[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              sum2 = __fadd2_rn(sum2, make_float2(v[c], v[c + 1]));
              packed[c >> 1] = pack_pair(v[c], v[c + 1]);
            }
            tmem_st16(p_row + (c0 >> 1), packed);      // two keys to a column
          };
#pragma unroll 1
          for (int c0 = 0; c0 < kTile; c0 += 64) {
            float a[32], b[32];
            tmem_ld32(s_row + c0, a);
            tmem_ld_wait32(a);
            tmem_ld32(s_row + c0 + 32, b);
            exps(a, kMasked ? (c0 ? seen[2] : seen[0]) : 0u, c0);
            tmem_ld_wait32(b);
            if (L::kOwnP && c0 > 0) {
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
              bar_arrive(s_free(g));
            }
            exps(b, kMasked ? (c0 ? seen[3] : seen[1]) : 0u, c0 + 32);
          }
          l_run += sum2.x + sum2.y;
        };
        if (all_visible) {
          walk(std::false_type{});
        } else {
          walk(std::true_type{});
          // values that are not finite, for the rows that see their keys
          const int c = first + j * s.step, stage = c % L::kVStages;
          ok = __all_sync(0xffffffffu, bar_wait_likely_done(v_checked(stage), (c / L::kVStages) & 1, p.status)) && ok;
#pragma unroll 1
          for (int word = 0; word < 4; ++word) {
            const uint32_t mine = cleared[stage * 4 + word] & seen[word];
            for (uint32_t rest = __reduce_or_sync(0xffffffffu, mine); rest; rest &= rest - 1) {
              const int bit = __ffs(rest) - 1, key = key0 + 32 * word + bit;
              const int page = p.block_table[(size_t)w.request * p.table_width + key / p.page_size];
              const bool add = (mine >> bit & 1u) && page >= 0 && page < p.num_pages;
              const __nv_bfloat16* value = static_cast<const __nv_bfloat16*>(p.v_cache) +
                  (((size_t)(add ? page : 0) * p.kv_heads + u.kv_head) * p.page_size + key % p.page_size) * D;
#pragma unroll 1
              for (int c0 = 0; c0 < D; c0 += 32) {
                float v[32];
                tmem_st_wait();
                tmem_ld32(o_row + c0, v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float x = add ? __bfloat162float(value[c0 + e]) : 0.f;
                  if (!isfinite(x)) v[e] += x;       // times a weight above zero
                }
                tmem_st32(o_row + c0, v);
              }
            }
          }
        }
        tmem_st_wait();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        bar_arrive(p_full(g));
      }
      if (ok && s.tiles > 0) {
        ok = __all_sync(0xffffffffu, bar_wait(o_done(g), (done - 1) & 1, p.status));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      // The row's sums: this slot's alone, or, where both slots had the same rows, both slots', half of the head each.
      float m = m_ref, l = l_run, mine = 1.f, other = 0.f;
      int d0 = 0, d1 = D;
      if (!s.pair) {
        xchg[g * 128 + r] = make_float2(m_ref, l_run);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        both_slots_sync();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float2 theirs = xchg[(g ^ 1) * 128 + r];
        m = fmaxf(m_ref, theirs.x);
        mine = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - m);
        other = theirs.x == -INFINITY ? 0.f : fast_exp2(theirs.x - m);
        l = (l_run == 0.f ? 0.f : l_run * mine) + (theirs.y == 0.f ? 0.f : theirs.y * other);
        d0 = g * (D / 2);
        d1 = d0 + D / 2;
      }
      const bool write = live && ok;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const uint32_t o_other = tmem_o(g ^ 1) + lane_addr;
      const size_t share = (size_t)w.share * p.unit_rows + row;
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + ((size_t)token * p.heads + u.first_head + (live ? r % u.heads : 0)) * D;
      if (warp_live) {
#pragma unroll 1
        for (int c0 = d0; c0 < d1; c0 += 32) {
          float v[32], x[32];
          tmem_ld32(o_row + c0, v);
          if (!s.pair) tmem_ld32(o_other + c0, x);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            v[c] = mine == 0.f ? 0.f : v[c] * mine;
            if (!s.pair && other != 0.f) v[c] += x[c] * other;
          }
          if (write && w.whole) {
#pragma unroll
            for (int d = 0; d < 32; d += 8) {
              uint4 raw;
              raw.x = pack_pair(v[d] * inv, v[d + 1] * inv);
              raw.y = pack_pair(v[d + 2] * inv, v[d + 3] * inv);
              raw.z = pack_pair(v[d + 4] * inv, v[d + 5] * inv);
              raw.w = pack_pair(v[d + 6] * inv, v[d + 7] * inv);
              *reinterpret_cast<uint4*>(dst + c0 + d) = raw;
            }
          } else if (write) {
#pragma unroll
            for (int d = 0; d < 32; d += 4)
              *reinterpret_cast<float4*>(p.part_o + share * D + c0 + d) = make_float4(v[d], v[d + 1], v[d + 2], v[d + 3]);
          }
          __syncwarp();
        }
      }
      if (write && !w.whole && d0 == 0) p.part_ml[share] = make_float2(m, l);
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
  e = launch_pdl(kernel, dim3(p.ctas), dim3(kTreeThreads), Layout<D>::kBytes, stream, map_q, map_k, map_v, run_k, run_v, p);
  if (e != cudaSuccess) return (int)e;
  return tree_merge<__nv_bfloat16>(p, stream);
}

}  // namespace einf

using namespace einf;

// The arguments of einf_tree_attention without a dtype.  part_o: [2 * ctas][rows][size] floats with
// rows = 2 * (128 / (heads / kv_heads)) * (heads / kv_heads), part_ml: [2 * ctas][rows][2], notes: [ctas][4].
extern "C" int einf_tree_attention_tcgen05(const void* q, const void* k_cache, const void* v_cache, const int* block_table,
                                           const int* q_start, const int* cached_lens, const void* mask, const int* positions,
                                           void* out, float* part_o, float* part_ml, int* notes, int requests, int tokens, int heads,
                                           int kv_heads, int size, int page_size, int num_pages, int table_width, int words,
                                           int window, float scale, float softcap, int ctas, int min_chunk, int* status,
                                           cudaStream_t stream) {
  if (requests == 0 || tokens == 0) return 0;
  if ((size != 64 && size != 128) || ctas < 1 || min_chunk < 1 || kv_heads < 1 || heads % kv_heads || heads / kv_heads > kTile ||
      page_size < 8 || page_size > 128 || (page_size & (page_size - 1)) || words < 1 || (window > 0 && !positions) ||
      ((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) % 16)
    return (int)cudaErrorInvalidValue;
  TreeParams p = tree_params(q, k_cache, v_cache, block_table, q_start, cached_lens, mask, positions, out, part_o, part_ml, notes,
                             requests, tokens, heads, kv_heads, size, page_size, num_pages, table_width, words, window, scale, softcap,
                             ctas, min_chunk, status);
  p.unit_heads = heads / kv_heads;
  p.unit_nodes = 2 * (kTile / p.unit_heads);
  p.unit_rows = p.unit_nodes * p.unit_heads;
  p.padded = size;
  p.tile_keys = kTile;
  return size == 64 ? launch_tree<64>(p, stream) : launch_tree<128>(p, stream);
}
