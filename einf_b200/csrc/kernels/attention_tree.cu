// Attention of drafted trees over the paged cache with 32-bit products: the 32-bit path, and in bfloat16 the head and
// page sizes that the tensor-core kernel (attention_tree_tcgen05.cu) does not take.
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax_j(cap(scale q_i . k_j)) over the keys that node i sees
//
// One pass over the keys, 32 at a time, with the running maximum and sum of every row.  Four warps have eight
// rows each.  Scores: lane j has key j, whose elements it reads once for its eight rows; the rows come as broadcasts.
// Sums: a lane has a few elements of the head, whose values it reads once for its eight rows.  Both products read 12
// 16-byte words of shared memory for 32 fused multiply-adds, so shared memory bounds the kernel at two thirds of
// the FMA rate.  Keys that no row of a tile is kept from run without masks; in the other tiles a value is added
// to the rows that see it and to no others, so that what stands in a masked place (a sibling's value, a row behind the
// last node) may be anything.  Between the products the scores change hands, so that a row's softmax is four lanes' work, eight
// keys each, done once for a warp's eight rows (a row after the other with a key a lane it was 2 us of a tile's 5: shuffles, and as
// many instructions to fetch again for every row).
//
// With few requests a CTA has one tile of keys, 3.2 us: its loads 1.2, scores 1, probabilities 0.4, sums 0.8, each at its latency with a
// warp on a scheduler; 2.5 us go before it, 4 are the second launch's.  15.7 us for 2 requests of up to 700 keys and 13 nodes
// with 14 and 2 heads of 64 in float32, where the bytes alone would take 0.2; 223 us for one of 8,192 and 32 with 28 and 4 of 128
// (17 TFLOP/s: the latency of shared memory between few warps).
#include "attention_tree.cuh"
#include "mma_sync.cuh"

namespace einf {

constexpr int kKeys = 32;
constexpr int kWarps = 4;
constexpr int kRowsPerWarp = 8;
constexpr int kRows = kWarps * kRowsPerWarp;
constexpr int kPitch = kKeys + 4;      // of a row's probabilities: four lanes a row meet no bank twice
static_assert(kKeys == 32 && kRowsPerWarp == 8, "four lanes a row, eight keys a lane");

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_pair(v.x, v.y), pack_pair(v.z, v.w));
}
// Four elements of a row from d on, wherever it starts; zeros behind its end.
template <typename T>
__device__ __forceinline__ float4 elements(const T* row, int d, int size) {
  return make_float4(d < size ? to_float(row[d]) : 0.f, d + 1 < size ? to_float(row[d + 1]) : 0.f, d + 2 < size ? to_float(row[d + 2]) : 0.f,
                     d + 3 < size ? to_float(row[d + 3]) : 0.f);
}

// VEC: elements of the head that a lane has (2, 4 or 8: heads of up to 64, 128, 256).  Launches have two CTAs an SM, and the compiler is
// told so: left to itself it took registers for one of three or four, and the products' loop came out up to a fifth slower with every
// change around it (one request of 8,192 keys and 32 nodes, 28 and 4 heads of 128 in float32: 223 us; 272 without, 229 for four).
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kWarps, 2) tree_attention_kernel(TreeParams p) {
  extern __shared__ __align__(16) float smem[];
  const int size4 = (p.size + 3) & ~3, pitch = size4 + 4;
  float* ks = smem;                                 // [keys][pitch]
  float* vs = ks + kKeys * pitch;                   // [keys][32 * VEC]
  float* qs = vs + kKeys * 32 * VEC;                // [rows][size4]
  float* ps = qs + kRows * size4;                   // [rows][pitch]: scores, then probabilities
  __shared__ long long places[kKeys];               // where a key's row starts in the caches, or -1
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const T* q = static_cast<const T*>(p.q);
  const T* k_cache = static_cast<const T*>(p.k_cache);
  const T* v_cache = static_cast<const T*>(p.v_cache);
  const bool aligned = p.size % 4 == 0 && (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)p.out) & 15) == 0;
  TreeWalk w;
  bool any = tree_first(p, blockIdx.x, &w);
  if (threadIdx.x == 0) tree_note(p, blockIdx.x, w, any);
  const float scale_log2 = p.scale * 1.4426950408889634f, cap_log2 = p.softcap * 1.4426950408889634f;
  for (; any; any = tree_next(p, blockIdx.x, &w)) {
    const TreeUnit u = tree_unit(p, w.t, w.unit);
    const int rows = u.nodes * u.heads;
    __syncthreads();
    const int pieces = size4 >> 2;                  // of a row, four elements each
    for (int e = threadIdx.x; e < kRows * pieces; e += 32 * kWarps) {
      const int row = divide(e, pieces), d = 4 * (e - row * pieces), node = divide(row, u.heads);
      const T* from = q + ((size_t)(w.t.first + u.first_node + node) * p.heads + u.first_head + row - node * u.heads) * p.size;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows) v = aligned ? load4(from + d) : elements(from, d, p.size);
      *reinterpret_cast<float4*>(qs + row * size4 + d) = v;
    }
    // elements beyond the head are zeros, once
    for (int e = threadIdx.x; e < kKeys * 32 * VEC; e += 32 * kWarps)
      if (e % (32 * VEC) >= size4) vs[e] = 0.f;
    const int my_rows = min(kRowsPerWarp, rows - warp * kRowsPerWarp), row = warp * kRowsPerWarp + (lane >> 2);
    float m = -INFINITY, l = 0.f, acc[kRowsPerWarp][VEC];      // maximum and sum of `row`
    bool some = false;                                         // it has seen a key
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[i][e] = 0.f;
    const int keys_end = w.t.cached + w.t.nodes;
    const int* table = p.block_table + (size_t)w.request * p.table_width;
    for (int tile = w.tile_begin; tile < w.tile_end; ++tile) {
      const int key0 = w.t.begin + tile * kKeys;
      __syncthreads();
      if (threadIdx.x < kKeys) {
        const int key = key0 + threadIdx.x;
        long long at = -1;
        if (key < keys_end) {
          const int page = table[key / p.page_size];
          if (page < 0 || page >= p.num_pages) atomicOr(p.status, kStatusBadPage);
          else at = (((long long)page * p.kv_heads + u.kv_head) * p.page_size + key % p.page_size) * p.size;
        }
        places[threadIdx.x] = at;
      }
      __syncthreads();
      // a key beyond the end, or without a page, is zeros
      constexpr int kAhead = 4;
      if (!aligned) {
#pragma unroll 1
        for (int e = threadIdx.x; e < kKeys * pieces; e += 32 * kWarps) {
          const int key = divide(e, pieces), d = 4 * (e - key * pieces);
          const long long at = places[key];
          const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(ks + key * pitch + d) = at < 0 ? zero : elements(k_cache + at, d, p.size);
          *reinterpret_cast<float4*>(vs + key * 32 * VEC + d) = at < 0 ? zero : elements(v_cache + at, d, p.size);
        }
      }
#pragma unroll 1
      for (int e0 = threadIdx.x; aligned && e0 < kKeys * pieces; e0 += kAhead * 32 * kWarps) {
        float4 k4[kAhead], v4[kAhead];
        int key[kAhead], d[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int e = e0 + a * 32 * kWarps;
          key[a] = divide(e, pieces);
          d[a] = 4 * (e - key[a] * pieces);
          const long long at = key[a] < kKeys ? places[key[a]] : -1;
          k4[a] = v4[a] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (at >= 0) {
            k4[a] = load4(k_cache + at + d[a]);
            v4[a] = load4(v_cache + at + d[a]);
          }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
          if (key[a] < kKeys) {
            *reinterpret_cast<float4*>(ks + key[a] * pitch + d[a]) = k4[a];
            *reinterpret_cast<float4*>(vs + key[a] * 32 * VEC + d[a]) = v4[a];
          }
      }
      __syncthreads();
      if (my_rows <= 0) continue;
      float s[kRowsPerWarp];
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) s[i] = 0.f;
      const float* kr = ks + lane * pitch;
      const float* qr = qs + warp * kRowsPerWarp * size4;
#pragma unroll 2
      for (int d = 0; d < size4; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; ++i) {
          const float4 q4 = *reinterpret_cast<const float4*>(qr + i * size4 + d);
          s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
        }
      }
      // the scores change hands: four lanes a row, eight keys each
      float* pr = ps + warp * kRowsPerWarp * kPitch;
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) pr[i * kPitch + lane] = s[i];
      uint32_t bits = row < rows ? 0xffffffffu : 0u;
      if (row < rows && (key0 + kKeys > w.t.cached || p.window > 0)) {
        const int token = w.t.first + u.first_node + divide(row, u.heads), position = tree_position(p, w.t, token);
        bits = tree_visible(p, w.t, token, tree_lowest(p, position), position, key0);
      }
      __syncwarp();
      const bool all = __all_sync(0xffffffffu, row >= rows || bits == 0xffffffffu);
      float* mine = ps + row * kPitch + 8 * (lane & 3);
      if (p.softcap > 0.f) {
#pragma unroll 1
        for (int c = 0; c < 8; ++c) mine[c] = cap_log2 * tanhf(mine[c] * p.scale / p.softcap);
      }
      const float factor = p.softcap > 0.f ? 1.f : scale_log2;
      some = some || bits != 0u;
      float x[8];
#pragma unroll
      for (int c = 0; c < 8; c += 4) {
        const float4 v = *reinterpret_cast<const float4*>(mine + c);
        x[c] = v.x, x[c + 1] = v.y, x[c + 2] = v.z, x[c + 3] = v.w;
      }
      float top = m, sum = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        x[c] = bits >> (8 * (lane & 3) + c) & 1u ? x[c] * factor : -INFINITY;
        top = fmaxf(top, x[c]);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float keep = m == -INFINITY ? 0.f : exp2f(m - top);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        x[c] = x[c] == -INFINITY ? 0.f : exp2f(x[c] - top);
        sum += x[c];
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      l = (l == 0.f ? 0.f : l * keep) + sum;
      m = top;
#pragma unroll
      for (int c = 0; c < 8; c += 4) *reinterpret_cast<float4*>(mine + c) = make_float4(x[c], x[c + 1], x[c + 2], x[c + 3]);
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) {
        const float factor_i = __shfl_sync(0xffffffffu, keep, 4 * i);
#pragma unroll
        for (int d = 0; d < VEC; ++d) acc[i][d] *= factor_i;
      }
      __syncwarp();
      auto value = [&](int j, float* v) {
        const float* vr = vs + j * 32 * VEC;
        if (VEC == 2) {
          const float2 a = *reinterpret_cast<const float2*>(vr + 2 * lane);
          v[0] = a.x, v[1] = a.y;
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e += 4) {
            const float4 a = *reinterpret_cast<const float4*>(vr + e * 32 + 4 * lane);
            v[e] = a.x, v[e + 1] = a.y, v[e + 2] = a.z, v[e + 3] = a.w;
          }
        }
      };
      if (all) {
#pragma unroll 2
        for (int j = 0; j < kKeys; j += 4) {
          float4 e4[kRowsPerWarp];
#pragma unroll
          for (int i = 0; i < kRowsPerWarp; ++i) e4[i] = *reinterpret_cast<const float4*>(pr + i * kPitch + j);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            float v[VEC];
            value(j + jj, v);
#pragma unroll
            for (int i = 0; i < kRowsPerWarp; ++i) {
              const float e = jj == 0 ? e4[i].x : jj == 1 ? e4[i].y : jj == 2 ? e4[i].z : e4[i].w;
#pragma unroll
              for (int d = 0; d < VEC; ++d) acc[i][d] = fmaf(e, v[d], acc[i][d]);
            }
          }
        }
      } else {
        uint32_t some = 0u, seen[kRowsPerWarp];
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; ++i) some |= seen[i] = __shfl_sync(0xffffffffu, bits, 4 * i);
        for (; some; some &= some - 1) {
          const int j = __ffs(some) - 1;
          float v[VEC];
          value(j, v);
#pragma unroll
          for (int i = 0; i < kRowsPerWarp; ++i)
            if (seen[i] >> j & 1u) {
              const float e = pr[i * kPitch + j];
#pragma unroll
              for (int d = 0; d < VEC; ++d) acc[i][d] = fmaf(e, v[d], acc[i][d]);
            }
        }
      }
      __syncwarp();
    }
    if (my_rows <= 0) continue;
    // the sums take the place of the warp's queries, and go out from there four elements at a time
    float* left = qs + warp * kRowsPerWarp * size4;
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
      if (VEC == 2) {
        if (2 * lane < size4) *reinterpret_cast<float2*>(left + i * size4 + 2 * lane) = make_float2(acc[i][0], acc[i][1]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
          if (e * 32 + 4 * lane < size4)
            *reinterpret_cast<float4*>(left + i * size4 + e * 32 + 4 * lane) = make_float4(acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]);
      }
    }
    __syncwarp();
    if (m == -INFINITY && l == 0.f && some) l = 1.f;
    const float inv = tree_inverse(m, l);
#pragma unroll 1
    for (int e0 = 0; e0 < my_rows * pieces; e0 += 32) {
      const int e = min(e0 + lane, my_rows * pieces - 1), i = divide(e, pieces), d = 4 * (e - i * pieces), r = warp * kRowsPerWarp + i;
      const float f = __shfl_sync(0xffffffffu, inv, 4 * i);
      float4 v = *reinterpret_cast<const float4*>(left + 4 * e);
      if (!w.whole) {
        *reinterpret_cast<float4*>(tree_share(p, w.share, r, d)) = v;
        continue;
      }
      const int node = divide(r, u.heads);
      T* to = static_cast<T*>(p.out) + ((size_t)(w.t.first + u.first_node + node) * p.heads + u.first_head + r - node * u.heads) * p.size + d;
      v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
      if (aligned) {
        store4(to, v);
      } else {
        to[0] = from_float<T>(v.x);
        if (d + 1 < p.size) to[1] = from_float<T>(v.y);
        if (d + 2 < p.size) to[2] = from_float<T>(v.z);
        if (d + 3 < p.size) to[3] = from_float<T>(v.w);
      }
    }
    if (!w.whole && (lane & 3) == 0 && row < rows) p.part_ml[(size_t)w.share * p.unit_rows + row] = make_float2(m, l);
  }
}

template <typename T, int VEC>
int launch_tree(const TreeParams& p, cudaStream_t stream) {
  const int size4 = (p.size + 3) & ~3;
  const size_t smem = sizeof(float) * ((size_t)kKeys * (size4 + 4) + kKeys * 32 * VEC + kRows * size4 + kRows * kPitch);
  cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  e = launch_pdl(tree_attention_kernel<T, VEC>, dim3(p.workers), dim3(32 * kWarps), smem, stream, p);
  if (e != cudaSuccess) return (int)e;
  return tree_merge<T>(p, stream);
}

template <typename T>
int dispatch_tree(const TreeParams& p, cudaStream_t stream) {
  return p.size <= 64 ? launch_tree<T, 2>(p, stream) : p.size <= 128 ? launch_tree<T, 4>(p, stream) : launch_tree<T, 8>(p, stream);
}

}  // namespace einf

using namespace einf;

// call: a TreeCall, on the host; a worker is a CTA.  part_o: [2 * workers][32][padded] floats with the size rounded up to four, part_ml:
// [2 * workers][32][2], notes: [workers][8].
extern "C" int einf_tree_attention(const char* call, cudaStream_t stream) {
  const TreeCall& c = *reinterpret_cast<const TreeCall*>(call);
  if (c.requests == 0 || c.tokens == 0) return 0;
  if (!tree_call_fits(c) || c.size > 256 || c.cluster != 1) return (int)cudaErrorInvalidValue;
  TreeParams p = tree_params(c);
  p.unit_heads = c.heads / c.kv_heads < kRows ? c.heads / c.kv_heads : kRows;
  p.unit_nodes = kRows / p.unit_heads;
  p.group = c.heads / c.kv_heads;
  p.head_blocks = (p.group + p.unit_heads - 1) / p.unit_heads;
  p.unit_rows = kRows;
  p.padded = (c.size + 3) & ~3;
  p.tile_shift = 5;
  static_assert(kKeys == 32, "a tile of keys");
  EINF_DISPATCH_2(c.dtype, T, return dispatch_tree<T>(p, stream);)
  return 0;
}
