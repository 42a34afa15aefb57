// Penalties for repeated tokens, biases and grammar masks on rows of logits, in one pass over them.
//
//   x = logits[row][v];  c = how often v stands among the answered tokens and, for a drafted node, on its path
//   if v stands in the prompt or c > 0:  x = x > 0 ? x / repetition : x * repetition
//   x = x - (frequency c + presence [c > 0]) + bias[v];  x = -inf where v's bit of the mask is 0
//
// A pass has to read and write the rows and to read their masks: it is bound by memory.  No table of counts over the
// vocabulary is kept between calls; a CTA has a piece of the vocabulary, counts the request's tokens that fall into it in
// shared memory (the history is read once per piece, from the L2) and then walks the request's rows.  The nodes of a
// request share these counts.  A row's path is a few tokens: their places are left out of the walk and done one by
// one at the end, so that a row may be shaped in place.
#include "common.cuh"

namespace einf {

constexpr int kShapeThreads = 256;
constexpr int kMostPlaces = 16384;            // of a CTA's piece of the vocabulary
constexpr uint32_t kInPrompt = 1u << 31;      // a place's word: in the prompt, some node's token, how often answered
constexpr uint32_t kDrafted = 1u << 30;
constexpr uint32_t kCount = kDrafted - 1;

// A call's arguments, as the caller packs them.
struct ShapeParams {
  const float* logits;         // [rows, vocab]
  float* out;
  int* status;
  const int* history_lens;     // [requests]
  const int* prompt_lens;      // [requests] or null: so many of the history's tokens are the prompt's
  const float* repetition;     // [requests] or null: 1
  const float* presence;       // [requests] or null: 0
  const float* frequency;
  const int* row_start;        // [requests + 1], or null: a row each
  const int* history;          // [requests, capacity] or null
  const int* node_tokens;      // [rows] or null
  const uint32_t* tree_mask;   // [rows, 2 * words]
  const int* bias_ids;         // [requests, biases], negative: none
  const float* bias;
  const uint32_t* allowed;     // [masks, mask_words] or null
  const int* allowed_rows;     // [rows] or null: row r has mask r
  int rows, vocab, requests, capacity, words, biases, masks, mask_words;
  int piece;                   // places of the vocabulary that a CTA has, a multiple of 32
  int row_ways;                // CTAs that take a request's rows in turn
};
static_assert(sizeof(ShapeParams) == 16 * 8 + 10 * 4, "as packed");

struct ShapeRequest {
  float repetition, presence, frequency;
};

__device__ __forceinline__ float shaped(float x, uint32_t word, int on_path, const ShapeRequest& s) {
  const int count = (int)(word & kCount) + on_path;
  if ((word & kInPrompt) || count > 0) x = x > 0.f ? x / s.repetition : x * s.repetition;
  if (count > 0) x -= fmaf(s.frequency, (float)count, s.presence);
  return x;
}

// Which mask a row has: its words, or null.
__device__ __forceinline__ const uint32_t* row_mask(const ShapeParams& p, int row) {
  if (!p.allowed) return nullptr;
  const int mask = p.allowed_rows ? p.allowed_rows[row] : row;
  if (mask >= p.masks) {
    atomicOr(p.status, kStatusBadIndex);
    return nullptr;
  }
  return mask < 0 ? nullptr : p.allowed + (size_t)mask * p.mask_words;
}

// VEC: elements of a row read together (4 where every row starts on 16 bytes); HAS_BIAS: the places' biases lie in
// shared memory behind their words.
template <int VEC, bool HAS_BIAS>
__global__ void __launch_bounds__(kShapeThreads) shape_logits_kernel(ShapeParams p) {
  extern __shared__ __align__(16) uint32_t words[];
  pdl_launch_dependents();
  pdl_wait();
  const int request = blockIdx.y, v0 = blockIdx.x * p.piece, length = min(p.piece, p.vocab - v0);
  const int first = p.row_start ? max(0, min(p.row_start[request], p.rows)) : request;
  const int nodes = p.row_start ? max(0, min(p.row_start[request + 1], p.rows) - first) : 1;
  if (nodes <= (int)blockIdx.z) return;
  uint32_t* which = words + p.piece;          // 1 + the place's entry in the list of biases, or 0
  for (int i = 4 * threadIdx.x; i < (HAS_BIAS ? 2 : 1) * p.piece; i += 4 * kShapeThreads)
    *reinterpret_cast<uint4*>(words + i) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  bool bad = false;
  if (p.history) {
    const int* history = p.history + (size_t)request * p.capacity;
    const int filled = max(0, min(p.history_lens[request], p.capacity)), prompt = p.prompt_lens ? p.prompt_lens[request] : 0;
    auto count = [&](int i, int token) {
      if ((unsigned)token >= (unsigned)p.vocab) {
        bad = true;
      } else if ((unsigned)(token - v0) < (unsigned)length) {
        if (i < prompt) atomicOr(words + token - v0, kInPrompt);
        else atomicAdd(words + token - v0, 1u);
      }
    };
    int done = 0;
    if (((uintptr_t)history & 15) == 0) {
      done = filled & ~3;
      for (int i = 4 * threadIdx.x; i < done; i += 4 * kShapeThreads) {
        const int4 t = *reinterpret_cast<const int4*>(history + i);
        count(i, t.x);
        count(i + 1, t.y);
        count(i + 2, t.z);
        count(i + 3, t.w);
      }
    }
    for (int i = done + threadIdx.x; i < filled; i += kShapeThreads) count(i, history[i]);
  }
  if (p.node_tokens)
    for (int k = threadIdx.x; k < nodes; k += kShapeThreads) {
      const int token = p.node_tokens[first + k];
      if ((unsigned)token >= (unsigned)p.vocab) bad = true;
      else if ((unsigned)(token - v0) < (unsigned)length) atomicOr(words + token - v0, kDrafted);
    }
  if (HAS_BIAS)
    for (int j = threadIdx.x; j < p.biases; j += kShapeThreads) {
      const int token = p.bias_ids[(size_t)request * p.biases + j];
      if (token >= p.vocab) bad = true;
      else if (token >= 0 && (unsigned)(token - v0) < (unsigned)length) atomicMax(which + token - v0, j + 1u);
    }
  if (bad && blockIdx.x == 0) atomicOr(p.status, kStatusBadToken);
  ShapeRequest s;
  s.repetition = p.repetition ? p.repetition[request] : 1.f;
  s.presence = p.presence ? p.presence[request] : 0.f;
  s.frequency = p.frequency ? p.frequency[request] : 0.f;
  const float* biases = p.bias + (size_t)request * p.biases;
  __syncthreads();

  constexpr int kAhead = 4;
  for (int node = blockIdx.z; node < nodes; node += gridDim.z) {
    const int row = first + node;
    const float* in = p.logits + (size_t)row * p.vocab + v0;
    float* out = p.out + (size_t)row * p.vocab + v0;
    const uint32_t* mask = row_mask(p, row);
    for (int i0 = VEC * threadIdx.x; i0 < length; i0 += kAhead * VEC * kShapeThreads) {
      float x[kAhead][VEC];
      uint32_t bits[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * VEC * kShapeThreads;
        bits[a] = 0xffffffffu;
        if (i < length) {
          if (VEC == 4) {
            const float4 v = *reinterpret_cast<const float4*>(in + i);
            x[a][0] = v.x, x[a][1] = v.y, x[a][2] = v.z, x[a][3] = v.w;
          } else {
            x[a][0] = in[i];
          }
          if (mask) bits[a] = mask[(v0 + i) >> 5] >> ((v0 + i) & 31);
        }
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * VEC * kShapeThreads;
        if (i >= length) break;
        uint32_t word[VEC], entry[VEC];
        if (VEC == 4) {
          *reinterpret_cast<uint4*>(word) = *reinterpret_cast<const uint4*>(words + i);
          if (HAS_BIAS) *reinterpret_cast<uint4*>(entry) = *reinterpret_cast<const uint4*>(which + i);
        } else {
          word[0] = words[i];
          if (HAS_BIAS) entry[0] = which[i];
        }
        uint32_t drafted = 0u;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          drafted |= word[e] & kDrafted;
          if (word[e]) x[a][e] = shaped(x[a][e], word[e], 0, s);
          if (HAS_BIAS && entry[e]) x[a][e] += biases[entry[e] - 1];
          if (!(bits[a] >> e & 1u)) x[a][e] = -INFINITY;
        }
        if (VEC == 4 && !drafted) {
          *reinterpret_cast<float4*>(out + i) = make_float4(x[a][0], x[a][1 % VEC], x[a][2 % VEC], x[a][3 % VEC]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (!(word[e] & kDrafted)) out[i + e] = x[a][e];
        }
      }
    }
  }
  if (!p.node_tokens) return;
  // the places of the nodes' tokens: (node whose token it is, row) pairs, a token that several nodes have at its first
  const int rows_here = (nodes - (int)blockIdx.z + (int)gridDim.z - 1) / (int)gridDim.z;
  for (int k = threadIdx.x >> 5; k < nodes; k += kShapeThreads / 32) {
    const int token = p.node_tokens[first + k];
    if ((unsigned)(token - v0) >= (unsigned)length || (unsigned)token >= (unsigned)p.vocab) continue;
    const int lane = threadIdx.x & 31;
    bool before = false;
    for (int k0 = 0; k0 < k; k0 += 32)
      before = before || __any_sync(0xffffffffu, k0 + lane < k && p.node_tokens[first + k0 + lane] == token);
    if (before) continue;
    const uint32_t word = words[token - v0];
    const uint32_t entry = HAS_BIAS ? which[token - v0] : 0u;
    for (int n = lane; n < rows_here; n += 32) {
      const int row = first + (int)blockIdx.z + n * (int)gridDim.z;
      const uint32_t* path = p.tree_mask + (size_t)row * 2 * p.words;
      int on_path = 0;
      for (int other = k; other < nodes && other < 64 * p.words; ++other)
        if ((path[other >> 5] >> (other & 31) & 1u) && p.node_tokens[first + other] == token) ++on_path;
      float x = shaped(p.logits[(size_t)row * p.vocab + token], word, on_path, s);
      if (entry) x += biases[entry - 1];
      const uint32_t* mask = row_mask(p, row);
      if (mask && !(mask[token >> 5] >> (token & 31) & 1u)) x = -INFINITY;
      p.out[(size_t)row * p.vocab + token] = x;
    }
  }
}

}  // namespace einf

using namespace einf;

// call: a ShapeParams, on the host.
extern "C" int einf_shape_logits(const char* call, cudaStream_t stream) {
  const ShapeParams& p = *reinterpret_cast<const ShapeParams*>(call);
  if (p.rows == 0 || p.requests == 0) return 0;
  if (p.vocab < 1 || p.piece < 32 || p.piece % 32 || p.piece > kMostPlaces || p.row_ways < 1 || p.row_ways > 65535 || p.requests > 65535 ||
      (p.node_tokens && !p.tree_mask) || (p.history && !p.history_lens))
    return (int)cudaErrorInvalidValue;
  const bool has_bias = p.biases > 0, vec = p.vocab % 4 == 0 && (((uintptr_t)p.logits | (uintptr_t)p.out) & 15) == 0;
  const auto kernel = vec ? (has_bias ? shape_logits_kernel<4, true> : shape_logits_kernel<4, false>)
                          : (has_bias ? shape_logits_kernel<1, true> : shape_logits_kernel<1, false>);
  const size_t smem = (size_t)p.piece * 4 * (has_bias ? 2 : 1);
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMostPlaces * 4);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kernel, dim3((p.vocab + p.piece - 1) / p.piece, p.requests, p.row_ways), dim3(kShapeThreads), smem, stream, p);
}
