// Penalties for repeated tokens, biases and grammar masks on rows of logits, in one pass over them.
//
//   x = logits[row][v];  c = how often v stands among the answered tokens and, for a drafted node, on its path
//   if v stands in the prompt or c > 0:  x = x > 0 ? x / repetition : x * repetition
//   x = x - (frequency c + presence [c > 0]) + bias[v];  x = -inf where v's bit of the mask is 0
//
// A pass has to read and write the rows and to read their masks: it is bound by memory.  No table of counts over the
// vocabulary is kept between calls; a CTA has a piece of the vocabulary, counts the request's tokens that fall into it in
// shared memory (the history is read once per piece, from the L2) and then walks the request's rows, a part of 2,048 places at
// a time.  Where rows start on 16 bytes the parts come to shared memory by bulk copies, four ahead, so that what is in flight
// depends neither on registers nor on how long a thread is at a part; other rows are read a float at a time, a part ahead.
// The nodes of a request share the counts.  A row's path is a few tokens: their places are left out of the walk and done
// one by one at the end, so that a row may be shaped in place.
//
// Measured with a vocabulary of 151,936, in captured graphs: 64 rows with histories of up to 4,096 tokens 21.5 us (3.7 TB/s;
// a plain copy would take 12: all of a row's parts are asked for at once and then wait for the counts, and each of a request's CTAs
// reads its whole history), 143 rows of eight trees with biases and masks 42.6 us (4.2 TB/s; 27 for a copy; the CTAs of the request
// with the most rows end alone), one row 3.3 us.
#include "tcgen05.cuh"

namespace einf {

constexpr int kShapeThreads = 256;
constexpr int kPart = 8 * kShapeThreads;      // places that a CTA has at a time
constexpr int kMostParts = 4;                 // of its piece of the vocabulary
constexpr int kStages = 4;                    // parts on their way or in work
constexpr uint32_t kInPrompt = 1u << 31;      // a place's word: in the prompt, some node's token, a token with a bias, how often answered
constexpr uint32_t kDrafted = 1u << 30;
constexpr uint32_t kBiased = 1u << 29;
constexpr uint32_t kCount = kBiased - 1;
constexpr int kMostWords = 64;                // of a node's mask: 4,096 nodes
static_assert(64 * kMostWords * 8 <= kStages * kPart * 4, "the hits take the place of the parts");

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
  int parts;                   // parts of the vocabulary that a CTA has: 1, 2 or 4
  int row_ways;                // CTAs that take a request's rows in turn
};
static_assert(sizeof(ShapeParams) == 16 * 8 + 10 * 4, "as packed");

struct ShapeRequest {
  float repetition, inverse, presence, frequency;
};

// Without branches: where one place in a warp's 128 has been seen, they all come here.  (x / repetition is x times its rounded
// reciprocal, two roundings of 2^-24 instead of one: a division here would be ten instructions for each of the 128.)
__device__ __forceinline__ float shaped(float x, uint32_t word, int on_path, const ShapeRequest& s) {
  const int count = (int)(word & kCount) + on_path;
  const float factor = x > 0.f ? s.inverse : s.repetition;
  const float off = count > 0 ? fmaf(s.frequency, (float)count, s.presence) : 0.f;
  return ((word & kInPrompt) || count > 0 ? x * factor : x) - off;
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

// What a CTA works on: rows first_row, first_row + ways, ... of a request and places v0 .. v0 + length of them.
struct Walk {
  int request, first, nodes, first_row, rows, v0, length, piece;
};
__device__ __forceinline__ Walk walk_of(const ShapeParams& p) {
  Walk w;
  w.piece = p.parts * kPart;
  w.request = blockIdx.y;
  w.v0 = blockIdx.x * w.piece;
  w.length = min(w.piece, p.vocab - w.v0);
  w.first = p.row_start ? max(0, min(p.row_start[w.request], p.rows)) : w.request;
  w.nodes = p.row_start ? max(0, min(p.row_start[w.request + 1], p.rows) - w.first) : 1;
  w.first_row = w.first + (int)blockIdx.z;
  w.rows = max(0, (w.nodes - (int)blockIdx.z + (int)gridDim.z - 1) / (int)gridDim.z);
  return w;
}

constexpr int kTokensAhead = 4;               // times four tokens of the history that a thread asks for at once

// The first tokens of the history: asked for before anything is known of how many there are.
__device__ __forceinline__ void ask_tokens(const ShapeParams& p, const Walk& w, int i0, int4 (&t)[kTokensAhead]) {
  const int* history = p.history + (size_t)w.request * p.capacity;
#pragma unroll
  for (int a = 0; a < kTokensAhead; ++a) {
    const int i = i0 + a * 4 * kShapeThreads;
    if (i + 4 <= p.capacity) t[a] = *reinterpret_cast<const int4*>(history + i);
  }
}

// The words of the CTA's places, and behind them (HAS_BIAS) 1 + a place's entry in the list of biases, or 0.
template <bool HAS_BIAS>
__device__ __forceinline__ ShapeRequest count_tokens(const ShapeParams& p, const Walk& w, uint32_t* words) {
  uint32_t* which = words + w.piece;
  const bool four = p.history && p.capacity % 4 == 0 && ((uintptr_t)p.history & 15) == 0;
  int4 t[kTokensAhead];
  if (four) ask_tokens(p, w, 4 * threadIdx.x, t);
  const int filled = p.history ? max(0, min(p.history_lens[w.request], p.capacity)) : 0, prompt = p.prompt_lens ? p.prompt_lens[w.request] : 0;
  ShapeRequest s;
  s.repetition = p.repetition ? p.repetition[w.request] : 1.f;
  s.presence = p.presence ? p.presence[w.request] : 0.f;
  s.frequency = p.frequency ? p.frequency[w.request] : 0.f;
  for (int i = 4 * threadIdx.x; i < (HAS_BIAS ? 2 : 1) * w.piece; i += 4 * kShapeThreads)
    *reinterpret_cast<uint4*>(words + i) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  bool bad = false;
  auto count = [&](int i, int token) {
    if (i >= filled) return;
    if ((unsigned)(token - w.v0) < (unsigned)w.length) {
      if (i < prompt) atomicOr(words + token - w.v0, kInPrompt);
      else atomicAdd(words + token - w.v0, 1u);
    } else if ((unsigned)token >= (unsigned)p.vocab) {
      bad = true;
    }
  };
  if (four) {
#pragma unroll 1
    for (int i0 = 4 * threadIdx.x; i0 < filled;) {
#pragma unroll
      for (int a = 0; a < kTokensAhead; ++a) {
        const int i = i0 + a * 4 * kShapeThreads;
        if (i >= filled) break;
        count(i, t[a].x);
        count(i + 1, t[a].y);
        count(i + 2, t[a].z);
        count(i + 3, t[a].w);
      }
      i0 += kTokensAhead * 4 * kShapeThreads;
      if (i0 < filled) ask_tokens(p, w, i0, t);
    }
  } else {
    for (int i = threadIdx.x; i < filled; i += kShapeThreads) count(i, p.history[(size_t)w.request * p.capacity + i]);
  }
  if (p.node_tokens)
    for (int k = threadIdx.x; k < min(w.nodes, 64 * p.words); k += kShapeThreads) {
      const int token = p.node_tokens[w.first + k];
      if ((unsigned)token >= (unsigned)p.vocab) bad = true;
      else if ((unsigned)(token - w.v0) < (unsigned)w.length) atomicOr(words + token - w.v0, kDrafted);
    }
  if (HAS_BIAS)
    for (int j = threadIdx.x; j < p.biases; j += kShapeThreads) {
      const int token = p.bias_ids[(size_t)w.request * p.biases + j];
      if (token >= p.vocab) bad = true;
      else if (token >= 0 && (unsigned)(token - w.v0) < (unsigned)w.length) {
        atomicMax(which + token - w.v0, j + 1u);
        atomicOr(words + token - w.v0, kBiased);
      }
    }
  if (bad && blockIdx.x == 0) atomicOr(p.status, kStatusBadToken);
  s.inverse = 1.f / s.repetition;
  __syncthreads();
  return s;
}

// The places of the nodes' tokens.  `hits` takes the nodes whose tokens are the CTA's (room for as many as a mask has bits), and the
// hits of one token are strung together, the lowest node first; then (hit, row) pairs, a token at its first hit: the row's count
// is the request's and that of the hits with this token on the row's path.
template <bool HAS_BIAS>
__device__ __forceinline__ void shape_drafted(const ShapeParams& p, const Walk& w, const ShapeRequest& s, const uint32_t* words, int2* hits) {
  __shared__ int hit_count;
  if (!p.node_tokens) return;
  const uint32_t* which = words + w.piece;
  if (threadIdx.x == 0) hit_count = 0;
  __syncthreads();
  for (int k = threadIdx.x; k < min(w.nodes, 64 * p.words); k += kShapeThreads) {
    const int token = p.node_tokens[w.first + k];
    if ((unsigned)(token - w.v0) < (unsigned)w.length) hits[atomicAdd(&hit_count, 1)] = make_int2(k, token);
  }
  __syncthreads();
  const int count = hit_count;
  // 12 bits: the node, 13 bits above: 1 + where the next hit of its token lies, or 0; the sign: it is not the first.  (What others
  // look at, the node's bits, does not change.)
  static_assert(64 * kMostWords <= 1 << 12, "a node in 12 bits");
  volatile int* entries = reinterpret_cast<volatile int*>(hits);
  for (int h = threadIdx.x; h < count; h += kShapeThreads) {
    const int node = entries[2 * h] & 0xfff, token = entries[2 * h + 1];
    int next = 0, next_node = 1 << 12, before = 0;
    for (int other = 0; other < count; ++other) {
      const int n = entries[2 * other] & 0xfff;
      if (entries[2 * other + 1] != token) continue;
      before |= n < node;
      if (n > node && n < next_node) next = other + 1, next_node = n;
    }
    entries[2 * h] = node | next << 12 | (before ? 1 << 31 : 0);
  }
  __syncthreads();
  for (int item = threadIdx.x; item < count * w.rows; item += kShapeThreads) {
    const int n = item / count, row = w.first_row + n * (int)gridDim.z;
    const int2 hit = hits[item - n * count];
    const uint32_t* path = p.tree_mask + (size_t)row * 2 * p.words;
    if (hit.x < 0) continue;
    int on_path = 0;
    for (int at = hit.x;; at = hits[(at >> 12 & 0x1fff) - 1].x) {
      on_path += path[(at & 0xfff) >> 5] >> (at & 31) & 1u;
      if (!(at >> 12 & 0x1fff)) break;
    }
    const uint32_t entry = HAS_BIAS ? which[hit.y - w.v0] : 0u;
    float x = shaped(p.logits[(size_t)row * p.vocab + hit.y], words[hit.y - w.v0], on_path, s);
    if (entry) x += p.bias[(size_t)w.request * p.biases + entry - 1];
    const uint32_t* mask = row_mask(p, row);
    if (mask && !(mask[hit.y >> 5] >> (hit.y & 31) & 1u)) x = -INFINITY;
    p.out[(size_t)row * p.vocab + hit.y] = x;
  }
}

// Rows that start on 16 bytes.
template <bool HAS_BIAS>
__global__ void __launch_bounds__(kShapeThreads) shape_logits_bulk_kernel(ShapeParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  float* ring = reinterpret_cast<float*>(smem);                                       // [stages][part]
  uint32_t* words = reinterpret_cast<uint32_t*>(smem + kStages * kPart * 4);
  __shared__ __align__(8) unsigned long long bars[kStages];
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) bar_init(saddr(bars + i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  const Walk w = walk_of(p);
  if (w.rows == 0) return;
  const int part_shift = __ffs(p.parts) - 1, steps = w.rows << part_shift;
  // parts beyond the end of the vocabulary are steps without work
  auto places = [&](int step) { return min(kPart, w.length - (step & (p.parts - 1)) * kPart); };
  auto fetch = [&](int step) {
    const int n = places(step);
    if (step >= steps || n <= 0) return;
    const int stage = step % kStages, row = w.first_row + (step >> part_shift) * (int)gridDim.z;
    const float* from = p.logits + (size_t)row * p.vocab + w.v0 + (step & (p.parts - 1)) * kPart;
    bar_expect_tx(saddr(bars + stage), n * 4);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(saddr(ring + stage * kPart)),
                 "l"(from), "r"(n * 4), "r"(saddr(bars + stage))
                 : "memory");
  };
  // a thread's two runs of four places, 32 words of the mask apart; asked for a step ahead
  const int i0 = 4 * threadIdx.x;
  struct Bits {
    uint32_t run[2];
  };
  auto ask_bits = [&](int step) {
    Bits b = {{0xffffffffu, 0xffffffffu}};
    if (!p.allowed || step >= steps) return b;
    const uint32_t* mask = row_mask(p, w.first_row + (step >> part_shift) * (int)gridDim.z);
    const int n = places(step), at = w.v0 + (step & (p.parts - 1)) * kPart + i0;
    if (mask && i0 < n) b.run[0] = mask[at >> 5];
    if (mask && i0 + 4 * kShapeThreads < n) b.run[1] = mask[(at >> 5) + kShapeThreads / 8];
    return b;
  };
  if (threadIdx.x == 0)
    for (int step = 0; step < kStages; ++step) fetch(step);      // on their way while the history is counted
  Bits ahead = ask_bits(0);
  const ShapeRequest s = count_tokens<HAS_BIAS>(p, w, words);
  const uint32_t* which = words + w.piece;
  const float* biases = p.bias + (size_t)w.request * p.biases;
  const int shift = (w.v0 + i0) & 31;                            // parts start on whole words
  uint32_t parity = 0u;                                          // a bit a stage
  int there = steps;                                             // the first step whose part did not come within the limit
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    const int stage = step % kStages, n = places(step), part0 = (step & (p.parts - 1)) * kPart;
    const Bits bits = ahead;
    ahead = ask_bits(step + 1);
    if (n > 0 && there == steps && !bar_wait_likely_done(saddr(bars + stage), parity >> stage & 1u, p.status)) there = step;
    if (n > 0 && there == steps) {
      float* out = p.out + (size_t)(w.first_row + (step >> part_shift) * (int)gridDim.z) * p.vocab + w.v0 + part0;
      parity ^= 1u << stage;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int i = i0 + a * 4 * kShapeThreads;
        if (i >= n) break;
        float4 x = *reinterpret_cast<const float4*>(ring + stage * kPart + i);
        const uint4 word = *reinterpret_cast<const uint4*>(words + part0 + i);
        const uint32_t any = word.x | word.y | word.z | word.w;
        if (any) {
          x.x = shaped(x.x, word.x, 0, s);
          x.y = shaped(x.y, word.y, 0, s);
          x.z = shaped(x.z, word.z, 0, s);
          x.w = shaped(x.w, word.w, 0, s);
          if (HAS_BIAS && (any & kBiased)) {
            const uint4 entry = *reinterpret_cast<const uint4*>(which + part0 + i);
            if (entry.x) x.x += biases[entry.x - 1];
            if (entry.y) x.y += biases[entry.y - 1];
            if (entry.z) x.z += biases[entry.z - 1];
            if (entry.w) x.w += biases[entry.w - 1];
          }
        }
        const uint32_t b = bits.run[a] >> shift;
        x.x = b & 1u ? x.x : -INFINITY;
        x.y = b & 2u ? x.y : -INFINITY;
        x.z = b & 4u ? x.z : -INFINITY;
        x.w = b & 8u ? x.w : -INFINITY;
        if (!(any & kDrafted)) {
          __stcs(reinterpret_cast<float4*>(out + i), x);
        } else {
          if (!(word.x & kDrafted)) out[i] = x.x;
          if (!(word.y & kDrafted)) out[i + 1] = x.y;
          if (!(word.z & kDrafted)) out[i + 2] = x.z;
          if (!(word.w & kDrafted)) out[i + 3] = x.w;
        }
      }
    }
    __syncthreads();                                             // the stage is read
    if (threadIdx.x == 0 && there == steps) fetch(step + kStages);
  }
  if (!__syncthreads_and(there == steps)) {
    // A thread that gave up asked for and wrote nothing more; no CTA ends with a copy under way.
    if (threadIdx.x == 0)
      for (int step = there; step < min(steps, there + kStages); ++step)
        if (places(step) > 0) bar_poll(saddr(bars + step % kStages), parity >> (step % kStages) & 1u);
    return;
  }
  shape_drafted<HAS_BIAS>(p, w, s, words, reinterpret_cast<int2*>(ring));
}

// Any rows.
template <bool HAS_BIAS>
__global__ void __launch_bounds__(kShapeThreads) shape_logits_kernel(ShapeParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  uint32_t* words = reinterpret_cast<uint32_t*>(smem);
  pdl_launch_dependents();
  pdl_wait();
  const Walk w = walk_of(p);
  if (w.rows == 0) return;
  const int part_shift = __ffs(p.parts) - 1, steps = w.rows << part_shift;
  struct Places {
    float x[8];
    bool allowed[8];
  };
  auto load = [&](int step, Places& t) {
    const int row = w.first_row + (step >> part_shift) * (int)gridDim.z, i0 = (step & (p.parts - 1)) * kPart + threadIdx.x;
    const float* in = p.logits + (size_t)row * p.vocab + w.v0;
    const uint32_t* mask = row_mask(p, row);
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      const int i = i0 + a * kShapeThreads;
      t.x[a] = i < w.length ? __ldcs(in + i) : 0.f;
      t.allowed[a] = !mask || i >= w.length || (mask[(w.v0 + i) >> 5] >> ((w.v0 + i) & 31) & 1u);
    }
  };
  Places now, next;
  load(0, now);                               // on their way while the history is counted
  const ShapeRequest s = count_tokens<HAS_BIAS>(p, w, words);
  const uint32_t* which = words + w.piece;
  const float* biases = p.bias + (size_t)w.request * p.biases;
  auto shape = [&](int step, Places& t) {
    const int row = w.first_row + (step >> part_shift) * (int)gridDim.z, i0 = (step & (p.parts - 1)) * kPart + threadIdx.x;
    float* out = p.out + (size_t)row * p.vocab + w.v0;
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      const int i = i0 + a * kShapeThreads;
      if (i >= w.length) break;
      const uint32_t word = words[i];
      float x = t.x[a];
      if (word) x = shaped(x, word, 0, s);
      if (HAS_BIAS && (word & kBiased)) x += biases[which[i] - 1];
      if (!(word & kDrafted)) __stcs(out + i, t.allowed[a] ? x : -INFINITY);
    }
  };
#pragma unroll 1
  for (int step = 0; step < steps; step += 2) {
    if (step + 1 < steps) load(step + 1, next);
    shape(step, now);
    if (step + 2 < steps) load(step + 2, now);
    if (step + 1 < steps) shape(step + 1, next);
  }
  __syncthreads();
  shape_drafted<HAS_BIAS>(p, w, s, words, reinterpret_cast<int2*>(words + (HAS_BIAS ? 2 : 1) * w.piece));
}

}  // namespace einf

using namespace einf;

// call: a ShapeParams, on the host.
extern "C" int einf_shape_logits(const char* call, cudaStream_t stream) {
  const ShapeParams& p = *reinterpret_cast<const ShapeParams*>(call);
  if (p.rows == 0 || p.requests == 0) return 0;
  if (p.vocab < 1 || p.parts < 1 || p.parts > kMostParts || (p.parts & (p.parts - 1)) || p.row_ways < 1 || p.row_ways > 65535 || p.requests > 65535 ||
      (p.node_tokens && (!p.tree_mask || p.words < 1 || p.words > kMostWords)) || (p.history && !p.history_lens))
    return (int)cudaErrorInvalidValue;
  const bool has_bias = p.biases > 0, bulk = p.vocab % 4 == 0 && (((uintptr_t)p.logits | (uintptr_t)p.out) & 15) == 0;
  const auto kernel = bulk ? (has_bias ? shape_logits_bulk_kernel<true> : shape_logits_bulk_kernel<false>)
                           : (has_bias ? shape_logits_kernel<true> : shape_logits_kernel<false>);
  const int piece = p.parts * kPart;
  const size_t smem = (size_t)piece * 4 * (has_bias ? 2 : 1) + (bulk ? kStages * kPart * 4 : p.node_tokens ? 64 * p.words * 8 : 0);
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * kMostParts + kStages) * kPart * 4);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kernel, dim3((p.vocab + piece - 1) / piece, p.requests, p.row_ways), dim3(kShapeThreads), smem, stream, p);
}
