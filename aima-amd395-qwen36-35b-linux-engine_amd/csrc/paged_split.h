// How attention over the paged cache is split, its partials in the workspace and
// the launch that joins them.
//
// The lengths are on the device, so every workgroup works the split out for
// itself; w is the number of 128-key blocks over all tiles of rows of a KV head.
//  * Prompts (tiles of 8 to 32 tokens): (tile, chunk of keys) items, the chunk
//    from an estimate of the time (paged_chunk) and w / target blocks at least:
//    at most target + tiles items, whatever the mixture of lengths.  The grid is
//    that bound, and workgroups without an item end.
//  * Single and few tokens (tiles of 2): the tiles' blocks in a row are cut into
//    one equal share for each workgroup that the GPU holds, so that all end
//    together; a share may end one tile and begin the next.
// A tile that one workgroup takes whole is written straight to the output.
#pragma once

#include "paged_common.h"

namespace q36 {

constexpr unsigned kSplitBlock = 128;    // keys; chunks are whole blocks
constexpr unsigned kMaxChunks = 256;

struct PagedOut {
  const bf16* gate;       // NULL, or q_gate's row 0
  bf16* out;
  float* ml;              // [slot][KV head][8 * tile tokens][2]: m (log2 domain), l
  float* o;               // [slot][KV head][8 * tile tokens][256]
  unsigned* head;         // [0]: blocks of a chunk or share, [1 + i]: first item or block of sequence i
  size_t gate_stride;
  unsigned slots;         // that the workspace holds; offsets that make more have none for the rest
};

struct PagedSplit {
  unsigned chunk;         // keys of a chunk
  unsigned seq, local;    // the item's sequence and its place there
};

template <unsigned kTile>
__device__ __forceinline__ unsigned paged_tiles(const PagedSeq& s) {
  return (unsigned)(s.z - s.a + (int)kTile - 1) / kTile;
}
__device__ __forceinline__ unsigned paged_blocks(const PagedSeq& s) {
  return ((unsigned)s.len + kSplitBlock - 1) / kSplitBlock;
}

// Over a KV head: blocks of all tiles, the tiles, the longest sequence's blocks (all
// threads call it; lds holds 52 words).
template <unsigned kTile>
__device__ __forceinline__ void paged_total(const PagedBatch& b, unsigned* lds, unsigned& w, unsigned& tiles,
                                            unsigned& longest) {
  const unsigned tid = threadIdx.x, n = blockDim.x, wave = tid >> 6, waves = n >> 6;
  if (b.seqs == 1) {
    const PagedSeq s = paged_seq(b, 0);
    longest = paged_blocks(s);
    tiles = paged_tiles<kTile>(s);
    w = tiles * longest;
    return;
  }
  w = tiles = longest = 0;
  for (unsigned i = tid; i < b.seqs; i += n) {
    const PagedSeq s = paged_seq(b, i);
    const unsigned t = paged_tiles<kTile>(s), l = t ? paged_blocks(s) : 0u;
    w += t * l;
    tiles += t;
    longest = max(longest, l);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    w += __shfl_xor(w, o, 64);
    tiles += __shfl_xor(tiles, o, 64);
    longest = max(longest, (unsigned)__shfl_xor(longest, o, 64));
  }
  if ((tid & 63) == 0) {
    lds[20 + wave] = w;
    lds[30 + wave] = longest;
    lds[40 + wave] = tiles;
  }
  __syncthreads();
  w = tiles = 0;
  for (unsigned i = 0; i < waves; ++i) {
    w += lds[20 + i];
    longest = max(longest, lds[30 + i]);
    tiles += lds[40 + i];
  }
  w = __builtin_amdgcn_readfirstlane(w);
  tiles = __builtin_amdgcn_readfirstlane(tiles);
  longest = __builtin_amdgcn_readfirstlane(longest);
}

// Blocks of a chunk: of 1 to 64 chunks for the longest sequence the number whose
// rounds of workgroups (`slots` of a KV head at once) end first, a lane for each,
// as if all sequences had the mean length.  A workgroup costs about one and a half
// blocks before its first product and after its last, a partial 1/100 in the join.
__device__ __forceinline__ unsigned paged_chunk(unsigned w, unsigned tiles, unsigned longest, unsigned slots,
                                                unsigned target) {
  const unsigned n = (threadIdx.x & 63) + 1;
  const float mean = tiles ? (float)w / (float)tiles : 0.f;
  const unsigned least = max((longest + kMaxChunks - 1) / kMaxChunks, (w + target - 1) / target);
  unsigned cb = max((unsigned)ceilf((float)longest / (float)n), max(least, 1u));
  const float items = (float)tiles * ceilf(mean / (float)cb);
  float cost = ceilf(items / (float)slots) * ((float)cb + 1.5f) + (n == 1 ? 0.f : 0.01f * items);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {   // the cheapest, of equals the fewest chunks
    const float c = __shfl_xor(cost, o, 64);
    const unsigned u = __shfl_xor(cb, o, 64);
    if (c < cost || (c == cost && u > cb)) cost = c, cb = u;
  }
  return __builtin_amdgcn_readfirstlane(cb);
}

// The item of this workgroup (all threads call it; lds holds 52 words); false
// if there is none.  Item 0 also writes the split down for the joining launch.
template <unsigned kTile>
__device__ __forceinline__ bool paged_split(const PagedBatch& b, unsigned item, unsigned slots, unsigned target,
                                            unsigned* head, unsigned* lds, PagedSplit& r) {
  unsigned w, tiles, longest;
  paged_total<kTile>(b, lds, w, tiles, longest);
  const unsigned cb = paged_chunk(w, tiles, longest, slots, target);
  r.chunk = cb * kSplitBlock;
  if (head != nullptr && threadIdx.x == 0) {
    head[0] = cb;
    if (b.seqs == 1) head[1] = 0;
  }
  return paged_find_item(b, item, lds, [&](unsigned i) {
    const PagedSeq s = paged_seq(b, i);
    return paged_tiles<kTile>(s) * ((paged_blocks(s) + cb - 1) / cb);
  }, r.seq, r.local, head != nullptr ? head + 1 : nullptr);
}

// Items of a KV head at most, for the grid and the workspace: the tiles and `target`
// more, and no more chunks of a tile than the page table has blocks of keys (17 rows
// over a page of 128: 0.5 MB of partials, not 136).
inline unsigned paged_items(const PagedBatch& b, unsigned tile, unsigned target) {
  const unsigned t = b.tokens / tile + b.seqs, tiles = t < b.tokens ? t : b.tokens;
  const size_t whole = (size_t)tiles * ((b.max_len + kSplitBlock - 1) / kSplitBlock);
  return whole < tiles + target ? (unsigned)whole : tiles + target;
}

// o * sigmoid(g) within a few fp32 ulps (rounded to bf16 by the caller): e^-g from
// the hardware exp2 with log2(e) split, as gate4_bf16_fast has it, but without its
// exact form next to a rounding border: the product is rounded once, so there is no
// sigmoid in bf16 to agree on.  Gates past 60 count as 60, where the sigmoid is 1; one
// below 2^-126 (gates under -87) may count as 0.  With expf and a division the epilogue
// of a 32-token tile took 13 us.
__device__ __forceinline__ float paged_gate(float o, bf16 gate) {
  float g = bf2f(gate);
  g = g > 60.f ? 60.f : g;
  const float th = __builtin_amdgcn_exp2f(g * -kLog2eHi);
  const float t = __builtin_fmaf(th, g * -kLn2Lo, th);
  return o * __builtin_amdgcn_rcpf(1.0f + t);
}

inline size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
inline size_t split_ws_bytes(unsigned seqs, size_t slots, unsigned heads, unsigned rows) {
  return round256(((size_t)seqs + 1) * 4) + round256(slots * heads * rows * 8) +
         slots * heads * rows * kD * 4;
}
inline void split_ws(void* ws, unsigned seqs, size_t slots, unsigned heads, unsigned rows, PagedOut& o) {
  char* p = static_cast<char*>(ws);
  o.slots = (unsigned)slots;
  o.head = reinterpret_cast<unsigned*>(p);
  p += round256(((size_t)seqs + 1) * 4);
  o.ml = reinterpret_cast<float*>(p);
  p += round256(slots * heads * rows * 8);
  o.o = reinterpret_cast<float*>(p);
}

// Joins the partials of tiles of `tile` tokens; listed_chunks != 0: every row
// has that many slots.  Rows of one chunk are already written.
int paged_combine(const PagedBatch& b, const PagedCache& c, const PagedOut& o, unsigned tile,
                  unsigned listed_chunks, void* stream);
// Tiles of 8, 16 or 32 tokens (paged_prefill.hip).
int paged_prefill(const void* q, const PagedCache& c, bool fp8, const PagedBatch& b, const PagedOut& o,
                  unsigned tile, unsigned items, unsigned slots, unsigned target, void* stream);

}  // namespace q36
