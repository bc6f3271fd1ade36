// How attention over the paged cache is split, its partials in the workspace and
// the launch that joins them.
//
// The lengths are on the device, so every workgroup works the split out for
// itself; w is the number of 128-key blocks over all tiles of rows of a KV head.
//  * Prompts (tiles of 8 to 32 tokens): (tile, chunk of keys) items, chunks of
//    max(1, w / target, longest / 256) blocks: at most target + tiles items,
//    whatever the mixture of lengths.  The grid is that bound, and workgroups
//    without an item end.
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

// Blocks of all tiles of a KV head, and of the longest sequence with a tile (all
// threads call it; lds holds 40 words).
template <unsigned kTile>
__device__ __forceinline__ void paged_total(const PagedBatch& b, unsigned* lds, unsigned& w, unsigned& longest) {
  if (b.seqs == 1) {
    const PagedSeq s = paged_seq(b, 0);
    longest = paged_blocks(s);
    w = paged_tiles<kTile>(s) * longest;
    return;
  }
  const unsigned tid = threadIdx.x, n = blockDim.x, wave = tid >> 6, waves = n >> 6;
  w = longest = 0;
  for (unsigned i = tid; i < b.seqs; i += n) {
    const PagedSeq s = paged_seq(b, i);
    const unsigned t = paged_tiles<kTile>(s), l = t ? paged_blocks(s) : 0u;
    w += t * l;
    longest = max(longest, l);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    w += __shfl_xor(w, o, 64);
    longest = max(longest, (unsigned)__shfl_xor(longest, o, 64));
  }
  if ((tid & 63) == 0) {
    lds[20 + wave] = w;
    lds[30 + wave] = longest;
  }
  __syncthreads();
  w = 0;
  for (unsigned i = 0; i < waves; ++i) {
    w += lds[20 + i];
    longest = max(longest, lds[30 + i]);
  }
  w = __builtin_amdgcn_readfirstlane(w);
  longest = __builtin_amdgcn_readfirstlane(longest);
}

// The item of this workgroup (all threads call it; lds holds 40 words); false
// if there is none.  Item 0 also writes the split down for the joining launch.
template <unsigned kTile>
__device__ __forceinline__ bool paged_split(const PagedBatch& b, unsigned item, unsigned target,
                                            unsigned* head, unsigned* lds, PagedSplit& r) {
  unsigned w, longest;
  paged_total<kTile>(b, lds, w, longest);
  const unsigned cb = max(1u, max((w + target - 1) / target, (longest + kMaxChunks - 1) / kMaxChunks));
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

// Items of a KV head at most, for the grid and the workspace.
inline unsigned paged_items(const PagedBatch& b, unsigned tile, unsigned target) {
  const unsigned t = b.tokens / tile + b.seqs;
  return (t < b.tokens ? t : b.tokens) + target;
}

__device__ __forceinline__ float paged_gate(float o, bf16 g) {
  return o * (1.0f / (1.0f + expf(-bf2f(g))));
}

inline size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
inline size_t split_ws_bytes(unsigned seqs, size_t slots, unsigned heads, unsigned rows) {
  return round256(((size_t)seqs + 1) * 4) + round256(slots * heads * rows * 8) +
         slots * heads * rows * kD * 4;
}
inline void split_ws(void* ws, unsigned seqs, size_t slots, unsigned heads, unsigned rows, PagedOut& o) {
  char* p = static_cast<char*>(ws);
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
                  unsigned tile, unsigned items, unsigned target, void* stream);

}  // namespace q36
