// A ragged batch whose sequences carry states in slots of a pool, as the entry
// points take it, and how work items over it are found.
//
// Device-side numbers (offsets, slots) are not trusted: offsets are cut to the
// call's rows, and a sequence whose slot lies outside the pool is padding.
#pragma once

#include "common.h"
#include "../../include/qwen36_attn.h"

namespace q36 {

struct RaggedBatch {
  const int* cu;
  const int* slots;
  const uint8_t* has;     // NULL: every sequence has a state
  unsigned seqs, tokens, n_slots;
};

// Rows [a, z) of the call, the slot (-1: padding), and whether the slot holds a state.
struct RaggedSeq {
  int a, z, slot;
  bool has;
};

__device__ __forceinline__ void ragged_rows(const RaggedBatch& b, unsigned i, int& a, int& z) {
  a = min(max(b.cu[i], 0), (int)b.tokens);
  z = min(max(b.cu[i + 1], a), (int)b.tokens);
}

__device__ __forceinline__ RaggedSeq ragged_seq(const RaggedBatch& b, unsigned i) {
  RaggedSeq s;
  ragged_rows(b, i, s.a, s.z);
  const int slot = b.slots[i];
  s.slot = slot >= 0 && (unsigned)slot < b.n_slots ? slot : -1;
  s.has = b.has == nullptr || b.has[i] != 0;
  return s;
}

// Tiles of kTile rows, counted from each sequence's first row.  Tile `local` of
// sequence i is item a_i / kTile + i + local: the items of two sequences never
// meet (a_{i+1} / kTile + 1 >= a_i / kTile + ceil(n_i / kTile) for whole offsets),
// so an item is found without a sum over the sequences before it, and
// tokens / kTile + seqs items hold every tile.  One wave; false where item holds
// no tile.
template <unsigned kTile>
__device__ __forceinline__ bool ragged_find_tile(const RaggedBatch& b, unsigned item, unsigned& seq,
                                                 unsigned& local) {
  const unsigned lane = threadIdx.x & 63;
  unsigned n = 0;   // sequences that begin at or before the item
  if (b.seqs > 1) {
    for (unsigned i0 = 0; i0 < b.seqs; i0 += 64) {
      const unsigned i = i0 + lane;
      const unsigned a = i < b.seqs ? (unsigned)min(max(b.cu[i], 0), (int)b.tokens) : 0u;
      const unsigned long long in = __ballot(i < b.seqs && a / kTile + i <= item);
      n += __popcll(in);
      if (in != ~0ull) break;
    }
    if (n == 0) return false;
    seq = __builtin_amdgcn_readfirstlane(n - 1);
  } else {
    seq = 0;
  }
  int a, z;
  ragged_rows(b, seq, a, z);
  local = item - ((unsigned)a / kTile + seq);
  return local < (unsigned)(z - a + (int)kTile - 1) / kTile;
}

inline bool ragged_batch_of(const qwen36_state_batch* b, RaggedBatch& o) {
  if (b == nullptr || b->cu_tokens == nullptr || b->slots == nullptr || b->seqs == 0 ||
      b->seqs > 65536 || b->tokens == 0 || b->tokens > kMaxTokens || b->num_slots == 0 ||
      b->num_slots > 0x7fffffffu)
    return false;
  o.cu = static_cast<const int*>(b->cu_tokens);
  o.slots = static_cast<const int*>(b->slots);
  o.has = static_cast<const uint8_t*>(b->has_state);
  o.seqs = b->seqs;
  o.tokens = b->tokens;
  o.n_slots = b->num_slots;
  return true;
}

}  // namespace q36
