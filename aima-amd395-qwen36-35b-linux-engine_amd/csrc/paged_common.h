// What the paged-cache kernels share: the cache and batch as the entry points
// take them, where a sequence's tokens stand, and how work items are found.
//
// A page holds page_tokens (16, 32, 64 or 128) tokens of every KV head,
// [KV head][token][256], in bf16 or in e4m3 with a power-of-two scale for each
// KV head of K and of V, kept as the byte e of 2^(e - 127).  A power of two
// costs e4m3 nothing (its relative step does not depend on the scale), makes
// e4m3 -> bf16 exact with the scale inside the conversion instruction, and lets
// a page's scale grow with at most the lowest bits of its subnormals lost.
//
// Device-side numbers (lengths, offsets, page ids) are not trusted: a sequence
// longer than its page table has no tokens, offsets are cut to the call's rows,
// and a page id outside the pool holds no tokens.
#pragma once

#include "common.h"
#include "../../include/qwen36_attn.h"

namespace q36 {

constexpr unsigned kScaleMin = 16;       // least scale byte: 2^-111
constexpr float kE4m3Max = 448.f;

struct PagedCache {
  char* k;
  char* v;
  uint8_t* k_exp;
  uint8_t* v_exp;
  int8_t* bounds;
  size_t k_stride, v_stride;   // bytes between pages
  unsigned pages, shift, heads;
};

struct PagedBatch {
  const int* table;
  const int* cu;
  const int* lens;
  size_t table_stride;
  unsigned seqs, tokens, width, max_len;
};

// A sequence of the batch: its rows [a, z) of the call and its length; row t is
// at position len - (z - t), and a row of negative position sees nothing.
struct PagedSeq {
  int a, z, len;
  __device__ __forceinline__ int pos(int t) const { return len - (z - t); }
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, unsigned i) {
  PagedSeq s;
  s.a = min(max(b.cu[i], 0), (int)b.tokens);
  s.z = min(max(b.cu[i + 1], s.a), (int)b.tokens);
  const int len = b.lens[i];
  s.len = len > 0 && len <= (int)b.max_len ? len : 0;
  return s;
}

// The sequence that holds row t, and where it stands; false where none does.
// By one wave: up to 64 sequences are looked at in one round of loads, more by a
// search with a load per 64 and a second round.
__device__ __forceinline__ bool paged_find_row(const PagedBatch& b, int t, unsigned& seq, PagedSeq& s) {
  if (b.seqs == 1) {
    seq = 0;
    s = paged_seq(b, 0);
    return t >= s.a && t < s.z;
  }
  if (b.seqs <= 64) {
    const unsigned i = min(threadIdx.x & 63, b.seqs - 1);
    const PagedSeq mine = paged_seq(b, i);
    const unsigned long long in = __ballot(t >= mine.a && t < mine.z);
    if (in == 0) return false;
    seq = __ffsll(in) - 1;
    s.a = __builtin_amdgcn_readlane(mine.a, seq);
    s.z = __builtin_amdgcn_readlane(mine.z, seq);
    s.len = __builtin_amdgcn_readlane(mine.len, seq);
    return true;
  }
  const unsigned lane = threadIdx.x & 63;
  unsigned n = 0;
  for (unsigned i0 = 0; i0 < b.seqs; i0 += 64) {
    const unsigned i = i0 + lane;
    const unsigned long long done = __ballot(i < b.seqs && b.cu[i + 1] <= t);
    n += __popcll(done);
    if (done != ~0ull) break;
  }
  seq = __builtin_amdgcn_readfirstlane(n);
  if (seq >= b.seqs) return false;
  s = paged_seq(b, seq);
  return t >= s.a && t < s.z;
}

__device__ __forceinline__ unsigned wave_scan_add(unsigned v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// Finds among the sequences' item counts the sequence that `item` falls into
// and its place there; false where there are fewer items.  All threads of the
// workgroup call it; `lds` holds 20 words.  `firsts`: NULL, or where every
// sequence's first item is written down.
template <class Count>
__device__ __forceinline__ bool paged_find_item(const PagedBatch& b, unsigned item, unsigned* lds,
                                                Count count, unsigned& seq, unsigned& local,
                                                unsigned* firsts = nullptr) {
  if (b.seqs == 1) {
    seq = 0;
    local = item;
    return item < count(0u);
  }
  const unsigned tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = blockDim.x;
  const unsigned waves = n >> 6;
  unsigned base = 0;
  bool found = false;
  for (unsigned i0 = 0; i0 < b.seqs; i0 += n) {
    const unsigned i = i0 + tid;
    const unsigned c = i < b.seqs ? count(i) : 0u;
    const unsigned in = wave_scan_add(c);
    if (lane == 63) lds[wave] = in;
    if (tid == 0) lds[16] = ~0u;
    __syncthreads();
    unsigned before = base, total = 0;
    for (unsigned w = 0; w < waves; ++w) {
      const unsigned s = lds[w];
      if (w < wave) before += s;
      total += s;
    }
    const unsigned lo = before + in - c;
    if (firsts != nullptr && i < b.seqs) firsts[i] = lo;
    if (item >= lo && item < lo + c) {
      lds[16] = i;
      lds[17] = item - lo;
    }
    __syncthreads();
    if (lds[16] != ~0u) {
      seq = __builtin_amdgcn_readfirstlane(lds[16]);
      local = __builtin_amdgcn_readfirstlane(lds[17]);
      found = true;
    }
    __syncthreads();
    if (found && firsts == nullptr) return true;
    base += total;
  }
  return found;
}

// Least byte e with amax <= 448 * 2^(e - 127), for finite amax >= 0.
__device__ __forceinline__ unsigned paged_scale_byte(float amax) {
  const unsigned u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);   // 448 = 1.75 * 2^8
  return (unsigned)max(e, (int)kScaleMin);
}
__device__ __forceinline__ float paged_scale(unsigned e) { return __uint_as_float(e << 23); }

// Two e4m3 values (one half of w) as bf16, times a power of two: exact.
template <bool kHi>
__device__ __forceinline__ unsigned cvt2(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHi));
}

// Ones over the bytes (e4m3) or halves (bf16) of u that are not finite.
template <bool kFp8>
__device__ __forceinline__ unsigned not_finite(unsigned u) {
  if constexpr (kFp8)
    return ((((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
  else
    return ((((u & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
}

// Adds to four dims what is not finite in the V rows of keys [lo, hi] from key
// `from` on: a weight above zero times it is itself.
template <bool kFp8>
__device__ __noinline__ f32x4 sum_not_finite(const char* v, size_t stride, const int* table, unsigned pages,
                                             unsigned shift, unsigned head, int lo, int hi, int d) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int key = lo; key <= hi; ++key) {
    const unsigned pid = (unsigned)table[key >> shift];
    if (pid >= pages) continue;
    const size_t at = ((size_t)head << (shift + 8)) + (size_t)(key & ((1 << shift) - 1)) * kD + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kFp8) {
        const unsigned x = *reinterpret_cast<const uint8_t*>(v + pid * stride + at + e);
        if ((x & 0x7fu) == 0x7fu) s[e] += NAN;
      } else {
        const float x = bf2f(*reinterpret_cast<const bf16*>(v + pid * stride + 2 * (at + e)));
        if (!(fabsf(x) < INFINITY)) s[e] += x;
      }
    }
  }
  return s;
}
template <bool kFp8>
__device__ __forceinline__ void add_not_finite(f32x4& o, const PagedCache& c, const int* table, unsigned head,
                                               int lo, int hi, int from, int d) {
  o += sum_not_finite<kFp8>(c.v, c.v_stride, table, c.pages, c.shift, head, max(lo, from), hi, d);
}

// Host side: the entry points' structures, checked.
inline bool paged_cache_of(const qwen36_paged_cache* c, PagedCache& o) {
  if (c == nullptr || c->k_pages == nullptr || c->v_pages == nullptr || c->num_pages == 0 ||
      c->num_pages > 0x7fffffffu || c->kv_heads == 0 || c->kv_heads > 16)
    return false;
  if (c->cache_type != QWEN36_PAGED_BF16 && c->cache_type != QWEN36_PAGED_E4M3) return false;
  const unsigned p = c->page_tokens;
  if (p != 16 && p != 32 && p != 64 && p != 128) return false;
  const size_t elem = c->cache_type == QWEN36_PAGED_E4M3 ? 1 : 2;
  const size_t least = (size_t)c->kv_heads * p * kD;
  if (c->k_page_stride < least || c->v_page_stride < least) return false;
  if ((c->k_page_stride * elem) % 16 || (c->v_page_stride * elem) % 16) return false;
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages) || !aligned16(c->bounds)) return false;
  if (elem == 1 && (c->k_exp == nullptr || c->v_exp == nullptr)) return false;
  if (c->bounds != nullptr && c->k_exp == nullptr) return false;
  o.k = static_cast<char*>(c->k_pages);
  o.v = static_cast<char*>(c->v_pages);
  o.k_exp = static_cast<uint8_t*>(c->k_exp);
  o.v_exp = static_cast<uint8_t*>(c->v_exp);
  o.bounds = static_cast<int8_t*>(c->bounds);
  o.k_stride = c->k_page_stride * elem;
  o.v_stride = c->v_page_stride * elem;
  o.pages = c->num_pages;
  o.shift = p == 16 ? 4 : p == 32 ? 5 : p == 64 ? 6 : 7;
  o.heads = c->kv_heads;
  return true;
}

inline bool paged_batch_of(const qwen36_paged_batch* b, unsigned page_tokens, PagedBatch& o) {
  if (b == nullptr || b->page_table == nullptr || b->cu_tokens == nullptr ||
      b->seq_lens == nullptr || b->seqs == 0 || b->seqs > 65536 || b->tokens == 0 ||
      b->tokens > kMaxTokens || b->table_width == 0 ||
      (size_t)b->table_width * page_tokens > kMaxTokens + 127u || b->table_stride < b->table_width)
    return false;
  o.table = static_cast<const int*>(b->page_table);
  o.cu = static_cast<const int*>(b->cu_tokens);
  o.lens = static_cast<const int*>(b->seq_lens);
  o.table_stride = b->table_stride;
  o.seqs = b->seqs;
  o.tokens = b->tokens;
  o.width = b->table_width;
  o.max_len = b->table_width * page_tokens;
  if (o.max_len > kMaxTokens) o.max_len = kMaxTokens;
  return true;
}

}  // namespace q36
