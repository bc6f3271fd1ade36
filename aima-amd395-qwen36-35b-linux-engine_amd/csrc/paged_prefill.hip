// Attention over the paged cache for many rows per sequence (prompts, chunks of
// prompts, many drafted tokens).
//
//   o = softmax(q k^T / 16) v over the positions up to the row's own.
//
// Work: an item is a tile of 8, 16 or 32 tokens x the 8 query heads of a KV head
// (32 matrix columns a wave) and a chunk of keys; bound by the matrix products
// (16,384 operations a (row's token, key) pair and KV head) and by LDS, which
// every wave reads whole.  8 tokens over e4m3 take four waves, two for each half of
// a stage's keys, joined at the end: 5 tokens of each of 16 sequences over 12K, two
// KV heads, 72 us with two waves, 65 with four.  Stages of 32 KB (64 keys of e4m3, 32 of bf16):
//  * K and V rows go from their pages straight to LDS in the pages' type (no
//    registers), a stage ahead of their use.  The 16-byte chunks of a row are
//    exchanged by its number on the way, which leaves the
//    row-wise K reads and the transposed V reads free of bank conflicts.
//  * per 32 keys: S^T = K Q^T, online softmax in fp32, O^T += V^T P^T.  A = K rows;
//    B = Q^T in registers; A = V^T by transposed LDS reads; B = P^T, the S^T
//    accumulator as it is.  bf16: 32x32x16 products throughout.  e4m3: K is taken as
//    it lies, by 32x32x64 products with the page's scale byte in the instruction,
//    against Q as the sum of two e4m3 values (as much matrix time as bf16, no
//    conversions); V becomes bf16 behind LDS, the scale inside the conversion.
//    2,048 tokens over 30K: with K converted too 6% more than with the parts, and
//    those 884 us, with the reads and products of e4m3 in a stated order 855; the
//    parts make a tile's prologue 1 us longer (93 tokens over 2K: 37.4 and 38.7).
// The reference maximum is the first visible tile's and is raised (with a
// rescale) only when a tile's probabilities sum past 2^20.
#include "paged_split.h"

#include <atomic>

namespace q36 {
namespace {

constexpr int kKeys = 32;
constexpr int kHalf = 16384, kStage = 2 * kHalf;   // K, V of a stage
constexpr int kLds = 2 * kStage;

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) void global_void;
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

// The exchange of a row's 16-byte chunks: chunk c of row r lies at c ^ swap(r).
// Rows 0-15 take 16 different places for one chunk (K reads, V of e4m3), rows
// r .. r + 3 disjoint ones for four chunks (V of bf16).
__device__ __forceinline__ int swap(int row) { return (row & 3) << 2 | ((row >> 2) & 3); }

constexpr float kScoreScale = 0.0625f * kLog2e;

// The compiler lets a transposed read wait for all loads to LDS under way, the next
// stage's among them, but not one whose memory is marked as its own.  (The barrier of
// a stage is what orders them.)  Two waves, which wait for memory most, gain by the
// mark: 5 tokens of each of 16 sequences 60.5 us, so 58.4; eight lose: 2,048 bf16 918, so 926.
__device__ __forceinline__ i16x4 tr16_own(lds_i16x4* __restrict__ at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
}
template <bool kOwn>
__device__ __forceinline__ i16x4 tr16(unsigned at) {
  lds_i16x4* p = (lds_i16x4*)(uintptr_t)at;
  if constexpr (kOwn)
    return tr16_own(p);
  else
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
}

// 32 bf16 values (and the 32 of lane ^ 32: one scale) as e4m3 sums
// v = 2^(e - 127) (a + 2^-kSplitDown b): a to nearest, b the rest, which has at most the
// 4 bits that a leaves of 8 and is at most half a step of a's, 16 of 448 (so 2^4 times
// it is in range).  What is not finite is a NaN.  Returns e.  The conversions divide by
// the scale that they are given.
constexpr unsigned kSplitDown = 4;
__device__ __forceinline__ unsigned split_e4m3(const u32x4 (&v)[4], i32x8& a, i32x8& b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  u16x2 top = {0, 0};   // magnitudes as bits; those past 0x7f7f are not finite
#pragma unroll
  for (int j = 0; j < 16; ++j)
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[j >> 2][j & 3] & 0x7fff7fffu));
  unsigned amax = max((unsigned)top[0], (unsigned)top[1]);
  amax = max(amax, (unsigned)__shfl_xor(amax, 32, 64));
  const bool strange = amax >= 0x7f80u;
  if (__any(strange)) {   // the largest finite one, the slow way
    amax = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const unsigned m = (v[j >> 3][(j >> 1) & 3] >> (16 * (j & 1))) & 0x7fffu;
      amax = max(amax, m < 0x7f80u ? m : 0u);
    }
    amax = max(amax, (unsigned)__shfl_xor(amax, 32, 64));
  }
  const unsigned e = paged_scale_byte(__uint_as_float(amax << 16));
  const float s1 = paged_scale(e), s2 = paged_scale(e - kSplitDown);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const unsigned lo = v[w >> 1][2 * (w & 1)], hi = v[w >> 1][2 * (w & 1) + 1];
    const float x0 = __uint_as_float(lo << 16), x1 = __uint_as_float(lo & 0xffff0000u);
    const float x2 = __uint_as_float(hi << 16), x3 = __uint_as_float(hi & 0xffff0000u);
    s16x2 p = {0, 0}, r = {0, 0};
    p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, x0, x1, s1, false);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, x2, x3, s1, true);
    const unsigned pw = __builtin_bit_cast(unsigned, p);
    const f32x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(pw, s1, false);
    const f32x2 a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(pw, s1, true);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, x0 - a0[0], x1 - a0[1], s2, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, x2 - a1[0], x3 - a1[1], s2, true);
    a[w] = (int)pw;
    b[w] = __builtin_bit_cast(int, r);
  }
  if (__any(strange)) {
#pragma unroll
    for (int w = 0; w < 8; ++w) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned m = (v[w >> 1][2 * (w & 1) + (j >> 1)] >> (16 * (j & 1))) & 0x7fffu;
        if (m >= 0x7f80u) a[w] |= 0x7f << (8 * j);
      }
    }
  }
  return e;
}

template <bool kFp8, int kWaves, int kParts>
__global__ __launch_bounds__(64 * kWaves, kWaves == 4 ? 2 : 1) void paged_prefill_kernel(
    const bf16* __restrict__ q, PagedCache c, PagedBatch b, PagedOut w, unsigned slots, unsigned target) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  __shared__ unsigned find[52];
  __shared__ float ml[kParts == 2 ? 64 : 1][2];   // maxima and sums of the second half
  __shared__ int odd;   // whether a V value that some rows must not see is not finite
  constexpr int kElem = kFp8 ? 1 : 2;
  constexpr int kTile = 4 * kWaves / kParts;
  constexpr int kRowB = kD * kElem, kStageKeys = kHalf / kRowB;   // bytes of a row, keys of a stage
  constexpr int kSubs = kStageKeys / kKeys, kGroups = kStageKeys / 16;
  static_assert(kParts == 1 || (kParts == 2 && kSubs == 2 && kWaves == 4));
  constexpr int kLoads = 16 / kWaves;                // 1 KB loads of K (and of V) a wave and stage
  constexpr int kBlockStages = 1024 / kStageKeys;    // stages of a 1,024-key block

  const unsigned head = blockIdx.x % c.heads, item = blockIdx.x / c.heads;
  const unsigned hq = c.heads * kGroup;
  PagedSplit sp;
  if (!paged_split<kTile>(b, item, slots, target, blockIdx.x == 0 ? w.head : nullptr, find, sp)) return;
  const PagedSeq s = paged_seq(b, sp.seq);
  const unsigned chunks = ((unsigned)s.len + sp.chunk - 1) / sp.chunk;
  const int n_rows = s.z - s.a;
  const int tiles = (n_rows + kTile - 1) / kTile;
  // the last tiles see most keys: they start first
  const int qt = tiles - 1 - (int)(sp.local / chunks);
  const unsigned chunk = sp.local % chunks;
  const int r0 = qt * kTile, n_tok = min(kTile, n_rows - r0);
  const int t0 = s.a + r0, pos0 = s.pos(t0);
  const int end = pos0 + n_tok;                    // keys the tile sees
  const int kv_first = (int)(chunk * sp.chunk);
  if (kv_first >= end) return;
  const int kv_stop = min(kv_first + (int)sp.chunk, end);
  const size_t slot = item - sp.local + (size_t)qt * chunks + chunk;
  const bool single = end <= (int)sp.chunk;
  if (slot >= w.slots) return;   // overlapping sequences: more tiles than rows

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lj = lane & 31, lg = lane >> 5;
  // wave w has rows w % kRowWaves of the tile and the part w / kRowWaves of each stage
  constexpr int kRowWaves = kWaves / kParts;
  const int part = wave / kRowWaves, first = wave % kRowWaves * 4;   // of its four tokens
  const int tok = first + (lj >> 3);               // of the tile
  const bool live = tok < n_tok;
  const int lim = live ? pos0 + tok : -1;          // this column's last key
  const int wave_first = pos0 + first;
  const int wave_lim = first < n_tok ? min(wave_first + 3, end - 1) : -1;

  f32x16 o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = f32x16{};
  float m = lim >= 0 ? -INFINITY : 0.f, l = 0.f;

  // ---- pages of the chunk: lane j holds what the 16 keys j of a 1,024-key block
  // need; the next block's are fetched in two steps while this one's are used.
  const int* table = b.table + sp.seq * b.table_stride;
  unsigned d_page = 0, d_exp = 0, n_page = 0, n_exp = 0;
  bool n_ok = false;
  unsigned long long d_ok = 0;
  const int page_mask = (1 << c.shift) - 1;
  const auto fetch_pages = [&](int key) {
    const int at = key + 16 * lane;
    n_page = at < kv_stop ? (unsigned)table[at >> c.shift] : ~0u;
  };
  const auto fetch_scales = [&]() {
    n_ok = n_page < c.pages;
    if (!n_ok) n_page = 0;
    if constexpr (kFp8) {
      const size_t e = (size_t)n_page * c.heads + head;
      n_exp = (unsigned)c.k_exp[e] | (unsigned)c.v_exp[e] << 8;
    }
  };

  // the first block's before the queries: loads return in order
  fetch_pages(kv_first);
  fetch_scales();
  // Q^T operand.  bf16: k-step i has dims 16 i + 8 lg.  e4m3: the sum of two e4m3
  // values with a scale for each 64 dims (step i: this lane has dims 64 i + 32 lg),
  // which holds a bf16 value exactly unless it is 2^-14 of the 64's largest or less
  // (then to 2^-22 of that).
  bf16x8 qf[kFp8 ? 1 : 16];
  i32x8 q1[kFp8 ? 4 : 1], q2[kFp8 ? 4 : 1];
  unsigned qs1 = 0, qs2 = 0;   // scale bytes of the 4 steps
  {
    const bf16* qp = q + ((size_t)(t0 + tok) * hq + head * kGroup + (lj & 7)) * kD + (kFp8 ? 32 : 8) * lg;
    if constexpr (kFp8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = lim >= 0 ? *reinterpret_cast<const u32x4*>(qp + 64 * i + 8 * j) : u32x4{};
        const unsigned e = split_e4m3(v, q1[i], q2[i]);
        qs1 |= e << (8 * i);
        qs2 |= (e - kSplitDown) << (8 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        qf[i] = lim >= 0 ? *reinterpret_cast<const bf16x8*>(qp + 16 * i) : bf16x8{};
    }
  }
  // ---- a stage's rows, 4 (e4m3) or 2 (bf16) a load: one page each
  unsigned ok = 0, ok_next = 0;            // bit g: the 16 keys g of the stage have a page
  unsigned e0 = 0, e1 = 0, e2 = 0, e3 = 0;  // scale bytes of the loaded stage's 16-key groups (K, V << 8)
  const size_t head_off = ((size_t)head << (c.shift + 8)) * kElem;
  const auto load_stage = [&](int i) {
    const int at = i % kBlockStages;
    if (at == 0) {
      d_page = n_page;
      d_exp = n_exp;
      d_ok = __ballot(n_ok);
    } else if (at == kBlockStages / 4) {
      fetch_pages(kv_first + (i - at + kBlockStages) * kStageKeys);
    } else if (at == kBlockStages * 5 / 8) {
      fetch_scales();
    }
    ok_next = (unsigned)(d_ok >> (kGroups * at)) & ((1u << kGroups) - 1);
    if constexpr (kFp8) {
      e0 = __builtin_amdgcn_readlane(d_exp, 4 * at);
      e1 = __builtin_amdgcn_readlane(d_exp, 4 * at + 1);
      e2 = __builtin_amdgcn_readlane(d_exp, 4 * at + 2);
      e3 = __builtin_amdgcn_readlane(d_exp, 4 * at + 3);
    }
    char* to = lds + (i & 1) * kStage;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int row0 = (j * kWaves + wave) * (1024 / kRowB);            // uniform
      const int row = row0 + lane / (kRowB / 16);
      const unsigned pid = __builtin_amdgcn_readlane(d_page, kGroups * at + (row0 >> 4));
      const int prow = (kv_first + i * kStageKeys + row0) & page_mask;
      const unsigned off = (row - row0) * kRowB + (((lane & (kRowB / 16 - 1)) ^ swap(row)) << 4);
      const char* kp = c.k + pid * c.k_stride + head_off + (size_t)prow * kRowB;
      const char* vp = c.v + pid * c.v_stride + head_off + (size_t)prow * kRowB;
      __builtin_amdgcn_global_load_lds((global_void*)(kp + off), (lds_void*)(to + row0 * kRowB), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((global_void*)(vp + off), (lds_void*)(to + kHalf + row0 * kRowB), 16, 0, 0);
    }
  };
  // Behind the tile's first position V may hold anything, and 0 * NaN is NaN: rows
  // that no token sees are cleared, and of the others what is not finite (the
  // tokens that do see it get it at the end).
  const auto clean_stage = [&](int i) {
    bool strange = false;
    for (int x = tid; x < kHalf / 16; x += 64 * kWaves) {
      const int row = x / (kRowB / 16), key = kv_first + i * kStageKeys + row;
      u32x4* p = reinterpret_cast<u32x4*>(lds + (i & 1) * kStage + kHalf) + x;
      const bool out = key >= kv_stop || !((ok >> (row >> 4)) & 1u), some = key > pos0;
      if (!out && !some) continue;
      u32x4 v = *p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned u = out ? 0u : v[e], bad = some ? not_finite<kFp8>(u) : 0u;
        v[e] = u & ~bad;
        strange |= bad != 0;
      }
      *p = v;
    }
    if (strange) odd = 1;
  };

  // per-lane LDS addresses; k-steps and dim tiles flip bits of the chunk number
  const unsigned lds0 = (unsigned)(uintptr_t)(lds_void*)lds;
  const unsigned kbase = lds0 + lj * kRowB + (((kFp8 ? 2 * lg : lg) ^ swap(lj)) << 4);
  const int grp = lane >> 4, m16 = lane & 15;
  const int vrow = kFp8 ? 8 * (m16 >> 3) + 4 * lg + ((m16 >> 1) & 3) : 4 * lg + (m16 >> 2);
  const int vchunk = kFp8 ? grp & 1 : 2 * (grp & 1) + ((m16 >> 1) & 1);
  const unsigned vbase = lds0 + kHalf + vrow * kRowB + ((vchunk ^ swap(vrow)) << 4) + 8 * (m16 & 1);

  const int n_stages = (kv_stop - kv_first + kStageKeys - 1) / kStageKeys;
  if (tid == 0) odd = 0;
  load_stage(0);
  for (int st = 0; st < n_stages; ++st) {
    ok = ok_next;
    const unsigned f0 = e0, f1 = e1, f2 = e2, f3 = e3;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();   // stage st is in LDS, stage st - 1 is used up
    const int key_st = kv_first + st * kStageKeys;
    if (key_st + kStageKeys - 1 > pos0 || ok != (1u << kGroups) - 1) {
      clean_stage(st);
      __syncthreads();
    }
    if (st + 1 < n_stages) load_stage(st + 1);
#pragma unroll 1
    for (int sub = part; sub < kSubs; sub += kParts) {
    const int kv0 = key_st + sub * kKeys;
    if (kv0 > wave_lim) continue;
    // (whole rows away: the exchanged bits stay as they are)
    const unsigned kp = kbase + (st & 1) * kStage + sub * kKeys * kRowB;
    const unsigned vp = vbase + (st & 1) * kStage + sub * kKeys * kRowB;
    const unsigned okh = ok >> (2 * sub), ea = sub ? f2 : f0, eb = sub ? f3 : f1;
    f32x16 x = f32x16{};
    // the wave with products to issue goes before the one in its softmax (2,048
    // tokens over 30K: 970 us without, 944 with)
    __builtin_amdgcn_s_setprio(1);
    if constexpr (kFp8) {
      // the page's scale byte of this lane's key goes into the product as it is
      const int ks = (int)((lj < 16 ? ea : eb) & 0xffu);
      i32x8 kr[2];
      const auto kread = [&](int i) {   // dims 64 i + 32 lg .. + 32
        const u32x4 lo = *(const lds_u32x4*)(uintptr_t)(kp ^ (i << 6)), hi = *(const lds_u32x4*)(uintptr_t)(kp ^ (i << 6) ^ 16);
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
      };
      kr[0] = kread(0);
      kr[1] = kread(1);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[0], q1[0], x, 0, 0, 0, ks, 0, (int)qs1);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[0], q2[0], x, 0, 0, 0, ks, 0, (int)qs2);
      kr[0] = kread(2);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[1], q1[1], x, 0, 0, 0, ks, 1, (int)qs1);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[1], q2[1], x, 0, 0, 0, ks, 1, (int)qs2);
      kr[1] = kread(3);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[0], q1[2], x, 0, 0, 0, ks, 2, (int)qs1);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[0], q2[2], x, 0, 0, 0, ks, 2, (int)qs2);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[1], q1[3], x, 0, 0, 0, ks, 3, (int)qs1);
      x = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kr[1], q2[3], x, 0, 0, 0, ks, 3, (int)qs2);
      // two steps of K ahead: left alone, each step's reads are issued and waited for
      // right before its products
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    } else {
      bf16x8 kr[4];
      const auto kread = [&](int i) { return __builtin_bit_cast(bf16x8, *(const lds_u32x4*)(uintptr_t)(kp ^ (i << 5))); };
#pragma unroll
      for (int i = 0; i < 4; ++i) kr[i] = kread(i);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x = mfma32x32x16(kr[i & 3], qf[i], x);
        if (i + 4 < 16) kr[i & 3] = kread(i + 4);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < 12; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    }
    __builtin_amdgcn_s_setprio(0);
    // lane: keys kv0 + 8 (r / 4) + 4 lg + r % 4 of its column
    const bool diag = kv0 + kKeys - 1 > wave_first;
    if (diag || (okh & 3u) != 3u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kv0 + 8 * (r >> 2) + 4 * lg + (r & 3);
        x[r] = key <= lim && ((okh >> (r >> 3)) & 1u) ? x[r] : -INFINITY;
      }
    }
    const auto col_max = [&]() {
      float mx = x[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
      return wave_max_xor(mx, 32) * kScoreScale;
    };
    if (__any(m == -INFINITY)) {   // no key seen so far
      const float mx = col_max();
      if (m == -INFINITY) m = mx;
    }
    float base = m == -INFINITY ? 0.f : m;
    float psum = 0.f;
    bf16x8 pb[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], kScoreScale, -base));
      psum += p;
      pb[r >> 3][r & 7] = f2bf(p);
    }
    if (__any(!(psum <= 1048576.0f))) {
      const float mx = fmaxf(m, col_max());
      const float a = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mx);
      l *= a;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] *= a;
      m = mx;
      base = m == -INFINITY ? 0.f : m;
      psum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], kScoreScale, -base));
        psum += p;
        pb[r >> 3][r & 7] = f2bf(p);
      }
    }
    l += psum;
    __builtin_amdgcn_s_setprio(1);

    if constexpr (kFp8) {
      // four V operands on their way, in this order (chunk of 2,048: 855 us; left to the
      // compiler 884, six in groups of sched_group_barrier 861)
      constexpr int kRing = 4;
      i32x2 va[kRing];
      const auto vread = [&](int i) {   // keys 16 (i / 8) .. + 16, dims 32 (i % 8) .. + 32
        return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_i32x2*)(uintptr_t)((vp ^ ((i & 7) << 5)) + (i >> 3) * 16 * kRowB));
      };
#pragma unroll
      for (int i = 0; i < kRing; ++i) va[i] = vread(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float vs = paged_scale((i < 8 ? ea : eb) >> 8);
        const i32x2 r = va[i % kRing];
        const u32x4 a = {cvt2<false>((unsigned)r[0], vs), cvt2<true>((unsigned)r[0], vs),
                         cvt2<false>((unsigned)r[1], vs), cvt2<true>((unsigned)r[1], vs)};
        o[i & 7] = mfma32x32x16(__builtin_bit_cast(bf16x8, a), pb[i >> 3], o[i & 7]);
        if (i + kRing < 16) va[i % kRing] = vread(i + kRing);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      i16x4 va[4][2];
      const auto vread = [&](int i, int to) {
        const unsigned at = vp ^ ((i & 7) << 6);
        va[to][0] = tr16<kWaves == 2>(at + (i >> 3) * 16 * kRowB);
        va[to][1] = tr16<kWaves == 2>((at ^ 32) + ((i >> 3) * 16 + 8) * kRowB);   // keys + 8: swap(8) is 2
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) vread(i, i);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[i & 7] = mfma32x32x16(cat_bf16x8(va[i & 3][0], va[i & 3][1]), pb[i >> 3], o[i & 7]);
        if (i + 4 < 16) vread(i + 4, i & 3);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
      for (int i = 0; i < 12; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 1);
    }
    __builtin_amdgcn_s_setprio(0);
    }
  }

  l += __shfl_xor(l, 32, 64);
  if constexpr (kParts == 2) {   // join the two halves of the keys
    __syncthreads();
    f32x4* ex = reinterpret_cast<f32x4*>(lds + wave % kRowWaves * 32768) + lane;
    if (part == 1) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        ex[i * 64] = f32x4{o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2],
                           o[i >> 2][4 * (i & 3) + 3]};
      if (lg == 0) {
        ml[wave % kRowWaves * 32 + lj][0] = l == 0.f ? -INFINITY : m;
        ml[wave % kRowWaves * 32 + lj][1] = l;
      }
    }
    __syncthreads();
    if (part == 0) {
      const float m1 = ml[wave * 32 + lj][0], l1 = ml[wave * 32 + lj][1];
      const float mx = fmaxf(l == 0.f ? -INFINITY : m, m1);
      const float a0 = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - mx);
      const float a1 = l1 == 0.f ? 0.f : __builtin_amdgcn_exp2f(m1 - mx);
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const f32x4 v = ex[i * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = o[i >> 2][4 * (i & 3) + e];
          o[i >> 2][4 * (i & 3) + e] = (l == 0.f ? 0.f : u * a0) + (l1 == 0.f ? 0.f : v[e] * a1);
        }
      }
      m = mx;
      l = l * a0 + l1 * a1;
    }
  }

  // ---- out through LDS in four rounds of 64 dims, so that stores are whole
  // 256-byte (fp32 partials) or 128-byte row segments
  const float inv = single ? (l == 0.f ? 0.f : 1.0f / l) : 1.0f;
  const size_t part0 = (slot * c.heads + head) * (8 * kTile);
  if (!single && lg == 0 && live && part == 0) {
    const size_t at = part0 + first * 8 + lj;
    w.ml[at * 2] = l == 0.f ? -INFINITY : m;   // what saw nothing weighs nothing
    w.ml[at * 2 + 1] = l;
  }
  const bool zero = l == 0.f;
  // bit j: column j saw nothing and is zeros whatever its gate (an attention of exactly
  // zero is not: its product with a NaN gate is a NaN)
  const unsigned none = (unsigned)__ballot(zero);
  // the gates of this wave's rows, all asked for at once (rows past the end read the
  // last row's)
  bf16x4 gt[4][8];
  if (single && w.gate != nullptr && part == 0) {
#pragma unroll
    for (int rd = 0; rd < 4; ++rd)
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int r = it * 4 + (lane >> 4);
        const size_t row = t0 + min(first + (r >> 3), n_tok - 1);
        gt[rd][it] = *reinterpret_cast<const bf16x4*>(w.gate + row * w.gate_stride + (head * kGroup + (r & 7)) * 2 * kD +
                                                      kD + rd * 64 + (lane & 15) * 4);
      }
  }
  __syncthreads();
  if (part != 0) return;
  const bool strange_v = odd != 0;
  char* stg = lds + wave * 8192;
#pragma unroll
  for (int rd = 0; rd < 4; ++rd) {
#pragma unroll
    for (int d2 = 0; d2 < 2; ++d2) {
      const int dt = 2 * rd + d2;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int ch = d2 * 8 + 2 * r4 + lg;
        f32x4 v = {o[dt][4 * r4], o[dt][4 * r4 + 1], o[dt][4 * r4 + 2], o[dt][4 * r4 + 3]};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = zero ? 0.f : v[e] * inv;
        *reinterpret_cast<f32x4*>(stg + lj * 256 + ((ch ^ (lj & 15)) * 16)) = v;
      }
    }
    // one wave's LDS operations are served in order
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int r = it * 4 + (lane >> 4), ch = lane & 15;
      f32x4 v = *reinterpret_cast<const f32x4*>(stg + r * 256 + ((ch ^ (r & 15)) * 16));
      const int rt = first + (r >> 3), d = rd * 64 + ch * 4;
      if (rt >= n_tok) continue;
      if (strange_v) add_not_finite<kFp8>(v, c, table, head, pos0 + 1, min(pos0 + rt, kv_stop - 1), kv_first, d);
      if (!single) {
        *reinterpret_cast<f32x4*>(w.o + (part0 + first * 8 + r) * kD + d) = v;
        continue;
      }
      const size_t row = t0 + rt, qh = head * kGroup + (r & 7);
      bf16x4 res;
      if (w.gate != nullptr) {
        const bool nothing = (none >> r) & 1u;
#pragma unroll
        for (int e = 0; e < 4; ++e) res[e] = f2bf(nothing ? 0.f : paged_gate(v[e], gt[rd][it][e]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) res[e] = f2bf(v[e]);
      }
      *reinterpret_cast<bf16x4*>(w.out + (row * hq + qh) * kD + d) = res;
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  }
}

// More than 64 KB of LDS has to be asked for once on each device.
int allow_lds(const void* kernel, std::atomic<bool> (&ready)[64]) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return Q36_EINVAL;
  if (ready[dev].load(std::memory_order_acquire)) return Q36_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (e == hipSuccess) ready[dev].store(true, std::memory_order_release);
  return static_cast<int>(e);
}

template <bool kFp8, int kWaves, int kParts = 1>
int launch(const bf16* q, const PagedCache& c, const PagedBatch& b, const PagedOut& o, unsigned items,
           unsigned slots, unsigned target, void* stream) {
  static std::atomic<bool> ready[64];
  const int e = allow_lds(reinterpret_cast<const void*>(&paged_prefill_kernel<kFp8, kWaves, kParts>), ready);
  if (e != Q36_OK) return e;
  hipLaunchKernelGGL((paged_prefill_kernel<kFp8, kWaves, kParts>), dim3(items * c.heads), dim3(64 * kWaves), kLds,
                     static_cast<hipStream_t>(stream), q, c, b, o, slots, target);
  return static_cast<int>(hipGetLastError());
}

}  // namespace

int paged_prefill(const void* q, const PagedCache& c, bool fp8, const PagedBatch& b, const PagedOut& o,
                  unsigned tile, unsigned items, unsigned slots, unsigned target, void* stream) {
  const bf16* p = static_cast<const bf16*>(q);
  switch (tile) {
    case 8:
      return fp8 ? launch<true, 4, 2>(p, c, b, o, items, slots, target, stream)
                 : launch<false, 2>(p, c, b, o, items, slots, target, stream);
    case 16:
      return fp8 ? launch<true, 4>(p, c, b, o, items, slots, target, stream)
                 : launch<false, 4>(p, c, b, o, items, slots, target, stream);
    default:
      return fp8 ? launch<true, 8>(p, c, b, o, items, slots, target, stream)
                 : launch<false, 8>(p, c, b, o, items, slots, target, stream);
  }
}

}  // namespace q36
