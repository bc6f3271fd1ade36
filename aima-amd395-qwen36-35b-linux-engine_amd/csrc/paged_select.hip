// Choosing the pages of a sparse attention: a score for each page from its
// keys' bounds, and the pages of the highest scores.
//
//   score(page) = 2^e max_h sum_d max(qi_hd kmax_d, qi_hd kmin_d)
//
// an estimate of the page's largest q.k, in whole numbers: qi and the bounds are
// int8, the sums stay below 2^22, and scores of different pages are compared as
// (integer, exponent), so no sum is rounded, no order of summation shows and ties
// are ties.  (No upper bound: q is rounded to qi, and the bounds are of the keys as
// appended, which e4m3 moves by up to half a step, 16 scales or 4 steps of a bound.)
//
// max(q a, q b) with a >= b is q+ a + q- b for q's positive and negative parts,
// so the score of 16 pages for 8 heads is a chain of 8 int8 matrix products of
// 64 dims.  Bound by the bounds' bytes (512 a page and KV head) and, for few
// rows, by latency: a launch that scores over the whole GPU and one workgroup
// per (row, KV head) that selects, its keys in registers, by halving their
// range.
#include "paged_common.h"

namespace q36 {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Orders (score, exponent) as an unsigned number; pages without keys are below
// all of these (1), pages behind the row's last are 0.
__device__ __forceinline__ unsigned score_key(int s, unsigned e) {
  if (s == 0) return 0x80000000u;
  const unsigned u = __float_as_uint((float)(s < 0 ? -s : s));   // exact: |s| < 2^23
  const unsigned mag = (((u >> 23) + e) << 22) | ((u & 0x7fffffu) >> 1);
  return s < 0 ? 0x7fffffffu - mag : 0x80000000u + mag;
}

// A wave scores 16 pages at a time: pages in the matrix rows, in the columns the 8
// heads of one row (twice) or, with kPair, of rows 2 i and 2 i + 1 where one sequence
// has both; else it takes the two in turn.
template <bool kPair>
__global__ __launch_bounds__(256) void paged_score_kernel(const bf16* __restrict__ q, PagedCache c,
                                                          PagedBatch b, unsigned* __restrict__ keys,
                                                          unsigned blocks, unsigned per_wave) {
  const unsigned head = blockIdx.x % c.heads, block = blockIdx.x / c.heads % blocks;
  const unsigned item = blockIdx.x / c.heads / blocks;
  const int lane = threadIdx.x & 63, col = lane & 7, row = lane & 15, g = lane >> 4;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned p0 = (block * 4 + wave) * per_wave * 16;
  const auto score = [&](unsigned t) {   // returns how many rows it took
    unsigned seq;
    PagedSeq s;
    if (!paged_find_row(b, (int)t, seq, s)) return 1u;
    const bool both = kPair && t % 2 == 0 && (int)t + 1 < s.z;
    const unsigned took = both ? 2 : 1;
    const int pos = s.pos((int)t) + (both ? 1 : 0);   // the last row's
    if (pos < 0) return took;
    const unsigned n = ((unsigned)pos >> c.shift) + 1;
    if (p0 >= n) return took;
    // this lane's column: its row of the call, the pages that it sees
    const unsigned second = both ? lane >> 3 & 1 : 0;
    const int my_pos = pos - (both ? 1 : 0) + (int)second;
    const unsigned my_t = t + second, my_n = my_pos < 0 ? 0 : ((unsigned)my_pos >> c.shift) + 1;

    const int* table = b.table + seq * b.table_stride;
    unsigned* kp = keys + ((size_t)my_t * c.heads + head) * b.width;
    i32x4 a[8];
    unsigned e;
    bool there;
    const auto load = [&](unsigned first) {   // 16 pages' bounds and scales; pages of none read page 0
      const unsigned mine = first + row;
      unsigned pid = mine < n ? (unsigned)table[mine] : ~0u;
      there = pid < c.pages;
      if (!there) pid = 0;
      const int8_t* bp = c.bounds + ((size_t)pid * c.heads + head) * 2 * kD + 16 * g;
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = *reinterpret_cast<const i32x4*>(bp + 64 * j);
      e = c.k_exp[(size_t)pid * c.heads + head];
    };
    load(p0);   // on the way while the queries are quantised

    // this lane's 64 dims of its head: 64 j + 16 g + [0, 16)
    const bf16* qp = q + ((size_t)my_t * c.heads * kGroup + head * kGroup + col) * kD + 16 * g;
    bf16x8 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const bf16x8*>(qp + 64 * (j >> 1) + 8 * (j & 1));
    unsigned amax = 0;   // bits of the largest finite magnitude
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned u = __float_as_uint(bf2f(x[j][e])) & 0x7fffffffu;
        if (u < 0x7f800000u) amax = max(amax, u);
      }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)   // (the columns of 8 .. 15 are another row's, or the same)
      if (o != 8) amax = max(amax, (unsigned)__shfl_xor(amax, o, 64));
    // in steps that put the largest in [64, 128) (and are 2^-127 at least)
    const float f = ldexpf(1.f, min(127 + 6 - (int)(amax >> 23), 127));
    i32x4 qpos[4], qneg[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        unsigned i[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = bf2f(x[2 * j + (w >> 1)][4 * (w & 1) + e]);
          i[e] = (unsigned)(int)(v == v ? __builtin_amdgcn_fmed3f(rintf(v * f), -127.f, 127.f) : 0.f);
        }
        const unsigned lo = __builtin_amdgcn_perm(i[1], i[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(i[3], i[2], 0x04000c0c);
        const unsigned all = lo | hi, sign = ((all >> 7) & 0x01010101u) * 0xffu;
        qpos[j][w] = (int)(all & ~sign);
        qneg[j][w] = (int)(all & sign);
      }

    for (unsigned i = 0; i < per_wave; ++i) {
      const unsigned first = p0 + 16 * i;
      if (first >= n) break;
      i32x4 d = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], qpos[j], d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[4 + j], qneg[j], d, 0, 0, 0);
      }
      const unsigned e_now = e;
      const bool there_now = there;
      if (i + 1 < per_wave && first + 16 < n) load(first + 16);
      // lane: pages 4 g + r of its head; the largest over the heads
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int v = d[r];
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) v = max(v, __shfl_xor(v, o, 64));
        const int from = 4 * g + r;
        const unsigned pe = __shfl(e_now, from, 64);
        const bool ok = __shfl((int)there_now, from, 64);
        if (col == r && (both || row == r) && first + from < my_n) kp[first + from] = ok ? score_key(v, pe) : 1u;
      }
    }
    return took;
  };
  if constexpr (kPair) {
    if (score(2 * item) == 1 && 2 * item + 1 < b.tokens) score(2 * item + 1);
  } else {
    score(item);
  }
}

// One workgroup of kWaves waves per (row, KV head); thread i holds the keys of
// pages [i kPer, + kPer).
template <int kPer, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void paged_pick_kernel(PagedCache c, PagedBatch b,
                                                         const unsigned* __restrict__ keys,
                                                         unsigned budget, unsigned sinks,
                                                         unsigned recents, int* __restrict__ pages,
                                                         unsigned first) {
  __shared__ unsigned cnt[2][kWaves];
  __shared__ unsigned scan[kWaves];
  const unsigned item = first + blockIdx.x, head = item % c.heads, t = item / c.heads, tid = threadIdx.x;
  const unsigned wave = tid >> 6;
  const unsigned* kp = keys + ((size_t)t * c.heads + head) * b.width;
  unsigned k[kPer];   // asked for before the row's length is known: what lies behind it is dropped below
#pragma unroll
  for (int j = 0; j < kPer; ++j) k[j] = kp[min(tid * kPer + j, b.width - 1)];
  unsigned seq;
  PagedSeq s;
  if (!paged_find_row(b, (int)t, seq, s)) return;
  const int pos = s.pos((int)t);
  const unsigned n = pos < 0 ? 0u : ((unsigned)pos >> c.shift) + 1;
  int* out = pages + ((size_t)t * c.heads + head) * budget;
  if (n <= budget) {
    for (unsigned i = tid; i < budget; i += 64 * kWaves) out[i] = i < n ? (int)i : -1;
    return;
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const unsigned p = tid * kPer + j;
    k[j] = p >= n ? 0u : p < sinks || p + recents >= n ? ~0u : k[j];
  }
  // Largest v with at least `budget` keys >= v, bit by bit below the bits that all
  // scores share: a ballot and a scalar bit count per 64 keys, one exchange between
  // the waves.
  unsigned hi = 0, lo = ~0u;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (k[j] != 0 && k[j] != ~0u) hi = max(hi, k[j]), lo = min(lo, k[j]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    hi = max(hi, (unsigned)__shfl_xor(hi, o, 64));
    lo = min(lo, (unsigned)__shfl_xor(lo, o, 64));
  }
  if ((tid & 63) == 0) {
    cnt[0][wave] = hi;
    cnt[1][wave] = lo;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    hi = max(hi, cnt[0][w]);
    lo = min(lo, cnt[1][w]);
  }
  __syncthreads();
  const int top = hi == lo ? -1 : 31 - __clz(hi ^ lo);   // the highest bit that differs
  unsigned v = top < 0 ? hi : hi >> top >> 1 << top << 1, equal = 0;
  for (int bit = top; bit >= 0; --bit) {
    const unsigned cand = v | (1u << bit);
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) m += __popcll(__ballot(k[j] >= cand));
    if ((tid & 63) == 0) cnt[bit & 1][wave] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m += cnt[bit & 1][w];
    if (m >= budget) v = cand;
    if (m == budget) break;   // exactly the keys >= v
  }
  // keys above v, and of those equal to it the lowest pages
  unsigned gt = 0, eq = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    gt += k[j] > v;
    eq += k[j] == v;
  }
  const unsigned own = (gt << 16) | eq;   // each at most 16384 over the workgroup
  unsigned in = wave_scan_add(own);
  if ((tid & 63) == 63) scan[wave] = in;
  __syncthreads();
  unsigned total = 0;
  for (unsigned w = 0; w < kWaves; ++w) {
    const unsigned x = scan[w];
    if (w < wave) in += x;
    total += x;
  }
  in -= own;
  equal = budget - (total >> 16);   // how many equal ones are taken
  unsigned eq_before = in & 0xffffu, at = (in >> 16) + min(eq_before, equal);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool tie = k[j] == v;
    if (k[j] > v || (tie && eq_before < equal)) out[at++] = (int)(tid * kPer + j);
    eq_before += tie;
  }
}

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT size_t qwen36_paged_select_workspace_bytes(const qwen36_paged_cache* cache,
                                                      const qwen36_paged_batch* batch) {
  PagedCache c;
  PagedBatch b;
  if (!paged_cache_of(cache, c) || !paged_batch_of(batch, cache->page_tokens, b)) return 0;
  return (size_t)b.tokens * c.heads * b.width * 4;
}

Q36_EXPORT int qwen36_paged_select(const void* q, const qwen36_paged_cache* cache,
                                   const qwen36_paged_batch* batch, unsigned budget,
                                   unsigned sink_pages, unsigned recent_pages, void* pages,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  PagedCache c;
  PagedBatch b;
  if (!paged_cache_of(cache, c) || !paged_batch_of(batch, cache->page_tokens, b) ||
      c.bounds == nullptr || q == nullptr || !aligned16(q) || pages == nullptr || budget == 0 ||
      budget > 1024 || recent_pages == 0 || sink_pages > budget || recent_pages > budget - sink_pages ||
      workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < qwen36_paged_select_workspace_bytes(cache, batch))
    return Q36_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  unsigned* keys = static_cast<unsigned*>(workspace);
  if (b.width > budget) {   // else every row takes all its pages
    // two rows at a time where sequences have two rows or more on average (300 rows of
    // one sequence over 512 pages: 14.2 us, one at a time 18.4)
    const bool pair = b.tokens >= 2 * b.seqs;
    const size_t rows = (size_t)(pair ? (b.tokens + 1) / 2 : b.tokens) * c.heads, groups = (b.width + 63) / 64;
    size_t per = rows * groups / 1024;   // 16-page groups a wave takes: the queries are quantised once
    per = per < 1 ? 1 : per > groups ? groups : per;
    const unsigned blocks = (unsigned)((groups + per - 1) / per);
    const auto score = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * blocks)), dim3(256), 0, st, static_cast<const bf16*>(q), c,
                         b, keys, blocks, (unsigned)per);
    };
    pair ? score(paged_score_kernel<true>) : score(paged_score_kernel<false>);
    const int e = static_cast<int>(hipGetLastError());
    if (e != Q36_OK) return e;
  }
  const unsigned items = b.tokens * c.heads;
  const auto pick = [&](auto kernel, unsigned threads) {
    const unsigned most = 0x80000000u / threads;   // a launch has less than 2^32 threads
    for (unsigned at = 0; at < items; at += most)
      hipLaunchKernelGGL(kernel, dim3(items - at < most ? items - at : most), dim3(threads), 0, st, c, b, keys,
                         budget, sink_pages, recent_pages, static_cast<int*>(pages), at);
  };
  // The whole call with its attention, graph us, one row and 16: up to 2,048 pages
  // 20.3 to 22.0 and 26.8 to 32.2, with 17 keys a thread 21.9 to 23.6 and 28.5 to
  // 33.6; 3,000 and 4,352 pages 22.2 and 23.5, 39.5 and 44.2, with 16 waves 27.0 and
  // 29.6, 46.0 and 50.6.
  if (b.width <= 2048)
    pick(paged_pick_kernel<8, 4>, 256);
  else if (b.width <= 4352)
    pick(paged_pick_kernel<17, 4>, 256);
  else                        // up to the longest sequence's 16,391
    pick(paged_pick_kernel<17, 16>, 1024);
  return static_cast<int>(hipGetLastError());
}
