// Attention over the paged cache for few rows per sequence (one token, drafted
// tokens, rows with page lists of their own), and the launch that joins split
// key ranges.
//
//   o = softmax(q k^T / 16) v over the positions up to the row's own.
//
// Work: an item is a tile of 2 tokens x the 8 query heads of a KV head (16
// matrix columns; a list has one token) and a chunk of keys, taken by 4 waves
// that deal its 32-key steps among them.  Bound by the cache's bytes (e4m3: 512
// a token and KV head), so nothing is staged and nothing passes through LDS in
// the loop:
//  * K: A operand of S^T = K Q^T straight from the page: lane l holds 16 bytes
//    of row l % 16 -- 16 dims of e4m3 (two k-steps; the reduction index may be
//    ordered freely) or 8 of bf16.
//  * S^T leaves lane l with column l % 16 and keys 4 (l / 16) + r of both
//    16-key tiles: the P^T operand of O^T += V^T P^T as it is.
//  * V: lane l reads 16 dims of exactly those 8 keys (whole rows of 16 lanes);
//    the operand of dims 16 i + t wants 8 keys of one dim a lane, which is a
//    byte (or half-word) exchange between registers of the same lane.
// e4m3 goes to bf16 with the page's power-of-two scale inside the conversion,
// exactly.  A step's V and the next step's K are asked for while its scores are
// formed (the compiler's order; V one step ahead as well, held there by fences,
// was 5% slower over 128K and 2% over 32 sequences).
// Scores, maximum, sum and accumulators are fp32; P is rounded to bf16 for the
// matrix product (its sum too is taken from the fp32 values).
#include "paged_split.h"

namespace q36 {
namespace {

constexpr int kCols = 16, kStep = 32, kWaves = 4;
constexpr int kNoKeys = 0x40000000;
constexpr float kScoreScale = 0.0625f * kLog2e;


// A cache streams through once: nontemporal 32.8 us over 128K of e4m3, plain 36.3 (32
// sequences 112 and 122; bf16 alike in both).  Listed pages are shared by rows: plain
// 113.5 us for a turn of 300 over bf16, nontemporal 208 (e4m3 70 and 94).
template <bool kOnce>
__device__ __forceinline__ u32x4 load16(const char* p) {
  const u32x4* x = reinterpret_cast<const u32x4*>(p);
  return kOnce ? __builtin_nontemporal_load(x) : *x;
}

__device__ __forceinline__ bf16x8 as_bf16x8(unsigned a, unsigned b, unsigned c, unsigned d) {
  const u32x4 v = {a, b, c, d};
  return __builtin_bit_cast(bf16x8, v);
}

struct ListArgs {
  const int* pages;     // [tokens][KV heads][listed]
  unsigned listed, chunks, chunk_keys;
};

__device__ __forceinline__ void paged_store(const PagedOut& w, unsigned hq, size_t t, unsigned qh, unsigned d,
                                            const f32x4& o, float l) {
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  bf16x4 r;
  if (w.gate != nullptr) {
    const bf16x4 g = *reinterpret_cast<const bf16x4*>(w.gate + t * w.gate_stride + qh * 2 * kD + kD + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = f2bf(l == 0.f ? 0.f : paged_gate(o[e] * inv, g[e]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = f2bf(l == 0.f ? 0.f : o[e] * inv);
  }
  *reinterpret_cast<bf16x4*>(w.out + (t * hq + qh) * kD + d) = r;
}

// What a workgroup takes at once: rows t0 .. t0 + n_tok and keys [key0, key1) of
// the sequence, or of the row's list.
struct Piece {
  unsigned seq, head;
  int t0, n_tok, pos0, key0, key1;
  size_t slot;
  bool single;
};

// The waves' accumulators, a column's 64-dim quarters 68 words apart: the four
// quarters and four neighbouring columns of a store then cover all banks.
constexpr int kQuarter = 68;
struct __attribute__((aligned(16))) Shared {
  float o[kWaves][kCols][4 * kQuarter];
  float ml[kWaves][kCols][2];
  int odd[kWaves];   // whether a V value that only the second token sees is not finite
};

template <bool kFp8, bool kList>
__device__ __forceinline__ void paged_piece(const bf16* __restrict__ q, const PagedCache& c, const PagedBatch& b,
                                            const PagedOut& w, const ListArgs& list, const Piece& pc, Shared& sh) {
  constexpr int kElem = kFp8 ? 1 : 2;
  constexpr int kKLoads = 4 * kElem, kVLoads = kElem;   // 16-byte loads of a K row part, a V row
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const unsigned hq = c.heads * kGroup, head = pc.head;
  // one piece for all lanes: scalar registers, so that loops and addresses are too
  const unsigned seq = __builtin_amdgcn_readfirstlane(pc.seq);
  const int t0 = __builtin_amdgcn_readfirstlane(pc.t0), n_tok = __builtin_amdgcn_readfirstlane(pc.n_tok);
  const int pos0 = __builtin_amdgcn_readfirstlane(pc.pos0);
  const int key0 = __builtin_amdgcn_readfirstlane(pc.key0), key1 = __builtin_amdgcn_readfirstlane(pc.key1);
  const int lim_max = pos0 + n_tok - 1;
  const int tok = col >> 3;
  const int lim = tok < n_tok ? pos0 + tok : -1;   // this column's last key

  bf16x8 qf[8];
  {
    const bf16* qp = q + ((size_t)(t0 + tok) * hq + head * kGroup + (col & 7)) * kD;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      // the dims of k-step s as the K operand below has them
      const int d = kFp8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
      qf[s] = lim >= 0 ? *reinterpret_cast<const bf16x8*>(qp + d) : bf16x8{};
    }
  }
  f32x4 o[16];
#pragma unroll
  for (int t = 0; t < 16; ++t) o[t] = f32x4{};
  float m = -INFINITY, l = 0.f;
  bool strange = false;

  const int n_steps = (key1 - key0 + kStep - 1) / kStep;
  const int my_steps = n_steps > wave ? (n_steps - wave + kWaves - 1) / kWaves : 0;
  const int* table = b.table + seq * b.table_stride;
  const int* mine = kList ? list.pages + ((size_t)t0 * c.heads + head) * list.listed : nullptr;
  const int page_mask = (1 << c.shift) - 1;
  const unsigned koff = col * kD * kElem + 16 * g;
  const unsigned voff = 4 * g * kD * kElem + 16 * kElem * col;
  const size_t head_off = (size_t)head << (c.shift + 8);   // elements

  // 32 steps (64 tiles of 16 keys) at a time: lane j holds what tile j needs
  for (int s0 = 0; s0 < my_steps; s0 += 32) {
    int d_key = kNoKeys, d_row = 0;
    unsigned d_page = 0, d_ke = 127, d_ve = 127;
    {
      const int step = wave + kWaves * (s0 + (lane >> 1));
      const int at = key0 + step * kStep + (lane & 1) * 16;   // of the sequence, or of the list
      if (at < key1) {
        int logical = at >> c.shift;
        bool any = true;
        if constexpr (kList) {
          logical = mine[logical];
          any = logical >= 0 && logical <= (pos0 >> c.shift);
        }
        if (any) {
          const unsigned pid = (unsigned)table[logical];
          const int first = (logical << c.shift) + (at & page_mask);
          if (pid < c.pages && first <= lim_max) {
            d_page = pid;
            d_row = at & page_mask;
            d_key = first;
            if constexpr (kFp8) {
              d_ke = c.k_exp[(size_t)pid * c.heads + head];
              d_ve = c.v_exp[(size_t)pid * c.heads + head];
            }
          }
        }
      }
    }
    // only the steps with a page: bit 2 i stands for step i
    const unsigned long long some = __ballot(d_key != kNoKeys);
    unsigned long long todo = (some | some >> 1) & 0x5555555555555555ull;
    if (todo == 0) continue;
    int i = (int)__builtin_ctzll(todo) >> 1;
    u32x4 kr[2][kKLoads], vr[2][4][kVLoads];
    const auto load_k = [&](int i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned pid = __builtin_amdgcn_readlane(d_page, 2 * i + h);
        const int row = __builtin_amdgcn_readlane(d_row, 2 * i + h);
        const char* p = c.k + pid * c.k_stride + (head_off + (size_t)row * kD) * kElem;
#pragma unroll
        for (int j = 0; j < kKLoads; ++j)
          kr[h][j] = load16<!kList>(p + koff + 64 * j);
      }
    };
    const auto load_v = [&](int i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned pid = __builtin_amdgcn_readlane(d_page, 2 * i + h);
        const int row = __builtin_amdgcn_readlane(d_row, 2 * i + h);
        const char* p = c.v + pid * c.v_stride + (head_off + (size_t)row * kD) * kElem;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int j = 0; j < kVLoads; ++j)
            vr[h][e][j] = load16<!kList>(p + voff + e * kD * kElem + 16 * j);
      }
    };
    load_k(i);
    load_v(i);
    for (;;) {
      const int ka = __builtin_amdgcn_readlane(d_key, 2 * i), kb = __builtin_amdgcn_readlane(d_key, 2 * i + 1);
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{};
        if constexpr (kFp8) {
          const float sc = paged_scale((unsigned)__builtin_amdgcn_readlane(d_ke, 2 * i + h));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const u32x4 x = kr[h][j];
            s[h] = mfma16x16x32(as_bf16x8(cvt2<false>(x[0], sc), cvt2<true>(x[0], sc), cvt2<false>(x[1], sc),
                                          cvt2<true>(x[1], sc)), qf[2 * j], s[h]);
            s[h] = mfma16x16x32(as_bf16x8(cvt2<false>(x[2], sc), cvt2<true>(x[2], sc), cvt2<false>(x[3], sc),
                                          cvt2<true>(x[3], sc)), qf[2 * j + 1], s[h]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) s[h] = mfma16x16x32(__builtin_bit_cast(bf16x8, kr[h][j]), qf[j], s[h]);
        }
      }
      todo &= todo - 1;
      const int ahead = todo ? (int)__builtin_ctzll(todo) >> 1 : i;   // the last step loads its own keys again
      load_k(ahead);
      // keys of this lane: ka + 4 g + r, kb + 4 g + r
      const bool edge = max(ka, kb) + 15 > lim_max - (n_tok - 1);
      if (edge) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[0][r] = ka + 4 * g + r <= lim ? s[0][r] : -INFINITY;
          s[1][r] = kb + 4 * g + r <= lim ? s[1][r] : -INFINITY;
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = wave_max_xor(mx, 16);
      mx = wave_max_xor(mx, 32);
      mx *= kScoreScale;
      if (__any(mx > m)) {
        const float mn = fmaxf(m, mx);
        const float a = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= a;
#pragma unroll
        for (int t = 0; t < 16; ++t) o[t] *= a;
      }
      const float base = m == -INFINITY ? 0.f : m;
      float p[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r >> 2][r & 3], kScoreScale, -base));
        l += p[r];
      }
      bf16x8 pb;
#pragma unroll
      for (int r = 0; r < 8; ++r) pb[r] = f2bf(p[r]);

      if (edge) {
        // Behind a row's position V may hold anything, and 0 * NaN is NaN: rows that
        // no token sees are cleared, and of the one that only the second token sees
        // what is not finite (it gets that at the end).
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = (h ? kb : ka) + 4 * g + e;
#pragma unroll
            for (int j = 0; j < kVLoads; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const unsigned u = key > lim_max ? 0u : vr[h][e][j][x];
                const unsigned bad = key > pos0 ? not_finite<kFp8>(u) : 0u;
                vr[h][e][j][x] = u & ~bad;
                strange |= bad != 0;
              }
          }
      }
      if constexpr (kFp8) {
        const float sa = paged_scale((unsigned)__builtin_amdgcn_readlane(d_ve, 2 * i));
        const float sb = paged_scale((unsigned)__builtin_amdgcn_readlane(d_ve, 2 * i + 1));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          // [key 0, key 1] of dims 4d, 4d+1 and 4d+2, 4d+3; [key 2, key 3] likewise
          unsigned x[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            x[h][0] = __builtin_amdgcn_perm(vr[h][1][0][d], vr[h][0][0][d], 0x05010400);
            x[h][1] = __builtin_amdgcn_perm(vr[h][3][0][d], vr[h][2][0][d], 0x05010400);
            x[h][2] = __builtin_amdgcn_perm(vr[h][1][0][d], vr[h][0][0][d], 0x07030602);
            x[h][3] = __builtin_amdgcn_perm(vr[h][3][0][d], vr[h][2][0][d], 0x07030602);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            o[4 * d + 2 * u] = mfma16x16x32(
                as_bf16x8(cvt2<false>(x[0][2 * u], sa), cvt2<false>(x[0][2 * u + 1], sa),
                          cvt2<false>(x[1][2 * u], sb), cvt2<false>(x[1][2 * u + 1], sb)),
                pb, o[4 * d + 2 * u]);
            o[4 * d + 2 * u + 1] = mfma16x16x32(
                as_bf16x8(cvt2<true>(x[0][2 * u], sa), cvt2<true>(x[0][2 * u + 1], sa),
                          cvt2<true>(x[1][2 * u], sb), cvt2<true>(x[1][2 * u + 1], sb)),
                pb, o[4 * d + 2 * u + 1]);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const auto word = [&](int h, int e) { return vr[h][e][d >> 2][d & 3]; };
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const unsigned sel = u ? 0x07060302 : 0x05040100;
            o[2 * d + u] = mfma16x16x32(
                as_bf16x8(__builtin_amdgcn_perm(word(0, 1), word(0, 0), sel),
                          __builtin_amdgcn_perm(word(0, 3), word(0, 2), sel),
                          __builtin_amdgcn_perm(word(1, 1), word(1, 0), sel),
                          __builtin_amdgcn_perm(word(1, 3), word(1, 2), sel)),
                pb, o[2 * d + u]);
          }
        }
      }
      load_v(ahead);
      if (todo == 0) break;
      i = ahead;
    }
  }

  // the waves' partials of each column, joined in LDS
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) {
    sh.ml[wave][col][0] = m;
    sh.ml[wave][col][1] = l;
  }
  if (!kList) {
    const int any = __any(strange);
    if (lane == 0) sh.odd[wave] = any;
  }
  if (col < 8 * n_tok) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < 16; t += 4) {
        const f32x4 v = {o[t][r], o[t + 1][r], o[t + 2][r], o[t + 3][r]};
        *reinterpret_cast<f32x4*>(&sh.o[wave][col][kQuarter * g + 16 * r + t]) = v;
      }
  }
  __syncthreads();
  const int oc = tid >> 4, od = (tid & 15) * 4;   // a column, 4 dims of each 64
  if (oc >= 8 * n_tok) return;
  float mm = sh.ml[0][oc][0];
#pragma unroll
  for (int x = 1; x < kWaves; ++x) mm = fmaxf(mm, sh.ml[x][oc][0]);
  const float base = mm == -INFINITY ? 0.f : mm;
  float f[kWaves], lsum = 0.f;
#pragma unroll
  for (int x = 0; x < kWaves; ++x) {
    f[x] = __builtin_amdgcn_exp2f(sh.ml[x][oc][0] - base);
    lsum += f[x] * sh.ml[x][oc][1];
  }
  const size_t row = t0 + (oc >> 3), qh = head * kGroup + (oc & 7);
  const unsigned rows = kList ? 8 : kCols;
  const size_t part = (pc.slot * c.heads + head) * rows + oc;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = 64 * j + od;
    f32x4 v = f32x4{};
#pragma unroll
    for (int x = 0; x < kWaves; ++x) v += f[x] * *reinterpret_cast<const f32x4*>(&sh.o[x][oc][kQuarter * j + od]);
    if (!kList && oc >= 8 && (sh.odd[0] | sh.odd[1] | sh.odd[2] | sh.odd[3]))
      add_not_finite<kFp8>(v, c, table, head, lim_max, key1 - 1, key0, d);
    if (pc.single) {
      paged_store(w, hq, row, qh, d, v, lsum);
    } else {
      *reinterpret_cast<f32x4*>(w.o + part * kD + d) = v;
    }
  }
  if (!pc.single && od == 0) {
    w.ml[part * 2] = mm;
    w.ml[part * 2 + 1] = lsum;
  }
}

// Rows with lists of their own: a workgroup per (row, KV head, chunk of the list);
// kPerCu of them share a CU.
template <bool kFp8, int kPerCu>
__global__ __launch_bounds__(64 * kWaves, kPerCu) void paged_list_kernel(
    const bf16* __restrict__ q, PagedCache c, PagedBatch b, PagedOut w, ListArgs list) {
  __shared__ Shared sh;
  const unsigned item = blockIdx.x / c.heads, chunk = item % list.chunks;
  Piece p;
  PagedSeq s;
  p.t0 = (int)(item / list.chunks);
  if (!paged_find_row(b, p.t0, p.seq, s)) return;
  p.head = blockIdx.x % c.heads;
  p.pos0 = s.pos(p.t0);
  p.single = list.chunks == 1;
  if (p.pos0 < 0 && !p.single) return;   // the joining launch writes its zeros
  p.n_tok = 1;
  p.key0 = (int)(chunk * list.chunk_keys);
  p.key1 = min(p.key0 + (int)list.chunk_keys, (int)(list.listed << c.shift));
  p.slot = item;
  paged_piece<kFp8, true>(q, c, b, w, list, p, sh);
}

// Tiles of two tokens over their sequences: workgroup i of a KV head takes blocks
// [i per, (i + 1) per) of all its tiles' in a row.
template <bool kFp8>
__global__ __launch_bounds__(64 * kWaves, kFp8 ? 2 : 1) void paged_rows_kernel(
    const bf16* __restrict__ q, PagedCache c, PagedBatch b, PagedOut w, unsigned shares) {
  __shared__ Shared sh;
  __shared__ unsigned find[52];
  const unsigned i = blockIdx.x / c.heads;
  unsigned total, tiles, longest, seq, local;
  paged_total<2>(b, find, total, tiles, longest);
  const unsigned per = max(1u, (total + shares - 1) / shares);
  unsigned* put = blockIdx.x == 0 ? w.head : nullptr;
  if (put != nullptr && threadIdx.x == 0) {
    put[0] = per;
    if (b.seqs == 1) put[1] = 0;
  }
  if (!paged_find_item(b, i * per, find, [&](unsigned j) {
        const PagedSeq s = paged_seq(b, j);
        return paged_tiles<2>(s) * paged_blocks(s);
      }, seq, local, put != nullptr ? put + 1 : nullptr))
    return;
  unsigned left = per;
  const ListArgs none = {};
  for (;; ++seq, local = 0) {
    if (seq >= b.seqs) return;
    const PagedSeq s = paged_seq(b, seq);
    const unsigned blocks = paged_blocks(s), n = paged_tiles<2>(s) * blocks;
    while (local < n) {
      const unsigned tile = local / blocks, at = local % blocks, take = min(left, blocks - at);
      Piece p;
      p.seq = seq;
      p.head = blockIdx.x % c.heads;
      p.t0 = s.a + 2 * (int)tile;
      p.n_tok = min(2, s.z - p.t0);
      p.pos0 = s.pos(p.t0);
      const int end = p.pos0 + p.n_tok;
      p.key0 = (int)(at * kSplitBlock);
      p.key1 = min((int)((at + take) * kSplitBlock), end);
      p.slot = (size_t)i + p.t0;   // grows with every step of a share or a tile
      p.single = p.key0 == 0 && p.key1 == end;
      if (p.key0 < p.key1) {
        paged_piece<kFp8, false>(q, c, b, w, none, p, sh);
        __syncthreads();
      }
      left -= take;
      local += take;
      if (left == 0) return;
    }
  }
}

// The partials of one row and head.
struct Parts {
  size_t first;     // of chunk 0
  unsigned n;       // chunks (0: the row sees nothing, 1: it is written already)
  unsigned stride;  // partials between chunks
};
__device__ __forceinline__ bool paged_parts(const PagedBatch& b, unsigned heads, const PagedOut& w, unsigned tile,
                                            unsigned listed_chunks, unsigned t, unsigned qh, Parts& p) {
  unsigned seq;
  PagedSeq s;
  if (!paged_find_row(b, (int)t, seq, s)) return false;
  size_t slot;
  unsigned r;
  if (listed_chunks != 0) {
    p.n = s.pos((int)t) < 0 ? 0 : listed_chunks;
    slot = (size_t)t * listed_chunks;
    r = qh % kGroup;
  } else {
    const unsigned per = w.head[0], own = t - s.a, in = own / tile, blocks = paged_blocks(s);
    const int end = s.len - (s.z - s.a) + min((int)((in + 1) * tile), s.z - s.a);
    const unsigned seen = end > 0 ? ((unsigned)end + kSplitBlock - 1) / kSplitBlock : 0;
    if (tile == 2) {   // shares of the tiles' blocks in a row
      const unsigned start = w.head[1 + seq] + in * blocks;
      p.n = seen ? (start + seen - 1) / per - start / per + 1 : 0;
      slot = (size_t)(start / per) + (s.a + in * tile);
    } else {
      p.n = (seen + per - 1) / per;
      slot = w.head[1 + seq] + (size_t)in * ((blocks + per - 1) / per);
    }
    r = own % tile * kGroup + qh % kGroup;
  }
  if (p.n > w.slots || slot > w.slots - p.n) return false;   // only where sequences overlap
  p.stride = heads * kGroup * tile;
  p.first = (slot * heads + qh / kGroup) * kGroup * tile + r;
  return true;
}

// Merges four chunks (absent ones: m = -inf, l = 0, o = 0) into (m, l, o).
__device__ __forceinline__ void paged_merge4(float& m, float& l, f32x4& o, const float (&cm)[4], const float (&cl)[4],
                                             const f32x4 (&co)[4]) {
  const float mn = fmaxf(fmaxf(fmaxf(cm[0], cm[1]), fmaxf(cm[2], cm[3])), m);
  const float base = mn == -INFINITY ? 0.f : mn;
  const float a = __builtin_amdgcn_exp2f(m - base);
  l *= a;
  o *= a;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float f = __builtin_amdgcn_exp2f(cm[u] - base);
    l += f * cl[u];
    o += f * co[u];
  }
  m = mn;
}

// Many rows of few chunks: a wave per kHeads query heads of a token, 4 dims a lane.
template <unsigned kHeads>
__global__ __launch_bounds__(256) void paged_combine_rows_kernel(PagedBatch b, unsigned heads, PagedOut w,
                                                                 unsigned tile, unsigned listed_chunks) {
  const unsigned hq = heads * kGroup;
  const unsigned i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned t = i * kHeads / hq, h0 = i * kHeads % hq;
  if (t >= b.tokens) return;
  Parts p;
  if (!paged_parts(b, heads, w, tile, listed_chunks, t, h0, p) || p.n == 1) return;
  const unsigned d = (threadIdx.x & 63) * 4;
#pragma unroll 4
  for (unsigned h = 0; h < kHeads; ++h) {   // a head's partials are the next rows of its KV head's
    float m = -INFINITY, l = 0.f;
    f32x4 o = f32x4{};
    for (unsigned i0 = 0; i0 < p.n; i0 += 4) {
      float cm[4], cl[4];
      f32x4 co[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool there = i0 + u < p.n;
        const size_t part = p.first + h + (size_t)(there ? i0 + u : i0) * p.stride;
        cm[u] = there ? w.ml[part * 2] : -INFINITY;
        cl[u] = there ? w.ml[part * 2 + 1] : 0.f;
        co[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(w.o + part * kD + d));
        if (!there) co[u] = f32x4{};
      }
      paged_merge4(m, l, o, cm, cl, co);
    }
    paged_store(w, hq, t, h0 + h, d, o, l);
  }
}

// Few rows of many chunks: a workgroup per row, head and 64 dims; 16 groups of
// 16 lanes take every 16th chunk each, 4 dims a lane.
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedBatch b, unsigned heads, PagedOut w,
                                                            unsigned tile, unsigned listed_chunks) {
  __shared__ float acc[4][16][4];
  __shared__ float stat[4][2];
  const unsigned hq = heads * kGroup;
  const unsigned slice = blockIdx.x & 3, qh = (blockIdx.x >> 2) % hq, t = (blockIdx.x >> 2) / hq;
  Parts p;
  if (!paged_parts(b, heads, w, tile, listed_chunks, t, qh, p) || p.n == 1) return;
  const int group = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  const unsigned d = slice * 64 + (threadIdx.x & 15) * 4;
  float m = -INFINITY, l = 0.f;
  f32x4 o = f32x4{};
  for (unsigned i0 = 0; i0 < p.n; i0 += 64) {   // 4 chunks a group at once
    float cm[4], cl[4];
    f32x4 co[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned i = i0 + 16 * u + group;
      cm[u] = -INFINITY;
      cl[u] = 0.f;
      co[u] = f32x4{};
      if (i < p.n) {
        const size_t part = p.first + (size_t)i * p.stride;
        cm[u] = w.ml[part * 2];
        cl[u] = w.ml[part * 2 + 1];
        co[u] = *reinterpret_cast<const f32x4*>(w.o + part * kD + d);
      }
    }
    paged_merge4(m, l, o, cm, cl, co);
  }
  // groups of a wave, then the waves
#pragma unroll
  for (int x = 16; x < 64; x <<= 1) {
    const float om = __shfl_xor(m, x, 64), mn = fmaxf(m, om);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - base), fo = __builtin_amdgcn_exp2f(om - base);
    l = l * f + __shfl_xor(l, x, 64) * fo;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f + __shfl_xor(o[e], x, 64) * fo;
    m = mn;
  }
  if ((threadIdx.x & 63) < 16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[wave][threadIdx.x & 15][e] = o[e];
    if ((threadIdx.x & 63) == 0) {
      stat[wave][0] = m;
      stat[wave][1] = l;
    }
  }
  __syncthreads();
  if (threadIdx.x >= 16) return;
  float mm = stat[0][0];
  for (int x = 1; x < 4; ++x) mm = fmaxf(mm, stat[x][0]);
  const float base = mm == -INFINITY ? 0.f : mm;
  float lsum = 0.f;
  f32x4 v = f32x4{};
  for (int x = 0; x < 4; ++x) {
    const float f = __builtin_amdgcn_exp2f(stat[x][0] - base);
    lsum += f * stat[x][1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += f * acc[x][threadIdx.x][e];
  }
  paged_store(w, hq, t, qh, d, v, lsum);
}

bool paged_out_of(const void* q, const PagedCache& c, const void* q_gate, unsigned stride, void* out,
                  const void* ws, PagedOut& o) {
  if (q == nullptr || out == nullptr || !aligned16(q) || (reinterpret_cast<uintptr_t>(out) & 7u) ||
      ws == nullptr || !aligned16(ws))
    return false;
  if (q_gate != nullptr && (stride < c.heads * kGroup * 2 * kD || stride % 4 ||
                            (reinterpret_cast<uintptr_t>(q_gate) & 7u)))
    return false;
  o.gate = static_cast<const bf16*>(q_gate);
  o.gate_stride = stride;
  o.out = static_cast<bf16*>(out);
  return true;
}

// How a call is cut: tokens of a tile, workgroups of a KV head that the GPU holds
// at once, items of a KV head aimed at, items (or slots of partials) at most.
// One tile for the whole call, by the mean rows of a sequence; graph us with tiles of
// 2 / 8 / 16 / 32 over two KV heads, first 16 sequences over 12,000, then 128 over 1,000:
//   rows    e4m3                            bf16
//    2   49  57  57  76   35  47  46  63    88  89  88  91   61  67  67  72
//    3   77  60  60  78   61  49  48  66   155  92  91  94  114  70  69  75
//    8  115  65  68  80  118  66  66  70   263  98  99  95  226  84  85  80
//    9  164  77  73  80  146  70  70  71   353 117 102  96  281 108  90  81
//   16  219  86  87  88  226  74  84  75   486 125 115 104  434 108 102  87
//   17  280 110 103 102  254 116  86  85   602 193 130 115  492 177 108  93
// The border of 2 is clear, those of 8 and 16 are e4m3's over long caches; bf16 would
// gain up to 15% by tiles of 32 from 8 rows on.  Sequences far from the mean pay for
// the one tile: 255 single tokens over 16,000 and one turn of 256 rows over 30,000
// together 1,184 us, alone 663 and 132; 63 single tokens and a prompt of 2,048 rows
// together 1,429, alone 175 and 836.
struct Plan {
  unsigned tile, slots, target, items;
};
Plan paged_plan(const PagedBatch& b, unsigned heads) {
  Plan p;
  const unsigned mean = (b.tokens + b.seqs - 1) / b.seqs;
  p.tile = mean <= 2 ? 2 : mean <= 8 ? 8 : mean <= 16 ? 16 : 32;
  if (p.tile == 2) {   // one share for each CU (512 shares: 38.0 us against 32.8 over 128K)
    p.slots = p.target = 256u / heads;
    p.items = p.target + b.tokens;
  } else {             // a workgroup of 8 waves a CU, two of 4 or of 2
    p.slots = (p.tile == 32 ? 256u : 512u) / heads;
    // (every workgroup of the grid costs its look at the lengths, also one without an item)
    p.target = p.tile == 32 ? 2 * p.slots : p.slots;
    p.items = paged_items(b, p.tile, p.target);
  }
  return p;
}

// Keys of a listed chunk: whole blocks, so that all rows' chunks fill the GPU.
void list_plan(const PagedBatch& b, const PagedCache& c, unsigned listed, ListArgs& l) {
  const size_t keys = (size_t)listed << c.shift;
  const size_t rows = (size_t)b.tokens * c.heads;
  const size_t blocks = (keys + kSplitBlock - 1) / kSplitBlock;
  const size_t want = rows >= 256 ? 1 : 256 / rows;   // chunks of a row: a workgroup a CU
  const size_t per = want >= blocks ? 1 : (blocks + want - 1) / want;
  l.chunk_keys = (unsigned)(per * kSplitBlock);
  l.chunks = (unsigned)((blocks + per - 1) / per);
  l.listed = listed;
}

}  // namespace

int paged_combine(const PagedBatch& b, const PagedCache& c, const PagedOut& o, unsigned tile,
                  unsigned listed_chunks, void* stream) {
  const unsigned hq = c.heads * kGroup;
  hipStream_t st = static_cast<hipStream_t>(stream);
  // 2,048 tokens of 2 chunks: 24 us with a wave per head (217 with a workgroup per 64
  // dims and 4 chunks).  Where thousands of tokens have one chunk a wave per 8 heads
  // ends sooner (4,020 tokens: 16 us and 5); 200 tokens of 18 chunks take 18 more so.
  const unsigned pairs = b.tokens * c.heads;
  const auto rows = [&](auto kernel, unsigned per) {
    hipLaunchKernelGGL(kernel, dim3((b.tokens * (hq / per) + 3) / 4), dim3(256), 0, st, b, c.heads, o, tile,
                       listed_chunks);
  };
  if (pairs >= 2048)
    rows(paged_combine_rows_kernel<kGroup>, kGroup);
  else if (pairs >= 256)
    rows(paged_combine_rows_kernel<1>, 1);
  else
    hipLaunchKernelGGL(paged_combine_kernel, dim3(b.tokens * hq * 4), dim3(256), 0, st, b, c.heads, o, tile,
                       listed_chunks);
  return static_cast<int>(hipGetLastError());
}

}  // namespace q36

using namespace q36;

Q36_EXPORT size_t qwen36_paged_attention_workspace_bytes(const qwen36_paged_cache* cache,
                                                         const qwen36_paged_batch* batch) {
  PagedCache c;
  PagedBatch b;
  if (!paged_cache_of(cache, c) || !paged_batch_of(batch, cache->page_tokens, b)) return 0;
  const Plan p = paged_plan(b, c.heads);
  return split_ws_bytes(b.seqs, p.items, c.heads, 8 * p.tile);
}

Q36_EXPORT int qwen36_paged_attention(const void* q, const qwen36_paged_cache* cache,
                                      const qwen36_paged_batch* batch, const void* q_gate,
                                      unsigned q_gate_row_stride, void* out, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  PagedCache c;
  PagedBatch b;
  PagedOut o;
  if (!paged_cache_of(cache, c) || !paged_batch_of(batch, cache->page_tokens, b) ||
      !paged_out_of(q, c, q_gate, q_gate_row_stride, out, workspace, o) ||
      workspace_bytes < qwen36_paged_attention_workspace_bytes(cache, batch))
    return Q36_EINVAL;
  const Plan p = paged_plan(b, c.heads);
  const bool fp8 = cache->cache_type == QWEN36_PAGED_E4M3;
  split_ws(workspace, b.seqs, p.items, c.heads, 8 * p.tile, o);
  int e;
  if (p.tile == 2) {
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(p.target * c.heads), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream),
                         static_cast<const bf16*>(q), c, b, o, p.target);
    };
    fp8 ? launch(paged_rows_kernel<true>) : launch(paged_rows_kernel<false>);
    e = static_cast<int>(hipGetLastError());
  } else {
    e = paged_prefill(q, c, fp8, b, o, p.tile, p.items, p.slots, p.target, stream);
  }
  return e != Q36_OK ? e : paged_combine(b, c, o, p.tile, 0, stream);
}

Q36_EXPORT size_t qwen36_paged_sparse_attention_workspace_bytes(const qwen36_paged_cache* cache,
                                                                const qwen36_paged_batch* batch,
                                                                unsigned listed) {
  PagedCache c;
  PagedBatch b;
  if (!paged_cache_of(cache, c) || !paged_batch_of(batch, cache->page_tokens, b) || listed == 0 ||
      listed > 1024)
    return 0;
  ListArgs l;
  list_plan(b, c, listed, l);
  return split_ws_bytes(0, (size_t)b.tokens * l.chunks, c.heads, 8);
}

Q36_EXPORT int qwen36_paged_sparse_attention(const void* q, const qwen36_paged_cache* cache,
                                             const qwen36_paged_batch* batch, const void* pages,
                                             unsigned listed, const void* q_gate,
                                             unsigned q_gate_row_stride, void* out, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  PagedCache c;
  PagedBatch b;
  PagedOut o;
  if (!paged_cache_of(cache, c) || !paged_batch_of(batch, cache->page_tokens, b) || listed == 0 ||
      listed > 1024 || pages == nullptr ||
      !paged_out_of(q, c, q_gate, q_gate_row_stride, out, workspace, o) ||
      workspace_bytes < qwen36_paged_sparse_attention_workspace_bytes(cache, batch, listed))
    return Q36_EINVAL;
  ListArgs l;
  list_plan(b, c, listed, l);
  l.pages = static_cast<const int*>(pages);
  split_ws(workspace, 0, (size_t)b.tokens * l.chunks, c.heads, 8, o);
  const unsigned grid = b.tokens * l.chunks * c.heads;
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream),
                       static_cast<const bf16*>(q), c, b, o, l);
  };
  // Two workgroups of bf16 a CU cost a few spilled registers, which pays where the grid
  // has more than one for each CU: 784 of them 60.9 us, so 57.9; 256 48.7, so 52.2.
  if (cache->cache_type == QWEN36_PAGED_E4M3)
    launch(paged_list_kernel<true, 2>);
  else if (grid > 256)
    launch(paged_list_kernel<false, 2>);
  else
    launch(paged_list_kernel<false, 1>);
  const int e = static_cast<int>(hipGetLastError());
  return e != Q36_OK || l.chunks == 1 ? e : paged_combine(b, c, o, 1, l.chunks, stream);
}
