// Attention over the paged cache for many rows per sequence (prompts, chunks of
// prompts, many drafted tokens).
//
//   o = softmax(q k^T / 16) v over the positions up to the row's own.
//
// Work: an item is a tile of 4 kWaves tokens x the 8 query heads of a KV head
// (32 matrix columns a wave) and a chunk of keys; bound by the matrix products
// (16,384 operations a (row's token, key) pair and KV head).  Per 32-key tile:
//  * K and V of the next tile leave their pages for registers, 16 bytes a lane,
//    become bf16 there (e4m3 with the page's scale inside the conversion, once
//    for all 8 heads and 4 kWaves tokens) and go to the other half of an LDS
//    double buffer, so that conversion costs 1/16 of what it would behind LDS;
//  * S^T = K Q^T, online softmax in fp32, O^T += V^T P^T on 32x32x16 products:
//    A = K rows from LDS, B = Q^T in registers; A = V^T by transposed LDS reads,
//    B = P^T, the S^T accumulator as it is.  LDS operands are read 4 products
//    ahead (the order is pinned by scheduling barriers).
// The reference maximum is the first visible tile's and is raised (with a
// rescale) only when a tile's probabilities sum past 2^20.
#include "paged_split.h"

namespace q36 {
namespace {

constexpr int kKeys = 32;
constexpr int kRowB = kD * 2;                      // a bf16 row in LDS
// LDS tile: block b (0..15) holds rows b and b + 16; 1040 (K) and 1088 (V) bytes
// apart, which keeps the 16-byte K reads and the transposed V reads free of bank
// conflicts.
constexpr int kKBlk = 1040, kVBlk = 1088;
constexpr int kKTile = 16 * kKBlk, kStage = kKTile + 16 * kVBlk;
constexpr int kLds = 2 * kStage;                   // 68,096 bytes
constexpr float kScoreScale = 0.0625f * kLog2e;

template <bool kFp8, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 4 ? 2 : 1) void paged_prefill_kernel(
    const bf16* __restrict__ q, PagedCache c, PagedBatch b, PagedOut w, unsigned target) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  __shared__ unsigned find[40];
  __shared__ int odd;   // whether a V value that some rows must not see is not finite
  constexpr int kElem = kFp8 ? 1 : 2;
  constexpr int kTile = 4 * kWaves, kPass = 8 / kWaves;   // 4 kWaves rows a pass

  const unsigned head = blockIdx.x % c.heads, item = blockIdx.x / c.heads;
  const unsigned hq = c.heads * kGroup;
  PagedSplit sp;
  if (!paged_split<kTile>(b, item, target, blockIdx.x == 0 ? w.head : nullptr, find, sp)) return;
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

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lj = lane & 31, lg = lane >> 5;
  const int tok = wave * 4 + (lj >> 3);            // of the tile
  const bool live = tok < n_tok;
  const int lim = live ? pos0 + tok : -1;          // this column's last key
  const int wave_first = pos0 + wave * 4;
  const int wave_lim = wave * 4 < n_tok ? min(wave_first + 3, end - 1) : -1;

  bf16x8 qf[16];
  {
    const bf16* qp = q + ((size_t)(t0 + tok) * hq + head * kGroup + (lj & 7)) * kD + 8 * lg;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      qf[i] = lim >= 0 ? *reinterpret_cast<const bf16x8*>(qp + 16 * i) : bf16x8{};
  }
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

  // ---- raw rows of the tile to come
  u32x4 rk[kPass][kElem], rv[kPass][kElem];
  unsigned rexp[kPass];
  unsigned r_ok = 0, ok = 0;     // bit h: the 16 keys h of the tile have a page
  int r_tile = 0;
  const size_t head_off = ((size_t)head << (c.shift + 8)) * kElem;
  const unsigned in_row = (lane & 15) * 16;
  const auto load_tile = [&](int i) {
    const int at = i & 31;
    if (at == 0) {
      if (i == 0) {
        fetch_pages(kv_first);
        fetch_scales();
      }
      d_page = n_page;
      d_exp = n_exp;
      d_ok = __ballot(n_ok);
    } else if (at == 8) {
      fetch_pages(kv_first + (i + 24) * kKeys);
    } else if (at == 20) {
      fetch_scales();
    }
    r_ok = (unsigned)(d_ok >> (2 * at)) & 3u;
    r_tile = i;
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
      const int row = p * 4 * kWaves + 4 * wave;       // first of this wave's 4
      const int from = 2 * at + (row >> 4);
      const unsigned pid = __builtin_amdgcn_readlane(d_page, from);
      const int prow = (kv_first + i * kKeys + row) & page_mask;
      rexp[p] = __builtin_amdgcn_readlane(d_exp, from);
      const unsigned voff = (lane >> 4) * kD * kElem + in_row;
      const char* kp = c.k + pid * c.k_stride + head_off + (size_t)prow * kD * kElem;
      const char* vp = c.v + pid * c.v_stride + head_off + (size_t)prow * kD * kElem;
#pragma unroll
      for (int e = 0; e < kElem; ++e) {
        rk[p][e] = *reinterpret_cast<const u32x4*>(kp + voff + 256 * e);
        rv[p][e] = *reinterpret_cast<const u32x4*>(vp + voff + 256 * e);
      }
    }
  };
  const auto store_tile = [&](int stage) {
    const int key0 = kv_first + r_tile * kKeys;
    const bool edge = key0 + kKeys - 1 > pos0 || r_ok != 3u;
    bool strange = false;
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
      const int row = p * 4 * kWaves + 4 * wave + (lane >> 4);
      if (edge) {
        // Behind the tile's first position V may hold anything, and 0 * NaN is NaN:
        // rows that no token sees are cleared, and of the others what is not finite
        // (the tokens that do see it get it at the end).
        const bool out = key0 + row >= kv_stop || !((r_ok >> (row >> 4)) & 1u);
        const bool some = key0 + row > pos0;
#pragma unroll
        for (int e = 0; e < kElem; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const unsigned u = out ? 0u : rv[p][e][x], bad = some ? not_finite<kFp8>(u) : 0u;
            rv[p][e][x] = u & ~bad;
            strange |= bad != 0;
          }
      }
      char* kb = lds + stage * kStage + (row & 15) * kKBlk + (row >> 4) * kRowB;
      char* vb = lds + stage * kStage + kKTile + (row & 15) * kVBlk + (row >> 4) * kRowB;
      if constexpr (kFp8) {
        const float ks = paged_scale(rexp[p] & 0xffu), vs = paged_scale(rexp[p] >> 8);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const unsigned k0 = rk[p][0][2 * x], k1 = rk[p][0][2 * x + 1];
          const unsigned v0 = rv[p][0][2 * x], v1 = rv[p][0][2 * x + 1];
          *reinterpret_cast<u32x4*>(kb + 2 * in_row + 16 * x) =
              u32x4{cvt2<false>(k0, ks), cvt2<true>(k0, ks), cvt2<false>(k1, ks), cvt2<true>(k1, ks)};
          *reinterpret_cast<u32x4*>(vb + 2 * in_row + 16 * x) =
              u32x4{cvt2<false>(v0, vs), cvt2<true>(v0, vs), cvt2<false>(v1, vs), cvt2<true>(v1, vs)};
        }
      } else {
#pragma unroll
        for (int e = 0; e < kElem; ++e) {
          *reinterpret_cast<u32x4*>(kb + in_row + 256 * e) = rk[p][e];
          *reinterpret_cast<u32x4*>(vb + in_row + 256 * e) = rv[p][e];
        }
      }
    }
    if (strange) odd = 1;
  };

  const int kbase = (lj & 15) * kKBlk + (lj >> 4) * kRowB + lg * 16;
  const int grp = lane >> 4, m16 = lane & 15;
  const int vbase = (4 * lg + (m16 >> 2)) * kVBlk + 32 * (grp & 1) + 8 * (m16 & 3);

  const int n_tiles = (kv_stop - kv_first + kKeys - 1) / kKeys;
  if (tid == 0) odd = 0;
  __syncthreads();
  load_tile(0);
  store_tile(0);
  unsigned ok_next = r_ok;
  if (n_tiles > 1) load_tile(1);
  for (int t = 0; t < n_tiles; ++t) {
    const int kv0 = kv_first + t * kKeys, stage = t & 1;
    ok = ok_next;
    __syncthreads();   // tile t is in LDS, tile t - 1 is used up
    if (t + 1 < n_tiles) {
      store_tile(stage ^ 1);
      ok_next = r_ok;
      if (t + 2 < n_tiles) load_tile(t + 2);
    }
    if (kv0 > wave_lim) continue;
    const char* kp = lds + stage * kStage + kbase;
    const char* vp = lds + stage * kStage + kKTile + vbase;

    bf16x8 kr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) kr[i] = *reinterpret_cast<const bf16x8*>(kp + i * 32);
    f32x16 x = f32x16{};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x = mfma32x32x16(kr[i & 3], qf[i], x);
      if (i + 4 < 16) kr[i & 3] = *reinterpret_cast<const bf16x8*>(kp + (i + 4) * 32);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    // lane: keys kv0 + 8 (r / 4) + 4 lg + r % 4 of its column
    const bool diag = kv0 + kKeys - 1 > wave_first;
    if (diag || ok != 3u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kv0 + 8 * (r >> 2) + 4 * lg + (r & 3);
        x[r] = key <= lim && ((ok >> (r >> 3)) & 1u) ? x[r] : -INFINITY;
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

    i16x4 va[4][2];
    const auto vread = [&](int i, int to) {
      const char* p = vp + (i >> 3) * kRowB + (i & 7) * 64;
      va[to][0] = lds_read_tr16(p);
      va[to][1] = lds_read_tr16(p + 8 * kVBlk);
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

  // ---- out through LDS in four rounds of 64 dims, so that stores are whole
  // 256-byte (fp32 partials) or 128-byte row segments
  l += __shfl_xor(l, 32, 64);
  const float inv = single ? (l == 0.f ? 0.f : 1.0f / l) : 1.0f;
  const size_t part0 = (slot * c.heads + head) * (8 * kTile);
  if (!single && lg == 0 && live) {
    const size_t part = part0 + wave * 32 + lj;
    w.ml[part * 2] = l == 0.f ? -INFINITY : m;   // what saw nothing weighs nothing
    w.ml[part * 2 + 1] = l;
  }
  const bool zero = l == 0.f;
  __syncthreads();
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
      const int rt = wave * 4 + (r >> 3), d = rd * 64 + ch * 4;
      if (rt >= n_tok) continue;
      if (strange_v) add_not_finite<kFp8>(v, c, table, head, pos0 + 1, min(pos0 + rt, kv_stop - 1), kv_first, d);
      if (!single) {
        *reinterpret_cast<f32x4*>(w.o + (part0 + wave * 32 + r) * kD + d) = v;
        continue;
      }
      const size_t row = t0 + rt, qh = head * kGroup + (r & 7);
      bf16x4 res;
      if (w.gate != nullptr) {
        const bf16x4 gt = *reinterpret_cast<const bf16x4*>(w.gate + row * w.gate_stride + qh * 2 * kD + kD + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) res[e] = f2bf(v[e] == 0.f ? 0.f : paged_gate(v[e], gt[e]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) res[e] = f2bf(v[e]);
      }
      *reinterpret_cast<bf16x4*>(w.out + (row * hq + qh) * kD + d) = res;
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  }
}

template <bool kFp8, int kWaves>
int launch(const bf16* q, const PagedCache& c, const PagedBatch& b, const PagedOut& o, unsigned items,
           unsigned target, void* stream) {
  // hipFuncSetAttribute is per device and idempotent
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_prefill_kernel<kFp8, kWaves>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (e != hipSuccess) return static_cast<int>(e);
  hipLaunchKernelGGL((paged_prefill_kernel<kFp8, kWaves>), dim3(items * c.heads), dim3(64 * kWaves), kLds,
                     static_cast<hipStream_t>(stream), q, c, b, o, target);
  return static_cast<int>(hipGetLastError());
}

}  // namespace

int paged_prefill(const void* q, const PagedCache& c, bool fp8, const PagedBatch& b, const PagedOut& o,
                  unsigned tile, unsigned items, unsigned target, void* stream) {
  const bf16* p = static_cast<const bf16*>(q);
  switch (tile) {
    case 8:
      return fp8 ? launch<true, 2>(p, c, b, o, items, target, stream)
                 : launch<false, 2>(p, c, b, o, items, target, stream);
    case 16:
      return fp8 ? launch<true, 4>(p, c, b, o, items, target, stream)
                 : launch<false, 4>(p, c, b, o, items, target, stream);
    default:
      return fp8 ? launch<true, 8>(p, c, b, o, items, target, stream)
                 : launch<false, 8>(p, c, b, o, items, target, stream);
  }
}

}  // namespace q36
