// Low-rank adapters of many requests beside a shared projection.
//
// The projection's weights are stacked slices (q | k | v, ...), y = x W^T.  A request
// with adapter i has y_s += scale_i (x A_i,s^T) B_i,s^T for every slice s, with A_i,s
// [rank, K] and B_i,s [width_s, rank].  Each adapter in use is read once per tile of its
// rows, x once and y read and written once: for prompts y's bytes are what bounds it
// (the 2 rank (K slices + N) operations a row are far below the matrix rate), for single
// tokens the adapters' bytes and the chain of two launches.
//
// Rows are taken in the order of their adapters (adapter_plan_kernel: once for all
// projections of a step), in tiles of 16 (few rows) or 64 (many).
//  * down: h = x A^T in fp32, split over K between the waves of a workgroup and, for few
//    tiles, between workgroups, whose partial sums the second launch adds in order.
//  * up: y + (scale h) B^T, rounded to bf16 once.  h enters the bf16 products as the sum
//    of two bf16 values (2^-17 of it).
// Results depend neither on the order of the requests nor on the tile: a row of a
// product is computed the same in whatever row of a tile it stands.
#include "gemm_tile.h"
#include "paged_common.h"

#include <mutex>

namespace q36 {
namespace {

constexpr unsigned kMaxSlices = 4, kMaxRank = 128, kMaxAdapters = 4096;
constexpr unsigned kFewRows = 1024;      // calls of up to so many rows take tiles of 16

struct Plan {
  const int* tiles;      // [0]: how many; from 4 on: first place in `rows`, rows, adapter, 0
  const int* rows;       // rows of the call, those of an adapter together
};

struct Adapters {
  const bf16* a;         // [n][slices][rank][k]
  const bf16* b;         // [n][sum of widths][rank]
  const int* ranks;
  const float* scales;
  unsigned n, rank, k, slices, total;
  unsigned begin[kMaxSlices + 1];        // first column of each slice
};

__device__ __forceinline__ unsigned adapter_rank(const Adapters& w, int i) {
  const int r = w.ranks != nullptr ? w.ranks[i] : (int)w.rank;
  return (unsigned)min(max(r, 0), (int)w.rank);
}

// ---- rows by adapter --------------------------------------------------------

// One workgroup: rows a adapter, their places, the tiles, the rows.  Sequences of an
// adapter take their places in any order, which no result depends on.
__global__ __launch_bounds__(1024) void adapter_plan_kernel(const int* __restrict__ cu, const int* __restrict__ ids,
                                                            unsigned seqs, unsigned tokens, unsigned n, unsigned tile,
                                                            unsigned max_tiles, int* __restrict__ tiles,
                                                            int* __restrict__ rows) {
  __shared__ unsigned count[kMaxAdapters], place[kMaxAdapters];
  __shared__ unsigned sums[16];
  const unsigned tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  auto rows_of = [&](unsigned i, int& a, int& z) {
    a = min(max(cu[i], 0), (int)tokens);
    z = min(max(cu[i + 1], a), (int)tokens);
  };
  for (unsigned j = tid; j < n; j += 1024) count[j] = 0;
  __syncthreads();
  for (unsigned i = tid; i < seqs; i += 1024) {
    int a, z;
    rows_of(i, a, z);
    const unsigned id = (unsigned)ids[i];
    if (id < n && z > a) atomicAdd(&count[id], (unsigned)(z - a));
  }
  __syncthreads();
  unsigned row0 = 0, tile0 = 0;
  for (unsigned j0 = 0; j0 < n; j0 += 1024) {
    const unsigned j = j0 + tid, c = j < n ? count[j] : 0u, m = (c + tile - 1) / tile;
    // the rows and tiles of the adapters before
    unsigned before[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const unsigned v = p ? m : c, in = wave_scan_add(v);
      __syncthreads();
      if (lane == 63) sums[wave] = in;
      __syncthreads();
      unsigned s = 0, total = 0;
      for (unsigned w = 0; w < 16; ++w) {
        if (w < wave) s += sums[w];
        total += sums[w];
      }
      before[p] = (p ? tile0 : row0) + s + in - v;
      (p ? tile0 : row0) += total;
    }
    if (j < n) {
      place[j] = before[0];
      for (unsigned t = 0; t < m && before[1] + t < max_tiles; ++t) {
        int* o = tiles + 4 * (1 + before[1] + t);
        o[0] = (int)(before[0] + t * tile);
        o[1] = (int)min(tile, c - t * tile);
        o[2] = (int)j;
        o[3] = 0;
      }
    }
  }
  if (tid == 0) tiles[0] = (int)min(tile0, max_tiles);
  __syncthreads();
  for (unsigned i = wave; i < seqs; i += 16) {
    int a, z;
    rows_of(i, a, z);
    const unsigned id = (unsigned)ids[i];
    if (id >= n || z <= a) continue;
    unsigned at = 0;
    if (lane == 0) at = atomicAdd(&place[id], (unsigned)(z - a));
    at = __builtin_amdgcn_readfirstlane(at);
    for (int t = a + (int)lane; t < z; t += 64)
      if (at + (t - a) < tokens) rows[at + (t - a)] = t;
  }
}

// A tile's adapter, first place and rows; false where there is none (offsets that
// overlap can make places behind the call's rows).
__device__ __forceinline__ bool plan_tile(const Plan& p, unsigned i, unsigned tokens, unsigned n, unsigned& first,
                                          unsigned& count, unsigned& id) {
  // both at once; what is asked for behind the plan's places (its rows follow) is none of them
  const int tiles = p.tiles[0];
  const unsigned most = (unsigned)(p.rows - p.tiles) / 4 - 1;
  const int4 t = *reinterpret_cast<const int4*>(p.tiles + 4 * min(1 + i, most));
  if (i >= (unsigned)tiles) return false;
  first = (unsigned)t.x;
  count = (unsigned)t.y;
  id = (unsigned)t.z;
  return id < n && first < tokens && count <= tokens - first;
}

// ---- down: h = x A^T ----------------------------------------------------------

constexpr int kDownPitch = 68;

// Workgroup: (tile, slice, 64 of the rank's rows, part of K); its waves a quarter of the
// part each.  h: [part][place][slice][rank] fp32, or, where K is in one part, what the
// second launch reads as operands: [tile][slice][16 rows][32 of the rank][high, low][lane].
template <int kTiles, bool kFinal>     // tiles of 16 rows
__global__ __launch_bounds__(256, 2) void adapter_down_kernel(const bf16* __restrict__ x, size_t ldx, Adapters w, Plan p,
                                                           unsigned tokens, unsigned parts, float* __restrict__ h) {
  constexpr int kPitch = kDownPitch;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  auto red = reinterpret_cast<float(*)[16 * kTiles][kPitch]>(smem);
  const unsigned groups = (w.rank + 63) / 64;
  // what reads the same rows of x is on one XCD
  const unsigned each = parts * groups * w.slices, tile = (blockIdx.x >> 3) / each * 8 + (blockIdx.x & 7);
  unsigned b = (blockIdx.x >> 3) % each;
  const unsigned part = b % parts;
  b /= parts;
  const unsigned group = b % groups, slice = b / groups;
  unsigned first, count, id;
  if (!plan_tile(p, tile, tokens, w.n, first, count, id)) return;
  const unsigned rank = adapter_rank(w, (int)id);
  if (64 * group >= rank) return;
  const int nt = (int)min((rank - 64 * group + 15) / 16, 4u);      // 16 rows of A each
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const unsigned len = w.k / (4 * parts), k0 = (part * 4 + wave) * len;
  const bf16* xp[kTiles];
#pragma unroll
  for (int m = 0; m < kTiles; ++m) {
    const unsigned row = (unsigned)p.rows[first + min((unsigned)(16 * m + li), count - 1)];
    xp[m] = x + (row < tokens ? row : 0u) * ldx + k0 + 8 * lg;
  }
  const bf16* ap[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const unsigned r = min(64 * group + 16 * c + li, w.rank - 1);
    ap[c] = w.a + ((size_t)id * w.slices + slice) * w.rank * w.k + (size_t)r * w.k + k0 + 8 * lg;
  }
  f32x4 acc[kTiles][4];
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[m][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const unsigned steps = len / 32;
  // operands are asked for three steps ahead
  bf16x8 xv[4][kTiles], av[4][4];
  auto load = [&](int s, unsigned k) {
#pragma unroll
    for (int m = 0; m < kTiles; ++m) xv[s][m] = *reinterpret_cast<const bf16x8*>(xp[m] + k);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < nt) av[s][c] = *reinterpret_cast<const bf16x8*>(ap[c] + k);
  };
#pragma unroll
  for (int s = 0; s < 3; ++s)
    if ((unsigned)s < steps) load(s, 32 * s);
#pragma unroll 1
  for (unsigned n = 0; n < steps; n += 4) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (n + s >= steps) break;
      if (n + s + 3 < steps) load((s + 3) & 3, 32 * (n + s + 3));
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c < nt) {
#pragma unroll
          for (int m = 0; m < kTiles; ++m) acc[m][c] = mfma16x16x32(av[s][c], xv[s][m], acc[m][c]);
        }
    }
  }
  // lane: h of row li, rank rows 16 c + 4 lg + r
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < nt) *reinterpret_cast<f32x4*>(&red[wave][16 * m + li][16 * c + 4 * lg]) = acc[m][c];
  __syncthreads();
  if (kFinal) {
    // the second launch's operands: 16 rows by 32 of the rank, high and low parts
    const float scale = w.scales != nullptr ? w.scales[id] : 1.0f;
    const unsigned nk = (w.rank + 31) / 32;
    bf16x8* o = reinterpret_cast<bf16x8*>(h) + ((size_t)tile * w.slices + slice) * kTiles * nk * 128;
    for (int it = wave; it < 2 * kTiles; it += 4) {
      const int m = it >> 1, kb = it & 1;
      if (64 * group + 32 * kb >= rank) continue;
      f32x4 s[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[e] = *reinterpret_cast<const f32x4*>(&red[0][16 * m + li][32 * kb + 8 * lg + 4 * e]);
#pragma unroll
        for (int u = 1; u < 4; ++u) s[e] += *reinterpret_cast<const f32x4*>(&red[u][16 * m + li][32 * kb + 8 * lg + 4 * e]);
      }
      bf16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = 64 * group + 32 * kb + 8 * lg + e < rank ? scale * s[e >> 2][e & 3] : 0.f;
        hi[e] = f2bf(v);
        lo[e] = f2bf(v - bf2f(hi[e]));
      }
      bf16x8* at = o + ((m * nk + 2 * group + kb) * 2) * 64 + lane;
      at[0] = hi;
      at[64] = lo;
    }
    return;
  }
  for (int it = tid; it < 16 * kTiles * 16; it += 256) {
    const unsigned row = it >> 4, c = 4 * (it & 15);
    if (row >= count || 64 * group + c >= rank) continue;
    f32x4 s = *reinterpret_cast<const f32x4*>(&red[0][row][c]);
#pragma unroll
    for (int u = 1; u < 4; ++u) s += *reinterpret_cast<const f32x4*>(&red[u][row][c]);
    *reinterpret_cast<f32x4*>(h + (((size_t)part * tokens + first + row) * w.slices + slice) * w.rank + 64 * group + c) = s;
  }
}

// The same for tiles of 64 rows by a ring of four stages in LDS, filled straight from
// memory, 128 bytes of a row at a time.  8,190 rows of K = 2048 beside three slices of rank
// 64: 23.6 us; 36 with operands from memory (adapter_down_kernel<4>, whatever its depth of
// prefetch and number of workgroups: a load of 16 rows 4 KB apart takes a CU some 80
// cycles), which is left for rows of x that reach behind 2^31 bytes.  Waves 2 x 2: 32 of
// the rank's rows by 32 rows of x.
using DownCfg = GemmCfg<1, 1, 2, 2, 2, 64, 4>;

template <bool kFinal>
__global__ __launch_bounds__(256, 2) void adapter_down_ring_kernel(const bf16* __restrict__ x, size_t ldx, Adapters w,
                                                                   Plan p, unsigned tokens, unsigned parts,
                                                                   float* __restrict__ h) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const unsigned groups = (w.rank + 63) / 64;
  const unsigned each = parts * groups * w.slices, tile = (blockIdx.x >> 3) / each * 8 + (blockIdx.x & 7);
  unsigned b = (blockIdx.x >> 3) % each;
  const unsigned part = b % parts;
  b /= parts;
  const unsigned group = b % groups, slice = b / groups;
  unsigned first, count, id;
  if (!plan_tile(p, tile, tokens, w.n, first, count, id)) return;
  const unsigned rank = adapter_rank(w, (int)id);
  if (64 * group >= rank) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave & 1, wn = wave >> 1, li = lane & 31;
  const unsigned len = w.k / parts;
  const u32x4 xr = g_rsrc(x + part * len, (unsigned)((((size_t)tokens - 1) * ldx + len) * 2));
  const u32x4 ar = g_rsrc(w.a + ((size_t)id * w.slices + slice) * w.rank * w.k + part * len,
                          ((rank - 1) * w.k + len) * 2);
  FetchPlan<DownCfg> fp;
#pragma unroll
  for (int j = 0; j < DownCfg::Instr; ++j) {
    const int srow = fetch_stage_row<DownCfg>(wave, j, lane);
    const unsigned at = fetch_chunk_off<DownCfg>(srow, lane);
    unsigned off = kGOob;
    if (srow < 64) {
      const unsigned r = 64 * group + srow;
      if (r < rank) off = r * w.k * 2 + at;
    } else if ((unsigned)(srow - 64) < count) {
      const unsigned r = (unsigned)p.rows[first + srow - 64];
      if (r < tokens) off = (unsigned)(r * ldx * 2) + at;
    }
    fp.off[j] = off;
    const bool mine = __builtin_amdgcn_readfirstlane(srow) < 64;     // a wave's rows are of one kind
    fp.rs[j] = mine ? ar : xr;
  }
  f32x16 acc[1][1];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[0][0][e] = 0.f;
  const int brow[1] = {64 + 32 * wn + li};
  gemm_mainloop<DownCfg>(smem, fp, (int)len, 32 * wm + li, brow, acc);
  // lane: row 32 wn + li of the tile, rank rows 64 group + 32 wm + 8 q + 4 kh + r
  const unsigned row = 32 * wn + li, kh = lane >> 5, r0 = 64 * group + 32 * wm + 4 * kh;
  if (kFinal) {
    const float scale = w.scales != nullptr ? w.scales[id] : 1.0f;
    const unsigned nk = (w.rank + 31) / 32, kb = 2 * group + wm;
    if (kb >= nk) return;
    bf16* o = reinterpret_cast<bf16*>(h) + (((size_t)tile * w.slices + slice) * 4 + (row >> 4)) * nk * 1024 + kb * 1024;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      bf16x4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = r0 + 8 * q + r < rank ? scale * acc[0][0][4 * q + r] : 0.f;
        hi[r] = f2bf(v);
        lo[r] = f2bf(v - bf2f(hi[r]));
      }
      bf16* at = o + (16 * q + (row & 15)) * 8 + 4 * kh;
      *reinterpret_cast<bf16x4*>(at) = hi;
      *reinterpret_cast<bf16x4*>(at + 512) = lo;
    }
  } else if (row < count) {
    float* o = h + (((size_t)part * tokens + first + row) * w.slices + slice) * w.rank;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (r0 + 8 * q < w.rank)
        *reinterpret_cast<f32x4*>(o + r0 + 8 * q) =
            f32x4{acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]};
  }
}

// ---- up: y += (scale h) B^T -----------------------------------------------------

constexpr unsigned kUpCols = 256;        // of a workgroup: 64 a wave, in two halves

// Workgroup: (tile, 256 columns of a slice).  The product is taken transposed (B's rows
// first), its row 4 j + r standing for column 8 j + 4 u + r of the pair u = 0, 1, so that
// a lane holds 8 columns in a row of y: 16-byte reads and writes.  All of y and B's
// first 64 of the rank are asked for at once; 16 waves a CU hide the rest.
template <int kTiles, int kParts>
__global__ __launch_bounds__(256, kTiles == 1 ? 4 : 3) void adapter_up_kernel(bf16* __restrict__ y, size_t ldy, Adapters w, Plan p,
                                                            unsigned tokens, unsigned chunks,
                                                            const float* __restrict__ h) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  bf16x8* hs = reinterpret_cast<bf16x8*>(smem);      // [tile of 16][32 of the rank][high, low][lane]
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const unsigned tile = blockIdx.x / chunks;
  unsigned chunk = blockIdx.x % chunks, slice = 0, first, count, id;
  if (!plan_tile(p, tile, tokens, w.n, first, count, id)) return;
  unsigned row[kTiles];
#pragma unroll
  for (int m = 0; m < kTiles; ++m) row[m] = (unsigned)p.rows[first + min((unsigned)(16 * m + li), count - 1)];
  const unsigned rank = adapter_rank(w, (int)id);
  if (rank == 0) return;
  while (slice + 1 < w.slices) {
    const unsigned n = (w.begin[slice + 1] - w.begin[slice] + kUpCols - 1) / kUpCols;
    if (chunk < n) break;
    chunk -= n;
    ++slice;
  }
  const unsigned end = w.begin[slice + 1], c0 = w.begin[slice] + chunk * kUpCols + 64 * wave;
  const unsigned nk = (rank + 31) / 32;
  const bf16* bp = w.b + (size_t)id * w.total * w.rank;
  // half g: columns from c0 + 32 g on; what is behind the slice, or a row that is none,
  // is read from where there is something
  bf16x8 yv[2][kTiles], bv[2][2][2];
  auto load_b = [&](int g, unsigned kb, bf16x8 (&o)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const unsigned col = min(c0 + 32 * g + 8 * (li >> 2) + 4 * u + (li & 3), end - 1);
      o[u] = *reinterpret_cast<const bf16x8*>(bp + (size_t)col * w.rank + min(32 * kb + 8 * lg, w.rank - 8));
    }
  };
#pragma unroll
  for (int m = 0; m < kTiles; ++m) {
    const bf16* yr = y + (row[m] < tokens ? row[m] : 0u) * ldy;
#pragma unroll
    for (int g = 0; g < 2; ++g)
      yv[g][m] = *reinterpret_cast<const bf16x8*>(yr + min(c0 + 32 * g + 8 * lg, end - 8));
  }
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    load_b(g, 0, bv[g][0]);
    if (nk > 1) load_b(g, 1, bv[g][1]);
  }
  if constexpr (kParts == 1) {
    const unsigned full = (w.rank + 31) / 32;
    const bf16x8* from = reinterpret_cast<const bf16x8*>(h) + ((size_t)tile * w.slices + slice) * kTiles * full * 128;
    for (unsigned it = tid; it < kTiles * nk * 128; it += 256) {
      const unsigned m = it / (nk * 128);
      hs[it] = from[it + m * (full - nk) * 128];
    }
  } else {
    // the scaled h as two bf16 values
    const float scale = w.scales != nullptr ? w.scales[id] : 1.0f;
    for (unsigned it = tid; it < 16 * kTiles * 4 * nk; it += 256) {
      const unsigned hr = it / (4 * nk), j = it % (4 * nk);       // 8 of the rank
      bf16x8 hi = {}, lo = {};
      if (8 * j < rank && hr < count) {
        f32x4 s[kParts][2];
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
          const f32x4* hp = reinterpret_cast<const f32x4*>(
              h + (((size_t)q * tokens + first + hr) * w.slices + slice) * w.rank + 8 * j);
          s[q][0] = hp[0];
          s[q][1] = hp[1];
        }
#pragma unroll
        for (int q = 1; q < kParts; ++q) {
          s[0][0] += s[q][0];
          s[0][1] += s[q][1];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = 8 * j + e < rank ? scale * s[0][e >> 2][e & 3] : 0.f;
          hi[e] = f2bf(v);
          lo[e] = f2bf(v - bf2f(hi[e]));
        }
      }
      bf16x8* o = hs + (((hr >> 4) * nk + (j >> 2)) * 2) * 64 + 16 * (j & 3) + (hr & 15);
      o[0] = hi;
      o[64] = lo;
    }
  }
  __syncthreads();
  if (c0 >= end) return;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    f32x4 acc[2][kTiles];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int m = 0; m < kTiles; ++m) acc[u][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto products = [&](unsigned kb, bf16x8 (&b)[2]) {
      if (32 * kb + 32 > rank) {           // what stands behind the adapter's rank may be anything
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (32 * kb + 8 * lg + e >= rank) b[u][e] = (bf16)0.f;
      }
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        const bf16x8 hi = hs[((m * nk + kb) * 2) * 64 + lane], lo = hs[((m * nk + kb) * 2 + 1) * 64 + lane];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          acc[u][m] = mfma16x16x32(b[u], lo, acc[u][m]);
          acc[u][m] = mfma16x16x32(b[u], hi, acc[u][m]);
        }
      }
    };
    products(0, bv[g][0]);
    if (nk > 1) products(1, bv[g][1]);
#pragma unroll 1
    for (unsigned kb = 2; kb < nk; ++kb) {
      bf16x8 b[2];
      load_b(g, kb, b);
      products(kb, b);
    }
    const unsigned col = c0 + 32 * g + 8 * lg;
    if (col >= end) continue;
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
      if ((unsigned)(16 * m + li) >= count || row[m] >= tokens) continue;
      bf16x8 o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = f2bf(bf2f(yv[g][m][e]) + acc[e >> 2][m][e & 3]);
      *reinterpret_cast<bf16x8*>(y + row[m] * ldy + col) = o;
    }
  }
}

unsigned tile_rows(unsigned tokens) { return tokens <= kFewRows ? 16 : 64; }
unsigned most_tiles(unsigned seqs, unsigned tokens, unsigned n) {
  return tokens / tile_rows(tokens) + (n < seqs ? n : seqs);
}

bool adapters_of(const qwen36_adapters* p, Adapters& w) {
  if (p == nullptr || p->a == nullptr || p->b == nullptr || !aligned16(p->a) || !aligned16(p->b) ||
      p->adapters == 0 || p->adapters > kMaxAdapters || p->rank == 0 || p->rank > kMaxRank || p->rank % 8 != 0 ||
      p->k == 0 || p->k > 16384 || p->k % 128 != 0 || p->slices == 0 || p->slices > kMaxSlices)
    return false;
  w.a = static_cast<const bf16*>(p->a);
  w.b = static_cast<const bf16*>(p->b);
  w.ranks = static_cast<const int*>(p->ranks);
  w.scales = static_cast<const float*>(p->scales);
  w.n = p->adapters;
  w.rank = p->rank;
  w.k = p->k;
  w.slices = p->slices;
  w.total = 0;
  for (unsigned s = 0; s < p->slices; ++s) {
    if (p->widths[s] == 0 || p->widths[s] % 8 != 0 || p->widths[s] > 65536) return false;
    w.begin[s] = w.total;
    w.total += p->widths[s];
  }
  for (unsigned s = p->slices; s <= kMaxSlices; ++s) w.begin[s] = w.total;
  return w.total <= 65536;
}

// Parts of K: for few tiles so many that 256 workgroups share the adapters' reads (61 rows of
// 17 adapters: 5.6 us and 6.7 for the sums and the second launch; with 512, 6.1 and 7.5).
unsigned k_parts(const Adapters& w, unsigned tiles) {
  unsigned parts = 1;
  while (parts < 8 && w.k % (256 * parts) == 0 && (size_t)tiles * w.slices * ((w.rank + 63) / 64) * parts < 256)
    parts *= 2;
  return parts;
}

bool batch_ok(unsigned seqs, unsigned tokens) {
  return seqs > 0 && seqs <= 65536 && tokens > 0 && tokens <= kMaxTokens;
}

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT size_t qwen36_adapter_plan_bytes(unsigned seqs, unsigned tokens, unsigned adapters) {
  if (!batch_ok(seqs, tokens) || adapters == 0 || adapters > kMaxAdapters) return 0;
  return ((size_t)4 * (1 + most_tiles(seqs, tokens, adapters)) + tokens) * 4;
}

Q36_EXPORT int qwen36_adapter_plan(const void* cu_tokens, const void* adapter_ids, unsigned seqs, unsigned tokens,
                                   unsigned adapters, void* plan, size_t plan_bytes, void* stream) {
  const size_t need = qwen36_adapter_plan_bytes(seqs, tokens, adapters);
  if (need == 0 || cu_tokens == nullptr || adapter_ids == nullptr || plan == nullptr || !aligned16(plan) ||
      plan_bytes < need)
    return Q36_EINVAL;
  const unsigned most = most_tiles(seqs, tokens, adapters);
  int* tiles = static_cast<int*>(plan);
  hipLaunchKernelGGL(adapter_plan_kernel, dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream),
                     static_cast<const int*>(cu_tokens), static_cast<const int*>(adapter_ids), seqs, tokens, adapters,
                     tile_rows(tokens), most, tiles, tiles + 4 * (1 + most));
  return static_cast<int>(hipGetLastError());
}

Q36_EXPORT size_t qwen36_adapter_workspace_bytes(const qwen36_adapters* adapters, unsigned seqs, unsigned tokens) {
  Adapters w;
  if (!adapters_of(adapters, w) || !batch_ok(seqs, tokens)) return 0;
  const unsigned most = most_tiles(seqs, tokens, w.n);
  const unsigned parts = k_parts(w, most);
  if (parts == 1) return (size_t)most * w.slices * tile_rows(tokens) * ((w.rank + 31) / 32) * 128;
  return (size_t)parts * tokens * w.slices * w.rank * 4;
}

Q36_EXPORT int qwen36_adapter_apply(const void* x, size_t x_row_stride, void* y, size_t y_row_stride,
                                    const qwen36_adapters* adapters, const void* plan, size_t plan_bytes,
                                    unsigned seqs, unsigned tokens, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  Adapters w;
  if (x == nullptr || y == nullptr || plan == nullptr || workspace == nullptr || !adapters_of(adapters, w) ||
      !batch_ok(seqs, tokens) || x_row_stride < w.k || y_row_stride < w.total || x_row_stride % 8 != 0 ||
      y_row_stride % 8 != 0 || !aligned16(x) || !aligned16(y) || !aligned16(plan) || !aligned16(workspace) ||
      plan_bytes < qwen36_adapter_plan_bytes(seqs, tokens, w.n) ||
      workspace_bytes < qwen36_adapter_workspace_bytes(adapters, seqs, tokens))
    return Q36_EINVAL;
  static std::once_flag once;
  static hipError_t attr = hipSuccess;
  std::call_once(once, [] {
    auto allow = [](const void* f, int bytes) {
      if (attr == hipSuccess) attr = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    allow(reinterpret_cast<const void*>(adapter_down_kernel<4, true>), 4 * 64 * kDownPitch * 4);
    allow(reinterpret_cast<const void*>(adapter_down_kernel<4, false>), 4 * 64 * kDownPitch * 4);
    allow(reinterpret_cast<const void*>(adapter_down_ring_kernel<true>), DownCfg::Lds);
    allow(reinterpret_cast<const void*>(adapter_down_ring_kernel<false>), DownCfg::Lds);
  });
  if (attr != hipSuccess) return static_cast<int>(attr);
  const unsigned most = most_tiles(seqs, tokens, w.n), parts = k_parts(w, most);
  unsigned chunks = 0;
  for (unsigned s = 0; s < w.slices; ++s) chunks += (w.begin[s + 1] - w.begin[s] + kUpCols - 1) / kUpCols;
  const int* tiles = static_cast<const int*>(plan);
  const Plan p = {tiles, tiles + 4 * (1 + most)};
  const bf16* xb = static_cast<const bf16*>(x);
  bf16* yb = static_cast<bf16*>(y);
  float* h = static_cast<float*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 down((most + 7) / 8 * 8 * w.slices * ((w.rank + 63) / 64) * parts), up(most * chunks);
  const unsigned index = (w.rank + 31) / 32 * 2048;      // bytes of 16 rows of h
  const unsigned tiles16 = tile_rows(tokens) / 16;
  // a ring's offsets into x are of 31 bits
  const bool ring = tiles16 == 4 && w.k / parts % 64 == 0 &&
                    (((size_t)tokens - 1) * x_row_stride + w.k) * 2 <= (size_t)kGOob;
  const unsigned lds = ring ? DownCfg::Lds : 4 * 16 * tiles16 * kDownPitch * 4;
  auto launch = [&](auto down_kernel, auto up_kernel) {
    hipLaunchKernelGGL(down_kernel, down, dim3(256), lds, st, xb, x_row_stride, w, p, tokens, parts, h);
    hipLaunchKernelGGL(up_kernel, up, dim3(256), tiles16 * index, st, yb, y_row_stride, w, p, tokens, chunks, h);
  };
  if (tiles16 == 1) {
    if (parts == 1) launch(adapter_down_kernel<1, true>, adapter_up_kernel<1, 1>);
    else if (parts == 2) launch(adapter_down_kernel<1, false>, adapter_up_kernel<1, 2>);
    else if (parts == 4) launch(adapter_down_kernel<1, false>, adapter_up_kernel<1, 4>);
    else launch(adapter_down_kernel<1, false>, adapter_up_kernel<1, 8>);
  } else {
    auto pair = [&](auto up_kernel) {
      if (parts == 1 && ring) launch(adapter_down_ring_kernel<true>, up_kernel);
      else if (parts == 1) launch(adapter_down_kernel<4, true>, up_kernel);
      else if (ring) launch(adapter_down_ring_kernel<false>, up_kernel);
      else launch(adapter_down_kernel<4, false>, up_kernel);
    };
    if (parts == 1) pair(adapter_up_kernel<4, 1>);
    else if (parts == 2) pair(adapter_up_kernel<4, 2>);
    else if (parts == 4) pair(adapter_up_kernel<4, 4>);
    else pair(adapter_up_kernel<4, 8>);
  }
  return static_cast<int>(hipGetLastError());
}
