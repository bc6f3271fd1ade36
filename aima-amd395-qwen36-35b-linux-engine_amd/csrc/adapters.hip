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
//    of two bf16 values (2^-17 of it), both in one product: the reduction index runs over
//    [high rank | low rank] against B twice, so that rank 16 fills one 16x16x32.
// Results depend neither on the order of the requests nor on the tile: a row of a
// product is computed the same in whatever row of a tile it stands.
#include "paged_common.h"

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
  if (i >= (unsigned)p.tiles[0]) return false;
  const int4 t = *reinterpret_cast<const int4*>(p.tiles + 4 * (1 + i));
  first = (unsigned)t.x;
  count = (unsigned)t.y;
  id = (unsigned)t.z;
  return id < n && first < tokens && count <= tokens - first;
}

// ---- down: h = x A^T ----------------------------------------------------------

// Workgroup: (tile, slice, 64 of the rank's rows, part of K); its waves a quarter of the
// part each.  h: [part][place][slice][rank] fp32.
template <int kTiles>     // of 16 rows
__global__ __launch_bounds__(256) void adapter_down_kernel(const bf16* __restrict__ x, size_t ldx, Adapters w, Plan p,
                                                           unsigned tokens, unsigned parts, float* __restrict__ h) {
  constexpr int kPitch = 68;
  __shared__ float red[3][16 * kTiles][kPitch];
  const unsigned groups = (w.rank + 63) / 64;
  unsigned b = blockIdx.x;
  const unsigned part = b % parts;
  b /= parts;
  const unsigned group = b % groups;
  b /= groups;
  const unsigned slice = b % w.slices;
  unsigned first, count, id;
  if (!plan_tile(p, b / w.slices, tokens, w.n, first, count, id)) return;
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
  for (unsigned k = 0; k < len; k += 32) {
    bf16x8 xv[kTiles], av[4];
#pragma unroll
    for (int m = 0; m < kTiles; ++m) xv[m] = *reinterpret_cast<const bf16x8*>(xp[m] + k);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < nt) av[c] = *reinterpret_cast<const bf16x8*>(ap[c] + k);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < nt) {
#pragma unroll
        for (int m = 0; m < kTiles; ++m) acc[m][c] = mfma16x16x32(av[c], xv[m], acc[m][c]);
      }
  }
  // lane: h of row li, rank rows 16 c + 4 lg + r
  if (wave > 0) {
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c < nt) *reinterpret_cast<f32x4*>(&red[wave - 1][16 * m + li][16 * c + 4 * lg]) = acc[m][c];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int m = 0; m < kTiles; ++m) {
    const unsigned row = 16 * m + li;
    if (row >= count) continue;
    float* o = h + (((size_t)part * tokens + first + row) * w.slices + slice) * w.rank + 64 * group + 4 * lg;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c >= nt) continue;
      f32x4 s = acc[m][c];
#pragma unroll
      for (int u = 0; u < 3; ++u) s += *reinterpret_cast<const f32x4*>(&red[u][row][16 * c + 4 * lg]);
      if (64 * group + 16 * c + 4 * lg < w.rank) *reinterpret_cast<f32x4*>(o + 16 * c) = s;
    }
  }
}

// ---- up: y += (scale h) B^T -----------------------------------------------------

constexpr unsigned kUpCols = 256;        // of a workgroup: 64 a wave

// Workgroup: (tile, 256 columns of a slice).  The product is taken transposed (B's rows
// first), its row 4 j + r standing for column 8 j + 4 u + r of the pair u = 0, 1, so that
// a lane holds 8 columns in a row of y: 16-byte reads and writes.
template <int kTiles>
__global__ __launch_bounds__(256) void adapter_up_kernel(bf16* __restrict__ y, size_t ldy, Adapters w, Plan p,
                                                         unsigned tokens, unsigned parts, unsigned chunks,
                                                         const float* __restrict__ h) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  bf16x8* hs = reinterpret_cast<bf16x8*>(smem);      // [tile of 16][32 of the index][lane]
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  unsigned chunk = blockIdx.x % chunks, slice = 0, first, count, id;
  if (!plan_tile(p, blockIdx.x / chunks, tokens, w.n, first, count, id)) return;
  const unsigned rank = adapter_rank(w, (int)id);
  if (rank == 0) return;
  while (slice + 1 < w.slices) {
    const unsigned n = (w.begin[slice + 1] - w.begin[slice] + kUpCols - 1) / kUpCols;
    if (chunk < n) break;
    chunk -= n;
    ++slice;
  }
  const unsigned end = w.begin[slice + 1], c0 = w.begin[slice] + chunk * kUpCols + 64 * wave;
  // y's values of this lane: row 16 m + li, columns c0 + 32 g + 8 lg .. + 7
  bf16* yp[kTiles];
  bf16x8 yv[kTiles][2];
#pragma unroll
  for (int m = 0; m < kTiles; ++m) {
    const unsigned at = 16 * m + li;
    const unsigned row = at < count ? (unsigned)p.rows[first + at] : tokens;
    yp[m] = row < tokens ? y + row * ldy + c0 + 8 * lg : nullptr;
#pragma unroll
    for (int g = 0; g < 2; ++g)
      if (yp[m] != nullptr && c0 + 32 * g + 8 * lg < end) yv[m][g] = *reinterpret_cast<const bf16x8*>(yp[m] + 32 * g);
  }
  // the scaled h as two bf16 values: [high, 0 to r8 | low, r8 to 2 r8 | zeros]
  const unsigned r8 = (rank + 7) & ~7u, nk = (2 * r8 + 31) / 32;
  const float scale = w.scales != nullptr ? w.scales[id] : 1.0f;
  const unsigned eights = 4 * nk;
  for (unsigned it = tid; it < 16 * kTiles * (eights - r8 / 8); it += 256) {
    const unsigned row = it % (16 * kTiles), j = it / (16 * kTiles);       // 8 of the rank, or zeros
    bf16x8 hi = {}, lo = {};
    if (j < r8 / 8 && row < count) {
      float s[8] = {};
      for (unsigned q = 0; q < parts; ++q) {
        const f32x4* hp = reinterpret_cast<const f32x4*>(
            h + (((size_t)q * tokens + first + row) * w.slices + slice) * w.rank + 8 * j);
        const f32x4 u = hp[0], v = hp[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[e] += u[e];
          s[4 + e] += v[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = 8 * j + e < rank ? scale * s[e] : 0.f;
        hi[e] = f2bf(v);
        lo[e] = f2bf(v - bf2f(hi[e]));
      }
    }
    auto put = [&](unsigned at, const bf16x8& v) {
      hs[((row >> 4) * nk + (at >> 2)) * 64 + 16 * (at & 3) + (row & 15)] = v;
    };
    if (j < r8 / 8) {
      put(j, hi);
      put(r8 / 8 + j, lo);
    } else {
      put(r8 / 8 + j, hi);
    }
  }
  __syncthreads();
  if (c0 >= end) return;
  f32x4 acc[2][2][kTiles];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int m = 0; m < kTiles; ++m) acc[g][u][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bf16* bp = w.b + (size_t)id * w.total * w.rank;
  for (unsigned kb = 0; kb < nk; ++kb) {
    const unsigned kk = 32 * kb + 8 * lg, at = kk < r8 ? kk : kk < 2 * r8 ? kk - r8 : 0u;
    bf16x8 bv[2][2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned col = min(c0 + 32 * g + 8 * (li >> 2) + 4 * u + (li & 3), end - 1);
        bv[g][u] = *reinterpret_cast<const bf16x8*>(bp + (size_t)col * w.rank + at);
        // what stands behind the adapter's rank, or against the zeros, may be anything
        if (at + 8 > rank || kk >= 2 * r8) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (at + e >= rank || kk >= 2 * r8) bv[g][u][e] = (bf16)0.f;
        }
      }
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
      const bf16x8 hv = hs[(m * nk + kb) * 64 + lane];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int u = 0; u < 2; ++u) acc[g][u][m] = mfma16x16x32(bv[g][u], hv, acc[g][u][m]);
    }
  }
#pragma unroll
  for (int m = 0; m < kTiles; ++m) {
    if (yp[m] == nullptr) continue;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (c0 + 32 * g + 8 * lg >= end) continue;
      bf16x8 o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = f2bf(bf2f(yv[m][g][e]) + acc[g][e >> 2][m][e & 3]);
      *reinterpret_cast<bf16x8*>(yp[m] + 32 * g) = o;
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

// Parts of K: for few tiles so many that 512 workgroups share the adapters' reads.
unsigned k_parts(const Adapters& w, unsigned tiles) {
  unsigned parts = 1;
  while (parts < 8 && w.k % (256 * parts) == 0 && (size_t)tiles * w.slices * ((w.rank + 63) / 64) * parts < 512)
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
  return (size_t)k_parts(w, most) * tokens * w.slices * w.rank * 4;
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
  const unsigned most = most_tiles(seqs, tokens, w.n), parts = k_parts(w, most);
  unsigned chunks = 0;
  for (unsigned s = 0; s < w.slices; ++s) chunks += (w.begin[s + 1] - w.begin[s] + kUpCols - 1) / kUpCols;
  const int* tiles = static_cast<const int*>(plan);
  const Plan p = {tiles, tiles + 4 * (1 + most)};
  const bf16* xb = static_cast<const bf16*>(x);
  bf16* yb = static_cast<bf16*>(y);
  float* h = static_cast<float*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 down(most * w.slices * ((w.rank + 63) / 64) * parts), up(most * chunks);
  const unsigned index = (2 * w.rank + 31) / 32 * 1024;      // bytes of 16 rows of h
  if (tile_rows(tokens) == 16) {
    hipLaunchKernelGGL(adapter_down_kernel<1>, down, dim3(256), 0, st, xb, x_row_stride, w, p, tokens, parts, h);
    hipLaunchKernelGGL(adapter_up_kernel<1>, up, dim3(256), index, st, yb, y_row_stride, w, p, tokens, parts, chunks, h);
  } else {
    hipLaunchKernelGGL(adapter_down_kernel<4>, down, dim3(256), 0, st, xb, x_row_stride, w, p, tokens, parts, h);
    hipLaunchKernelGGL(adapter_up_kernel<4>, up, dim3(256), 4 * index, st, yb, y_row_stride, w, p, tokens, parts,
                       chunks, h);
  }
  return static_cast<int>(hipGetLastError());
}
