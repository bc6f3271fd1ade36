// Who holds which page of a paged cache: giving rows up, forking and growing them,
// and moving the held pages together.
//
// refs[p] counts the table entries that name page p; a page of no count is free.
// Every call works on rows of the whole table, so that no row can be named twice:
//  * trim: rows keep at most keep[i] tokens; pages behind them lose a count.
//  * fork: an empty row becomes parent[i]'s, whose pages gain a count each.
//  * extend: rows grow by add[i] tokens.  A last page that is not full and not held
//    alone is never written: the row gets a copy of it.  Free pages are given out in
//    ascending order to the rows in theirs, to each row all or nothing.
//  * compact: with n pages held, those at n or behind go to the free ones before n,
//    in ascending order.
// The numbers are whole and every choice goes by order, not by timing.
//
// trim and fork are a workgroup a row (a chain of three dependent loads); extend and
// compact do their bookkeeping in one workgroup, which scans 16,384 counts a step,
// and a second launch copies the pages.  Copies are bound by their bytes (6 layers'
// compaction of 461 MB: 97 us, 4.8 TB/s); the bookkeeping by latency (5 to 12 us a step,
// which holds any pool of a few thousand pages; 400K pages take 25, once for all layers).
#include "paged_common.h"

namespace q36 {
namespace {

struct Tables {
  int* refs;
  int* table;
  int* lens;
  size_t stride;
  unsigned pages, page, width, rows;
  int max_len;
};

// Tokens of a row; -1 where the number is none (the row is left alone).
__device__ __forceinline__ int row_len(const Tables& t, unsigned i) {
  const int n = t.lens[i];
  return n >= 0 && n <= t.max_len ? n : -1;
}
__device__ __forceinline__ int pages_of(int tokens, unsigned page) { return (tokens + (int)page - 1) / (int)page; }

__global__ __launch_bounds__(256) void pages_trim_kernel(Tables t, const int* __restrict__ keep) {
  const unsigned i = blockIdx.x;
  const int len = row_len(t, i), kept = max(keep[i], 0);
  __syncthreads();   // the length is written below
  if (len < 0 || kept >= len) return;
  int* row = t.table + i * t.stride;
  for (int c = pages_of(kept, t.page) + (int)threadIdx.x; c < pages_of(len, t.page); c += 256) {
    const int p = row[c];
    if ((unsigned)p < t.pages) atomicSub(&t.refs[p], 1);
    row[c] = -1;
  }
  if (threadIdx.x == 0) t.lens[i] = kept;
}

__global__ __launch_bounds__(256) void pages_fork_kernel(Tables t, const int* __restrict__ parent) {
  const unsigned i = blockIdx.x;
  const int p = parent[i];
  if ((unsigned)p >= t.rows || (unsigned)p == i) return;
  // a parent is no child of the same call, so its row stays as it is
  const int mine = row_len(t, i), len = row_len(t, p);
  const bool ok = parent[p] < 0 && mine == 0 && len > 0;
  __syncthreads();   // the length is written below
  if (!ok) return;
  const int* from = t.table + p * t.stride;
  int* row = t.table + i * t.stride;
  for (int c = threadIdx.x; c < pages_of(len, t.page); c += 256) {
    const int x = from[c];
    row[c] = x;
    if ((unsigned)x < t.pages) atomicAdd(&t.refs[x], 1);
  }
  if (threadIdx.x == 0) t.lens[i] = len;
}

constexpr unsigned kBlock = 1024, kPer = 16, kStep = kBlock * kPer;   // counts a step
constexpr unsigned kRowsInLds = 4096;

// Inclusive sum over the workgroup, and the whole.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* lds, unsigned& total) {
  const unsigned wave = threadIdx.x >> 6;
  const unsigned in = wave_scan_add(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[wave] = in;
  __syncthreads();
  unsigned before = 0;
  total = 0;
#pragma unroll
  for (unsigned w = 0; w < kBlock / 64; ++w) {
    const unsigned s = lds[w];
    if (w < wave) before += s;
    total += s;
  }
  return before + in;
}

// This thread's counts of the step at page `at` (behind the pool: held).
__device__ __forceinline__ void read_counts(const int* refs, unsigned pages, unsigned at, int (&r)[kPer]) {
  const unsigned p0 = at + threadIdx.x * kPer;
  if (p0 + kPer <= pages && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
#pragma unroll
    for (unsigned u = 0; u < kPer / 4; ++u) {
      const int4 v = reinterpret_cast<const int4*>(refs + p0)[u];
      r[4 * u] = v.x;
      r[4 * u + 1] = v.y;
      r[4 * u + 2] = v.z;
      r[4 * u + 3] = v.w;
    }
  } else {
#pragma unroll
    for (unsigned u = 0; u < kPer; ++u) r[u] = p0 + u < pages ? refs[p0 + u] : 1;
  }
}

// Where a call's second launch finds its copies: moves[0] of them, from src to dst.
struct Moves {
  unsigned* count;
  int* src;
  int* dst;
};

// until[i]: pages that rows 0 .. i ask for together; first[i]: the first column that
// gets one (its top bit: that page is copied).
__global__ __launch_bounds__(kBlock) void pages_extend_kernel(Tables t, const int* __restrict__ add,
                                                              int* __restrict__ granted, int* until_ws, int* first,
                                                              int* src_of, int* dst_of, Moves m) {
  __shared__ unsigned sums[16];
  __shared__ int until_lds[kRowsInLds];
  int* until = t.rows <= kRowsInLds ? until_lds : until_ws;
  const unsigned tid = threadIdx.x;
  int r[kPer];
  read_counts(t.refs, t.pages, 0, r);      // a pool of one step is read once, and before all else
  unsigned need = 0;
  for (unsigned i0 = 0; i0 < t.rows; i0 += kBlock) {
    const unsigned i = i0 + tid;
    unsigned mine = 0;
    if (i < t.rows) {
      const int len = row_len(t, i), grow = add[i];
      int at = 0;
      if (len >= 0 && grow > 0 && grow <= t.max_len - len) {
        const int have = pages_of(len, t.page), want = pages_of(len + grow, t.page);
        const int last = have > 0 && len % (int)t.page ? t.table[i * t.stride + have - 1] : -1;
        const bool copy = (unsigned)last < t.pages && t.refs[last] > 1;
        mine = want - have + copy;
        at = (have - copy) | (copy ? (int)0x80000000 : 0);
        if (copy) src_of[i] = last;
      }
      first[i] = at;
    }
    unsigned total;
    const unsigned in = block_scan(mine, sums, total);
    if (i < t.rows) until[i] = (int)(need + in);
    need += total;
  }
  __syncthreads();
  // free pages: all there are, or as many as are asked for
  unsigned there = 0;
  for (unsigned at = 0; at < t.pages && there < need; at += kStep) {
    if (at > 0) read_counts(t.refs, t.pages, at, r);
    unsigned n = 0, total;
#pragma unroll
    for (unsigned u = 0; u < kPer; ++u) n += r[u] <= 0;
    block_scan(n, sums, total);
    there += total;
  }
  // give them out: the k-th free page is the k-th that is asked for
  unsigned base = 0;
  for (unsigned at = 0; at < t.pages && base < need; at += kStep) {
    if (t.pages > kStep) read_counts(t.refs, t.pages, at, r);
    unsigned n = 0, total;
#pragma unroll
    for (unsigned u = 0; u < kPer; ++u) n += r[u] <= 0;
    unsigned k = base + block_scan(n, sums, total) - n;
    // the first row with until > k; for the thread's next pages it is this one or one behind
    unsigned lo = 0, hi = t.rows - 1;
    if (n > 0 && k < need)
      while (lo < hi) {
        const unsigned mid = (lo + hi) / 2;
        if ((unsigned)until[mid] > k) hi = mid; else lo = mid + 1;
      }
    // (the scan's barriers stand between the step's reads and the counts written below)
#pragma unroll
    for (unsigned u = 0; u < kPer; ++u) {
      if (r[u] > 0 || k >= need) continue;
      while ((unsigned)until[lo] <= k) ++lo;
      if ((unsigned)until[lo] <= there) {
        const unsigned before = lo ? (unsigned)until[lo - 1] : 0u;
        const int page = (int)(at + tid * kPer + u);
        const int f = first[lo];
        t.table[lo * t.stride + (f & 0x7fffffff) + (k - before)] = page;
        t.refs[page] = 1;
        if (f < 0 && k == before) dst_of[lo] = page;
      }
      ++k;
    }
    base += total;
  }
  __syncthreads();
  unsigned moved = 0;
  for (unsigned i0 = 0; i0 < t.rows; i0 += kBlock) {
    const unsigned i = i0 + tid;
    bool copy = false;
    if (i < t.rows) {
      const int len = row_len(t, i), grow = add[i];
      const unsigned before = i ? (unsigned)until[i - 1] : 0u, mine = (unsigned)until[i] - before;
      const bool fits = len >= 0 && grow > 0 && grow <= t.max_len - len;
      const bool ok = fits && (mine == 0 || (unsigned)until[i] <= there);
      if (ok) t.lens[i] = len + grow;
      granted[i] = ok || (len >= 0 && grow <= 0);
      copy = ok && first[i] < 0;
      if (copy) atomicSub(&t.refs[src_of[i]], 1);
    }
    unsigned total;
    const unsigned in = block_scan(copy, sums, total);
    if (copy) {
      m.src[moved + in - 1] = src_of[i];
      m.dst[moved + in - 1] = dst_of[i];
    }
    moved += total;
  }
  if (tid == 0) *m.count = moved;
}

// The same where a row is a thread and the pool one step: rows stay in registers, and one
// exchange sums the pages asked for, the free ones and the copies.  86 rows over 3,300
// pages: 7.5 us, 12.2 by the form above; 5 rows over 512: 5.3 and 8.4.
__global__ __launch_bounds__(kBlock) void pages_extend_few_kernel(Tables t, const int* __restrict__ add,
                                                                  int* __restrict__ granted, Moves m) {
  __shared__ uint2 sums[16];
  __shared__ unsigned until[kBlock];
  __shared__ int first[kBlock], dst_of[kBlock];
  __shared__ unsigned moved;
  const unsigned tid = threadIdx.x, wave = tid >> 6;
  int r[kPer];
  read_counts(t.refs, t.pages, 0, r);
  int len = -1, grow = 0, at = 0, src = -1;
  bool fits = false, copy = false;
  unsigned mine = 0;
  if (tid < t.rows) {
    len = row_len(t, tid);
    grow = add[tid];
    fits = len >= 0 && grow > 0 && grow <= t.max_len - len;
    if (fits) {
      const int have = pages_of(len, t.page), want = pages_of(len + grow, t.page);
      src = have > 0 && len % (int)t.page ? t.table[tid * t.stride + have - 1] : -1;
      copy = (unsigned)src < t.pages && t.refs[src] > 1;
      mine = want - have + copy;
      at = (have - copy) | (copy ? (int)0x80000000 : 0);
    }
  }
  unsigned n = 0;
#pragma unroll
  for (unsigned u = 0; u < kPer; ++u) n += r[u] <= 0;
  // free pages (at most 2^14) below the copies (2^10)
  const unsigned a = wave_scan_add(mine), b = wave_scan_add(n | (copy ? 1u << 16 : 0u));
  if ((tid & 63) == 63) sums[wave] = uint2{a, b};
  if (tid == 0) moved = 0;
  __syncthreads();
  unsigned need = 0, other = 0, mine_to = a, other_to = b;
#pragma unroll
  for (unsigned w = 0; w < kBlock / 64; ++w) {
    const uint2 s = sums[w];
    if (w < wave) {
      mine_to += s.x;
      other_to += s.y;
    }
    need += s.x;
    other += s.y;
  }
  const unsigned there = other & 0xffffu;
  until[tid] = mine_to;
  first[tid] = at;
  __syncthreads();
  // give them out: the k-th free page is the k-th that is asked for
  unsigned k = (other_to & 0xffffu) - n, lo = 0, hi = t.rows - 1;
  if (n > 0 && k < need)
    while (lo < hi) {
      const unsigned mid = (lo + hi) / 2;
      if (until[mid] > k) hi = mid; else lo = mid + 1;
    }
#pragma unroll
  for (unsigned u = 0; u < kPer; ++u) {
    if (r[u] > 0 || k >= need) continue;
    while (until[lo] <= k) ++lo;
    if (until[lo] <= there) {
      const unsigned before = lo ? until[lo - 1] : 0u;
      const int page = (int)(tid * kPer + u), f = first[lo];
      t.table[lo * t.stride + (f & 0x7fffffff) + (k - before)] = page;
      t.refs[page] = 1;
      if (f < 0 && k == before) dst_of[lo] = page;
    }
    ++k;
  }
  __syncthreads();
  if (tid < t.rows) {
    // a row that gets its pages has them after all rows before it, their copies among them
    const bool ok = fits && (mine == 0 || mine_to <= there);
    if (ok) t.lens[tid] = len + grow;
    granted[tid] = ok || (len >= 0 && grow <= 0);
    if (ok && copy) {
      atomicSub(&t.refs[src], 1);
      m.src[(other_to >> 16) - 1] = src;
      m.dst[(other_to >> 16) - 1] = dst_of[tid];
      atomicAdd(&moved, 1u);
    }
  }
  __syncthreads();
  if (tid == 0) *m.count = moved;
}

// map[p]: where page p >= n goes (p itself where nothing holds it).
__global__ __launch_bounds__(kBlock) void pages_compact_kernel(const int* refs, unsigned pages, int* refs_out,
                                                               int* __restrict__ map, unsigned* held, Moves m) {
  __shared__ unsigned sums[16];
  const unsigned tid = threadIdx.x;
  int r[kPer];
  unsigned n = 0;
#pragma unroll 1
  for (unsigned at = 0; at < pages; at += kStep) {
    read_counts(refs, pages, at, r);
    unsigned mine = 0, total;
    const unsigned p0 = at + tid * kPer;
#pragma unroll
    for (unsigned u = 0; u < kPer; ++u) mine += r[u] > 0 && p0 + u < pages;
    block_scan(mine, sums, total);
    n += total;
  }
  unsigned moved = 0, holes = 0;
#pragma unroll 1
  for (unsigned at = 0; at < pages; at += kStep) {
    if (pages > kStep) read_counts(refs, pages, at, r);
    const unsigned p0 = at + tid * kPer;
    unsigned a = 0, h = 0, total;
#pragma unroll
    for (unsigned u = 0; u < kPer; ++u) {
      a += r[u] > 0 && p0 + u >= n && p0 + u < pages;
      h += r[u] <= 0 && p0 + u < n;
    }
    // both counts of a step fit 16 bits
    const unsigned in = block_scan(a | h << 16, sums, total);
    unsigned ka = moved + (in & 0xffffu) - a, kh = holes + (in >> 16) - h;
#pragma unroll
    for (unsigned u = 0; u < kPer; ++u) {
      const unsigned p = p0 + u;
      if (p >= n && p < pages) {
        if (r[u] > 0) m.src[ka++] = (int)p;
        map[p] = (int)p;
      } else if (r[u] <= 0) {
        m.dst[kh++] = (int)p;
      }
    }
    moved += total & 0xffffu;
    holes += total >> 16;
  }
  __syncthreads();
  // as many holes before n as held pages behind it; refs_out may be refs, so the
  // counts that move are read before any place behind n is cleared
  for (unsigned k = tid; k < moved; k += kBlock) {
    const int s = m.src[k], d = m.dst[k];
    map[s] = d;
    refs_out[d] = refs[s];
  }
  __syncthreads();
  if (refs_out != refs)
    for (unsigned p = tid; p < n; p += kBlock)
      if (refs[p] > 0) refs_out[p] = refs[p];
  for (unsigned p = n + tid; p < pages; p += kBlock) refs_out[p] = 0;
  if (tid == 0) {
    *m.count = moved;
    *held = n;
  }
}

// ---- copies ----------------------------------------------------------------

constexpr unsigned kCaches = 16, kPiece = 32768;

struct CopyCaches {
  PagedCache c[kCaches];
  unsigned n, elem_shift[kCaches];
};

struct Remap {            // table == NULL: nothing to remap
  const int* table;
  int* out;
  const int* lens;
  const int* map;
  const unsigned* held;
  size_t stride, out_stride;
  unsigned pages, page, width, rows;
  int max_len;
};

// 32 KB by 256 threads have 8 loads each in flight; the rest of a row goes 4 KB a step.
__device__ __forceinline__ void copy16(char* to, const char* from, unsigned bytes) {
  const unsigned o = threadIdx.x * 16;
  if (bytes == kPiece) {
    u32x4 x[8];
#pragma unroll
    for (unsigned u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const u32x4*>(from + o + u * 4096);
#pragma unroll
    for (unsigned u = 0; u < 8; ++u) *reinterpret_cast<u32x4*>(to + o + u * 4096) = x[u];
    return;
  }
#pragma unroll 1
  for (unsigned at = o; at < bytes; at += 4096)
    *reinterpret_cast<u32x4*>(to + at) = *reinterpret_cast<const u32x4*>(from + at);
}

// Item: (copy, cache, K or V, piece of 32 KB).  No page is both read and written.
__global__ __launch_bounds__(256, 8) void pages_copy_kernel(CopyCaches cs, unsigned pieces, Moves m, Remap r) {
  if (r.table != nullptr) {
    const unsigned n = *r.held;
    for (unsigned i = blockIdx.x; i < r.rows; i += gridDim.x) {
      // a row of no valid length keeps its entries, whose pages are counted still
      const int len = r.lens[i];
      const int have = len >= 0 && len <= r.max_len ? pages_of(len, r.page) : (int)r.width;
      for (unsigned c = threadIdx.x; c < r.width; c += 256) {
        int p = (int)c < have ? r.table[i * r.stride + c] : -1;
        if ((unsigned)p >= n && (unsigned)p < r.pages) p = r.map[p];
        r.out[i * r.out_stride + c] = p;
      }
    }
  }
  const unsigned per = cs.n * 2 * pieces;
  const size_t items = (size_t)*m.count * per;
  for (size_t it = blockIdx.x; it < items; it += gridDim.x) {
    const unsigned k = (unsigned)(it / per), j = (unsigned)(it % per);
    const unsigned piece = j % pieces, kv = (j / pieces) & 1, ci = j / pieces >> 1;
    const PagedCache& c = cs.c[ci];
    const unsigned page_bytes = (c.heads << c.shift) * kD << cs.elem_shift[ci];
    const size_t s = (size_t)m.src[k], d = (size_t)m.dst[k];
    const unsigned off = piece * kPiece;
    char* base = kv ? c.v : c.k;
    const size_t stride = kv ? c.v_stride : c.k_stride;
    if (off < page_bytes)
      copy16(base + d * stride + off, base + s * stride + off, min(kPiece, page_bytes - off));
    if (piece == 0) {
      uint8_t* e = kv ? c.v_exp : c.k_exp;
      if (e != nullptr && threadIdx.x < c.heads) e[d * c.heads + threadIdx.x] = e[s * c.heads + threadIdx.x];
      if (kv == 0 && c.bounds != nullptr) {
        const unsigned n = c.heads * 2 * kD;
        copy16(reinterpret_cast<char*>(c.bounds) + d * n, reinterpret_cast<const char*>(c.bounds) + s * n, n);
      }
    }
  }
}

// ---- slots -----------------------------------------------------------------

// A workgroup for every slot and 32 KB of it, forked or not: 30 layers' pools of 64 slots take
// 31 us where nothing is forked, 39 for one child (64 MB each way, 27 at a copy's rate), 359
// for 21 of one parent, which is read from caches then (566 at a copy's rate).
constexpr unsigned kPools = 64;
struct SlotPools {
  char* at[kPools];
  size_t stride[kPools];     // bytes
  size_t bytes[kPools];      // of a slot
  unsigned first[kPools + 1];   // pieces before pool j
  unsigned n;
};

__global__ __launch_bounds__(256, 8) void slots_fork_kernel(SlotPools s, const int* __restrict__ parent, unsigned slots) {
  const unsigned per = s.first[s.n];
  const unsigned i = blockIdx.x / per;
  unsigned piece = blockIdx.x % per;
  const int p = parent[i];
  if ((unsigned)p >= slots || (unsigned)p == i || parent[p] >= 0) return;
  unsigned j = 0;
  while (piece >= s.first[j + 1]) ++j;
  const size_t off = (size_t)(piece - s.first[j]) * kPiece;
  const size_t left = s.bytes[j] - off;
  copy16(s.at[j] + i * s.stride[j] + off, s.at[j] + (size_t)p * s.stride[j] + off,
         left < kPiece ? (unsigned)left : kPiece);
}

bool tables_of(const qwen36_page_tables* p, Tables& t) {
  if (p == nullptr || p->refs == nullptr || p->page_table == nullptr || p->seq_lens == nullptr ||
      p->num_pages == 0 || p->num_pages > 0x7fffffffu || p->rows == 0 || p->rows > 65536 || p->table_width == 0 ||
      p->table_stride < p->table_width ||
      (p->page_tokens != 16 && p->page_tokens != 32 && p->page_tokens != 64 && p->page_tokens != 128) ||
      (size_t)p->table_width * p->page_tokens > kMaxTokens + 127u)
    return false;
  t.refs = static_cast<int*>(p->refs);
  t.table = static_cast<int*>(p->page_table);
  t.lens = static_cast<int*>(p->seq_lens);
  t.stride = p->table_stride;
  t.pages = p->num_pages;
  t.page = p->page_tokens;
  t.width = p->table_width;
  t.rows = p->rows;
  t.max_len = (int)(p->table_width * p->page_tokens);
  if (t.max_len > (int)kMaxTokens) t.max_len = (int)kMaxTokens;
  return true;
}

bool caches_of(const qwen36_paged_cache* caches, unsigned n, const Tables& t) {
  if ((n > 0 && caches == nullptr) || n > 1024) return false;
  for (unsigned i = 0; i < n; ++i) {
    PagedCache c;
    if (!paged_cache_of(caches + i, c) || c.pages != t.pages || (1u << c.shift) != t.page) return false;
  }
  return true;
}

// The copies, 16 caches a launch; the remapping with the first.
int copy_launches(const qwen36_paged_cache* caches, unsigned n, const Moves& m, Remap r, size_t most, hipStream_t st) {
  for (unsigned i0 = 0; i0 < n || r.table != nullptr; i0 += kCaches) {
    CopyCaches cs = {};
    unsigned pieces = 1;
    for (unsigned i = i0; i < n && i < i0 + kCaches; ++i) {
      PagedCache& c = cs.c[cs.n];
      if (!paged_cache_of(caches + i, c)) return Q36_EINVAL;
      cs.elem_shift[cs.n] = caches[i].cache_type == QWEN36_PAGED_BF16 ? 1 : 0;
      const unsigned bytes = (c.heads << c.shift) * kD << cs.elem_shift[cs.n];
      if ((bytes + kPiece - 1) / kPiece > pieces) pieces = (bytes + kPiece - 1) / kPiece;
      ++cs.n;
    }
    // 8 workgroups a CU go on through the items
    size_t grid = most * cs.n * 2 * pieces;
    if (grid > 2048) grid = 2048;
    if (r.table != nullptr && grid < r.rows) grid = r.rows < 2048 ? r.rows : 2048;
    if (grid > 0)
      hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)grid), dim3(256), 0, st, cs, pieces, m, r);
    r.table = nullptr;
  }
  return static_cast<int>(hipGetLastError());
}

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT int qwen36_pages_trim(const qwen36_page_tables* tables, const void* keep, void* stream) {
  Tables t;
  if (!tables_of(tables, t) || keep == nullptr) return Q36_EINVAL;
  hipLaunchKernelGGL(pages_trim_kernel, dim3(t.rows), dim3(256), 0, static_cast<hipStream_t>(stream), t,
                     static_cast<const int*>(keep));
  return static_cast<int>(hipGetLastError());
}

Q36_EXPORT int qwen36_pages_fork(const qwen36_page_tables* tables, const void* parent, void* stream) {
  Tables t;
  if (!tables_of(tables, t) || parent == nullptr) return Q36_EINVAL;
  hipLaunchKernelGGL(pages_fork_kernel, dim3(t.rows), dim3(256), 0, static_cast<hipStream_t>(stream), t,
                     static_cast<const int*>(parent));
  return static_cast<int>(hipGetLastError());
}

Q36_EXPORT size_t qwen36_pages_extend_workspace_bytes(const qwen36_page_tables* tables) {
  Tables t;
  if (!tables_of(tables, t)) return 0;
  return 16 + 6 * round16((size_t)t.rows * 4);
}

Q36_EXPORT int qwen36_pages_extend(const qwen36_page_tables* tables, const void* add, void* granted,
                                   const qwen36_paged_cache* caches, unsigned n_caches, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  Tables t;
  if (!tables_of(tables, t) || add == nullptr || granted == nullptr || !caches_of(caches, n_caches, t) ||
      workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < qwen36_pages_extend_workspace_bytes(tables))
    return Q36_EINVAL;
  char* w = static_cast<char*>(workspace);
  const size_t row = round16((size_t)t.rows * 4);
  int* part[6];
  for (int i = 0; i < 6; ++i) part[i] = reinterpret_cast<int*>(w + 16 + i * row);
  const Moves m = {reinterpret_cast<unsigned*>(w), part[4], part[5]};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (t.rows <= kBlock && t.pages <= kStep)
    hipLaunchKernelGGL(pages_extend_few_kernel, dim3(1), dim3(kBlock), 0, st, t, static_cast<const int*>(add),
                       static_cast<int*>(granted), m);
  else
    hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(kBlock), 0, st, t, static_cast<const int*>(add),
                       static_cast<int*>(granted), part[0], part[1], part[2], part[3], m);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return static_cast<int>(e);
  return copy_launches(caches, n_caches, m, Remap{}, t.rows, st);
}

Q36_EXPORT size_t qwen36_pages_compact_workspace_bytes(const qwen36_page_tables* tables) {
  Tables t;
  if (!tables_of(tables, t)) return 0;
  return 16 + 3 * round16((size_t)t.pages * 4);
}

Q36_EXPORT int qwen36_pages_compact(const qwen36_page_tables* tables, void* refs_out, void* table_out,
                                    size_t table_out_stride, const qwen36_paged_cache* caches, unsigned n_caches,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  Tables t;
  if (!tables_of(tables, t) || refs_out == nullptr || table_out == nullptr || table_out_stride < t.width ||
      !caches_of(caches, n_caches, t) || workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < qwen36_pages_compact_workspace_bytes(tables))
    return Q36_EINVAL;
  char* w = static_cast<char*>(workspace);
  const size_t part = round16((size_t)t.pages * 4);
  unsigned* head = reinterpret_cast<unsigned*>(w);
  int* map = reinterpret_cast<int*>(w + 16);
  const Moves m = {head, reinterpret_cast<int*>(w + 16 + part), reinterpret_cast<int*>(w + 16 + 2 * part)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(kBlock), 0, st, t.refs, t.pages,
                     static_cast<int*>(refs_out), map, head + 1, m);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return static_cast<int>(e);
  const Remap r = {t.table, static_cast<int*>(table_out), t.lens, map, head + 1, t.stride, table_out_stride,
                   t.pages, t.page, t.width, t.rows, t.max_len};
  return copy_launches(caches, n_caches, m, r, (t.pages + 1) / 2, st);
}

Q36_EXPORT int qwen36_slots_fork(const qwen36_slot_pool* pools, unsigned n_pools, unsigned slots,
                                 const void* parent, void* stream) {
  if (pools == nullptr || n_pools == 0 || n_pools > 1024 || slots == 0 || slots > 65536 || parent == nullptr)
    return Q36_EINVAL;
  for (unsigned j = 0; j < n_pools; ++j)
    if (pools[j].data == nullptr || !aligned16(pools[j].data) || pools[j].slot_bytes == 0 ||
        pools[j].slot_bytes % 16 != 0 || pools[j].slot_bytes > ((size_t)1 << 30) ||
        pools[j].slot_stride_bytes % 16 != 0 || pools[j].slot_stride_bytes < pools[j].slot_bytes)
      return Q36_EINVAL;
  for (unsigned j0 = 0; j0 < n_pools;) {
    // as many pools as one grid and one argument hold
    SlotPools s = {};
    while (j0 < n_pools && s.n < kPools) {
      const size_t pieces = (pools[j0].slot_bytes + kPiece - 1) / kPiece;
      if (s.n > 0 && (s.first[s.n] + pieces) * slots > ((size_t)1 << 23)) break;
      if (pieces * slots > ((size_t)1 << 23)) return Q36_EINVAL;
      s.at[s.n] = static_cast<char*>(pools[j0].data);
      s.stride[s.n] = pools[j0].slot_stride_bytes;
      s.bytes[s.n] = pools[j0].slot_bytes;
      s.first[s.n + 1] = s.first[s.n] + (unsigned)pieces;
      ++s.n;
      ++j0;
    }
    hipLaunchKernelGGL(slots_fork_kernel, dim3(s.first[s.n] * slots), dim3(256), 0,
                       static_cast<hipStream_t>(stream), s, static_cast<const int*>(parent), slots);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return static_cast<int>(e);
  }
  return Q36_OK;
}
