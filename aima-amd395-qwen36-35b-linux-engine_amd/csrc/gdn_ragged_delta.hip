// The gated delta rule over a ragged batch with its states in slots.
//
// Per value head (key head h * qk_heads / 32) and token, with the state S [128 k]
// [128 v] in fp32:
//   q, k <- x / sqrt(sum x^2 + 1e-6), q *= 1/sqrt(128)
//   S <- e^g S;  d = beta (v - k S);  S <- S + k (x) d;  o = q S
// (or q and k as given, q /= sqrt(128); or S kept as [128 v] [128 k]).  A sequence begins
// with its slot's state (zeros where it has none) and leaves its last one there.
#include "gemm_tile.h"
#include "ragged.h"

#include <mutex>

namespace q36 {
namespace {

constexpr unsigned kMaxStride = 1u << 24;          // 64 rows within 32 bits of bytes
constexpr float kQScale = 0.08838834764831845f;   // 1/sqrt(128)

struct DeltaArgs {
  const bf16 *q, *k, *v;
  const float *g, *beta;
  float* states;
  bf16* out;
  size_t slot_stride;
  unsigned qk_heads, qk_stride, v_stride;
  bool normalized;         // q and k are used as given
  int row_step, col_step;  // elements between rows (of k) and columns (of v) of a state
};

// ---------------------------------------------------------------------------
// Token by token: sequences of up to `limit` tokens.
// Bound by the states' bytes (4.2 MB a sequence, read and written: 53 us for 64
// sequences of a token, 5.1 TB/s; 81 where states are by columns, whose rows are loads of 4
// bytes).  Both reductions of a token, S^T k and S^T q, are taken of the state before it:
// o = e^g S_old^T q + d (k.q), so that a token costs one exchange between waves (64
// sequences of 2 tokens 63 us, of 4 90, of 7 131).
// One workgroup owns 32 columns of a head: thread (rg, cq) rows rg + 32 i and
// columns 4 cq .. +3, a row of the 32 columns being one 128-byte line.
// ---------------------------------------------------------------------------
struct StepLds {
  f32x4 red[2][4][2][8];    // [parity][wave][k | q][column quad]
  float dots[2][4][4];      // [parity][wave][k.k, q.q, k.q]
};

__device__ __forceinline__ void step_rows(const DeltaArgs& p, const RaggedBatch& b, unsigned block, unsigned limit,
                                          StepLds& lds) {
  auto& red = lds.red;
  auto& dots = lds.dots;
  const unsigned seq = block >> 7;
  const int h = (block >> 2) & 31, cg = block & 3;
  const RaggedSeq s = ragged_seq(b, seq);
  const unsigned len = (unsigned)(s.z - s.a);
  if (s.slot < 0 || len == 0 || len > limit) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int rg = tid >> 3, cq = tid & 7;
  const int col = 32 * cg + 4 * cq;
  const int kh = h * (int)p.qk_heads / kGdnHv;
  float* sp = p.states + (size_t)s.slot * p.slot_stride + (size_t)h * kGdnDk * kGdnDv + rg * p.row_step + col * p.col_step;
  f32x4 st[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s.has && p.col_step == 1) {
      st[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(sp + 32 * i * kGdnDv));
    } else if (s.has) {
#pragma unroll
      for (int e = 0; e < 4; ++e) st[i][e] = sp[32 * i + e * kGdnDk];
    }
  }
  for (int t = s.a; t < s.z; ++t) {
    const bf16* qp = p.q + (size_t)t * p.qk_stride + kh * kGdnDk + rg;
    const bf16* kp = p.k + (size_t)t * p.qk_stride + kh * kGdnDk + rg;
    const bf16x4 v4 = *reinterpret_cast<const bf16x4*>(p.v + (size_t)t * p.v_stride + h * kGdnDv + col);
    const float gt = p.g[(size_t)t * kGdnHv + h], bt = p.beta[(size_t)t * kGdnHv + h];
    float kr[4], qr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kr[i] = bf2f(kp[32 * i]);
      qr[i] = bf2f(qp[32 * i]);
    }
    f32x4 pk = {0.f, 0.f, 0.f, 0.f}, pq = pk;
    float kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pk += st[i] * kr[i];
      pq += st[i] * qr[i];
      kk += kr[i] * kr[i];
      qq += qr[i] * qr[i];
      kq += kr[i] * qr[i];
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pk[e] += __shfl_xor(pk[e], o, 64);
        pq[e] += __shfl_xor(pq[e], o, 64);
      }
      kk += __shfl_xor(kk, o, 64);
      qq += __shfl_xor(qq, o, 64);
      kq += __shfl_xor(kq, o, 64);
    }
    const int par = t & 1;
    if (lane < 8) {
      red[par][wave][0][cq] = pk;
      red[par][wave][1][cq] = pq;
    }
    if (lane == 0) {
      dots[par][wave][0] = kk;
      dots[par][wave][1] = qq;
      dots[par][wave][2] = kq;
    }
    lds_barrier();
    f32x4 sk = red[par][0][0][cq], sq = red[par][0][1][cq];
    float nk = dots[par][0][0], nq = dots[par][0][1], nkq = dots[par][0][2];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      sk += red[par][w][0][cq];
      sq += red[par][w][1][cq];
      nk += dots[par][w][0];
      nq += dots[par][w][1];
      nkq += dots[par][w][2];
    }
    const float kinv = p.normalized ? 1.0f : 1.0f / sqrtf(nk + 1e-6f);
    const float qn = p.normalized ? kQScale : kQScale / sqrtf(nq + 1e-6f);
    const float eg = expf(gt), dot = nkq * kinv * qn;
    f32x4 d, o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      d[e] = (bf2f(v4[e]) - eg * (sk[e] * kinv)) * bt;
      o[e] = eg * (sq[e] * qn) + d[e] * dot;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) st[i] = st[i] * eg + d * (kr[i] * kinv);
    if (rg == 0) {
      bf16x4 ob;
#pragma unroll
      for (int e = 0; e < 4; ++e) ob[e] = f2bf(o[e]);
      *reinterpret_cast<bf16x4*>(p.out + ((size_t)t * kGdnHv + h) * kGdnDv + col) = ob;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (p.col_step == 1) {
      __builtin_nontemporal_store(st[i], reinterpret_cast<f32x4*>(sp + 32 * i * kGdnDv));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) sp[32 * i + e * kGdnDk] = st[i][e];
    }
  }
}

__global__ __launch_bounds__(256) void gdn_ragged_step_kernel(DeltaArgs p, RaggedBatch b) {
  __shared__ StepLds lds;
  step_rows(p, b, blockIdx.x, ~0u, lds);
}

// ---------------------------------------------------------------------------
// Chunks of 64 tokens: longer sequences.
//
// With G the sum of g from the chunk's first token on, S the state before it:
//   L = strictly lower part of diag(beta) (k k^T) e^(Gi - Gj),  T = (I + L)^-1
//   v' = T diag(beta) (v - diag(e^G) k S)
//   o  = diag(e^G) q S + A v',  A = lower part of (q k^T) e^(Gi - Gj)
//   S <- e^Glast S + k^T diag(e^(Glast - G)) v'
// The norms of q and k and the decays are row factors in fp32; products with S are
// taken of the raw q and k.
//
// Precision.  S, v', its decayed rows and beta (v - ..) are fp32; into products that the
// state comes from they enter as the sum of two fp16 values (22 bits), each column scaled
// by a power of two that brings its largest to 2^13 .. 2^14: what is lost of a value is
// 2^-22 of it or, for small ones beside large, 2^-38 of the column's largest (half of
// fp16's least step).  Sums are fp32, so that only the operands have to stay within fp16.  k
// and q (8 bits in bf16) are exact in fp16 once a row is scaled by a power of two to a norm
// of 8 to 16: values below 2^-20 of their row's norm lose bits, 2^-28 of it at most.  T has
// two such parts, of 2^8 T (with 0 <= beta <= 2 and g <= 0 its values are at most 2:
// T_ij is -beta_i k_i (reflections, which lengthen nothing) k_j): what is lost is 2^-22 of a
// value or 2^-33.  Low by low parts are left out (2^-22 of a term).  A against v', which
// only the output comes from, takes two bf16 values of each (2^-17 of a term): decays of
// any size meet there, and rows that are all decayed keep their bits.
// (Three bf16 parts throughout, which need no scales, take 182 products a chunk and column
// tile where this takes 132: 157 us where the scan then took 134.)
//
// Times below are of 13 prompts of 9,903 rows, 161 chunks, the longest of 24.
//  * gdn_ragged_prep_kernel, a workgroup a (chunk, key head): T and A of its value heads,
//    which do not depend on the state, as the scan's operands, and the row factors: a
//    record of 26,368 bytes a value head.  53 us, of which reading q and k once and writing
//    the records (217 MB) take 48 at 4.5 TB/s; four workgroups a CU hide most of its steps'
//    latencies (two, with L and T as whole matrices in LDS, took 81 us).  The short sequences'
//    workgroups are behind them (a launch of their own takes 4.8 us even where there are none).
//  * gdn_ragged_scan_kernel, a workgroup a (sequence, head or part of its columns),
//    chunk after chunk.  A wave owns 16 columns of v with all 128 rows of their
//    state, in registers: the layout of a product's result is that of the next one's
//    right operand, so that nothing of a column's recurrence leaves its wave, and waves
//    meet once a chunk, where the next chunk's k, q, v, T and A are ready in LDS.
//    117 us: a chunk takes 4.7 us, 4.3 without its fetches.  Products hold a SIMD's vector
//    instructions up for half of their 16 cycles: 132 x 8 and 656 x 4 cycles of two waves are
//    3.1 us; LDS is read for 1.7.  What is left is the chain's latency.  (131 us with the
//    fetches in the eight waves that own columns; 4 such waves of 32 columns each 128.)
// ---------------------------------------------------------------------------

typedef _Float16 f16;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kC = 64;
// Longer sequences go by chunks.  Token by token and by chunks, us, over three inputs and
// their states in turn: one sequence of 8 tokens 12.7 and 15.1, of 12 17.7 and 15.2; 16
// sequences of 8 48 and 40, of 12 63 and 39; 64 of 7 131 and 142, of 8 152 and 136, of 12 212
// and 139.  A call of up to 12 rows goes token by token whatever its lengths, without a
// workspace (2.5 us more for one sequence of 12).
constexpr unsigned kShort = 7, kFewRows = 12;
constexpr int kPitchR = 136;              // 16-bit row pitch of [64][128] tiles: 272 bytes
// g below this is taken as this: e^g is zero in fp32 either way (below -104), and sums of 64
// stay finite and small enough for what comes after to keep its bits.
constexpr float kGateMin = -128.0f;

// A record.  T and A as operands: tokens 16 i .. by 32 tokens k, lane 16 g + m of row m the
// columns 32 k + 4 g .. + 3 and 32 k + 16 + 4 g .. + 3, which is how two tiles of a product's
// result are the right operand of the next; fragments i + k for i < 2, 2 + 2 (i - 2) + k
// else.  Then the factors of each token.
constexpr int kFragA = 12, kFrags = 24;   // 2^8 T: high, low of each fragment; then A so, bf16
enum {
  kBeta = 0,
  kBcy = kC,                // beta e^G / |k'|
  kRsq = 2 * kC,            // e^G / (|q'| sqrt(128))
  kRsk = 3 * kC,            // 2^-8 e^(Glast - G) / |k'|
  kScanFactors = 4 * kC,
  kKs = 4 * kC,             // k' = ks k, q' = qs q
  kQs = 5 * kC,
  kEgl = 6 * kC,            // e^Glast
  kFactors = 7 * kC
};
struct Record {
  f16x8 frag[kFrags * 64];
  float f[kFactors];
};
static_assert(sizeof(Record) == 26368, "record");

// The long sequences are counted in their order; record a_i / 64 + (long sequences before
// i) + c is chunk c of sequence i: no two meet, as for tiles of rows (ragged.h).
__device__ __forceinline__ bool find_record(const RaggedBatch& b, unsigned rec, RaggedSeq& s, unsigned& chunk) {
  const unsigned lane = threadIdx.x & 63;
  unsigned longs = 0;
  for (unsigned i0 = 0; i0 < b.seqs; i0 += 64) {
    const unsigned i = i0 + lane;
    int a = 0, z = 0;
    if (i < b.seqs) ragged_rows(b, i, a, z);
    const bool is = (unsigned)(z - a) > kShort;
    const unsigned long long mask = __ballot(is);
    const unsigned first = (unsigned)a / kC + longs + __popcll(mask & ((1ull << lane) - 1));
    const unsigned long long hit = __ballot(is && rec >= first && rec - first < (unsigned)(z - a + kC - 1) / kC);
    if (hit != 0) {
      const int at = __ffsll((long long)hit) - 1;
      s = ragged_seq(b, i0 + at);
      chunk = rec - (unsigned)__builtin_amdgcn_readlane((int)first, at);
      return s.slot >= 0;
    }
    longs += __popcll(mask);
  }
  return false;
}

// The n-th long sequence and its first record; among up to 64 sequences the n-th longest,
// so that the longest begin first.  Of sequences that overlap there may be more than the
// `most` that records are kept for: those behind have none.
__device__ __forceinline__ bool find_long(const RaggedBatch& b, unsigned n, unsigned most, RaggedSeq& s,
                                          unsigned& rec) {
  const unsigned lane = threadIdx.x & 63;
  unsigned longs = 0;
  for (unsigned i0 = 0; i0 < b.seqs; i0 += 64) {
    const unsigned i = i0 + lane;
    int a = 0, z = 0;
    if (i < b.seqs) ragged_rows(b, i, a, z);
    const int len = z - a;
    const bool is = (unsigned)len > kShort;
    const unsigned long long mask = __ballot(is);
    const unsigned before = longs + __popcll(mask & ((1ull << lane) - 1));
    unsigned place = before;
    if (b.seqs <= 64) {
      place = 0;
      for (unsigned long long m = mask; m != 0; m &= m - 1) {
        const int j = __ffsll((long long)m) - 1, other = __builtin_amdgcn_readlane(len, j);
        place += other > len || (other == len && j < (int)lane);
      }
    }
    const unsigned long long hit = __ballot(is && place == n && before < most);
    if (hit != 0) {
      const int at = __ffsll((long long)hit) - 1;
      s = ragged_seq(b, i0 + at);
      rec = (unsigned)__builtin_amdgcn_readlane((int)((unsigned)a / kC + before), at);
      return s.slot >= 0;
    }
    longs += __popcll(mask);
  }
  return false;
}

__device__ __forceinline__ bf16x8 ld8(const bf16* p) { return *reinterpret_cast<const bf16x8*>(p); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(const __amdgpu_buffer_rsrc_t& r, unsigned off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0);
}
__device__ __forceinline__ f32x4 ld4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }

// e^x from the hardware's 2^x: the rounding of x log2(e), and its low bits, come
// in to first order (2 units of 2^-24 in all; below 2^-126 zero).
__device__ __forceinline__ float exp_fast(float x) {
  const float h = x * kLog2e;
  const float l = __builtin_fmaf(x, kLog2e, -h) + x * 1.925963033500e-08f;
  const float e = __builtin_amdgcn_exp2f(h);
  return __builtin_fmaf(e, l * 0.693147180559945f, e);
}

template <int kHeads>      // value heads of a key head
struct PrepLds {
  union {
    struct {
      bf16 k[kC * kPitchR], q[kC * kPitchR];
    } rows;                                      // dead once k k^T and q k^T are in registers
    struct {
      float l[kHeads][10][256], t[kHeads][4][256];      // L and T's diagonal, tiles as at `tile_at`
    } tiles;
  } u;
  float gs[kHeads][kC], gl[kHeads][kC];         // G = gs + gl: differences of fast decays keep their bits
  // e^(Gi - Gj) in tiles of 16 below the diagonal: near[i] far[tile of i][j], by the first
  // token of i's tile
  float near[kHeads][kC], far[kHeads][3][48];
  float bs[kHeads][kC];
  float kinv[kC], qinv[kC];             // 1 where rows are taken as given
  float kscale[kC], qscale[kC];
};

// A 16x16 tile of a lower matrix, transposed: column c, row r of it.  Four rows of the 16
// columns, as a product's left operand reads them, lie in different banks.
__device__ __forceinline__ int tile_at(int c, int r) { return 16 * c + ((r & 12) ^ (c & 12)) + (r & 3); }

// C += A B: A a tile in LDS (transposed, as it is kept), B a product's result.
__device__ __forceinline__ f32x4 mm16(const float* a, const f32x4& b, f32x4 acc, int li, int lg) {
  const f32x4 x = *reinterpret_cast<const f32x4*>(a + tile_at(li, 4 * lg));
#pragma unroll
  for (int s = 0; s < 4; ++s) acc = mfma16x16x4f32(x[s], b[s], acc);
  return acc;
}

__device__ __forceinline__ int frag_of(int i, int k) { return i < 2 ? i : 2 * i - 2 + k; }

// The power of two that brings a row of inverse norm `inv` to a norm of 8 to 16.
__device__ __forceinline__ float row_scale(float inv) {
  const int e = min(max((int)(__float_as_uint(inv) >> 23) - 127, -100), 100);
  return __uint_as_float((unsigned)(e + 127 + 4) << 23);
}

template <int kHeads>
__global__ __launch_bounds__(256, 4) void gdn_ragged_prep_kernel(DeltaArgs p, RaggedBatch b, Record* __restrict__ ws,
                                                               unsigned blocks) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if (blockIdx.x >= blocks) {      // the batch's short sequences
    step_rows(p, b, blockIdx.x - blocks, kShort, *reinterpret_cast<StepLds*>(smem));
    return;
  }
  PrepLds<kHeads>& s = *reinterpret_cast<PrepLds<kHeads>*>(smem);
  // a key head's chunks on the XCD where the scan reads their records
  constexpr unsigned kEach = 4 / kHeads;       // key heads an XCD
  const unsigned slot = blockIdx.x >> 3, rec_i = slot / kEach;
  const int kh = kEach * (blockIdx.x & 7) + slot % kEach, h0 = kh * kHeads;
  RaggedSeq q;
  unsigned chunk;
  if (!find_record(b, rec_i, q, chunk)) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const unsigned tok0 = (unsigned)q.a + chunk * kC, rows = min((unsigned)kC, (unsigned)q.z - tok0);
  Record* rec = ws + (size_t)rec_i * kGdnHv + h0;
  // rows behind the sequence read as zeros
  const unsigned range = ((rows - 1) * p.qk_stride + kGdnDk) * 2;
  const __amdgpu_buffer_rsrc_t qrs = rows_rsrc(p.q + (size_t)tok0 * p.qk_stride + kh * kGdnDk, range);
  const __amdgpu_buffer_rsrc_t krs = rows_rsrc(p.k + (size_t)tok0 * p.qk_stride + kh * kGdnDk, range);
  const int r1 = tid >> 2, p1 = tid & 3;
  bf16x8 k8[4], q8[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned off = (r1 * p.qk_stride + 32 * p1 + 8 * i) * 2;
    k8[i] = __builtin_bit_cast(bf16x8, load16(krs, off));
    q8[i] = __builtin_bit_cast(bf16x8, load16(qrs, off));
  }
  if ((wave & 1) < kHeads) {      // waves 0, 1: G; 2, 3: beta
    const int hd = wave & 1;
    const float* from = wave < 2 ? p.g : p.beta;
    const float v = (unsigned)lane < rows ? from[(size_t)(tok0 + lane) * kGdnHv + h0 + hd] : 0.f;
    if (wave < 2) {
      double sum = v < kGateMin ? kGateMin : v;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(sum, o, 64);
        if (lane >= o) sum += u;
      }
      s.gs[hd][lane] = (float)sum;
      s.gl[hd][lane] = (float)(sum - (double)(float)sum);
    } else {
      s.bs[hd][lane] = v;
    }
  }
  float kss = 0.f, qss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    *reinterpret_cast<bf16x8*>(&s.u.rows.k[r1 * kPitchR + 32 * p1 + 8 * i]) = k8[i];
    *reinterpret_cast<bf16x8*>(&s.u.rows.q[r1 * kPitchR + 32 * p1 + 8 * i]) = q8[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float kx = bf2f(k8[i][e]), qx = bf2f(q8[i][e]);
      kss += kx * kx;
      qss += qx * qx;
    }
  }
  kss += __shfl_xor(kss, 1, 64);
  kss += __shfl_xor(kss, 2, 64);
  qss += __shfl_xor(qss, 1, 64);
  qss += __shfl_xor(qss, 2, 64);
  if (p1 == 0) {
    const float ki = 1.0f / sqrtf(kss + 1e-6f), qi = 1.0f / sqrtf(qss + 1e-6f);
    s.kscale[r1] = row_scale(ki);
    s.qscale[r1] = row_scale(qi);
    s.kinv[r1] = p.normalized ? 1.0f : ki;
    s.qinv[r1] = p.normalized ? 1.0f : qi;
  }
  lds_barrier();
  auto decay = [&](int hd, int i, int j) { return (s.gs[hd][i] - s.gs[hd][j]) + (s.gl[hd][i] - s.gl[hd][j]); };
  if (wave < kHeads) {
    const int hd = wave, i = lane;
    const float ki = s.kinv[i], qi = s.qinv[i], ks = s.kscale[i], qs = s.qscale[i];
    const float eg = expf(s.gs[hd][i]), bt = s.bs[hd][i];
    const float kn = ki / ks, qn = qi / qs;        // by powers of two
    Record& r = rec[hd];
    r.f[kBeta + i] = bt;
    r.f[kBcy + i] = bt * (eg * kn);
    r.f[kRsq + i] = eg * (qn * kQScale);
    r.f[kRsk + i] = kn * expf(decay(hd, kC - 1, i)) * 0.00390625f;
    r.f[kKs + i] = ks;
    r.f[kQs + i] = qs;
    r.f[kEgl + i] = expf(s.gs[hd][kC - 1]);
    s.near[hd][i] = expf(decay(hd, i, i & ~15));
  } else {
    for (int n = tid - 64 * kHeads; n < 96 * kHeads; n += 256 - 64 * kHeads) {
      const int hd = n / 96, at = n % 96, rt = at < 16 ? 1 : at < 48 ? 2 : 3, j = at - (rt == 1 ? 0 : rt == 2 ? 16 : 48);
      s.far[hd][rt - 1][j] = expf(decay(hd, 16 * rt, j));
    }
  }
  // k k^T and q k^T by fragments of A (two tiles of a row of tiles, the second not behind the
  // diagonal), transposed: lane columns 4 lg + r of row li.  Waves 0, 1 take fragments 2 wave
  // and the next, 2 and 3 fragments 4 and 5: 3, 3, 2 and 2 tiles.
  const int f0 = wave < 2 ? 2 * wave : wave + 2, n_frags = wave < 2 ? 2 : 1;
  auto frag_row = [](int f) { return f < 2 ? f : f < 4 ? 2 : 3; };
  auto frag_col = [](int f) { return f < 2 ? 0 : f & 1; };
  f32x4 kk[2][2], qk[2][2];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int rt = frag_row(f0 + n), ct = 2 * frag_col(f0 + n) + u;
      kk[n][u] = f32x4{0.f, 0.f, 0.f, 0.f};
      qk[n][u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (n >= n_frags || ct > rt) continue;
      const int jrow = (16 * ct + li) * kPitchR + 8 * lg, irow = (16 * rt + li) * kPitchR + 8 * lg;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bf16x8 kj = ld8(s.u.rows.k + jrow + 32 * k);
        kk[n][u] = mfma16x16x32(kj, ld8(s.u.rows.k + irow + 32 * k), kk[n][u]);
        qk[n][u] = mfma16x16x32(kj, ld8(s.u.rows.q + irow + 32 * k), qk[n][u]);
      }
    }
  lds_barrier();     // the rows make room for L
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    if (n >= n_frags) continue;
    const int rt = frag_row(f0 + n), i = 16 * rt + li;
    const float ki = s.kinv[i], qi = s.qinv[i] * kQScale;
#pragma unroll
    for (int hd = 0; hd < kHeads; ++hd) {
      bf16x8 hi = {}, lo = {};
      const float bi = s.bs[hd][i];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int ct = 2 * frag_col(f0 + n) + u, j0 = 16 * ct + 4 * lg;
        if (ct > rt) continue;
        const f32x4 kj = ld4(s.kinv + j0);
        f32x4 d;
        if (rt == ct) {      // behind the diagonal anything, chosen against below
#pragma unroll
          for (int r = 0; r < 4; ++r) d[r] = exp_fast(decay(hd, i, j0 + r));
        } else {
          d = ld4(s.far[hd][rt - 1] + j0) * s.near[hd][i];
        }
        float* lt = s.u.tiles.l[hd][rt * (rt + 1) / 2 + ct];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lt[tile_at(4 * lg + r, li)] = j0 + r < i ? (((ki * kj[r]) * kk[n][u][r]) * bi) * d[r] : 0.f;
          const float av = j0 + r <= i ? ((qi * kj[r]) * qk[n][u][r]) * d[r] : 0.f;
          const bf16 ah = f2bf(av);
          hi[4 * u + r] = ah;
          lo[4 * u + r] = f2bf(av - bf2f(ah));
        }
      }
      f16x8* to = rec[hd].frag + (kFragA + 2 * (f0 + n)) * 64 + lane;
      to[0] = __builtin_bit_cast(f16x8, hi);
      to[64] = __builtin_bit_cast(f16x8, lo);
    }
  }
  lds_barrier();
  // (I + L)^-1: diagonal 16x16 blocks by substitution, a block a wave, a column a lane
  if (lane < 16 * kHeads) {
    const int hd = lane >> 4;
    const float* lm = s.u.tiles.l[hd][wave * (wave + 3) / 2];
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = i == li ? 1.f : 0.f;
#pragma unroll
    for (int m = 0; m < 15; ++m)
#pragma unroll
      for (int i4 = (m + 1) & 12; i4 < 16; i4 += 4) {
        const f32x4 x = ld4(lm + tile_at(m, i4));
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i4 + r > m) t[i4 + r] -= x[r] * t[m];
      }
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<f32x4*>(s.u.tiles.t[hd][wave] + tile_at(li, i)) = f32x4{t[i], t[i + 1], t[i + 2], t[i + 3]};
  }
  lds_barrier();
  // Row i of blocks from the diagonal on, T_ij = -(sum_{j < k <= i} T_ik L_kj) T_jj, transposed:
  // a wave's results are its next products' right operands, and the record's layout.
#pragma unroll
  for (int hd = 0; hd < kHeads; ++hd) {
    const int own = hd == 0 ? wave : 3 - wave;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (own != i) continue;
      f32x4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 4; ++r) x[i][r] = s.u.tiles.t[hd][i][tile_at(4 * lg + r, li)];
#pragma unroll
      for (int j = i - 1; j >= 0; --j) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = i; k > j; --k) sum = mm16(s.u.tiles.l[hd][k * (k + 1) / 2 + j], x[k], sum, li, lg);
        x[j] = -mm16(s.u.tiles.t[hd][j], sum, f32x4{0.f, 0.f, 0.f, 0.f}, li, lg);
      }
#pragma unroll
      for (int k = 0; k < (i < 2 ? 1 : 2); ++k) {
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = x[2 * k + (e >> 2)][e & 3] * 256.0f;
          hi[e] = (f16)v;
          lo[e] = (f16)(v - (float)hi[e]);
        }
        f16x8* to = rec[hd].frag + 2 * frag_of(i, k) * 64 + lane;
        to[0] = hi;
        to[64] = lo;
      }
    }
  }
}

// ---- scan --------------------------------------------------------------------

__device__ __forceinline__ f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

#define kFence __builtin_amdgcn_sched_barrier(0)
#define kPin(x) asm volatile("" : "+v"(x))
// The reads of LDS, then `m` products with `n` vector instructions behind each.
#define kBeside(m, n)                                                 \
  do {                                                                \
    __builtin_amdgcn_sched_group_barrier(0x100, 16, 0);               \
    for (int q_ = 0; q_ < (m); ++q_) {                                \
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);                \
      __builtin_amdgcn_sched_group_barrier(0x2, n, 0);                \
    }                                                                 \
    kFence;                                                           \
  } while (0)
// s_waitcnt: at most n vector-memory operations outstanding.
constexpr int kVmcnt(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

// Rows of k', q' and v in LDS: chunk j (8 values) of a row stands at j ^ row_key, so that
// what one cycle takes of a 16-byte read (lanes 0-3, 12-15, 20-27 and so on: eight rows of one
// chunk, the eight others of the next) lies in different banks.
__device__ __forceinline__ int row_key(int row) {
  const int x = (row >> 2) & 3;
  return (row & 3) << 2 | ((x ^ x >> 1) & 1) << 1 | x >> 1;
}
__device__ __forceinline__ int row_at(int row, int chunk) { return row * kGdnDk + 8 * (chunk ^ row_key(row)); }

struct ScanBuf {
  float f[kScanFactors];
  f16x8 frag[kFrags * 64];
  f16 kr[kC * kGdnDk], qr[kC * kGdnDk];       // k', q'
  bf16 vr[kC * kGdnDk];                       // v; then the output, which the fetching waves store
};
static_assert(sizeof(ScanBuf) % 256 == 0 && offsetof(ScanBuf, kr) % 256 == 0, "rows begin at bank 0");

// Lane i's 16 bytes at byte `off` of the range to `to` + 16 i, without registers.  (The
// compiler does not see the load: fetches are waited for where the chunk ends.)
__device__ __forceinline__ void to_lds(const u32x4& range, unsigned off, void* to) {
  g_fetch((unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)to, (int)off, range);
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight values times s as the sum of two fp16 values, by conversions of pairs: the form that
// multiplies, adds and converts one value (which the pin keeps the compiler from) takes twice
// a vector instruction's time.
__device__ __forceinline__ void split8(const f32x4& a, const f32x4& b, float s, f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const f32x4& v = e < 4 ? a : b;
    const f32x2 x = {v[e & 2], v[(e & 2) + 1]};
    const f16x2 h = __builtin_convertvector(x * s, f16x2);
    float l0 = __builtin_fmaf(x[0], s, -(float)h[0]), l1 = __builtin_fmaf(x[1], s, -(float)h[1]);
    kPin(l0);
    kPin(l1);
    const f16x2 l = __builtin_convertvector(f32x2{l0, l1}, f16x2);
    hi[e] = h[0];
    hi[e + 1] = h[1];
    lo[e] = l[0];
    lo[e + 1] = l[1];
  }
}

// The same as two bf16 values, without a scale.
__device__ __forceinline__ void split8(const f32x4& a, const f32x4& b, bf16x8& hi, bf16x8& lo) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x4& v = e < 2 ? a : b;
    const float x0 = v[2 * (e & 1)], x1 = v[2 * (e & 1) + 1];
    const bf16x2 y = __builtin_convertvector(f32x2{x0, x1}, bf16x2);
    const unsigned u = __builtin_bit_cast(unsigned, y);
    const bf16x2 z = __builtin_convertvector(f32x2{x0 - __uint_as_float(u << 16), x1 - __uint_as_float(u & 0xffff0000u)}, bf16x2);
    hi[2 * e] = y[0];
    hi[2 * e + 1] = y[1];
    lo[2 * e] = z[0];
    lo[2 * e + 1] = z[1];
  }
}

// A column's largest magnitude: over the lane's values and the four lanes of it.
struct ColumnMax {
  float top = 0.f;
  __device__ __forceinline__ void take(const f32x4& x) {
#pragma unroll
    for (int r = 0; r < 4; ++r) top = __builtin_fmaxf(top, __builtin_fabsf(x[r]));
  }
  __device__ __forceinline__ unsigned bits() const {
    unsigned m = __float_as_uint(top);
    const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return max(b[0], b[1]);
  }
};

// The power of two that brings the value of bits m into [2^13, 2^14), and its inverse.
__device__ __forceinline__ void scale_of(unsigned m, float& s, float& inv) {
  const int e = min(max((int)(m >> 23), 27), 253) - 13;      // biased
  s = __uint_as_float((unsigned)(254 - e) << 23);
  inv = __uint_as_float((unsigned)e << 23);
}

// Eight bf16 values times a power of two in fp16.
__device__ __forceinline__ f16x8 to_f16(const u32x4& x, float s) {
  f16x8 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f16x2 y =
        __builtin_convertvector(f32x2{__uint_as_float(x[e] << 16), __uint_as_float(x[e] & 0xffff0000u)} * s, f16x2);
    o[2 * e] = y[0];
    o[2 * e + 1] = y[1];
  }
  return o;
}

// The workgroup's first kWaves waves own 16 columns each, the others only fetch.
constexpr int scan_waves(int chains) { return chains == 8 ? 12 : 8; }

template <int kWaves>
__global__ __launch_bounds__(64 * scan_waves(kWaves), 1) void gdn_ragged_scan_kernel(
    DeltaArgs p, RaggedBatch b, const Record* __restrict__ ws, unsigned most) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  ScanBuf* buf = reinterpret_cast<ScanBuf*>(smem);
  constexpr unsigned kGroups = 8 / kWaves;
  const unsigned slot = blockIdx.x >> 3, rest = slot >> 2;
  const int h = 4 * (blockIdx.x & 7) + (slot & 3);
  RaggedSeq s;
  unsigned rec0;
  if (!find_long(b, rest / kGroups, most, s, rec0)) return;
  const int kh = h * (int)p.qk_heads / kGdnHv;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const unsigned len = (unsigned)(s.z - s.a), chunks = (len + kC - 1) / kC, last = chunks - 1;

  // ---- fetching a chunk ahead, into the other buffer: v, fragments and factors straight
  // to LDS; k and q, where they become fp16, by way of registers, two chunks ahead.  And what
  // the chunk two before left of output there goes out.
  if (wave >= kWaves) {
    constexpr int kFetch = scan_waves(kWaves) - kWaves;      // waves
    constexpr int kRowIts = (16 + kFetch - 1) / kFetch, kFragIts = (kFrags + 1 + kFetch - 1) / kFetch;
    const int fw = __builtin_amdgcn_readfirstlane(wave) - kWaves;
    __builtin_assume(fw < kFetch);
    u32x4 fk[kRowIts], fq[kRowIts], out[kRowIts];
    float sk[kRowIts], sq[kRowIts];
    auto load_kq = [&](unsigned c) {
      const unsigned t0 = (unsigned)s.a + c * kC, rows = min((unsigned)kC, (unsigned)s.z - t0);
      const Record* rec = ws + (size_t)(rec0 + c) * kGdnHv + h;
      const unsigned range = ((rows - 1) * p.qk_stride + kGdnDk) * 2;
      const __amdgpu_buffer_rsrc_t qrs = rows_rsrc(p.q + (size_t)t0 * p.qk_stride + kh * kGdnDk, range);
      const __amdgpu_buffer_rsrc_t krs = rows_rsrc(p.k + (size_t)t0 * p.qk_stride + kh * kGdnDk, range);
#pragma unroll
      for (int n = 0; n < kRowIts; ++n) {        // behind row 63: behind the ranges, zeros
        const unsigned row = 4 * (fw + n * kFetch) + lg, off = (row * p.qk_stride + 8 * li) * 2;
        fk[n] = load16(krs, off);
        fq[n] = load16(qrs, off);
        sk[n] = rec->f[kKs + (row & 63)];
        sq[n] = rec->f[kQs + (row & 63)];
      }
    };
    auto stage_kq = [&](unsigned c) {
      ScanBuf& o = buf[c & 1];
#pragma unroll
      for (int n = 0; n < kRowIts; ++n) {
        const int i = fw + n * kFetch, at = row_at((4 * i + lg) & 63, li);
        if (i < 16) {
          *reinterpret_cast<f16x8*>(o.kr + at) = to_f16(fk[n], sk[n]);
          *reinterpret_cast<f16x8*>(o.qr + at) = to_f16(fq[n], sq[n]);
        }
      }
    };
    // a lane's 16 bytes of a row of the output are those of v that it fetches next
    const __amdgpu_buffer_rsrc_t ors =
        rows_rsrc(p.out + ((size_t)s.a * kGdnHv + h) * kGdnDv, ((len - 1) * kGdnHv + 1) * (unsigned)(kGdnDv * 2));
    auto read_out = [&](unsigned c) {
#pragma unroll
      for (int n = 0; n < kRowIts; ++n)
        out[n] = *reinterpret_cast<const u32x4*>(buf[c & 1].vr + 4 * min(fw + n * kFetch, 15) * kGdnDk + 8 * lane);
    };
    auto store_out = [&](unsigned c) {
#pragma unroll
      for (int n = 0; n < kRowIts; ++n) {       // rows behind the sequence fall outside the range and are dropped
        const int i = fw + n * kFetch, row = 4 * i + lg, chunk = li ^ row_key(row);
        const bool own = i < 16 && (unsigned)chunk / (2 * kWaves) == rest % kGroups;      // the workgroup's columns
        const unsigned off = own ? (c * kC + row) * (kGdnHv * kGdnDv * 2) + 16 * chunk : ~15u;
        __builtin_amdgcn_raw_buffer_store_b128(out[n], ors, (int)off, 0, 0);
      }
    };
    auto fetch = [&](unsigned c) {
      const unsigned t0 = (unsigned)s.a + c * kC, rows = min((unsigned)kC, (unsigned)s.z - t0);
      ScanBuf& o = buf[c & 1];
      const u32x4 rrs = g_rsrc(ws + (size_t)(rec0 + c) * kGdnHv + h, sizeof(Record));
#pragma unroll
      for (int n = 0; n < kFragIts; ++n) {       // (the factors follow the fragments)
        const int i = fw + n * kFetch;
        if (i <= kFrags) to_lds(rrs, 1024 * i + 16 * lane, i < kFrags ? (void*)(o.frag + i * 64) : (void*)o.f);
      }
      const u32x4 vrs =
          g_rsrc(p.v + (size_t)t0 * p.v_stride + h * kGdnDv, ((rows - 1) * p.v_stride + kGdnDv) * 2);
#pragma unroll
      for (int n = 0; n < kRowIts; ++n) {        // four rows of v; behind the sequence its last again (beta is 0)
        const int i = fw + n * kFetch, row = 4 * i + lg;
        if (i < 16)
          to_lds(vrs, (min((unsigned)row, rows - 1) * p.v_stride + 8 * (li ^ row_key(row))) * 2, o.vr + 4 * i * kGdnDk);
      }
    };
    load_kq(0);
    fetch(0);
    stage_kq(0);
    load_kq(min(1u, last));
    __builtin_amdgcn_s_waitcnt(kVmcnt(0));
    lds_barrier();
    for (unsigned c = 0; c < chunks; ++c) {      // beside chunk c
      if (c >= 1) read_out(c - 1);
      if (c < last) {
        stage_kq(c + 1);
        load_kq(min(c + 2, last));
        __builtin_amdgcn_s_waitcnt(0xC07F);       // what was read of v's place, before v is fetched there
        fetch(c + 1);
      }
      if (c >= 1) {
        store_out(c - 1);
        __builtin_amdgcn_s_waitcnt(kVmcnt(kRowIts));      // all but the stores
      } else {
        __builtin_amdgcn_s_waitcnt(kVmcnt(0));
      }
      lds_barrier();      // chunk c is done with, c + 1 is there
    }
    read_out(last);
    store_out(last);
    return;
  }

  // ---- the wave's columns
  const int col0 = 16 * ((int)(rest % kGroups) * kWaves + wave);
  float* sp = p.states + (size_t)s.slot * p.slot_stride + (size_t)h * kGdnDk * kGdnDv + 8 * lg * p.row_step +
              (col0 + li) * p.col_step;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  auto state_row = [&](int i, int r) { return (32 * (i >> 1) + 4 * (i & 1) + r) * p.row_step; };
  f32x4 state[8];      // state[2 k + u][r]: row 32 k + 8 lg + 4 u + r
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) state[i][r] = s.has ? sp[state_row(i, r)] : 0.f;

  // The lane's places in the buffer, in bytes: chunk j ^ 4 n of a row is n << 6 away by XOR,
  // 16 rows 4096 by addition.
  const int w2 = 2 * (col0 >> 4);
  unsigned at_row = 256 * li + 16 * (lg ^ row_key(li));                                          // row li, chunk lg
  unsigned at_kt = 256 * (4 * lg + (li >> 2)) + 16 * ((li & 3) ^ row_key(4 * lg + (li >> 2)));   // row 4 lg + li / 4
  unsigned at_v = offsetof(ScanBuf, vr) + 256 * (4 * lg + (li >> 2)) +
                  16 * ((w2 + ((li & 3) >> 1)) ^ row_key(4 * lg + (li >> 2))) + 8 * (li & 1);
  unsigned at_o = offsetof(ScanBuf, vr) + 256 * (4 * lg) + 16 * ((w2 + (li >> 3)) ^ row_key(4 * lg)) + 2 * (li & 7);
  unsigned at_f = 16 * lg, at_frag = offsetof(ScanBuf, frag) + 16 * lane;
  int step = sizeof(ScanBuf);
  constexpr unsigned kKr = offsetof(ScanBuf, kr), kQr = offsetof(ScanBuf, qr);
  f16x8 kf[2][4];
  auto read_rows = [&](unsigned m, int k, f16x8 (&o)[4]) {
    const char* from = smem + (at_row ^ (k << 6));
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = *reinterpret_cast<const f16x8*>(from + m + 4096 * i);
  };
  auto factors = [&](int which, int i) { return *reinterpret_cast<const f32x4*>(smem + at_f + 4 * which + 64 * i); };
  // fragments 2 part, 2 part + 1 of T or A, in their order: tokens 16 i .. by 32 k ..
  f16x8 fa[4], fb[4];
  auto read_frags = [&](int first, int part, f16x8 (&o)[4]) {
#pragma unroll
    for (int n = 0; n < 4; ++n) o[n] = *reinterpret_cast<const f16x8*>(smem + at_frag + 1024 * (first + 4 * part + n));
  };
  auto frag_i = [](int f) { return f < 2 ? f : 2 + ((f - 2) >> 1); };
  auto frag_k = [](int f) { return f < 2 ? 0 : f & 1; };

  // The chain of a chunk is S -> k S -> rows -> T rows -> decayed v' -> S.  What does not wait
  // for it (q S, A v', the output) stands beside products or vector instructions
  // that would stand alone, and LDS is read a step ahead; fences and group orders hold the
  // compiler to that.  What still stands alone runs beside the SIMD's other wave.
  ColumnMax top;
#pragma unroll
  for (int i = 0; i < 8; ++i) top.take(state[i]);
  float egl_next = (ws + (size_t)rec0 * kGdnHv + h)->f[kEgl];
  __builtin_amdgcn_s_waitcnt(kVmcnt(0));       // here, not in every round of the loop
  lds_barrier();
  for (unsigned c = 0; c < chunks; ++c) {
    const float egl = egl_next;
    f16x8 sh[4], sl[4];
    f32x4 ks[4], qs[4];
    float ss, si;
    read_rows(kKr, 0, kf[0]);
    scale_of(top.bits(), ss, si);
    split8(state[0], state[1], ss, sh[0], sl[0]);
    kFence;
    egl_next = (ws + (size_t)(rec0 + min(c + 1, last)) * kGdnHv + h)->f[kEgl];
    // k' S, S in parts
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      read_rows(k < 3 ? kKr : kQr, (k + 1) & 3, kf[(k + 1) & 1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) ks[i] = mfma_f16(kf[k & 1][i], sl[k], k == 0 ? zero : ks[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) ks[i] = mfma_f16(kf[k & 1][i], sh[k], ks[i]);
      if (k < 3) split8(state[2 * k + 2], state[2 * k + 3], ss, sh[k + 1], sl[k + 1]);
      kBeside(8, 3);
    }
    // q' S, rows beta (v - e^G k S)
    ColumnMax ztop;
    i16x4 v4[4];
    f32x4 bt[4], cy[4];
    auto read_in = [&](int i) {
      v4[i] = lds_read_tr16(reinterpret_cast<const bf16*>(smem + at_v + 4096 * i));
      bt[i] = factors(kBeta, i);
      cy[i] = factors(kBcy, i);
    };
    read_in(0);
    kFence;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k < 3) {
        read_rows(kQr, k + 1, kf[(k + 1) & 1]);
        read_in(k + 1);
      }
      if (k >= 2) read_frags(0, k - 2, k == 2 ? fa : fb);
#pragma unroll
      for (int i = 0; i < 4; ++i) qs[i] = mfma_f16(kf[k & 1][i], sl[k], k == 0 ? zero : qs[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) qs[i] = mfma_f16(kf[k & 1][i], sh[k], qs[i]);
      cy[k] *= si;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        ks[k][r] = __builtin_fmaf(-cy[k][r], ks[k][r],
                                  bt[k][r] * __uint_as_float((unsigned)(unsigned short)v4[k][r] << 16));
      ztop.take(ks[k]);
      kBeside(8, 3);
    }
    float zs, zi;
    f16x8 xh[2], xl[2];
    scale_of(ztop.bits(), zs, zi);
#pragma unroll
    for (int k = 0; k < 2; ++k) split8(ks[2 * k], ks[2 * k + 1], zs, xh[k], xl[k]);
    f32x4 rq[4], rk[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rq[i] = factors(kRsq, i);
    kFence;
    // v' = T rows, times 2^8 and the rows' scale: low T by high rows, high by low, high by high
    auto t_rows = [&](int part, const f16x8 (&m)[4]) {
#pragma unroll
      for (int n = 0; n < 3; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = frag_i(2 * part + j), k = frag_k(2 * part + j);
          ks[i] = mfma_f16(m[2 * j + (n == 0)], n == 1 ? xl[k] : xh[k], n == 0 && k == 0 ? zero : ks[i]);
        }
    };
    t_rows(0, fa);
    kBeside(6, 0);
    t_rows(1, fb);
    read_frags(0, 2, fa);
#pragma unroll
    for (int i = 0; i < 2; ++i) qs[i] *= rq[i] * si;
    kBeside(6, 3);
    t_rows(2, fa);
    read_frags(kFragA, 0, fb);
#pragma unroll
    for (int i = 2; i < 4; ++i) qs[i] *= rq[i] * si;
    kBeside(6, 3);
    // decayed v', A v'
    bf16x8 vh[2], vl[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) split8(ks[2 * k], ks[2 * k + 1], vh[k], vl[k]);
#pragma unroll
    for (int i = 0; i < 4; ++i) rk[i] = factors(kRsk, i);
    kFence;
    f32x4 av[4];
    auto a_rows = [&](int part, const f16x8 (&m)[4]) {
#pragma unroll
      for (int n = 0; n < 3; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = frag_i(2 * part + j), k = frag_k(2 * part + j);
          av[i] = mfma16x16x32(__builtin_bit_cast(bf16x8, m[2 * j + (n == 0)]), n == 1 ? vl[k] : vh[k],
                               n == 0 && k == 0 ? zero : av[i]);
        }
    };
    f16x8 kt[2][4];
    auto read_kt = [&](int g) {        // rows 64 (g / 2) .. of S, tokens 32 (g % 2) ..
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 4 * (g >> 1) + j;
        const bf16* from =
            reinterpret_cast<const bf16*>(smem + (at_kt ^ ((i >> 1) << 6)) + kKr + 8 * (i & 1) + 8192 * (g & 1));
        kt[g & 1][j] = __builtin_bit_cast(f16x8, cat_bf16x8(lds_read_tr16(from), lds_read_tr16(from + 2048)));
      }
    };
    ColumnMax wtop;
    float wsc, wi;
    a_rows(0, fb);
    read_frags(kFragA, 1, fa);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ks[i] *= rk[i];
      wtop.take(ks[i]);
    }
    kBeside(6, 4);
    a_rows(1, fa);
    read_frags(kFragA, 2, fb);
    scale_of(wtop.bits(), wsc, wi);
    split8(ks[0], ks[1], wsc, xh[0], xl[0]);
    wi *= zi;
    kBeside(6, 6);
    a_rows(2, fb);
    read_kt(0);
    split8(ks[2], ks[3], wsc, xh[1], xl[1]);
    kBeside(6, 4);
    // S <- e^Glast S + k'^T decayed v'; the output e^G q S + A v', in place of the columns' v
    const float ai = zi * 0.00390625f;
    top = ColumnMax{};
    f32x4 up[2][4];
    auto update = [&](int i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) state[i][r] = __builtin_fmaf(up[i >> 2][i & 3][r], wi, egl * state[i][r]);
      top.take(state[i]);
    };
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (g < 3) read_kt(g + 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) up[g >> 1][j] = mfma_f16(kt[g & 1][j], xl[g & 1], (g & 1) == 0 ? zero : up[g >> 1][j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) up[g >> 1][j] = mfma_f16(kt[g & 1][j], xh[g & 1], up[g >> 1][j]);
#pragma unroll
      for (int i = 2 * (g & 1); i < 2 * (g & 1) + 2; ++i) {
        if (g < 2) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            *reinterpret_cast<bf16*>(smem + (at_o ^ (r << 6)) + 256 * r + 4096 * i) =
                f2bf(__builtin_fmaf(av[i][r], ai, qs[i][r]));
        } else {
          update(i);
        }
      }
      kBeside(8, 3);
    }
#pragma unroll
    for (int i = 4; i < 8; ++i) update(i);
    lds_barrier();
    at_row += step;
    at_kt += step;
    at_v += step;
    at_o += step;
    at_f += step;
    at_frag += step;
    step = -step;
    kPin(at_row);
    kPin(at_kt);
    kPin(at_v);
    kPin(at_o);
    kPin(at_f);
    kPin(at_frag);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) sp[state_row(i, r)] = state[i][r];
}

// Sequences that can be long, and records for their chunks.
unsigned most_long(const RaggedBatch& b) {
  const unsigned n = b.tokens / (kShort + 1);
  return n < b.seqs ? n : b.seqs;
}
unsigned most_records(const RaggedBatch& b) { return b.tokens / kC + most_long(b); }
// Chunks are not needed where the host knows that no sequence is long (one that is all
// the same goes token by token).
bool by_chunks(const RaggedBatch& b, unsigned longest) {
  return b.tokens > kFewRows && (longest == 0 || longest > kShort);
}

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT size_t qwen36_gdn_ragged_delta_workspace_bytes(const qwen36_state_batch* batch, unsigned longest) {
  RaggedBatch b;
  if (!ragged_batch_of(batch, b) || !by_chunks(b, longest)) return 0;
  return (size_t)most_records(b) * kGdnHv * sizeof(Record);
}

Q36_EXPORT int qwen36_gdn_ragged_delta_ex(const void* q, const void* k, const void* v, unsigned qk_heads,
                                          unsigned qk_token_stride, unsigned v_token_stride, const void* g,
                                          const void* beta, void* states, size_t slot_stride,
                                          const qwen36_state_batch* batch, unsigned longest, unsigned flags,
                                          void* out, void* workspace, size_t workspace_bytes, void* stream) {
  RaggedBatch b;
  if (q == nullptr || k == nullptr || v == nullptr || g == nullptr || beta == nullptr || states == nullptr ||
      out == nullptr || !ragged_batch_of(batch, b) || (qk_heads != 16u && qk_heads != 32u) ||
      qk_token_stride < qk_heads * kGdnDk || qk_token_stride % 8 != 0 || qk_token_stride > kMaxStride ||
      v_token_stride > kMaxStride || v_token_stride < (unsigned)(kGdnHv * kGdnDv) || v_token_stride % 8 != 0 ||
      slot_stride < (size_t)kGdnHv * kGdnDk * kGdnDv || slot_stride % 4 != 0 || !aligned16(q) ||
      !aligned16(k) || !aligned16(v) || !aligned16(states) || !aligned16(out) ||
      (flags & ~(QWEN36_GDN_QK_NORMALIZED | QWEN36_GDN_STATE_VK)) != 0)
    return Q36_EINVAL;
  const bool vk = (flags & QWEN36_GDN_STATE_VK) != 0;
  const size_t need = qwen36_gdn_ragged_delta_workspace_bytes(batch, longest);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) return Q36_EINVAL;
  const DeltaArgs p = {static_cast<const bf16*>(q),  static_cast<const bf16*>(k),
                       static_cast<const bf16*>(v),  static_cast<const float*>(g),
                       static_cast<const float*>(beta), static_cast<float*>(states),
                       static_cast<bf16*>(out), slot_stride, qk_heads, qk_token_stride, v_token_stride,
                       (flags & QWEN36_GDN_QK_NORMALIZED) != 0, vk ? 1 : kGdnDv, vk ? kGdnDk : 1};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool chunks = by_chunks(b, longest);
  if (!chunks) {
    hipLaunchKernelGGL(gdn_ragged_step_kernel, dim3(b.seqs * 128), dim3(256), 0, st, p, b);
    return static_cast<int>(hipGetLastError());
  }
  static std::once_flag once;
  static hipError_t attr = hipSuccess;
  std::call_once(once, [] {
    auto allow = [](const void* f, size_t bytes) {
      if (attr == hipSuccess) attr = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    };
    allow(reinterpret_cast<const void*>(gdn_ragged_scan_kernel<2>), 2 * sizeof(ScanBuf));
    allow(reinterpret_cast<const void*>(gdn_ragged_scan_kernel<4>), 2 * sizeof(ScanBuf));
    allow(reinterpret_cast<const void*>(gdn_ragged_scan_kernel<8>), 2 * sizeof(ScanBuf));
    allow(reinterpret_cast<const void*>(gdn_ragged_prep_kernel<1>), sizeof(PrepLds<1>));
    allow(reinterpret_cast<const void*>(gdn_ragged_prep_kernel<2>), sizeof(PrepLds<2>));
  });
  if (attr != hipSuccess) return static_cast<int>(attr);
  Record* ws = static_cast<Record*>(workspace);
  const unsigned blocks = most_records(b) * (qk_heads == 16 ? 16 : 32);
  const dim3 grid(blocks + b.seqs * 128);
  if (qk_heads == 16)
    hipLaunchKernelGGL(gdn_ragged_prep_kernel<2>, grid, dim3(256), sizeof(PrepLds<2>), st, p, b, ws, blocks);
  else
    hipLaunchKernelGGL(gdn_ragged_prep_kernel<1>, grid, dim3(256), sizeof(PrepLds<1>), st, p, b, ws, blocks);
  // Few sequences leave CUs, one a workgroup: their columns in two or four.  Sequences of
  // 2,000 tokens, all in all, by 2, 4 and 8 chains a workgroup, us: one 90, 93 and 134; two 98,
  // 104 and 144; three 183, 123 and 160; four 198, 145 and 173; five 282, 236 and 185; eight
  // 394, 290 and 245.  Two of 4,096: 193, 215 and 282.
  // n is how many sequences may be long, as the host knows no more.  A prompt beside many
  // single tokens goes by 8 chains: 2,000 beside 40 take 159 us (116 by 2 chains), 8,192 beside
  // 63 541 (364).
  const unsigned n = most_long(b);
  const unsigned lds = 2 * sizeof(ScanBuf);
  if (n <= 2)
    hipLaunchKernelGGL(gdn_ragged_scan_kernel<2>, dim3(n * kGdnHv * 4), dim3(512), lds, st, p, b, ws, n);
  else if (n <= 4)
    hipLaunchKernelGGL(gdn_ragged_scan_kernel<4>, dim3(n * kGdnHv * 2), dim3(512), lds, st, p, b, ws, n);
  else
    hipLaunchKernelGGL(gdn_ragged_scan_kernel<8>, dim3(n * kGdnHv), dim3(64 * scan_waves(8)), lds, st, p, b, ws, n);
  return static_cast<int>(hipGetLastError());
}

Q36_EXPORT int qwen36_gdn_ragged_delta(const void* q, const void* k, const void* v, unsigned qk_heads,
                                       unsigned qk_token_stride, unsigned v_token_stride, const void* g,
                                       const void* beta, void* states, size_t slot_stride,
                                       const qwen36_state_batch* batch, unsigned longest, void* out,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  return qwen36_gdn_ragged_delta_ex(q, k, v, qk_heads, qk_token_stride, v_token_stride, g, beta, states, slot_stride,
                                    batch, longest, 0, out, workspace, workspace_bytes, stream);
}
