// The gated delta rule over a ragged batch with its states in slots.
//
// Per value head (key head h * qk_heads / 32) and token, with the state S [128 k]
// [128 v] in fp32:
//   q, k <- x / sqrt(sum x^2 + 1e-6), q *= 1/sqrt(128)
//   S <- e^g S;  d = beta (v - k S);  S <- S + k (x) d;  o = q S
// A sequence begins with its slot's state (zeros where it has none) and leaves its
// last one there.
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
};

// ---------------------------------------------------------------------------
// Token by token: sequences of up to `limit` tokens.
// Bound by the states' bytes (4.2 MB a sequence, read and written).  Both
// reductions of a token, S^T k and S^T q, are taken of the state before it:
// o = e^g S_old^T q + d (k.q), so that a token costs one exchange between waves.
// One workgroup owns 32 columns of a head: thread (rg, cq) rows rg + 32 i and
// columns 4 cq .. +3, a row of the 32 columns being one 128-byte line.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void gdn_ragged_step_kernel(DeltaArgs p, RaggedBatch b, unsigned limit) {
  __shared__ f32x4 red[2][4][2][8];    // [parity][wave][k | q][column quad]
  __shared__ float dots[2][4][4];      // [parity][wave][k.k, q.q, k.q]
  const unsigned seq = blockIdx.x >> 7;
  const int h = (blockIdx.x >> 2) & 31, cg = blockIdx.x & 3;
  const RaggedSeq s = ragged_seq(b, seq);
  const unsigned len = (unsigned)(s.z - s.a);
  if (s.slot < 0 || len == 0 || len > limit) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int rg = tid >> 3, cq = tid & 7;
  const int col = 32 * cg + 4 * cq;
  const int kh = h * (int)p.qk_heads / kGdnHv;
  float* sp = p.states + (size_t)s.slot * p.slot_stride + ((size_t)h * kGdnDk + rg) * kGdnDv + col;
  f32x4 st[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    st[i] = s.has ? __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(sp + 32 * i * kGdnDv))
                  : f32x4{0.f, 0.f, 0.f, 0.f};
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
    const float kinv = 1.0f / sqrtf(nk + 1e-6f), qn = kQScale / sqrtf(nq + 1e-6f);
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
  for (int i = 0; i < 4; ++i) __builtin_nontemporal_store(st[i], reinterpret_cast<f32x4*>(sp + 32 * i * kGdnDv));
}

// ---------------------------------------------------------------------------
// Chunks of 64 tokens: longer sequences.
//
// With G the sum of g from the chunk's first token on, S the state before it:
//   L = strictly lower part of diag(beta) (k k^T) e^(Gi - Gj),  T = (I + L)^-1 diag(beta)
//   v' = T (v - diag(e^G) k S)
//   o  = diag(e^G) q S + A v',  A = lower part of (q k^T) e^(Gi - Gj)
//   S <- e^Glast S + k^T diag(e^(Glast - G)) v'
// The norms of q and k and the decays are row factors in fp32; products are taken of
// the raw q and k, which bf16 holds.
//
// Precision: an fp32 operand enters bf16 products as the sum of three bf16 values
// (24 bits together) wherever the state is computed from it: S, v' and the rows
// v - .. against exact k, six products of T by those rows (all above 2^-24).  What
// only reaches the output, which is rounded to bf16, takes two (2^-17): S against q,
// A and v' against each other.
//
//  * gdn_ragged_prep_kernel, a workgroup a (chunk, head): T and A, which do not
//    depend on the state, in fp32, and the row factors: a record of 25,600 bytes.
//  * gdn_ragged_scan_kernel, a workgroup a (sequence, head or part of its columns),
//    chunk after chunk.  A wave owns 16 columns of v with all 128 rows of their
//    state, in registers: the layout of a product's result is that of the next one's
//    right operand, so that nothing of a column's recurrence leaves its wave, and waves
//    meet once a chunk, where the next chunk's k, q, T and A are ready in LDS.
// ---------------------------------------------------------------------------

constexpr int kC = 64;
constexpr unsigned kShort = 12;           // longer sequences go by chunks
constexpr int kPitchR = 136;              // bf16 row pitch of [64][128] tiles: 272 bytes
constexpr int kPitchF = 68;               // fp32 row pitch of [64][64] matrices

// A record: T and A as fp32 rows (0 .. 31: 32 columns, 32 .. 63: all 64), then
// e^G / |k|, e^G / (|q| sqrt(128)), e^(Glast - G) / |k| of each token and e^Glast.
constexpr unsigned kRecM = 32 * 32 + 32 * 64;
constexpr unsigned kRecS = 2 * kRecM;
constexpr unsigned kRecFloats = kRecS + 4 * kC;
constexpr size_t kRecBytes = kRecFloats * 4;

__device__ __forceinline__ unsigned rec_row(unsigned i) { return i < 32 ? 32 * i : 1024 + 64 * (i - 32); }

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

struct PrepLds {
  union {
    bf16 kr[kC * kPitchR];      // k rows; dead once k k^T is in registers
    float lm[kC * kPitchF];     // L
  } u;
  float tm[kC * kPitchF];       // (I + L)^-1; its upper blocks hold sums on the way
  float gs[kC], gl[kC];         // G = gs + gl: differences of fast decays keep their bits
  float bs[kC], kinv[kC], qinv[kC];
};

// C += A B of 16x16 fp32 blocks of [64][kPitchF] matrices.
__device__ __forceinline__ f32x4 mm16(const float* a, int ar, int ac, const float* b, int br, int bc, f32x4 acc,
                                      int li, int lg) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
    acc = mfma16x16x4f32(a[(ar + li) * kPitchF + ac + 4 * s + lg], b[(br + 4 * s + lg) * kPitchF + bc + li], acc);
  return acc;
}

// Lower 16x16 tile t (0 .. 9): its row and column of tiles.
__device__ __forceinline__ int tri_row(int t) { return (t >= 1) + (t >= 3) + (t >= 6); }
__device__ __forceinline__ int tri_col(int t) {
  const int r = tri_row(t);
  return t - r * (r + 1) / 2;
}

__global__ __launch_bounds__(256, 4) void gdn_ragged_prep_kernel(DeltaArgs p, RaggedBatch b, float* __restrict__ ws) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  PrepLds& s = *reinterpret_cast<PrepLds*>(smem);
  // the heads of a key head on one XCD, as in the scan
  const unsigned slot = blockIdx.x >> 3, rec_i = slot >> 2;
  const int h = 4 * (blockIdx.x & 7) + (slot & 3);
  RaggedSeq q;
  unsigned chunk;
  if (!find_record(b, rec_i, q, chunk)) return;
  const int kh = h * (int)p.qk_heads / kGdnHv;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const unsigned tok0 = (unsigned)q.a + chunk * kC, rows = min((unsigned)kC, (unsigned)q.z - tok0);
  float* rec = ws + ((size_t)rec_i * kGdnHv + h) * kRecFloats;
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
  if (wave < 2) {
    const float* from = wave == 0 ? p.g : p.beta;
    const float v = (unsigned)lane < rows ? from[(size_t)(tok0 + lane) * kGdnHv + h] : 0.f;
    if (wave == 0) {
      double sum = v;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(sum, o, 64);
        if (lane >= o) sum += u;
      }
      s.gs[lane] = (float)sum;
      s.gl[lane] = (float)(sum - (double)(float)sum);
    } else {
      s.bs[lane] = v;
    }
  }
  float kss = 0.f, qss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    *reinterpret_cast<bf16x8*>(&s.u.kr[r1 * kPitchR + 32 * p1 + 8 * i]) = k8[i];
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
    s.kinv[r1] = 1.0f / sqrtf(kss + 1e-6f);
    s.qinv[r1] = kQScale / sqrtf(qss + 1e-6f);
  }
  lds_barrier();
  if (tid < kC) {
    const float gi = s.gs[tid], eg = expf(gi), left = (s.gs[kC - 1] - gi) + (s.gl[kC - 1] - s.gl[tid]);
    rec[kRecS + tid] = eg * s.kinv[tid];
    rec[kRecS + kC + tid] = eg * s.qinv[tid];
    rec[kRecS + 2 * kC + tid] = s.kinv[tid] * expf(left);
    rec[kRecS + 3 * kC + tid] = expf(s.gs[kC - 1]);
  }
  // k k^T and q k^T of the lower tiles, five a wave; q straight from memory
  f32x4 job[5];
#pragma unroll
  for (int jj = 0; jj < 5; ++jj) {
    const int j = wave + 4 * jj, t = j >= 10 ? j - 10 : j, rt = tri_row(t), ct = tri_col(t);
    const bf16* brow = s.u.kr + (16 * ct + li) * kPitchR + 8 * lg;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (j >= 10) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {     // transposed: row 4 lg + r is column j
        const u32x4 qf = load16(qrs, ((16 * rt + li) * p.qk_stride + 32 * k + 8 * lg) * 2);
        acc = mfma16x16x32(ld8(brow + 32 * k), __builtin_bit_cast(bf16x8, qf), acc);
      }
    } else {
      const bf16* arow = s.u.kr + (16 * rt + li) * kPitchR + 8 * lg;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc = mfma16x16x32(ld8(arow + 32 * k), ld8(brow + 32 * k), acc);
    }
    job[jj] = acc;
  }
  lds_barrier();     // the k rows make room for L
#pragma unroll
  for (int jj = 0; jj < 5; ++jj) {
    const int j = wave + 4 * jj, t = j >= 10 ? j - 10 : j, rt = tri_row(t), ct = tri_col(t);
    // decays behind the diagonal may overflow: chosen against, not multiplied by zero
    if (j >= 10) {
      const int i = 16 * rt + li, j0 = 16 * ct + 4 * lg;
      const float gi = s.gs[i], hi = s.gl[i], qi = s.qinv[i];
      const f32x4 gj = *reinterpret_cast<const f32x4*>(s.gs + j0), hj = *reinterpret_cast<const f32x4*>(s.gl + j0);
      const f32x4 kj = *reinterpret_cast<const f32x4*>(s.kinv + j0);
      f32x4 a;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        a[r] = j0 + r <= i ? ((qi * kj[r]) * job[jj][r]) * expf((gi - gj[r]) + (hi - hj[r])) : 0.f;
      *reinterpret_cast<f32x4*>(rec + kRecM + rec_row(i) + j0) = a;
    } else {
      const int c = 16 * ct + li, i0 = 16 * rt + 4 * lg;
      const float gj = s.gs[c], hj = s.gl[c], kj = s.kinv[c];
      const f32x4 gi = *reinterpret_cast<const f32x4*>(s.gs + i0), hi = *reinterpret_cast<const f32x4*>(s.gl + i0);
      const f32x4 ki = *reinterpret_cast<const f32x4*>(s.kinv + i0);
      const f32x4 bi = *reinterpret_cast<const f32x4*>(s.bs + i0);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s.u.lm[(i0 + r) * kPitchF + c] =
            c < i0 + r ? (((ki[r] * kj) * job[jj][r]) * bi[r]) * expf((gi[r] - gj) + (hi[r] - hj)) : 0.f;
    }
  }
  // upper tiles that the rows of a record hold: (0, 1) and (2, 3)
  if (tid < 128) {
    const unsigned i = 32 * (tid >> 6) + li, j0 = 32 * (tid >> 6) + 16 + 4 * lg;
    *reinterpret_cast<f32x4*>(rec + kRecM + rec_row(i) + j0) = f32x4{0.f, 0.f, 0.f, 0.f};
    *reinterpret_cast<f32x4*>(rec + rec_row(i) + j0) = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  lds_barrier();
  // (I + L)^-1: diagonal 16x16 blocks by forward substitution, a block a wave, a column a lane
  if (lane < 16) {
    const int d = 16 * wave;
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float acc = 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) acc += s.u.lm[(d + i) * kPitchF + d + m] * t[m];
      t[i] = i == lane ? 1.f : i > lane ? -acc : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s.tm[(d + i) * kPitchF + d + lane] = t[i];
  }
  lds_barrier();
  // the others by distance: T_ij = -T_ii sum_{j <= k < i} L_ik T_kj; the sum lies in block (j, i)
  for (int d = 1; d < 4; ++d) {
    const int bj = wave, bi = wave + d;
    if (bi < 4) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      for (int kb = bj; kb < bi; ++kb) x = mm16(s.u.lm, 16 * bi, 16 * kb, s.tm, 16 * kb, 16 * bj, x, li, lg);
#pragma unroll
      for (int r = 0; r < 4; ++r) s.tm[(16 * bj + 4 * lg + r) * kPitchF + 16 * bi + li] = x[r];
      // (a wave's own writes to LDS are read back in order)
      const f32x4 y = mm16(s.tm, 16 * bi, 16 * bi, s.tm, 16 * bj, 16 * bi, f32x4{0.f, 0.f, 0.f, 0.f}, li, lg);
#pragma unroll
      for (int r = 0; r < 4; ++r) s.tm[(16 * bi + 4 * lg + r) * kPitchF + 16 * bj + li] = -y[r];
    }
    lds_barrier();
  }
  for (int idx = tid; idx < 10 * 64; idx += 256) {
    const int t = idx >> 6, i = 16 * tri_row(t) + ((idx >> 2) & 15), j0 = 16 * tri_col(t) + 4 * (idx & 3);
    const f32x4 v = *reinterpret_cast<const f32x4*>(s.tm + i * kPitchF + j0);
    *reinterpret_cast<f32x4*>(rec + rec_row(i) + j0) = v * *reinterpret_cast<const f32x4*>(s.bs + j0);
  }
}

// ---- scan --------------------------------------------------------------------

// Products of 32 of the reduction index, as LDS holds their left operands: T and A of
// token tiles (t, u) (tokens 32 t + 8 (m / 4) + 4 u + m % 4 for row m) by 32 tokens k:
// fragment 0, 1: (0, u) k = 0; 2 .. 5: (1, u) k = 0, 1.
struct ScanBuf {
  bf16 kr[kC * kPitchR], qr[kC * kPitchR];
  bf16x8 tf[6][3][64], af[6][2][64];
  float sc[4 * kC];
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// x as kParts bf16 values, each of what the ones before leave.
template <int kParts>
__device__ __forceinline__ void split8(const f32x4& a, const f32x4& b, bf16x8 (&o)[kParts]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x4& v = e < 2 ? a : b;
    float x0 = v[2 * (e & 1)], x1 = v[2 * (e & 1) + 1];
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      const bf16x2 y = __builtin_convertvector(f32x2{x0, x1}, bf16x2);
      o[n][2 * e] = y[0];
      o[n][2 * e + 1] = y[1];
      const unsigned u = __builtin_bit_cast(unsigned, y);
      x0 -= __uint_as_float(u << 16);
      x1 -= __uint_as_float(u & 0xffff0000u);
    }
  }
}

// kWaves of the workgroup's 8 waves own 16 columns each; where these are not all, the
// others only fetch.
template <int kWaves>
__global__ __launch_bounds__(512, 1) void gdn_ragged_scan_kernel(DeltaArgs p, RaggedBatch b,
                                                                 const float* __restrict__ ws, unsigned most) {
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
  const unsigned len = (unsigned)(s.z - s.a), chunks = (len + kC - 1) / kC;

  // ---- fetching: a chunk ahead in registers, then in the other buffer
  constexpr int kFirst = kWaves < 8 ? 64 * kWaves : 0, kFetch = 512 - kFirst;
  constexpr int kRowIts = (1024 + kFetch - 1) / kFetch, kFragIts = (384 + kFetch - 1) / kFetch;
  const bool fetches = tid >= kFirst;
  const int ft = tid - kFirst;
  u32x4 fk[kRowIts], fq[kRowIts];
  f32x4 fT[kFragIts][2], fA[kFragIts][2], fs;
  auto fetch = [&](unsigned c) {
    const unsigned t0 = (unsigned)s.a + c * kC, rows = min((unsigned)kC, (unsigned)s.z - t0);
    const unsigned range = ((rows - 1) * p.qk_stride + kGdnDk) * 2;
    const __amdgpu_buffer_rsrc_t qrs = rows_rsrc(p.q + (size_t)t0 * p.qk_stride + kh * kGdnDk, range);
    const __amdgpu_buffer_rsrc_t krs = rows_rsrc(p.k + (size_t)t0 * p.qk_stride + kh * kGdnDk, range);
    const float* rec = ws + ((size_t)(rec0 + c) * kGdnHv + h) * kRecFloats;
#pragma unroll
    for (int n = 0; n < kRowIts; ++n) {
      const unsigned i = ft + n * kFetch;        // behind row 63: behind the range, zeros
      const unsigned off = ((i >> 4) * p.qk_stride + 8 * (i & 15)) * 2;
      fk[n] = load16(krs, off);
      fq[n] = load16(qrs, off);
    }
#pragma unroll
    for (int n = 0; n < kFragIts; ++n) {
      const unsigned i = min(ft + n * kFetch, 383), f = i >> 6, l = i & 63, m = l & 15;
      const unsigned row = (f >= 2 ? 32 : 0) + 8 * (m >> 2) + 4 * (f & 1) + (m & 3);
      const unsigned at = rec_row(row) + (f >= 4 ? 32 : 0) + 8 * (l >> 4);
      fT[n][0] = *reinterpret_cast<const f32x4*>(rec + at);
      fT[n][1] = *reinterpret_cast<const f32x4*>(rec + at + 4);
      fA[n][0] = *reinterpret_cast<const f32x4*>(rec + kRecM + at);
      fA[n][1] = *reinterpret_cast<const f32x4*>(rec + kRecM + at + 4);
    }
    fs = *reinterpret_cast<const f32x4*>(rec + kRecS + 4 * (ft & 63));
  };
  auto stage = [&](unsigned c) {
    ScanBuf& o = buf[c & 1];
#pragma unroll
    for (int n = 0; n < kRowIts; ++n) {
      const int i = ft + n * kFetch, at = (i >> 4) * kPitchR + 8 * (i & 15);
      if (i < 1024) {
        *reinterpret_cast<u32x4*>(o.kr + at) = fk[n];
        *reinterpret_cast<u32x4*>(o.qr + at) = fq[n];
      }
    }
#pragma unroll
    for (int n = 0; n < kFragIts; ++n) {
      const int i = ft + n * kFetch;
      if (i < 384) {
        bf16x8 t3[3], a2[2];
        split8<3>(fT[n][0], fT[n][1], t3);
        split8<2>(fA[n][0], fA[n][1], a2);
#pragma unroll
        for (int e = 0; e < 3; ++e) o.tf[i >> 6][e][i & 63] = t3[e];
#pragma unroll
        for (int e = 0; e < 2; ++e) o.af[i >> 6][e][i & 63] = a2[e];
      }
    }
    if (ft < 64) *reinterpret_cast<f32x4*>(o.sc + 4 * ft) = fs;
  };
  const unsigned last = chunks - 1;
  if (fetches) {
    fetch(0);
    stage(0);
    fetch(min(1u, last));
  }
  if (kWaves < 8 && wave >= kWaves) {
    lds_barrier();
    for (unsigned c = 0; c < chunks; ++c) {
      if (c < last) {
        stage(c + 1);
        fetch(min(c + 2, last));
      }
      lds_barrier();
    }
    return;
  }

  // ---- the wave's columns
  const int col = 16 * ((int)(rest % kGroups) * kWaves + wave) + li;
  float* sp = p.states + (size_t)s.slot * p.slot_stride + (size_t)h * kGdnDk * kGdnDv + col;
  // state[2 k + u][r]: row 32 k + 8 lg + 4 u + r
  f32x4 state[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      state[i][r] = s.has ? sp[(32 * (i >> 1) + 8 * lg + 4 * (i & 1) + r) * kGdnDv] : 0.f;
  unsigned short vn[16];
  auto fetch_v = [&](unsigned c) {
    const unsigned t0 = (unsigned)s.a + c * kC, rows = min((unsigned)kC, (unsigned)s.z - t0);
    const __amdgpu_buffer_rsrc_t vrs =
        rows_rsrc(p.v + (size_t)t0 * p.v_stride + h * kGdnDv, ((rows - 1) * p.v_stride + kGdnDv) * 2);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const unsigned row = 32 * (i >> 3) + 8 * lg + (i & 7);
      vn[i] = __builtin_amdgcn_raw_buffer_load_b16(vrs, (int)((row * p.v_stride + col) * 2), 0, 0);
    }
  };
  fetch_v(0);
  const __amdgpu_buffer_rsrc_t ors =
      rows_rsrc(p.out + (size_t)s.a * kGdnHv * kGdnDv, len * (unsigned)(kGdnHv * kGdnDv * 2));
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int m4 = 8 * (li >> 2) + (li & 3);       // token (or dim) of operand row li, without 32 t + 4 u
  lds_barrier();
  for (unsigned c = 0; c < chunks; ++c) {
    const ScanBuf& x = buf[c & 1];
    if (kWaves == 8 && c < last) {
      stage(c + 1);
      fetch(min(c + 2, last));
    }
    // k S and q S: tiles (t, u)
    bf16x8 sb[4][3];
#pragma unroll
    for (int k = 0; k < 4; ++k) split8<3>(state[2 * k], state[2 * k + 1], sb[k]);
    f32x4 ks[4] = {zero, zero, zero, zero}, qs[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (32 * (i >> 1) + m4 + 4 * (i & 1)) * kPitchR + 32 * k + 8 * lg;
        const bf16x8 kf = ld8(x.kr + at), qf = ld8(x.qr + at);
#pragma unroll
        for (int e = 2; e >= 0; --e) ks[i] = mfma16x16x32(kf, sb[k][e], ks[i]);
#pragma unroll
        for (int e = 1; e >= 0; --e) qs[i] = mfma16x16x32(qf, sb[k][e], qs[i]);
      }
    // rows v - e^G k S
    f32x4 zr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 cy = *reinterpret_cast<const f32x4*>(x.sc + 32 * (i >> 1) + 8 * lg + 4 * (i & 1));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        zr[i][r] = bf2f(__builtin_bit_cast(bf16, vn[8 * (i >> 1) + 4 * (i & 1) + r])) - cy[r] * ks[i][r];
    }
    fetch_v(min(c + 1, last));
    bf16x8 zb[2][3];
#pragma unroll
    for (int t = 0; t < 2; ++t) split8<3>(zr[2 * t], zr[2 * t + 1], zb[t]);
    // v' = T rows
    f32x4 vp[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 2 * k; i < 4; ++i) {
        const int f = i < 2 ? i : 2 + 2 * k + (i & 1);
        const bf16x8 t0 = x.tf[f][0][lane], t1 = x.tf[f][1][lane], t2 = x.tf[f][2][lane];
        vp[i] = mfma16x16x32(t1, zb[k][1], vp[i]);
        vp[i] = mfma16x16x32(t2, zb[k][0], vp[i]);
        vp[i] = mfma16x16x32(t0, zb[k][2], vp[i]);
        vp[i] = mfma16x16x32(t1, zb[k][0], vp[i]);
        vp[i] = mfma16x16x32(t0, zb[k][1], vp[i]);
        vp[i] = mfma16x16x32(t0, zb[k][0], vp[i]);
      }
    // o = e^G q S + A v'
    bf16x8 vb[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) split8<2>(vp[2 * t], vp[2 * t + 1], vb[t]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qs[i] *= *reinterpret_cast<const f32x4*>(x.sc + kC + 32 * (i >> 1) + 8 * lg + 4 * (i & 1));
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 2 * k; i < 4; ++i) {
        const int f = i < 2 ? i : 2 + 2 * k + (i & 1);
        const bf16x8 a0 = x.af[f][0][lane], a1 = x.af[f][1][lane];
        qs[i] = mfma16x16x32(a1, vb[k][0], qs[i]);
        qs[i] = mfma16x16x32(a0, vb[k][1], qs[i]);
        qs[i] = mfma16x16x32(a0, vb[k][0], qs[i]);
      }
    // S = e^Glast S + k^T e^(Glast - G) v'
    bf16x8 wb[2][3];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      vp[i] *= *reinterpret_cast<const f32x4*>(x.sc + 2 * kC + 32 * (i >> 1) + 8 * lg + 4 * (i & 1));
#pragma unroll
    for (int t = 0; t < 2; ++t) split8<3>(vp[2 * t], vp[2 * t + 1], wb[t]);
    const float egl = x.sc[3 * kC];
#pragma unroll
    for (int i = 0; i < 8; ++i) state[i] *= egl;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bf16* ra = x.kr + (32 * t + 8 * lg + (li >> 2)) * kPitchR + 32 * (i >> 1) + 8 * (li & 3) + 4 * (i & 1);
        const bf16x8 kt = cat_bf16x8(lds_read_tr16(ra), lds_read_tr16(ra + 4 * kPitchR));
#pragma unroll
        for (int e = 2; e >= 0; --e) state[i] = mfma16x16x32(kt, wb[t][e], state[i]);
      }
    // rows behind the sequence fall outside the range and are dropped
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned row = c * kC + 32 * (i >> 1) + 8 * lg + 4 * (i & 1) + r;
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, f2bf(qs[i][r])), ors,
                                              (int)(((row * kGdnHv + h) * kGdnDv + col) * 2), 0, 0);
      }
    lds_barrier();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) sp[(32 * (i >> 1) + 8 * lg + 4 * (i & 1) + r) * kGdnDv] = state[i][r];
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
  return most_long(b) > 0 && (longest == 0 || longest > kShort);
}

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT size_t qwen36_gdn_ragged_delta_workspace_bytes(const qwen36_state_batch* batch, unsigned longest) {
  RaggedBatch b;
  if (!ragged_batch_of(batch, b) || !by_chunks(b, longest)) return 0;
  return (size_t)most_records(b) * kGdnHv * kRecBytes;
}

Q36_EXPORT int qwen36_gdn_ragged_delta(const void* q, const void* k, const void* v, unsigned qk_heads,
                                       unsigned qk_token_stride, unsigned v_token_stride, const void* g,
                                       const void* beta, void* states, size_t slot_stride,
                                       const qwen36_state_batch* batch, unsigned longest, void* out,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  RaggedBatch b;
  if (q == nullptr || k == nullptr || v == nullptr || g == nullptr || beta == nullptr || states == nullptr ||
      out == nullptr || !ragged_batch_of(batch, b) || (qk_heads != 16u && qk_heads != 32u) ||
      qk_token_stride < qk_heads * kGdnDk || qk_token_stride % 8 != 0 || qk_token_stride > kMaxStride ||
      v_token_stride > kMaxStride || v_token_stride < (unsigned)(kGdnHv * kGdnDv) || v_token_stride % 8 != 0 ||
      slot_stride < (size_t)kGdnHv * kGdnDk * kGdnDv || slot_stride % 4 != 0 || !aligned16(q) ||
      !aligned16(k) || !aligned16(v) || !aligned16(states) || !aligned16(out))
    return Q36_EINVAL;
  const size_t need = qwen36_gdn_ragged_delta_workspace_bytes(batch, longest);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) return Q36_EINVAL;
  const DeltaArgs p = {static_cast<const bf16*>(q),  static_cast<const bf16*>(k),
                       static_cast<const bf16*>(v),  static_cast<const float*>(g),
                       static_cast<const float*>(beta), static_cast<float*>(states),
                       static_cast<bf16*>(out), slot_stride, qk_heads, qk_token_stride, v_token_stride};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool chunks = by_chunks(b, longest);
  hipLaunchKernelGGL(gdn_ragged_step_kernel, dim3(b.seqs * 128), dim3(256), 0, st, p, b, chunks ? kShort : ~0u);
  if (!chunks) return static_cast<int>(hipGetLastError());
  static std::once_flag once;
  static hipError_t attr = hipSuccess;
  std::call_once(once, [] {
    const void* scans[] = {reinterpret_cast<const void*>(gdn_ragged_scan_kernel<1>),
                           reinterpret_cast<const void*>(gdn_ragged_scan_kernel<2>),
                           reinterpret_cast<const void*>(gdn_ragged_scan_kernel<4>),
                           reinterpret_cast<const void*>(gdn_ragged_scan_kernel<8>)};
    for (const void* f : scans)
      if (attr == hipSuccess)
        attr = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)(2 * sizeof(ScanBuf)));
    if (attr == hipSuccess)
      attr = hipFuncSetAttribute(reinterpret_cast<const void*>(gdn_ragged_prep_kernel),
                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(PrepLds));
  });
  if (attr != hipSuccess) return static_cast<int>(attr);
  float* ws = static_cast<float*>(workspace);
  hipLaunchKernelGGL(gdn_ragged_prep_kernel, dim3(most_records(b) * kGdnHv), dim3(256), sizeof(PrepLds), st, p, b, ws);
  // few sequences: their columns in several workgroups, one a CU
  const unsigned n = most_long(b);
  const unsigned lds = 2 * sizeof(ScanBuf);
  if (n <= 1)
    hipLaunchKernelGGL(gdn_ragged_scan_kernel<1>, dim3(n * kGdnHv * 8), dim3(512), lds, st, p, b, ws, n);
  else if (n <= 2)
    hipLaunchKernelGGL(gdn_ragged_scan_kernel<2>, dim3(n * kGdnHv * 4), dim3(512), lds, st, p, b, ws, n);
  else if (n <= 4)
    hipLaunchKernelGGL(gdn_ragged_scan_kernel<4>, dim3(n * kGdnHv * 2), dim3(512), lds, st, p, b, ws, n);
  else
    hipLaunchKernelGGL(gdn_ragged_scan_kernel<8>, dim3(n * kGdnHv), dim3(512), lds, st, p, b, ws, n);
  return static_cast<int>(hipGetLastError());
}
