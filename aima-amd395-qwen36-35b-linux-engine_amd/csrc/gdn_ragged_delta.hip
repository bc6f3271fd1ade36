// The gated delta rule over a ragged batch with its states in slots.
//
// Per value head (key head h * qk_heads / 32) and token, with the state S [128 k]
// [128 v] in fp32:
//   q, k <- x / sqrt(sum x^2 + 1e-6), q *= 1/sqrt(128)
//   S <- e^g S;  d = beta (v - k S);  S <- S + k (x) d;  o = q S
// A sequence begins with its slot's state (zeros where it has none) and leaves its
// last one there.
#include "ragged.h"

namespace q36 {
namespace {

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

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT size_t qwen36_gdn_ragged_delta_workspace_bytes(const qwen36_state_batch* batch, unsigned longest) {
  (void)batch;
  (void)longest;
  return 0;
}

Q36_EXPORT int qwen36_gdn_ragged_delta(const void* q, const void* k, const void* v, unsigned qk_heads,
                                       unsigned qk_token_stride, unsigned v_token_stride, const void* g,
                                       const void* beta, void* states, size_t slot_stride,
                                       const qwen36_state_batch* batch, unsigned longest, void* out,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  RaggedBatch b;
  if (q == nullptr || k == nullptr || v == nullptr || g == nullptr || beta == nullptr || states == nullptr ||
      out == nullptr || !ragged_batch_of(batch, b) || (qk_heads != 16u && qk_heads != 32u) ||
      qk_token_stride < qk_heads * kGdnDk || qk_token_stride % 8 != 0 ||
      v_token_stride < (unsigned)(kGdnHv * kGdnDv) || v_token_stride % 8 != 0 ||
      slot_stride < (size_t)kGdnHv * kGdnDk * kGdnDv || slot_stride % 4 != 0 || !aligned16(q) ||
      !aligned16(k) || !aligned16(v) || !aligned16(states) || !aligned16(out))
    return Q36_EINVAL;
  const size_t need = qwen36_gdn_ragged_delta_workspace_bytes(batch, longest);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) return Q36_EINVAL;
  const DeltaArgs p = {static_cast<const bf16*>(q),  static_cast<const bf16*>(k),
                       static_cast<const bf16*>(v),  static_cast<const float*>(g),
                       static_cast<const float*>(beta), static_cast<float*>(states),
                       static_cast<bf16*>(out), slot_stride, qk_heads, qk_token_stride, v_token_stride};
  hipLaunchKernelGGL(gdn_ragged_step_kernel, dim3(b.seqs * 128), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p, b, ~0u);
  return static_cast<int>(hipGetLastError());
}
