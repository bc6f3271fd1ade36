// The Gated-DeltaNet convolution over a ragged batch with its states in slots.
//
// Per channel: y_t = SiLU(bf16(sum_j w_j x_{t-3+j})), j = 0..3, where the three
// inputs before a sequence's first row come from its slot (zeros where it has no
// state); the slot then holds the sequence's last three inputs.  The arithmetic
// is that of qwen36_gdn_conv1d: products and sums rounded one by one, the sum
// rounded to bf16 before SiLU (four_layer_mini_engine.py:5368-5386), the result
// to bf16.
//
// Bound by its bytes (32 KB a row) for prompts (9,903 rows 73 us, 4.4 TB/s) and by the
// chain offsets -> slot -> state -> store for single tokens (64 sequences 7 us).  A thread
// takes 8 channels (16-byte loads) of a tile of 4 rows counted from the sequence's first
// row, so that only a sequence's first tile reads its slot, and that tile alone writes it:
// the state is read before it is written by the same thread, whatever the order of tiles.
#include "ragged.h"

namespace q36 {
namespace {

constexpr unsigned kRows = 4;

__device__ __forceinline__ float silu_exact(float x) { return x / (1.0f + expf(-x)); }

// bf16(SiLU(x)) for a bf16 x: silu_fast unless it could round to another value.
__device__ __forceinline__ bf16 silu_bf16(float x) {
  const float f = silu_fast(x);
  const int mid = (int)(__float_as_uint(f) & 0xffffu) - 0x8000;
  const bool slow = (mid >= -kSiluMid && mid <= kSiluMid) || !(fabsf(x) <= 60.0f);
  return f2bf(slow ? silu_exact(x) : f);
}

__global__ __launch_bounds__(256) void gdn_ragged_conv_kernel(
    const bf16* __restrict__ x, unsigned x_row_stride, const bf16* __restrict__ weight, bf16* states,
    size_t slot_stride, RaggedBatch b, bf16* __restrict__ out) {
  const int c0 = ((blockIdx.x & 3) * 256 + threadIdx.x) * 8;
  unsigned i, local;
  if (!ragged_find_tile<kRows>(b, blockIdx.x >> 2, i, local)) return;
  const RaggedSeq s = ragged_seq(b, i);
  if (s.slot < 0) return;
  const int t0 = s.a + (int)(local * kRows), n = min((int)kRows, s.z - t0);
  bf16* st = states + (size_t)s.slot * slot_stride + c0 * 3;
  bf16x8 rows[3 + kRows];       // window rows t0 - 3 .. t0 + 3 (behind the end: the last again)
#pragma unroll
  for (int j = 0; j < (int)kRows; ++j)
    rows[3 + j] = *reinterpret_cast<const bf16x8*>(x + (size_t)min(t0 + j, s.z - 1) * x_row_stride + c0);
  if (local > 0) {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      rows[j] = *reinterpret_cast<const bf16x8*>(x + (size_t)(t0 - 3 + j) * x_row_stride + c0);
  } else {
    bf16 h[24] = {};
    if (s.has) {
#pragma unroll
      for (int u = 0; u < 3; ++u) {
        const bf16x8 v = reinterpret_cast<const bf16x8*>(st)[u];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[8 * u + e] = v[e];
      }
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) rows[j][e] = h[3 * e + j];
  }
  float w[8][kGdnConvK];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const bf16x8 wv = *reinterpret_cast<const bf16x8*>(weight + c0 * kGdnConvK + 8 * u);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[2 * u + e / 4][e % 4] = bf2f(wv[e]);
  }
#pragma unroll
  for (int j = 0; j < (int)kRows; ++j) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float acc = __fmul_rn(bf2f(rows[j][e]), w[e][0]);
      acc = __fadd_rn(acc, __fmul_rn(bf2f(rows[j + 1][e]), w[e][1]));
      acc = __fadd_rn(acc, __fmul_rn(bf2f(rows[j + 2][e]), w[e][2]));
      acc = __fadd_rn(acc, __fmul_rn(bf2f(rows[j + 3][e]), w[e][3]));
      o[e] = silu_bf16(bf2f(f2bf(acc)));
    }
    if (j < n) *reinterpret_cast<bf16x8*>(out + (size_t)(t0 + j) * kGdnConvDim + c0) = o;
  }
  if (local == 0) {
    // the last three of [state | rows]
    const int len = s.z - s.a;
    bf16x8 last[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      if (len >= 3) {
        last[j] = *reinterpret_cast<const bf16x8*>(x + (size_t)(s.z - 3 + j) * x_row_stride + c0);
      } else {
        last[j] = len == 1 ? rows[1 + j] : rows[2 + j];
      }
    }
    bf16 h[24];
#pragma unroll
    for (int j = 0; j < 3; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[3 * e + j] = last[j][e];
#pragma unroll
    for (int u = 0; u < 3; ++u) {
      bf16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = h[8 * u + e];
      reinterpret_cast<bf16x8*>(st)[u] = v;
    }
  }
}

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT int qwen36_gdn_ragged_conv1d(const void* x, unsigned x_row_stride, const void* weight,
                                        void* states, size_t slot_stride,
                                        const qwen36_state_batch* batch, void* out, void* stream) {
  RaggedBatch b;
  if (x == nullptr || weight == nullptr || states == nullptr || out == nullptr ||
      !ragged_batch_of(batch, b) || x_row_stride < (unsigned)kGdnConvDim || x_row_stride % 8 != 0 ||
      slot_stride < (size_t)kGdnConvDim * 3 || slot_stride % 8 != 0 || !aligned16(x) ||
      !aligned16(weight) || !aligned16(states) || !aligned16(out))
    return Q36_EINVAL;
  hipLaunchKernelGGL(gdn_ragged_conv_kernel, dim3(kGdnConvDim / 2048 * (b.tokens / kRows + b.seqs)),
                     dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const bf16*>(x), x_row_stride,
                     static_cast<const bf16*>(weight), static_cast<bf16*>(states), slot_stride, b,
                     static_cast<bf16*>(out));
  return static_cast<int>(hipGetLastError());
}
