// Appending to the paged KV cache: head norm and rotation of the queries and
// keys of a ragged batch's new tokens, the keys and raw values written to their
// pages in the page's type.
//
//   y = bf16(x / sqrt(mean(x^2) + 1e-6) * (w + 1)), dims [0, 64) rotated by the
//   tables' cos/sin at the token's position, rounded to bf16: the arithmetic of
//   the dense path's head norm, value for value.
//
// Work: an item per (page that gets rows, KV head) and a wave per (row, 4 query
// heads), in one launch.  A page's scale is one number for all its tokens, so
// the workgroup of a page holds its new rows in registers (packed bf16, at most
// 16 rows a wave, 4 registers each), takes their largest magnitude, settles the
// scale and writes.  Rows that were in the page are rescaled only where the
// scale grew: a shift by a power of two, exact but for subnormals.
// The keys' bounds (int8, in steps of four scales) are rounded outwards: the
// ceiling of a ceiling over powers of two is the ceiling, so they do not depend
// on the steps in which a page was filled.
#include "paged_common.h"

namespace q36 {
namespace {

struct AppendArgs {
  const bf16* q_gate;
  const bf16* k;
  const bf16* v;
  const bf16* q_weight;
  const bf16* k_weight;
  const float* cosv;
  const float* sinv;
  bf16* q_out;
  size_t q_stride, k_stride, v_stride;
  unsigned items;       // page items of one KV head, at most
};

constexpr int kRowsPerWave = 16;

// cos/sin of this lane's four dims (lanes 0-15), as rope_cos_sin_wave deals
// them, from the tables' row.
__device__ __forceinline__ void rope_from_tables(const float* cosv, const float* sinv, size_t pos,
                                                 float (&c)[4], float (&s)[4]) {
  const int p = (4 * (threadIdx.x & 63)) & (kRotaryPairs - 1);
  const f32x4 cv = *reinterpret_cast<const f32x4*>(cosv + pos * kRotaryPairs + p);
  const f32x4 sv = *reinterpret_cast<const f32x4*>(sinv + pos * kRotaryPairs + p);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    c[e] = cv[e];
    s[e] = sv[e];
  }
}

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// Four values to e4m3, rounded to nearest even; what is not finite is a NaN.
__device__ __forceinline__ unsigned pack_e4m3(const float (&x)[4], float inv) {
  int r = 0;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = finite(x[e]) ? x[e] * inv : 0.f;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (!finite(x[e])) r |= 0x7f << (8 * e);
  return (unsigned)r;
}

// Four e4m3 values times 2^-down.
__device__ __forceinline__ unsigned rescale_e4m3(unsigned w, float factor) {
  float x[4];
  x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
  x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
  x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
  x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
  return pack_e4m3(x, factor);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

template <bool kFp8>
__global__ __launch_bounds__(512) void paged_append_kernel(AppendArgs g, PagedCache c, PagedBatch b) {
  __shared__ unsigned find[20];
  __shared__ float amax[2][8];
  __shared__ float edge[2][8][kD];
  const unsigned waves = blockDim.x >> 6;
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const unsigned hq = c.heads * kGroup;
  const unsigned kv_blocks = g.items * c.heads;

  if (blockIdx.x >= kv_blocks) {   // queries: a wave takes 4 heads of a row
    const unsigned w = (blockIdx.x - kv_blocks) * waves + wave;
    const unsigned quads = hq / 4, t = w / quads, h0 = w % quads * 4;
    if (t >= b.tokens) return;
    bf16x4 xin[4];
#pragma unroll
    for (int h = 0; h < 4; ++h)
      xin[h] = *reinterpret_cast<const bf16x4*>(g.q_gate + t * g.q_stride + (h0 + h) * 2 * kD + 4 * lane);
    float wp1[4], cs[4], sn[4];
    head_norm_wp1(g.q_weight, wp1);
    const unsigned i = paged_find_row(b, (int)t);
    if (i >= b.seqs) return;
    const PagedSeq s = paged_seq(b, i);
    const int pos = s.pos((int)t);
    if ((int)t < s.a || (int)t >= s.z || pos < 0) return;
    rope_from_tables(g.cosv, g.sinv, (size_t)pos, cs, sn);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = bf2f(xin[h][e]);
      head_norm_rope_wave_wp1(x, wp1, cs, sn, y);
      bf16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = f2bf(y[e]);
      *reinterpret_cast<bf16x4*>(g.q_out + ((size_t)t * hq + h0 + h) * kD + 4 * lane) = o;
    }
    return;
  }

  const unsigned head = blockIdx.x % c.heads, item = blockIdx.x / c.heads;
  const int page = 1 << c.shift;
  unsigned i, local;
  const bool some = paged_find_item(b, item, find, [&](unsigned j) {
    const PagedSeq s = paged_seq(b, j);
    const int p0 = max(s.pos(s.a), 0);   // the first new position
    return s.z > s.a && s.len > p0 ? (unsigned)(((s.len - 1) >> c.shift) - (p0 >> c.shift) + 1) : 0u;
  }, i, local);
  if (!some) return;
  const PagedSeq s = paged_seq(b, i);
  const int p0 = max(s.pos(s.a), 0);
  const unsigned logical = (unsigned)(p0 >> c.shift) + local;
  const unsigned pid = (unsigned)b.table[i * b.table_stride + logical];
  if (pid >= c.pages) return;
  const int first = (int)(logical << c.shift);
  const int lo = max(p0, first), hi = min(s.len, first + page);
  const int kept = lo - first, rows = hi - lo;
  const int t0 = s.z - (s.len - lo);   // the row of position lo

  float wp1[4];
  head_norm_wp1(g.k_weight, wp1);
  bf16x4 kr[kRowsPerWave], vr[kRowsPerWave];
#pragma unroll
  for (int j = 0; j < kRowsPerWave; ++j) {
    const int r = (int)wave + j * (int)waves;
    if (r < rows) {
      const size_t t = (size_t)(t0 + r);
      kr[j] = *reinterpret_cast<const bf16x4*>(g.k + t * g.k_stride + head * kD + 4 * lane);
      vr[j] = *reinterpret_cast<const bf16x4*>(g.v + t * g.v_stride + head * kD + 4 * lane);
    }
  }
  float ka = 0.f, va = 0.f, top[4], low[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    top[e] = -INFINITY;
    low[e] = INFINITY;
  }
#pragma unroll
  for (int j = 0; j < kRowsPerWave; ++j) {
    const int r = (int)wave + j * (int)waves;
    if (r >= rows) break;
    float x[4], y[4], cs[4], sn[4];
    rope_from_tables(g.cosv, g.sinv, (size_t)(lo + r), cs, sn);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = bf2f(kr[j][e]);
    head_norm_rope_wave_wp1(x, wp1, cs, sn, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      kr[j][e] = f2bf(y[e]);
      const float k = bf2f(kr[j][e]), v = bf2f(vr[j][e]);
      if (finite(k)) ka = fmaxf(ka, fabsf(k));
      if (finite(v)) va = fmaxf(va, fabsf(v));
      const float z = k == k ? k : 0.f;
      top[e] = fmaxf(top[e], z);
      low[e] = fminf(low[e], z);
    }
  }
  const bool scaled = kFp8 || c.bounds != nullptr;
  unsigned ke = 0, ve = 0, ke_old = 0, ve_old = 0;
  const size_t es = (size_t)pid * c.heads + head;
  if (scaled) {
    ka = wave_max(ka);
    va = wave_max(va);
    if (lane == 0) {
      amax[0][wave] = ka;
      amax[1][wave] = va;
    }
    if (c.bounds != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        edge[0][wave][4 * lane + e] = top[e];
        edge[1][wave][4 * lane + e] = low[e];
      }
    }
    ke_old = c.k_exp[es];
    if (kFp8) ve_old = c.v_exp[es];
    __syncthreads();
    for (unsigned w = 0; w < waves; ++w) {
      ka = fmaxf(ka, amax[0][w]);
      va = fmaxf(va, amax[1][w]);
    }
    ke = paged_scale_byte(ka);
    ve = paged_scale_byte(va);
    if (kept > 0) {
      ke = max(ke, ke_old);
      ve = max(ve, ve_old);
    }
    // every thread holds the old bytes (read before the barrier)
    if (threadIdx.x == 0) {
      c.k_exp[es] = (uint8_t)ke;
      if (kFp8) c.v_exp[es] = (uint8_t)ve;
    }
  }
  if (c.bounds != nullptr) {
    int8_t* bp = c.bounds + es * 2 * kD;
    const float inv = paged_scale(252u - ke);   // 1 / (4 * 2^(ke - 127))
    const unsigned down = kept > 0 ? min(ke - ke_old, 31u) : 0u;
    for (unsigned d = threadIdx.x; d < kD; d += blockDim.x) {
      float t = -INFINITY, l = INFINITY;
      for (unsigned w = 0; w < waves; ++w) {
        t = fmaxf(t, edge[0][w][d]);
        l = fminf(l, edge[1][w][d]);
      }
      int ti = (int)fminf(fmaxf(ceilf(t * inv), -127.f), 127.f);
      int li = (int)fminf(fmaxf(floorf(l * inv), -127.f), 127.f);
      if (kept > 0) {
        ti = max(ti, -((-(int)bp[d]) >> down));
        li = min(li, (int)bp[kD + d] >> down);
      }
      bp[d] = (int8_t)ti;
      bp[kD + d] = (int8_t)li;
    }
  }
  constexpr size_t kElem = kFp8 ? 1 : 2;
  char* kp = c.k + (size_t)pid * c.k_stride + (size_t)head * page * kD * kElem;
  char* vp = c.v + (size_t)pid * c.v_stride + (size_t)head * page * kD * kElem;
  if (kFp8 && kept > 0) {
    const int n = kept * kD / 16;
    for (int p = 0; p < 2; ++p) {
      const unsigned up = p ? ve - ve_old : ke - ke_old;
      if (up == 0) continue;
      const float f = paged_scale(127u - min(up, 126u));
      u32x4* x = reinterpret_cast<u32x4*>(p ? vp : kp);
      for (int j = threadIdx.x; j < n; j += blockDim.x) {
        u32x4 w = x[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = rescale_e4m3(w[e], f);
        x[j] = w;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kRowsPerWave; ++j) {
    const int r = (int)wave + j * (int)waves;
    if (r >= rows) break;
    const size_t at = (size_t)(kept + r) * kD + 4 * lane;
    if constexpr (kFp8) {
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = bf2f(kr[j][e]);
        y[e] = bf2f(vr[j][e]);
      }
      *reinterpret_cast<unsigned*>(kp + at) = pack_e4m3(x, paged_scale(254u - ke));
      *reinterpret_cast<unsigned*>(vp + at) = pack_e4m3(y, paged_scale(254u - ve));
    } else {
      *reinterpret_cast<bf16x4*>(kp + 2 * at) = kr[j];
      *reinterpret_cast<bf16x4*>(vp + 2 * at) = vr[j];
    }
  }
}

}  // namespace
}  // namespace q36

using namespace q36;

Q36_EXPORT int qwen36_paged_append(const void* q_gate, unsigned q_row_stride, const void* k_raw,
                                   unsigned k_row_stride, const void* v_raw, unsigned v_row_stride,
                                   const void* q_weight, const void* k_weight, const float* cosv,
                                   const float* sinv, unsigned positions,
                                   const qwen36_paged_cache* cache, const qwen36_paged_batch* batch,
                                   void* q_out, void* stream) {
  PagedCache c;
  PagedBatch b;
  if (!paged_cache_of(cache, c) || !paged_batch_of(batch, cache->page_tokens, b)) return Q36_EINVAL;
  const unsigned hq = c.heads * kGroup;
  const auto a8 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; };
  if (q_gate == nullptr || k_raw == nullptr || v_raw == nullptr || q_weight == nullptr ||
      k_weight == nullptr || cosv == nullptr || sinv == nullptr || q_out == nullptr ||
      q_row_stride < hq * 2 * kD || k_row_stride < c.heads * kD || v_row_stride < c.heads * kD ||
      q_row_stride % 4 || k_row_stride % 4 || v_row_stride % 4 || !a8(q_gate) || !a8(k_raw) ||
      !a8(v_raw) || !a8(q_out) || !aligned16(cosv) || !aligned16(sinv) || positions == 0)
    return Q36_EINVAL;
  if (b.max_len > positions) b.max_len = positions;
  AppendArgs g;
  g.q_gate = static_cast<const bf16*>(q_gate);
  g.k = static_cast<const bf16*>(k_raw);
  g.v = static_cast<const bf16*>(v_raw);
  g.q_weight = static_cast<const bf16*>(q_weight);
  g.k_weight = static_cast<const bf16*>(k_weight);
  g.cosv = cosv;
  g.sinv = sinv;
  g.q_out = static_cast<bf16*>(q_out);
  g.q_stride = q_row_stride;
  g.k_stride = k_row_stride;
  g.v_stride = v_row_stride;
  // n new tokens touch at most n pages and (n - 1) / page + 2
  const unsigned page = cache->page_tokens;
  const unsigned most = b.tokens / page + 2 * b.seqs;
  g.items = b.tokens < most ? b.tokens : most;
  // 16 rows a wave: a wave for each 16 tokens of a page
  const unsigned waves = page / kRowsPerWave;
  const unsigned blocks = g.items * c.heads + (b.tokens * (hq / 4) + waves - 1) / waves;
  if (cache->cache_type == QWEN36_PAGED_E4M3)
    hipLaunchKernelGGL(paged_append_kernel<true>, dim3(blocks), dim3(64 * waves), 0,
                       static_cast<hipStream_t>(stream), g, c, b);
  else
    hipLaunchKernelGGL(paged_append_kernel<false>, dim3(blocks), dim3(64 * waves), 0,
                       static_cast<hipStream_t>(stream), g, c, b);
  return static_cast<int>(hipGetLastError());
}
