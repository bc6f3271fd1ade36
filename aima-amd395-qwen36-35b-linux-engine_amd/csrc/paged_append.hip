// Appending to the paged KV cache: head norm and rotation of the queries and
// keys of a ragged batch's new tokens, the keys and raw values written to their
// pages in the page's type.
//
//   y = bf16(x / sqrt(mean(x^2) + 1e-6) * (w + 1)), dims [0, 64) rotated by the
//   tables' cos/sin at the token's position, rounded to bf16: the arithmetic of
//   the dense path's head norm, value for value.
//
// Work: a workgroup of 4 waves per (page that gets rows, KV head), and a wave per
// (row, 8 query heads), in one launch.  A page's scale is one number for all its
// tokens, so its workgroup holds the new rows in registers (packed bf16, a
// quarter of the page a wave), takes their largest magnitude, settles the scale
// and writes.  Rows that were in the page are rescaled only where the scale grew:
// a shift by a power of two, exact but for subnormals.
// The keys' bounds (int8, in steps of four scales) are rounded outwards: the
// ceiling of a ceiling over powers of two is the ceiling, so they do not depend
// on the steps in which a page was filled.
// Norms are taken four heads (or rows) at once: each level of the sum's tree
// halves the values a lane carries, and the square root and division in 64 bits
// run once for four heads instead of once each, which bounded the first form
// (8,192 tokens: 41 us; bytes alone 34).
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

constexpr int kWaves = 4;

// The factors 1 / sqrt(mean(x^2) + 1e-6) of four 256-wide heads, lane l holding
// dims 4l .. 4l + 3 of each: head_norm_rope_wave_wp1's sums (four neighbours, then
// lanes 32, 16, 8, 4, 2, 1 apart; an exchanged addition is the same), with the
// heads dealt to quarters of the wave at the first two levels.
__device__ __forceinline__ void head_inv4(const float (&x)[4][4], float (&inv)[4]) {
  const int lane = threadIdx.x & 63;
  float s[4];
#pragma unroll
  for (int h = 0; h < 4; ++h)
    s[h] = __fadd_rn(__fadd_rn(__fmul_rn(x[h][0], x[h][0]), __fmul_rn(x[h][1], x[h][1])),
                     __fadd_rn(__fmul_rn(x[h][2], x[h][2]), __fmul_rn(x[h][3], x[h][3])));
  const bool up = lane & 32, odd = lane & 16;
  const float a = __fadd_rn(up ? s[2] : s[0], __shfl_xor(up ? s[0] : s[2], 32, 64));
  const float b = __fadd_rn(up ? s[3] : s[1], __shfl_xor(up ? s[1] : s[3], 32, 64));
  float c = __fadd_rn(odd ? b : a, __shfl_xor(odd ? a : b, 16, 64));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) c = __fadd_rn(c, __shfl_xor(c, o, 64));
  const float var = __fmul_rn(c, 1.0f / 256.0f);
  const float r = (float)(1.0 / sqrt((double)__fadd_rn(var, 1e-6f)));
#pragma unroll
  for (int h = 0; h < 4; ++h)
    inv[h] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(r), 16 * h));
}

// The rest of head_norm_rope_wave_wp1: scaled, rounded, rotated, rounded.
__device__ __forceinline__ bf16x4 head_rope(const float (&x)[4], float inv, const float (&wp1)[4],
                                            const float (&cs)[4], const float (&sn)[4]) {
  const int lane = threadIdx.x & 63;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = bf2f(f2bf(__fmul_rn(__fmul_rn(x[e], inv), wp1[e])));
  bf16x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // lane ^ 8: a rotation by 8 of 16 lanes
    const float mate = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(y[e]), 0x128, 0xf, 0xf, false));
    const float a = __fmul_rn(y[e], cs[e]), b = __fmul_rn(mate, sn[e]);
    const float r = lane < 8 ? __fsub_rn(a, b) : __fadd_rn(a, b);
    o[e] = f2bf(lane < 16 ? r : y[e]);
  }
  return o;
}

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

template <bool kFp8, int kRows>   // kRows: rows of a page that a wave takes
__global__ __launch_bounds__(64 * kWaves) void paged_append_kernel(AppendArgs g, PagedCache c, PagedBatch b) {
  __shared__ unsigned find[20];
  __shared__ float amax[2][kWaves];
  __shared__ float edge[2][kWaves][kD];
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const unsigned kv_blocks = g.items * c.heads;

  if (blockIdx.x >= kv_blocks) {   // queries: a wave takes the 8 heads of a KV head in a row
    const unsigned w = (blockIdx.x - kv_blocks) * kWaves + wave;
    const unsigned t = w / c.heads, h0 = w % c.heads * kGroup;
    if (t >= b.tokens) return;
    bf16x4 xin[kGroup];
#pragma unroll
    for (int h = 0; h < kGroup; ++h)
      xin[h] = *reinterpret_cast<const bf16x4*>(g.q_gate + t * g.q_stride + (h0 + h) * 2 * kD + 4 * lane);
    float wp1[4], cs[4], sn[4];
    head_norm_wp1(g.q_weight, wp1);
    unsigned i;
    PagedSeq s;
    if (!paged_find_row(b, (int)t, i, s)) return;
    const int pos = s.pos((int)t);
    if (pos < 0) return;
    rope_from_tables(g.cosv, g.sinv, (size_t)pos, cs, sn);
    bf16* out = g.q_out + ((size_t)t * c.heads * kGroup + h0) * kD + 4 * lane;
#pragma unroll
    for (int h = 0; h < kGroup; h += 4) {
      float x[4][4], inv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = bf2f(xin[h + j][e]);
      head_inv4(x, inv);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<bf16x4*>(out + (h + j) * kD) = head_rope(x[j], inv[j], wp1, cs, sn);
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
  // row j of this wave is wave + 4 j of the new ones
  bf16x4 kr[kRows], vr[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int r = (int)wave + j * kWaves;
    if (r < rows) {
      const size_t t = (size_t)(t0 + r);
      kr[j] = *reinterpret_cast<const bf16x4*>(g.k + t * g.k_stride + head * kD + 4 * lane);
      vr[j] = *reinterpret_cast<const bf16x4*>(g.v + t * g.v_stride + head * kD + 4 * lane);
    } else {
      kr[j] = vr[j] = bf16x4{};
    }
  }
  float ka = 0.f, va = 0.f, top[4], low[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    top[e] = -INFINITY;
    low[e] = INFINITY;
  }
#pragma unroll
  for (int j0 = 0; j0 < kRows; j0 += 4) {
    if ((int)wave + j0 * kWaves >= rows) break;
    float x[4][4], inv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = bf2f(kr[j0 + j][e]);
    head_inv4(x, inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = (int)wave + (j0 + j) * kWaves;
      if (r >= rows) break;
      float cs[4], sn[4];
      rope_from_tables(g.cosv, g.sinv, (size_t)(lo + r), cs, sn);
      kr[j0 + j] = head_rope(x[j], inv[j], wp1, cs, sn);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float k = bf2f(kr[j0 + j][e]), v = bf2f(vr[j0 + j][e]);
        if (finite(k)) ka = fmaxf(ka, fabsf(k));
        if (finite(v)) va = fmaxf(va, fabsf(v));
        const float z = k == k ? k : 0.f;
        top[e] = fmaxf(top[e], z);
        low[e] = fminf(low[e], z);
      }
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
    for (int w = 0; w < kWaves; ++w) {
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
      for (int w = 0; w < kWaves; ++w) {
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
  for (int j = 0; j < kRows; ++j) {
    const int r = (int)wave + j * kWaves;
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
  const unsigned blocks = g.items * c.heads + (b.tokens * c.heads + kWaves - 1) / kWaves;
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), g, c, b);
  };
  const bool fp8 = cache->cache_type == QWEN36_PAGED_E4M3;
  switch (page) {
    case 16: fp8 ? launch(paged_append_kernel<true, 4>) : launch(paged_append_kernel<false, 4>); break;
    case 32: fp8 ? launch(paged_append_kernel<true, 8>) : launch(paged_append_kernel<false, 8>); break;
    case 64: fp8 ? launch(paged_append_kernel<true, 16>) : launch(paged_append_kernel<false, 16>); break;
    default: fp8 ? launch(paged_append_kernel<true, 32>) : launch(paged_append_kernel<false, 32>); break;
  }
  return static_cast<int>(hipGetLastError());
}
