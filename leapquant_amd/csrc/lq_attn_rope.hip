// Norms of each head's queries and keys, rotation by the token's position, keys and values into their pages (lq_rope_norm).
//
// y = x rsqrt(mean x^2 + eps) (offset + w); the pair (a, b) of rotation i turns by phi = t f_i: (a cos - b sin, b cos + a sin).
// One pass: an element is read once, stays in fp32 registers through norm and rotation and is rounded once.  Bound by memory:
// 4 bytes an element.
//
// A head's D elements lie in D / 8 lanes of 8 neighbours (16-byte loads).  The other half of a pair (i, i + rot / 2) is in
// another lane of the head: four lane exchanges bring its raw elements, which this lane scales by their own weights.  An angle
// is formed in turns, t (f / 2 pi) in fp64 less its whole part, so that a far position keeps its fraction of a turn (2^-21
// of one at t = 2^31); the hardware's sine and cosine take turns.  Without a table of them a token's chain is one load shorter.
//
// A workgroup takes U times its vectors (heads of q, k and v) of one token.
#include "lq_attn.h"

namespace {

constexpr int TH = 256;

__device__ __forceinline__ void unpack8(const u32x4& w, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = bf_lo(w[i]); f[2 * i + 1] = bf_hi(w[i]); }
}
__device__ __forceinline__ u32x4 pack8(const float* f) {
  return u32x4{pk_bf16(f[0], f[1]), pk_bf16(f[2], f[3]), pk_bf16(f[4], f[5]), pk_bf16(f[6], f[7])};
}
// offset + weight of 8 neighbours
__device__ __forceinline__ void weight8(const void* w, bool bf16, int d, float offset, float* f) {
  if (bf16) {
    unpack8(*(const u32x4*)((const bf16_t*)w + d), f);
  } else {
    const f32x4 a = *(const f32x4*)((const float*)w + d), b = *(const f32x4*)((const float*)w + d + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] += offset;
}
template <int LANES> __device__ __forceinline__ float lanes_sum(float x) {
  x = sum8(x);
  if (LANES >= 16) x += dpp<DPP_MIRROR>(x);
  if (LANES >= 32) x = xor16_sum(x);
  return x;
}
template <int LANES> __device__ __forceinline__ float lanes_max(float x) {
  x = max8(x);
  if (LANES >= 16) x = fmaxf(x, dpp<DPP_MIRROR>(x));
  if (LANES >= 32) x = xor16_max(x);
  return x;
}

// the sequence that holds the packed token t: the last n with loc[n] <= t, looked for by a whole wave, 64 a step; -1: none
__device__ __forceinline__ int token_seq(const lq_batch& b, int t) {
  const int lane = threadIdx.x & 63;
  int a = 0, len = b.N;
  while (len > 1) {
    const int step = (len + 63) >> 6;
    const bool below = lane * step < len && batch_at(b, a + lane * step) <= t;
    const int at = max((int)__popcll(__ballot(below)) - 1, 0) * step;
    a += at;
    len = min(step, len - at);
  }
  return batch_at(b, a) <= t && t < batch_at(b, a + 1) ? a : -1;
}

template <int D, int U>
__global__ __launch_bounds__(TH) void rope_norm_kernel(lq_rope r, lq_pages p, lq_batch b, PageDiv div) {
  constexpr int LANES = D / 8, SLOTS = TH / LANES;
  const int t = blockIdx.x, lane = threadIdx.x & (LANES - 1), d0 = 8 * lane;
  const int n = __builtin_amdgcn_readfirstlane(token_seq(b, t));
  if (n < 0) return;
  const int pos = batch_len(b, p, n) - (batch_at(b, n + 1) - t);
  const int heads = r.HQ + 2 * p.HK, first = blockIdx.y * U * SLOTS + threadIdx.x / LANES;
  u32x4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = first + u * SLOTS;
    const bool isq = h < r.HQ, isk = h < r.HQ + p.HK;
    const lq_rows& from = isq ? r.q : isk ? r.k : r.v;
    const int hh = isq ? h : isk ? h - r.HQ : h - r.HQ - p.HK;
    raw[u] = u32x4(0u);
    if (h < heads) raw[u] = *(const u32x4*)((const bf16_t*)from.p + (long long)t * from.ld + (long long)hh * from.hd + d0);
  }
  if (pos < 0) {                                   // before the sequence's first token: no place, a zero output
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = first + u * SLOTS;
      if (h < r.HQ) *(u32x4*)((bf16_t*)r.out.p + (long long)t * r.out.ld + (long long)h * r.out.hd + d0) = u32x4(0u);
    }
    return;
  }
  const int pg = page_of(div, pos), in = pos - pg * p.page;
  const int page = b.table[(long long)n * b.table_ld + pg];
  const bool held = page >= 0 && page < p.NP;
  const int half = r.rot >> 1;
  const bool turns = d0 < r.rot;
  const int other = r.interleaved || !turns ? d0 : d0 < half ? d0 + half : d0 - half;      // elements of the pairs' other halves
  const float sign = d0 < half ? -1.f : 1.f;
  float cs[8], sn[8];                              // interleaved: 4 of each
  const int i0 = r.interleaved ? d0 >> 1 : min(d0, other), ni = r.interleaved ? 4 : 8;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
    if (turns && e < ni) {
      const double f = r.freq64 ? ((const double*)r.inv_freq)[i0 + e] : (double)((const float*)r.inv_freq)[i0 + e];
      const double x = (double)pos * (f * 0.15915494309189535);
      const float y = (float)(x - __builtin_rint(x));
      cs[e] = __builtin_amdgcn_cosf(y);
      sn[e] = __builtin_amdgcn_sinf(y);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = first + u * SLOTS;
    const bool isq = h < r.HQ, isk = !isq && h < r.HQ + p.HK;
    float f[8], y[8];
    unpack8(raw[u], f);
    if (__any(isq || isk)) {
      const void* weight = isq ? r.q_weight : r.k_weight;
      const bool wide = !(r.weight_bf16 & (isq ? 1 : 2));
      float w[8], wo[8], g[8], sum = 0.f;
      weight8(weight, !wide, d0, r.offset, w);
      weight8(weight, !wide, other, r.offset, wo);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(f[e], f[e], sum);
      const float inv = rsqrtf_rn(lanes_sum<LANES>(sum) * (1.f / D) + r.eps);
      if (r.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = f[e] * inv * w[e];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = y[2 * e], c = y[2 * e + 1];
          y[2 * e] = fmaf(a, cs[e], -c * sn[e]);
          y[2 * e + 1] = fmaf(c, cs[e], a * sn[e]);
        }
      } else {
        u32x4 away;
        const int from = ((threadIdx.x & 63) - lane + other / 8) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) away[i] = __builtin_amdgcn_ds_bpermute(from, raw[u][i]);
        unpack8(away, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = f[e] * inv * w[e], c = g[e] * inv * wo[e] * sign;
          y[e] = turns ? fmaf(a, cs[e], c * sn[e]) : a;
        }
      }
      if (!isq && !isk) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = f[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = f[e];
    }
    if (isq) *(u32x4*)((bf16_t*)r.out.p + (long long)t * r.out.ld + (long long)h * r.out.hd + d0) = pack8(y);
    const int hk = isk ? h - r.HQ : h - r.HQ - p.HK;
    void* to = isk ? p.k : p.v;
    if (!p.int8) {
      if (!isq && h < heads && held)
        *(u32x4*)((bf16_t*)to + (long long)page * p.page_ld + in * p.row_ld + hk * p.head_ld + d0) = pack8(y);
    } else if (__any(!isq && h < heads)) {
      float big = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(y[e]));
      big = lanes_max<LANES>(big);
      const float scale = big > 1e-30f ? big * (1.f / 127.f) : 0.f;
      const float inv = big > 1e-30f && big < INFINITY ? 127.f / big : 0.f;
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float c = __builtin_rintf(y[e] * inv);
        const int code = c == c ? (int)fminf(fmaxf(c, -127.f), 127.f) : 0;
        w[e >> 2] |= (uint32_t)(code & 255) << (8 * (e & 3));
      }
      if (!isq && h < heads && held) {
        *(u32x2*)((int8_t*)to + (long long)page * p.page_ld + in * p.row_ld + hk * p.head_ld + d0) = u32x2{w[0], w[1]};
        if (lane == 0)
          (isk ? p.k_scale : p.v_scale)[(long long)page * p.s_page_ld + in * p.s_row_ld + hk * p.s_head_ld] = scale;
      }
    }
  }
}

template <int D> int launch(const lq_rope* r, const lq_pages* p, const lq_batch* b, hipStream_t s) {
  const int heads = r->HQ + 2 * p->HK, slots = TH / (D / 8), per = (heads + slots - 1) / slots;
  const PageDiv div = page_div(p->page);
  auto go = [&](auto kernel, int u) {
    const dim3 grid((unsigned)b->T, (unsigned)((per + u - 1) / u));
    if (grid.y > 65535u) return LQ_ERR_ARG;
    kernel<<<grid, TH, 0, s>>>(*r, *p, *b, div);
    return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
  };
  if ((long long)b->T * per <= 8ll * lq_attn_cus() || per == 1) return go(rope_norm_kernel<D, 1>, 1);
  if (per == 2) return go(rope_norm_kernel<D, 2>, 2);
  return go(rope_norm_kernel<D, 3>, 3);
}

}  // namespace

extern "C" int lq_rope_norm(const lq_rope* r, const lq_pages* p, const lq_batch* b, void* stream) {
  if (!r || !pages_ok(p) || !batch_ok(b, p)) return LQ_ERR_ARG;
  if (r->HQ <= 0 || r->HQ > 1 << 20 || p->HK > 1 << 20 || r->rot < 0 || r->rot > p->D || r->rot % 16) return LQ_ERR_ARG;
  if ((r->weight_bf16 & ~3) || (r->freq64 & ~1) || (r->interleaved & ~1) || !(r->eps >= 0.f)) return LQ_ERR_ARG;
  if (b->N == 0 || b->T == 0) return LQ_OK;
  if (!rows_ok(r->q) || !rows_ok(r->k) || !rows_ok(r->v) || !rows_ok(r->out)) return LQ_ERR_ARG;
  if (!r->q.p || !r->k.p || !r->v.p || !r->out.p || !r->q_weight || !r->k_weight || (r->rot && !r->inv_freq)) return LQ_ERR_ARG;
  if (((uintptr_t)r->q_weight | (uintptr_t)r->k_weight) & 15 || (uintptr_t)r->inv_freq & (r->freq64 ? 7 : 3)) return LQ_ERR_ARG;
  if (!rows_apart(r->out, b->T, r->HQ, p->D)) return LQ_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (p->D == 64) return launch<64>(r, p, b, s);
  if (p->D == 128) return launch<128>(r, p, b, s);
  return launch<256>(r, p, b, s);
}
