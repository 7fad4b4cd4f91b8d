// Norms of each head's queries and keys, rotation by the token's position, keys and values into their pages (lq_rope_norm).
//
// y = x rsqrt(mean x^2 + eps) (offset + w); the pair (a, b) of rotation i turns by phi = t f_i: (a cos - b sin, b cos + a sin).
// One pass: an element is read once, stays in fp32 registers through norm and rotation and is rounded once.  Bound by memory:
// 4 bytes an element.
//
// A head's D elements lie in D / 8 lanes of 8 neighbours (16-byte loads), a wave's GROUP heads beside each other.  The other half of
// a pair (i, i + rot / 2) is in another lane of the head: four lane exchanges bring its raw elements, which this lane scales by their
// own weights.  An angle is formed in turns, t (f / 2 pi) in fp64 less its whole part, so that a far position keeps its fraction of
// a turn (2^-21 of one at t = 2^31); the hardware's sine and cosine take turns.
//
// Many tokens: a workgroup takes TOK of them.  Its threads share out their angles, whose cosines and sines lie in LDS for all heads;
// then a wave takes GROUP heads of all of them at a time, their loads on their way together, the weights loaded once.
// Few: a workgroup takes one token, a wave GROUP heads of it, and each lane forms its own angles: no barrier in the chain.
//
// Measured (MI355X): 41530 tokens of 16 + 2 + 2 heads of 256 175 us (4.9 TB/s; a large copy 5.2), into
// 8-bit pages 177, 8192 of 16 + 8 + 8 of 128 32 us
// (4.2 TB/s); a wave's 159 vector instructions for 64 x 8 elements are the next bound.  A decode batch of 64 tokens 5 us: its chain of
// three loads and the launch.  Per wave 4 tokens at a time 192 us, 16 at a time in two halves 191, 128 threads 196, 512 209.
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

// A token's place.  Its sequence is the last n with loc[n] <= t, looked for by a whole wave, 64 a step: one round of loads up to 64.
struct Place {
  int pos;                 // position; below 0: before the first, or of no sequence
  int page, in;            // page and place there; page < 0: not to be written
  int held;                // of a sequence
};
__device__ __forceinline__ Place place_of(const lq_batch& b, const lq_pages& p, const PageDiv& div, int t) {
  const int lane = threadIdx.x & 63;
  int a = 0, len = b.N, step = 1;
  int lo = 0, hi = 0, all = 0;
  do {
    step = (len + 63) >> 6;
    const int n = min(a + lane * step, b.N - 1);
    lo = batch_at(b, n);
    if (step == 1) { hi = batch_at(b, n + 1); all = batch_len(b, p, n); }
    const bool below = lane * step < len && lo <= t;
    const int at = max((int)__popcll(__ballot(below)) - 1, 0);
    if (step == 1) {
      a += at;
      lo = __shfl(lo, at);
      hi = __shfl(hi, at);
      all = __shfl(all, at);
    } else {
      a += at * step;
      len = min(step, len - at * step);
    }
  } while (step > 1);
  Place r;
  r.held = lo <= t && t < hi;
  r.pos = r.held ? all - (hi - t) : -1;
  r.page = -1;
  r.in = 0;
  if (r.pos >= 0) {
    const int pg = page_of(div, r.pos), page = b.table[(long long)a * b.table_ld + pg];
    r.in = r.pos - pg * p.page;
    r.page = page >= 0 && page < p.NP ? page : -1;
  }
  return r;
}

template <int D, int TOK>
__global__ __launch_bounds__(TH) void rope_norm_kernel(lq_rope r, lq_pages p, lq_batch b, PageDiv div) {
  constexpr int LANES = D / 8, GROUP = 64 / LANES, WAVES = TH / 64;
  constexpr bool FEW = TOK == 1;
  __shared__ Place places[TOK];
  __shared__ f32x4 cosine[FEW ? 1 : TOK][D / 8], sine[FEW ? 1 : TOK][D / 8];
  const int t0 = blockIdx.x * TOK, tokens = min(TOK, b.T - t0), lane = threadIdx.x & (LANES - 1), d0 = 8 * lane;
  const int wave = threadIdx.x >> 6, heads = r.HQ + 2 * p.HK, groups = (heads + GROUP - 1) / GROUP, half = r.rot >> 1;

  const bool turns = d0 < r.rot;
  const int other = r.interleaved || !turns ? d0 : d0 < half ? d0 + half : d0 - half;      // elements of the pairs' other halves
  const float sign = !r.interleaved && d0 < half ? -1.f : 1.f;
  const int i0 = !turns ? 0 : r.interleaved ? d0 >> 1 : min(d0, other);
  auto angle = [&](int i, int pos, float& c, float& s) {
    const double f = r.freq64 ? ((const double*)r.inv_freq)[i] : (double)((const float*)r.inv_freq)[i];
    const double phi = (double)pos * (f * 0.15915494309189535);
    const float turn = (float)(phi - __builtin_rint(phi));
    c = __builtin_amdgcn_cosf(turn);
    s = __builtin_amdgcn_sinf(turn);
  };

  int group = FEW ? blockIdx.y * WAVES + wave : wave;
  int h, kind;                                                 // kind 0: q, 1: k, 2: v, 3: none; h its head
  u32x4 raw[TOK];
  auto load = [&]() {
    h = group * GROUP + ((threadIdx.x & 63) / LANES);
    kind = h < r.HQ ? 0 : h < r.HQ + p.HK ? 1 : h < heads ? 2 : 3;
    h = kind == 3 ? p.HK - 1 : h - (kind == 0 ? 0 : kind == 1 ? r.HQ : r.HQ + p.HK);
    const lq_rows& from = kind == 0 ? r.q : kind == 1 ? r.k : r.v;
    const bf16_t* at = (const bf16_t*)from.p + (long long)h * from.hd + d0;
#pragma unroll
    for (int k = 0; k < TOK; ++k) raw[k] = *(const u32x4*)(at + (long long)min(t0 + k, b.T - 1) * from.ld);
  };
  if (group < groups) load();

  Place mine;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  if (FEW) {
    mine = place_of(b, p, div, t0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (turns && e < (r.interleaved ? 4 : 8)) angle(i0 + e, mine.pos, cs[e], sn[e]);
    }
  } else {
    for (int k = wave; k < tokens; k += WAVES) {
      const Place w = place_of(b, p, div, t0 + k);
      if ((threadIdx.x & 63) == 0) places[k] = w;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < tokens * half; x += TH) {
      const int k = x / half, i = x - k * half;
      angle(i, places[k].pos, ((float*)cosine[k])[i], ((float*)sine[k])[i]);
    }
    __syncthreads();
  }

  while (group < groups) {
    float w[8], wo[8];
    const bool norms = __any(kind < 2);
    if (norms) {
      const void* weight = kind == 0 ? r.q_weight : r.k_weight;
      const bool wide = !(r.weight_bf16 & (kind == 0 ? 1 : 2));
      weight8(weight, !wide, d0, r.offset, w);
      weight8(weight, !wide, other, r.offset, wo);
#pragma unroll
      for (int e = 0; e < 8; ++e) wo[e] = turns ? wo[e] * sign : 0.f;
    }
#pragma unroll
    for (int k = 0; k < TOK; ++k) {
      if (!FEW && k >= tokens) break;
      const Place at = FEW ? mine : places[k];
      float y[8];
      unpack8(raw[k], y);
      if (norms) {
        if (!FEW && turns) {
          const int x = i0 >> 2;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            cs[e] = cosine[k][x][e];
            sn[e] = sine[k][x][e];
            cs[4 + e] = cosine[k][(x + 1) & (D / 8 - 1)][e];
            sn[4 + e] = sine[k][(x + 1) & (D / 8 - 1)][e];
          }
        }
        float f[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[e] = y[e];
          sum = fmaf(f[e], f[e], sum);
        }
        const float inv = rsqrtf_rn(lanes_sum<LANES>(sum) * (1.f / D) + r.eps);
        if (r.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = f[e] * inv * w[e];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = f[2 * e], c = f[2 * e + 1];
            f[2 * e] = turns ? fmaf(a, cs[e], -c * sn[e]) : a;
            f[2 * e + 1] = turns ? fmaf(c, cs[e], a * sn[e]) : c;
          }
        } else {
          u32x4 away;
          float g[8];
          const int from = ((threadIdx.x & 63) - lane + other / 8) * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) away[i] = __builtin_amdgcn_ds_bpermute(from, raw[k][i]);
          unpack8(away, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = f[e] * inv * w[e], c = g[e] * inv * wo[e];
            f[e] = fmaf(a, cs[e], c * sn[e]);                  // lanes that do not turn: a 1 + 0
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = kind < 2 ? f[e] : y[e];
      }
      const long long t = t0 + k;
      if (kind == 0 && at.held) {
        u32x4 o = pack8(y);
        if (at.pos < 0) o = u32x4(0u);                         // before the sequence's first token: no place, a zero output
        *(u32x4*)((bf16_t*)r.out.p + t * r.out.ld + (long long)h * r.out.hd + d0) = o;
      }
      const bool write = (kind == 1 || kind == 2) && at.page >= 0;
      void* to = kind == 1 ? p.k : p.v;
      if (!p.int8) {
        if (write) *(u32x4*)((bf16_t*)to + (long long)at.page * p.page_ld + at.in * p.row_ld + h * p.head_ld + d0) = pack8(y);
      } else if (__any(write)) {
        float big = 0.f;
        bool nan = false;                                      // a maximum drops it
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          big = fmaxf(big, fabsf(y[e]));
          nan |= y[e] != y[e];
        }
        big = lanes_max<LANES>(big);
        nan = (__ballot(nan) >> ((threadIdx.x & 63) - lane)) & ((1ull << LANES) - 1);
        const float scale = nan ? NAN : big > 1e-30f ? big * (1.f / 127.f) : 0.f;
        const float inv = !nan && big > 1e-30f && big < INFINITY ? 127.f / big : 0.f;
        uint32_t o[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float c = __builtin_rintf(y[e] * inv);
          const int code = c == c ? (int)fminf(fmaxf(c, -127.f), 127.f) : 0;
          o[e >> 2] |= (uint32_t)(code & 255) << (8 * (e & 3));
        }
        if (write) {
          *(u32x2*)((int8_t*)to + (long long)at.page * p.page_ld + at.in * p.row_ld + h * p.head_ld + d0) = u32x2{o[0], o[1]};
          if (lane == 0) (kind == 1 ? p.k_scale : p.v_scale)[(long long)at.page * p.s_page_ld + at.in * p.s_row_ld + h * p.s_head_ld] = scale;
        }
      }
    }
    if (FEW) break;
    group += WAVES;
    if (group < groups) load();
  }
}

template <int D> int launch(const lq_rope* r, const lq_pages* p, const lq_batch* b, hipStream_t s) {
  const int heads = r->HQ + 2 * p->HK, group = 64 / (D / 8), groups = (heads + group - 1) / group, waves = TH / 64;
  const PageDiv div = page_div(p->page);
  auto go = [&](auto kernel, int tokens, int parts) {
    if (parts > 65535) return LQ_ERR_ARG;
    kernel<<<dim3((unsigned)((b->T + (long long)tokens - 1) / tokens), (unsigned)parts), TH, 0, s>>>(*r, *p, *b, div);
    return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
  };
  const int parts = (groups + waves - 1) / waves;
  // By tokens, whatever the heads (us, one token a workgroup / 8, 16 + 16 heads on 256 CUs): 1024 tokens of 64 6.4 / 9.4, of 256
  // 16 / 24; 2048 of 64 10.5 / 10.5, of 128 17.0 / 18.6, of 256 27.4 / 25.7; 8192 of 128 52 / 32, of 256 126 / 61
  if (b->T <= 8ll * lq_attn_cus()) return go(rope_norm_kernel<D, 1>, 1, parts);
  return go(rope_norm_kernel<D, 8>, 8, 1);
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
