// The gated delta rule token by token (lq_delta_steps): the form for single tokens and short sequences.
//
//   u = beta (v - S diag(alpha) k),   o = S diag(alpha) q + (k.q) u,   S' = S diag(alpha) + u k^T
//
// (GDN: one alpha a head and token; KDA: one a key channel.)  The state is read once and written once a sequence: 8 K V bytes a
// head, which bounds it at one token; each token adds 6 K V operations on the vector units.
//
// Rows of S (value channels) do not meet, so a workgroup owns 32 ROWS of them: 8 lanes a row, each with K / 8 key channels
// in float4 groups 32 channels apart (a wave's load covers 128-byte pieces of 8 rows), ROWS rows of each lane in registers
// across the tokens.  Both dot products run on the old state, so their 8-lane sums do not wait for the update.  The next
// token's inputs are requested before the current one is worked on.
#include "lq_seq.h"

namespace {

// the log-gate of a token: GDN and KDA's unbounded form, or KDA's bounded one.  Below -128 its exponential is zero in fp32
// either way.  A NaN stays one.
__device__ __forceinline__ float log_gate(float x, float ea, float glb) {
  return glb != 0.f ? glb / (1.0f + expf(-ea * x)) : -ea * softplus20f(x);
}

template <int K, bool KDA> struct Token {        // a token's inputs as loaded
  uint2 q[K / 32], k[K / 32], a[KDA ? K / 32 : 1];
  bf16_t b, ag;
};

template <int K, int V, int ROWS, bool KDA>
__global__ __launch_bounds__(256) void steps_kernel(lq_delta p, lq_seqs s) {
  constexpr int E = K / 32;                      // float4 groups a lane
  constexpr int PARTS = V / (32 * ROWS);         // workgroups a head
  const int part = blockIdx.x % PARTS, hn = blockIdx.x / PARTS, n = hn / p.HV, hv = hn - n * p.HV;
  const int hk = hv / (p.HV / p.H);
  const int lane = threadIdx.x & 7, row0 = part * 32 * ROWS + (threadIdx.x >> 3) * ROWS;
  const int lo = seq_at(s, n), hi = max(lo, seq_at(s, n + 1));
  const int dst = seq_dst(s, n, p.NS), src = seq_src(s, n, p.NS);
  bf16_t* out = (bf16_t*)p.out + (long long)hv * V + row0;
  const long long old = (long long)p.HV * V;
  if (dst == 0) {
    if (lane < ROWS)
      for (int t = lo; t < hi; ++t) out[t * old + lane] = 0;
    return;
  }
  const long long head = (long long)hv * V * K + (long long)row0 * K + 4 * lane;
  float S[ROWS][4 * E];
  {
    const float* f = p.S + src * p.slot_stride + head;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float4 x = src ? *(const float4*)(f + r * K + 32 * e) : make_float4(0.f, 0.f, 0.f, 0.f);
        S[r][4 * e] = x.x; S[r][4 * e + 1] = x.y; S[r][4 * e + 2] = x.z; S[r][4 * e + 3] = x.w;
      }
  }
  const float ea = expf(gate_param(p.A_log, p.gate_bf16 & 1, hv));
  float dt[KDA ? 4 * E : 1];
  if (KDA) {
#pragma unroll
    for (int i = 0; i < 4 * E; ++i)
      dt[KDA ? i : 0] = gate_param(p.dt_bias, p.gate_bf16 & 2, (long long)hv * K + 4 * lane + 32 * (i >> 2) + (i & 3));
  } else {
    dt[0] = gate_param(p.dt_bias, p.gate_bf16 & 2, hv);
  }
  const bf16_t* mixed = (const bf16_t*)p.mixed + 4 * lane;
  const bf16_t* vrow = (const bf16_t*)p.mixed + 2ll * p.H * K + (long long)hv * V + row0;
  Token<K, KDA> next;
  bf16_t vnext[ROWS];
  auto request = [&](int t) {
    const bf16_t* m = mixed + t * p.mixed_ld + hk * K;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      next.q[e] = *(const uint2*)(m + 32 * e);
      next.k[e] = *(const uint2*)(m + p.H * K + 32 * e);
      if (KDA) next.a[KDA ? e : 0] = *(const uint2*)((const bf16_t*)p.a + t * p.a_ld + hv * K + 4 * lane + 32 * e);
    }
    if (!KDA) next.ag = ((const bf16_t*)p.a)[t * p.a_ld + hv];
    next.b = ((const bf16_t*)p.b)[t * p.b_ld + hv];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) vnext[r] = vrow[t * p.mixed_ld + r];
  };
  if (lo < hi) request(lo);
  for (int t = lo; t < hi; ++t) {
    const Token<K, KDA> now = next;
    float v[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) v[r] = bf2f(vnext[r]);
    if (t + 1 < hi) request(t + 1);
    float q[4 * E], k[4 * E], nq = 0.f, nk = 0.f, kq = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t qw[2] = {now.q[e].x, now.q[e].y}, kw[2] = {now.k[e].x, now.k[e].y};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        q[4 * e + 2 * i] = bf_lo(qw[i]); q[4 * e + 2 * i + 1] = bf_hi(qw[i]);
        k[4 * e + 2 * i] = bf_lo(kw[i]); k[4 * e + 2 * i + 1] = bf_hi(kw[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4 * E; ++i) {
      nq = fmaf(q[i], q[i], nq); nk = fmaf(k[i], k[i], nk); kq = fmaf(k[i], q[i], kq);
    }
    nq = sum8(nq); nk = sum8(nk); kq = sum8(kq);
    const float iq = rsqrtf_rn(nq + 1e-6f) * p.scale, ik = rsqrtf_rn(nk + 1e-6f);
    kq *= iq * ik;
    const float beta = 1.0f / (1.0f + expf(-bf2f(now.b)));
    float al[KDA ? 4 * E : 1];
    if (KDA) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t aw[2] = {now.a[KDA ? e : 0].x, now.a[KDA ? e : 0].y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = (i & 1) ? bf_hi(aw[i >> 1]) : bf_lo(aw[i >> 1]);
          al[KDA ? 4 * e + i : 0] = expf(log_gate(x + dt[KDA ? 4 * e + i : 0], ea, p.glb));
        }
      }
    } else {
      al[0] = expf(log_gate(bf2f(now.ag) + dt[0], ea, 0.f));
    }
    float keep = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float m = 0.f, y = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * E; ++i) {
        S[r][i] *= al[KDA ? i : 0];
        m = fmaf(S[r][i], k[i], m); y = fmaf(S[r][i], q[i], y);
      }
      m = sum8(m) * ik; y = sum8(y) * iq;
      const float u = beta * (v[r] - m), uk = u * ik;
#pragma unroll
      for (int i = 0; i < 4 * E; ++i) S[r][i] = fmaf(uk, k[i], S[r][i]);
      y = fmaf(kq, u, y);
      if (lane == r) keep = y;
    }
    if (lane < ROWS) out[t * old + lane] = f2bf(keep);
  }
  float* f = p.S + dst * p.slot_stride + head;
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int e = 0; e < E; ++e)
      *(float4*)(f + r * K + 32 * e) = make_float4(S[r][4 * e], S[r][4 * e + 1], S[r][4 * e + 2], S[r][4 * e + 3]);
}

template <int K, int V, int ROWS, bool KDA>
int launch(const lq_delta* d, const lq_seqs* s, hipStream_t st) {
  const long long grid = (long long)s->N * d->HV * (V / (32 * ROWS));
  if (grid > 0x7fffffffll) return LQ_ERR_ARG;
  steps_kernel<K, V, ROWS, KDA><<<(unsigned)grid, 256, 0, st>>>(*d, *s);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
}

}  // namespace

__attribute__((visibility("hidden"))) int lq_check_delta(const lq_delta* d, const lq_seqs* s) {
  if (!d || !seqs_ok(s)) return LQ_ERR_ARG;
  const bool dims = (d->K == 128 && d->V == 128) || (!d->kda && d->K == 64 && (d->V == 128 || d->V == 64));
  if (!dims || d->NS <= 0 || d->H <= 0 || d->HV <= 0 || d->HV % d->H != 0) return LQ_ERR_ARG;
  if ((d->kda != 0 && d->kda != 1) || d->gate_bf16 < 0 || d->gate_bf16 > 3 || (!d->kda && d->glb != 0.f)) return LQ_ERR_ARG;
  if (!d->S || ((uintptr_t)d->S & 15) || d->slot_stride % 4 || d->slot_stride < (long long)d->HV * d->V * d->K)
    return LQ_ERR_ARG;
  const int KA = d->kda ? d->K : 1;
  if (d->mixed_ld < 2ll * d->H * d->K + (long long)d->HV * d->V || d->mixed_ld % 8 || d->a_ld < (long long)d->HV * KA ||
      d->b_ld < d->HV || (d->kda && d->a_ld % 4))
    return LQ_ERR_ARG;
  if (((uintptr_t)d->mixed & 15) || ((uintptr_t)d->out & 15) || (d->kda && ((uintptr_t)d->a & 7))) return LQ_ERR_ARG;
  if (!d->A_log || !d->dt_bias) return LQ_ERR_ARG;
  if (s->N > 0 && s->T > 0 && (!d->mixed || !d->a || !d->b || !d->out)) return LQ_ERR_ARG;
  return LQ_OK;
}

extern "C" int lq_delta_steps(const lq_delta* d, const lq_seqs* s, void* stream) {
  if (int rc = lq_check_delta(d, s)) return rc;
  if (s->N == 0) return LQ_OK;
  hipStream_t st = (hipStream_t)stream;
  if (d->kda) return launch<128, 128, 4, true>(d, s, st);
  if (d->K == 128) return launch<128, 128, 4, false>(d, s, st);
  if (d->V == 128) return launch<64, 128, 4, false>(d, s, st);
  return launch<64, 64, 2, false>(d, s, st);
}
