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
//
// GDN's decay is kept beside the state, S = scale S', and goes into the sums' and the update's factors, so that an element
// costs three operations a token; the factor is multiplied out before it falls below 2^-20.  KDA's gates, a log, two
// exponentials and a reciprocal for each key channel, are the same for all rows: the workgroup forms those of 8 tokens at once.
//
// Measured, heads of 128 x 128: 256 sequences of one token and 32 heads 205 us (1.07 GB: 5.2 TB/s, a copy's rate), 64 of one
// 68 us (3.9 TB/s), 64 of 8 tokens 90 us, where the vector units take over (2 us a token); one sequence of one token 5 us, the
// chain of its loads, of 32 tokens 26 us.  (Caches full of other data; 40, 61 and 21 us where they hold states.)  Norms, gates
// and beta come from the hardware's reciprocal square root, exp2, log and reciprocal, 1 ulp each: with the library's 7 to
// 10% of a token's time more.
#include "lq_seq.h"

namespace {

// the gate of a token: GDN and KDA's unbounded form, or KDA's bounded one.  A NaN stays one.
__device__ __forceinline__ float gate_of(float x, float ea, float glb) {
  return exp_f(glb != 0.f ? glb * __builtin_amdgcn_rcpf(1.0f + exp_f(-ea * x)) : -ea * softplus_f(x));
}

constexpr int BLOCK = 8;                         // tokens whose KDA gates a workgroup forms at once

template <int K, int V, int ROWS, bool KDA, bool PAST>
__global__ __launch_bounds__(256) void steps_kernel(lq_delta p, lq_seqs s) {
  constexpr int E = K / 32;                      // float4 groups a lane
  constexpr int PARTS = V / (32 * ROWS);         // workgroups a head
  __shared__ f32x4 gates[KDA ? BLOCK : 1][KDA ? K / 4 : 1];
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
  const bf16_t* mixed = (const bf16_t*)p.mixed + 4 * lane + hk * K;
  const bf16_t* vrow = (const bf16_t*)p.mixed + 2ll * p.H * K + (long long)hv * V + row0;
  u32x2 qn[E], kn[E];                            // the next token's inputs as loaded
  bf16_t vn[ROWS], bn = 0, an = 0;
  auto request = [&](int t) {
    const bf16_t* m = mixed + t * p.mixed_ld;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      qn[e] = *(const u32x2*)(m + 32 * e);
      kn[e] = *(const u32x2*)(m + p.H * K + 32 * e);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) vn[r] = vrow[t * p.mixed_ld + r];
    if (!KDA) an = ((const bf16_t*)p.a)[t * p.a_ld + hv];
    bn = ((const bf16_t*)p.b)[t * p.b_ld + hv];
  };
  if (lo < hi) request(lo);
  const long long head = (long long)hv * V * K + (long long)row0 * K + 4 * lane;
  float S[ROWS][4 * E];
  {
    const float* f = p.S + src * p.slot_stride + head;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f32x4 x = {};
        if (src) x = *(const f32x4*)(f + r * K + 32 * e);
#pragma unroll
        for (int i = 0; i < 4; ++i) S[r][4 * e + i] = x[i];
      }
  }
  const float ea = expf(gate_param(p.A_log, p.gate_bf16 & 1, hv));
  const int channel = threadIdx.x % K;
  const float dt = gate_param(p.dt_bias, p.gate_bf16 & 2, KDA ? (long long)hv * K + channel : hv);
  float scale = 1.f;                             // GDN: the state is scale S
  for (int t = lo; t < hi; ++t) {
    if (KDA && (t - lo) % BLOCK == 0) {
      const bf16_t* a = (const bf16_t*)p.a + hv * K + channel;
      if (t > lo) __syncthreads();
      for (int i = threadIdx.x / K; i < min(BLOCK, hi - t); i += 256 / K)
        ((float*)gates[i])[channel] = gate_of(bf2f(a[(t + i) * p.a_ld]) + dt, ea, p.glb);
      __syncthreads();
    }
    float q[4 * E], k[4 * E], v[ROWS], nq = 0.f, nk = 0.f, kq = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        q[4 * e + 2 * i] = bf_lo(qn[e][i]); q[4 * e + 2 * i + 1] = bf_hi(qn[e][i]);
        k[4 * e + 2 * i] = bf_lo(kn[e][i]); k[4 * e + 2 * i + 1] = bf_hi(kn[e][i]);
      }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) v[r] = bf2f(vn[r]);
    const float beta = __builtin_amdgcn_rcpf(1.0f + exp_f(-bf2f(bn)));
    float al[KDA ? 4 * E : 1];
    if (KDA) {
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) al[KDA ? 4 * e + i : 0] = gates[KDA ? (t - lo) % BLOCK : 0][KDA ? lane + 8 * e : 0][i];
    } else {
      scale *= gate_of(bf2f(an) + dt, ea, 0.f);
    }
    if (t + 1 < hi) request(t + 1);
#pragma unroll
    for (int i = 0; i < 4 * E; ++i) {
      nq = fmaf(q[i], q[i], nq); nk = fmaf(k[i], k[i], nk); kq = fmaf(k[i], q[i], kq);
    }
    nq = sum8(nq); nk = sum8(nk); kq = sum8(kq);
    const float iq = __builtin_amdgcn_rsqf(nq + 1e-6f) * p.scale, ik = __builtin_amdgcn_rsqf(nk + 1e-6f);
    kq *= iq * ik;
    if (!KDA && scale < 0x1p-20f) {              // before 1 / scale grows large
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < 4 * E; ++i) S[r][i] *= scale;
      scale = 1.f;
    }
    const float up = KDA ? ik : ik * __builtin_amdgcn_rcpf(scale), sk = ik * scale, sq = iq * scale;
    float keep = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float m = 0.f, y = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * E; ++i) {
        if (KDA) S[r][i] *= al[KDA ? i : 0];
        m = fmaf(S[r][i], k[i], m); y = fmaf(S[r][i], q[i], y);
      }
      m = sum8(m) * sk; y = sum8(y) * sq;
      const float u = beta * (v[r] - m), uk = u * up;
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
    for (int e = 0; e < E; ++e) {
      const float* x = &S[r][4 * e];
      const f32x4 y = f32x4{x[0], x[1], x[2], x[3]} * scale;
      f32x4* to = (f32x4*)(f + r * K + 32 * e);
      if (PAST) __builtin_nontemporal_store(y, to);
      else *to = y;
    }
}

// Rows a lane.  One asks for the state in the shortest chain of loads; all rows of a head's workgroup in one share a token's
// norms and sums among 4.  One | four rows, 32 heads of 128 x 128: 1 x 1 token 5.4 | 6.8 us, 64 x 1 69 | 75, 1 x 4
// 7.9 | 9.7, 1 x 32 28 | 41, 8 x 4 17.8 | 15.3, 64 x 8 143 | 94.
int rows_of(const lq_delta* d, const lq_seqs* s) {
  return s->T <= s->N || (long long)s->N * d->HV * (d->V / 32) <= 2 * lq_seq_cus() ? 1 : d->V / 32;
}
long long grid_of(const lq_delta* d, const lq_seqs* s) { return (long long)s->N * d->HV * (d->V / (32 * rows_of(d, s))); }

template <int K, int V, int ROWS, bool KDA>
int launch_rows(const lq_delta* d, const lq_seqs* s, hipStream_t st) {
  const long long grid = grid_of(d, s);
  // States that fit the shared cache are written past it, which leaves it to those that are read.  With the hint | without, 32
  // heads of 128 x 128, to other slots: 64 sequences of 4 tokens 47 | 54 us, 32 of 4 27 | 29 (where other data fill the cache,
  // the same).  In place, where the next call reads what this one wrote: four layers in turn, as a model has them, 54 | 61 and
  // 29.5 | 30; one layer over and over 53 | 48 and 30 | 28; with the 8-bit quantize of all states right after it 98 | 95 and
  // 53 | 52; single tokens the same either way.  Beyond the cache's size it gains nothing, and after other writes 256
  // sequences lose 18%.
  if (4ll * s->N * d->HV * V * K <= 256ll << 20) steps_kernel<K, V, ROWS, KDA, true><<<(unsigned)grid, 256, 0, st>>>(*d, *s);
  else steps_kernel<K, V, ROWS, KDA, false><<<(unsigned)grid, 256, 0, st>>>(*d, *s);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
}
template <int K, int V, bool KDA>
int launch(const lq_delta* d, const lq_seqs* s, hipStream_t st) {
  return rows_of(d, s) == 1 ? launch_rows<K, V, 1, KDA>(d, s, st) : launch_rows<K, V, V / 32, KDA>(d, s, st);
}

}  // namespace

__attribute__((visibility("hidden"))) int lq_seq_cus() {
  static int cache[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cache[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

extern "C" int lq_seq_abi_version(void) { return LQ_SEQ_ABI_VERSION; }

extern "C" int lq_delta_check(const lq_delta* d, const lq_seqs* s, int chunks) {
  if (!d || !seqs_ok(s) || (chunks != 0 && (chunks != 1 || d->kda))) return LQ_ERR_ARG;
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
  if (s->N == 0) return LQ_OK;
  if (chunks) return lq_prefill_fits(d, s) ? LQ_OK : LQ_ERR_ARG;
  return grid_of(d, s) > 0x7fffffffll ? LQ_ERR_ARG : LQ_OK;
}

extern "C" int lq_delta_steps(const lq_delta* d, const lq_seqs* s, void* stream) {
  if (int rc = lq_delta_check(d, s, 0)) return rc;
  if (s->N == 0) return LQ_OK;
  hipStream_t st = (hipStream_t)stream;
  if (d->kda) return launch<128, 128, true>(d, s, st);
  if (d->K == 128) return launch<128, 128, false>(d, s, st);
  if (d->V == 128) return launch<64, 128, false>(d, s, st);
  return launch<64, 64, false>(d, s, st);
}
