// Depthwise causal conv1d over a ragged batch (lq_conv_seq): y_t = act(w0 x_{t-3} + w1 x_{t-2} + w2 x_{t-1} + w3 x_t + bias).
//
// Reads 2 and writes 2 bytes an element; ~11 vector instructions an element keep it bound by memory.  A thread owns VEC
// neighbouring channels of a run of RUN tokens of one sequence and carries the last three inputs in registers, so each
// input is requested once and the three before the run once more.
// The workgroup of a sequence's first run also moves its taps: it reads them before it writes them, and no other
// workgroup touches them, so a call can run in place.
#include "lq_seq.h"

namespace {

constexpr int RUN = 16;

template <int VEC> struct Elems;
template <> struct Elems<8> {
  typedef uint4 raw;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = bf_lo(w[i]); f[2 * i + 1] = bf_hi(w[i]); }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pk_bf16(f[0], f[1]), pk_bf16(f[2], f[3]), pk_bf16(f[4], f[5]), pk_bf16(f[6], f[7]));
  }
  static __device__ __forceinline__ uint4 zero() { return make_uint4(0, 0, 0, 0); }
};
template <> struct Elems<1> {
  typedef bf16_t raw;
  static __device__ __forceinline__ void unpack(const bf16_t& u, float* f) { f[0] = bf2f(u); }
  static __device__ __forceinline__ bf16_t pack(const float* f) { return f2bf(f[0]); }
  static __device__ __forceinline__ bf16_t zero() { return 0; }
};

template <int VEC>
__global__ __launch_bounds__(256) void conv_seq_kernel(lq_conv cv, lq_seqs s, const bf16_t* __restrict__ x, long long ld,
                                                       bf16_t* __restrict__ out, int C) {
  typedef Elems<VEC> E;
  typedef typename E::raw raw_t;
  const SeqRun r = seq_run<RUN>(s, blockIdx.x);
  const int t0 = r.lo + r.j * RUN, n = min(RUN, r.hi - t0);
  if (n <= 0 && r.j > 0) return;
  const int c = (blockIdx.y * 256 + threadIdx.x) * VEC;
  if (c >= C) return;
  const int dst = seq_dst(s, r.n, cv.NS), src = seq_src(s, r.n, cv.NS);
  if (dst == 0) {
    for (int i = 0; i < n; ++i) *(raw_t*)(out + (long long)(t0 + i) * C + c) = E::zero();
    return;
  }
  const bf16_t* p = x + (long long)t0 * ld + c;
  float h[3][VEC];                               // the three inputs before the run, oldest first
  if (r.j == 0) {
    bf16_t tap[3][VEC];
    const bf16_t* S = (const bf16_t*)cv.state + (long long)src * cv.slot_stride + (long long)c * cv.ch_stride;
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        tap[i][e] = src ? S[e * cv.ch_stride + i * cv.tap_stride] : (bf16_t)0;
        h[i][e] = bf2f(tap[i][e]);
      }
    const int len = r.hi - r.lo;                 // the last three inputs: of the sequence, and of the taps where it is short
    bf16_t* D = (bf16_t*)cv.state + (long long)dst * cv.slot_stride + (long long)c * cv.ch_stride;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int at = len - 3 + i;                // -3 + i .. : a tap where negative
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        bf16_t v = at == -3 ? tap[0][e] : at == -2 ? tap[1][e] : tap[2][e];
        if (at >= 0) v = p[(long long)at * ld + e];
        D[e * cv.ch_stride + i * cv.tap_stride] = v;
      }
    }
    if (n <= 0) return;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) E::unpack(*(const raw_t*)(p + (long long)(i - 3) * ld), h[i]);
  }
  float w[4][VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const uint2 u = ((const uint2*)cv.weight)[c + e];
    w[0][e] = bf_lo(u.x); w[1][e] = bf_hi(u.x); w[2][e] = bf_lo(u.y); w[3][e] = bf_hi(u.y);
    b[e] = cv.bias ? bf2f(((const bf16_t*)cv.bias)[c + e]) : 0.f;
  }
  bf16_t* o = out + (long long)t0 * C + c;
  const bool silu = cv.silu;
  auto token = [&](const raw_t& u, int i) {
    float f[VEC], y[VEC];
    E::unpack(u, f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      y[e] = fmaf(w[3][e], f[e], fmaf(w[2][e], h[2][e], fmaf(w[1][e], h[1][e], fmaf(w[0][e], h[0][e], b[e]))));
      if (silu) y[e] *= fast_sigmoid(y[e]);
      h[0][e] = h[1][e]; h[1][e] = h[2][e]; h[2][e] = f[e];
    }
    *(raw_t*)(o + (long long)i * C) = E::pack(y);
  };
  if (n == RUN) {                                // all loads of the run in flight before its arithmetic
    raw_t u[RUN];
#pragma unroll
    for (int i = 0; i < RUN; ++i) u[i] = *(const raw_t*)(p + i * ld);
#pragma unroll
    for (int i = 0; i < RUN; ++i) token(u[i], i);
  } else {
    for (int i = 0; i < n; ++i) token(*(const raw_t*)(p + i * ld), i);
  }
}

}  // namespace

extern "C" int lq_conv_seq(const lq_conv* cv, const lq_seqs* s, const void* x, long long x_ld, void* out, int C,
                           void* stream) {
  if (!cv || !seqs_ok(s) || C <= 0 || x_ld < C) return LQ_ERR_ARG;
  if (!cv->state || !cv->weight || cv->W != 4 || (cv->silu != 0 && cv->silu != 1) || cv->NS <= 0) return LQ_ERR_ARG;
  if (cv->ch_stride <= 0 || cv->tap_stride <= 0 || (C - 1) * cv->ch_stride + 2 * cv->tap_stride >= cv->slot_stride)
    return LQ_ERR_ARG;
  if ((uintptr_t)cv->weight & 7) return LQ_ERR_ARG;
  if (s->N == 0) return LQ_OK;
  if (s->T > 0 && (!x || !out)) return LQ_ERR_ARG;
  const bool wide = C % 8 == 0 && x_ld % 8 == 0 && (((uintptr_t)x | (uintptr_t)out) & 15) == 0;
  const int per = 256 * (wide ? 8 : 1);
  const dim3 grid((unsigned)seq_runs<RUN>(s), (unsigned)((C + per - 1) / per));
  if (grid.y > 65535u) return LQ_ERR_ARG;
  if (wide)
    conv_seq_kernel<8><<<grid, 256, 0, (hipStream_t)stream>>>(*cv, *s, (const bf16_t*)x, x_ld, (bf16_t*)out, C);
  else
    conv_seq_kernel<1><<<grid, 256, 0, (hipStream_t)stream>>>(*cv, *s, (const bf16_t*)x, x_ld, (bf16_t*)out, C);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
}
