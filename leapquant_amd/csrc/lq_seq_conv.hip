// Depthwise causal conv1d over a ragged batch (lq_conv_seq): y_t = act(w0 x_{t-3} + w1 x_{t-2} + w2 x_{t-1} + w3 x_t + bias).
//
// Reads 2 and writes 2 bytes an element; ~11 vector instructions an element keep it bound by memory.  A thread owns VEC
// neighbouring channels of a run of RUN tokens of one sequence: all of the run's loads are in flight before its arithmetic,
// the three inputs before the run are requested once more (out of a cache), and the last three move through registers.
// The workgroup of a sequence's first run also moves its taps: it reads them before it writes them, and no other
// workgroup touches them, so a call can run in place.
//
// VEC = 8 where the call is large (WIDE): a workgroup's rows are then 4 KiB pieces, and 32768 tokens of 8192 channels take
// 212 us (1.07 GB: 5.1 TB/s, past a large copy's rate; 218 without the outputs' hint, 223 with one on the inputs, which
// other runs read again), against 276 us with VEC = 2.  VEC = 2 below: a thread moves 2 channels'
// taps and not 8, and there are four times the waves: 64 tokens 4.5 us against 9.4, 333 tokens 6.4 against 10.8, 8000
// tokens 66 against 70, which is about where they meet.  Small calls are bound by their chain of loads: the run's
// sequence, its slots, the taps.
#include "lq_seq.h"

namespace {

constexpr int RUN = 8;
static_assert(RUN >= 3, "the three inputs before a later run belong to its own sequence");
constexpr long long WIDE = 1ll << 27;            // elements of a call

template <int VEC> struct Elems {
  typedef uint32_t raw __attribute__((ext_vector_type(VEC / 2)));
  static __device__ __forceinline__ void unpack(const raw& u, float* f) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) { f[2 * i] = bf_lo(u[i]); f[2 * i + 1] = bf_hi(u[i]); }
  }
  static __device__ __forceinline__ raw pack(const float* f) {
    raw u;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) u[i] = pk_bf16(f[2 * i], f[2 * i + 1]);
    return u;
  }
  static __device__ __forceinline__ raw zero() { return raw(0); }
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
  const bf16_t* p = x + (long long)t0 * ld + c;
  raw_t u[RUN];                                  // all loads of the run in flight before its arithmetic
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < RUN; ++i) u[i] = *(const raw_t*)(p + (long long)min(i, n - 1) * ld);
  }
  float w[4][VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const uint2 v = ((const uint2*)cv.weight)[c + e];
    w[0][e] = bf_lo(v.x); w[1][e] = bf_hi(v.x); w[2][e] = bf_lo(v.y); w[3][e] = bf_hi(v.y);
    b[e] = cv.bias ? bf2f(((const bf16_t*)cv.bias)[c + e]) : 0.f;
  }
  const int dst = seq_dst(s, r.n, cv.NS), src = seq_src(s, r.n, cv.NS);
  float h[3][VEC];                               // the three inputs before the run, oldest first
  if (r.j == 0) {
    const bf16_t* S = (const bf16_t*)cv.state + (long long)src * cv.slot_stride + (long long)c * cv.ch_stride;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      h[0][e] = h[1][e] = h[2][e] = 0.f;
      if (src) {
        const bf16_t* f = S + e * cv.ch_stride;
        h[0][e] = bf2f(f[0]); h[1][e] = bf2f(f[cv.tap_stride]); h[2][e] = bf2f(f[2 * cv.tap_stride]);
      }
    }
    if (dst) {                                   // the last three inputs: of the sequence, and of the taps where it is short
      const int len = r.hi - r.lo;
      bf16_t* D = (bf16_t*)cv.state + (long long)dst * cv.slot_stride + (long long)c * cv.ch_stride;
      const bf16_t* last = p + (long long)(len - 3) * ld;
      float f[3][VEC] = {};
      if (len >= 3) E::unpack(*(const raw_t*)last, f[0]);
      if (len >= 2) E::unpack(*(const raw_t*)(last + ld), f[1]);
      if (len >= 1) E::unpack(*(const raw_t*)(last + 2 * ld), f[2]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float a0 = h[0][e], a1 = h[1][e], a2 = h[2][e];
        const float f0 = len >= 3 ? f[0][e] : len == 2 ? a2 : len == 1 ? a1 : a0;
        const float f1 = len >= 2 ? f[1][e] : len == 1 ? a2 : a1;
        const float f2 = len >= 1 ? f[2][e] : a2;
        bf16_t* to = D + e * cv.ch_stride;
        to[0] = (bf16_t)(__float_as_uint(f0) >> 16);
        to[cv.tap_stride] = (bf16_t)(__float_as_uint(f1) >> 16);
        to[2 * cv.tap_stride] = (bf16_t)(__float_as_uint(f2) >> 16);
      }
    }
    if (n <= 0) return;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) E::unpack(*(const raw_t*)(p + (long long)(i - 3) * ld), h[i]);
  }
  bf16_t* o = out + (long long)t0 * C + c;
  const bool silu = cv.silu;
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    float f[VEC], y[VEC];
    E::unpack(u[i], f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      y[e] = fmaf(w[3][e], f[e], fmaf(w[2][e], h[2][e], fmaf(w[1][e], h[1][e], fmaf(w[0][e], h[0][e], b[e]))));
      if (silu) y[e] *= fast_sigmoid(y[e]);
      h[0][e] = h[1][e]; h[1][e] = h[2][e]; h[2][e] = f[e];
    }
    if (i < n) {
      const raw_t r = dst ? E::pack(y) : E::zero();
      raw_t* to = (raw_t*)(o + (long long)i * C);
      if (VEC == 8) __builtin_nontemporal_store(r, to);      // more than the caches hold
      else *to = r;
    }
  }
}

template <int VEC>
int launch(const lq_conv* cv, const lq_seqs* s, const void* x, long long x_ld, void* out, int C, hipStream_t st) {
  const dim3 grid((unsigned)seq_runs<RUN>(s), (unsigned)((C + 256 * VEC - 1) / (256 * VEC)));
  if (grid.y > 65535u) return LQ_ERR_ARG;
  conv_seq_kernel<VEC><<<grid, 256, 0, st>>>(*cv, *s, (const bf16_t*)x, x_ld, (bf16_t*)out, C);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
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
  const uintptr_t where = (uintptr_t)x | (uintptr_t)out;
  hipStream_t st = (hipStream_t)stream;
  if (C % 8 == 0 && x_ld % 8 == 0 && where % 16 == 0 && (long long)s->T * C >= WIDE)
    return launch<8>(cv, s, x, x_ld, out, C, st);
  if (C % 2 == 0 && x_ld % 2 == 0 && where % 4 == 0) return launch<2>(cv, s, x, x_ld, out, C, st);
  return launch<1>(cv, s, x, x_ld, out, C, st);
}
