// Shared device helpers of liblq_seq: ragged batches and the gates of a token.
#pragma once
#include "../../include/lq_seq.h"
#include "lq_common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__attribute__((visibility("hidden"))) int lq_seq_cus();      // compute units of the current GPU
// a prefill's grids and 32-bit offsets hold what it is given
__attribute__((visibility("hidden"))) bool lq_prefill_fits(const lq_delta* d, const lq_seqs* s);

struct SeqRun {      // a run of a sequence's tokens, as its workgroup finds it
  int n, j;          // sequence, run of it
  int lo, hi;        // the sequence's packed tokens
};

// Start of sequence n, held to the packed tokens whatever loc says.
__device__ __forceinline__ int seq_at(const lq_seqs& s, int n) { return min(max(s.loc[n], 0), s.T); }

// Runs of RUN tokens of a ragged batch, numbered without a scan over the batch: run j of sequence n has the number
// loc[n] / RUN + n + j.  Sequence n owns loc[n+1] / RUN - loc[n] / RUN + 1 numbers, which is at least its ceil(len / RUN)
// runs and at least one; the numbers left over, and those before the first sequence, find an empty run past the end.  The
// batch has T / RUN + N of them.  A whole wave looks for its run at once, 64 sequences a step: one load up to 64 of them.
template <int RUN>
__device__ __forceinline__ SeqRun seq_run(const lq_seqs& s, int number) {
  const int lane = threadIdx.x & 63;
  int a = 0, len = s.N;                          // the last n of a .. a + len - 1 whose first number is not above `number`
  while (len > 1) {
    const int step = (len + 63) >> 6, m = a + lane * step;
    const bool below = lane * step < len && seq_at(s, m) / RUN + m <= number;
    const int at = max((int)__popcll(__ballot(below)) - 1, 0) * step;     // the count is unsigned
    a += at;
    len = min(step, len - at);
  }
  SeqRun r;
  r.n = a;
  r.lo = seq_at(s, a);
  r.hi = max(r.lo, seq_at(s, a + 1));
  r.j = number - (r.lo / RUN + a);
  if (r.j < 0 || r.j > s.T / RUN) { r.j = 1; r.lo = r.hi; }
  return r;
}
template <int RUN>
static inline long long seq_runs(const lq_seqs* s) { return (long long)s->T / RUN + s->N; }

// slot of a cache with NS slots, or 0 where the sequence has none
__device__ __forceinline__ int seq_slot(int i, int NS) { return i > 0 && i < NS ? i : 0; }
__device__ __forceinline__ int seq_dst(const lq_seqs& s, int n, int NS) { return seq_slot(s.idx[n], NS); }
__device__ __forceinline__ int seq_src(const lq_seqs& s, int n, int NS) {
  return seq_slot((s.src ? s.src : s.idx)[n], NS);
}
static inline bool seqs_ok(const lq_seqs* s) {
  return s && s->N >= 0 && s->T >= 0 && (s->N == 0 || (s->loc && s->idx));
}

// a gate parameter, fp32 or bf16
__device__ __forceinline__ float gate_param(const void* p, int bf16, long long i) {
  return bf16 ? bf2f(((const bf16_t*)p)[i]) : ((const float*)p)[i];
}
// e^x and 1 / (1 + e^-x) from the hardware's exp2 and reciprocal (1 ulp each): for results that are rounded to bf16
__device__ __forceinline__ float fast_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
// e^x, the argument's product with log2 e carried in two parts (a few 1e-7 for any x; __expf loses |x| 1e-7)
__device__ __forceinline__ float exp_f(float x) {
  const float t = x * 1.44269504f, r = fmaf(x, 1.44269504f, -t) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return fabsf(t) < 150.f ? e * fmaf(r, 0.693147181f, 1.0f) : e;             // zero, infinity and NaN as they are
}
// log(1 + e^x), x above the threshold itself; log(1 + u) as log(w) u / (w - 1), w = 1 + u, which has w's rounding cancel
__device__ __forceinline__ float softplus_f(float x) {
  const float u = exp_f(fminf(x, (float)LQ_SOFTPLUS_THRESHOLD)), w = 1.0f + u, d = w - 1.0f;
  const float y = __builtin_amdgcn_logf(w) * 0.693147181f * u * __builtin_amdgcn_rcpf(d);
  const float z = d == 0.f ? u : y;
  return x <= (float)LQ_SOFTPLUS_THRESHOLD ? z : x;
}
