// Shared device helpers of liblq_seq: ragged batches and the gates of a token.
#pragma once
#include "../../include/lq_seq.h"
#include "lq_common.h"

struct SeqRun {      // a run of a sequence's tokens, as its workgroup finds it
  int n, j;          // sequence, run of it
  int lo, hi;        // the sequence's packed tokens
};

// Start of sequence n, held to the packed tokens whatever loc says.
__device__ __forceinline__ int seq_at(const lq_seqs& s, int n) { return min(max(s.loc[n], 0), s.T); }

// Runs of RUN tokens of a ragged batch, numbered without a scan over the batch: run j of sequence n has the number
// loc[n] / RUN + n + j.  Sequence n owns loc[n+1] / RUN - loc[n] / RUN + 1 numbers, which is at least its ceil(len / RUN)
// runs and at least one; the numbers left over find j past the end.  The batch has T / RUN + N of them.
template <int RUN>
__device__ __forceinline__ SeqRun seq_run(const lq_seqs& s, int number) {
  int a = 0, b = s.N - 1;                        // the last n whose first number is not above `number`
  while (a < b) {
    const int m = (a + b + 1) >> 1;
    if (seq_at(s, m) / RUN + m <= number) a = m; else b = m - 1;
  }
  SeqRun r;
  r.n = a;
  r.lo = seq_at(s, a);
  r.hi = max(r.lo, seq_at(s, a + 1));
  r.j = number - (r.lo / RUN + a);
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
