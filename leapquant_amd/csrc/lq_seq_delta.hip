// The gated delta rule over prompts (lq_delta_prefill).
#include "lq_seq.h"

__attribute__((visibility("hidden"))) int lq_check_delta(const lq_delta* d, const lq_seqs* s);

extern "C" long long lq_delta_workspace(const lq_delta* d, const lq_seqs* s) { return 0; }

extern "C" int lq_delta_prefill(const lq_delta* d, const lq_seqs* s, void* work, long long work_bytes, void* stream) {
  if (d && d->kda) return LQ_ERR_ARG;
  return lq_delta_steps(d, s, stream);
}
