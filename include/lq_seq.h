/* liblq_seq -- C ABI of the operators that take whole sequences through a linear-attention layer on MI355X (gfx950): the
 * gated delta rule over a ragged batch (chunked, and token by token), the causal conv1d before it, and the norms before
 * and after the block.  They run beside the decode path of liblq (lq.h): same tensors, dtypes and status codes.
 *
 * Every entry point takes plain device pointers, sizes and a hipStream_t (as void*), launches on that stream, allocates
 * nothing, never synchronises, and returns 0 or a negative lq_status.
 */
#ifndef LQ_SEQ_H
#define LQ_SEQ_H

#include "lq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Raised with every change of a structure's layout or an entry point's arguments, as LQ_ABI_VERSION of lq.h. */
#define LQ_SEQ_ABI_VERSION 1
int lq_seq_abi_version(void);

/* A ragged batch: sequence n holds the packed tokens loc[n] .. loc[n + 1] - 1 of T.  The kernels hold every offset to
 * 0 <= loc[n] <= loc[n + 1] <= T.  It starts from slot src[n] of the state (or conv) cache and leaves its last state in slot
 * idx[n]; a src outside 1 .. NS - 1 starts from zero, an idx outside makes a padding sequence: its outputs are zero and
 * no slot is written.  A sequence of no tokens copies its state.  No slot that one sequence of a call writes may be read or
 * written by another.  Rows of `out` that no sequence holds are not written. */
typedef struct lq_seqs {
  const int* loc;         /* [N + 1] */
  const int* idx;         /* [N] */
  const int* src;         /* [N], or NULL: idx (in place) */
  int N, T;
} lq_seqs;

/* One gated delta rule layer: S_t = S_{t-1} diag(e^g) + u k^T, u = beta (v - S_{t-1} diag(e^g) k), o = S_t q, with
 * q = q / sqrt(|q|^2 + 1e-6) scale, k = k / sqrt(|k|^2 + 1e-6), beta = sigmoid(b) and
 * g = -exp(A_log) softplus(a + dt_bias), or, KDA with glb != 0, glb sigmoid(exp(A_log) (a + dt_bias)).
 * KDA (kda = 1) has a gate for each key channel, GDN one for each value head. */
typedef struct lq_delta {
  float* S;               /* fp32 [NS][HV][V][K], slots slot_stride floats apart (divisible by 4), 16-byte aligned */
  long long slot_stride;
  int NS, HV, H, K, V;    /* (K, V) = (128, 128), (64, 128) or (64, 64); KDA (128, 128).  HV % H == 0 */
  const void* mixed;      /* bf16 [T] rows of mixed_ld elements (divisible by 8, 16-byte aligned): q | k | v, after the conv */
  const void* a;          /* bf16 [T] rows of a_ld elements: GDN [HV]; KDA [HV][K], 8-byte aligned, a_ld divisible by 4 */
  const void* b;          /* bf16 [T] rows of b_ld elements: [HV] */
  const void* A_log;      /* [HV], fp32 or bf16 (gate_bf16 bit 0) */
  const void* dt_bias;    /* GDN [HV]; KDA [HV][K], fp32 or bf16 (gate_bf16 bit 1) */
  void* out;              /* bf16 [T][HV][V], 16-byte aligned */
  long long mixed_ld, a_ld, b_ld;
  float scale;
  int gate_bf16, kda;
  float glb;
} lq_delta;

/* Token by token: a state is read and written once a sequence, the time grows with its longest sequence.  For single
 * tokens, drafted tokens and short prompts; any length is right. */
int lq_delta_steps(const lq_delta* d, const lq_seqs* s, void* stream);

/* The same result in chunks of tokens on the matrix cores (GDN), for prompts.  `work`: lq_delta_workspace(d, s) bytes of device
 * memory, 16-byte aligned, whose contents do not matter before and after the call. */
int lq_delta_prefill(const lq_delta* d, const lq_seqs* s, void* work, long long work_bytes, void* stream);
long long lq_delta_workspace(const lq_delta* d, const lq_seqs* s);

/* What lq_delta_steps (chunks = 0) or lq_delta_prefill (chunks = 1) answers to these arguments, workspace aside, without a
 * launch: for a caller with work to do before the call that must not be done if the call is refused. */
int lq_delta_check(const lq_delta* d, const lq_seqs* s, int chunks);

/* Depthwise causal conv1d (W = 4) of the packed tokens x (bf16, rows x_ld elements apart) into out (bf16 [T][C], not
 * overlapping x): the conv of lq.h's lq_conv for each token, the taps before a sequence's first token read from its slot, its
 * last three inputs left there. */
int lq_conv_seq(const lq_conv* cv, const lq_seqs* s, const void* x, long long x_ld, void* out, int C, void* stream);

/* Norm of the rows of D <= 16384 elements, of `heads` consecutive vectors each: element (row, h, d) of x at
 * x[row * x_ld + h * x_hd + d], z and out likewise; vectors of out (o_ld, o_hd) may not overlap each other.  `weight` [D], fp32
 * or bf16 (weight_bf16). */
typedef struct lq_norm {
  const void* x;
  const void* z;          /* lq_gated_norm: the gate; lq_add_norm: what is added */
  const void* weight;
  void* res;              /* lq_add_norm: bf16, laid out as out */
  void* out;              /* bf16 */
  long long x_ld, x_hd, z_ld, z_hd, o_ld, o_hd;
  int rows, heads, D;
  float eps, scale, offset;
  int act;                /* lq_gated_norm: 0 SiLU, 1 sigmoid */
  int weight_bf16;
} lq_norm;

/* out = x rsqrt(mean(x^2) + eps) (offset + weight) act(z) */
int lq_gated_norm(const lq_norm* n, void* stream);
/* res = x + scale z;  out = res rsqrt(mean(res^2) + eps) (offset + weight), of the sum before it is rounded.  res may be
 * x or z. */
int lq_add_norm(const lq_norm* n, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LQ_SEQ_H */
