/* liblq_attn -- C ABI of the operators that take sequences through a softmax-attention layer with a paged cache on MI355X
 * (gfx950): the norms of each head's queries and keys with the rotation by position, which also fill the cache, and the
 * attention of new tokens over it.  They stand beside the linear-attention layers' operators of lq_seq.h: packed ragged
 * batches, bf16, the status codes of lq.h.
 *
 * Every entry point takes plain device pointers, sizes and a hipStream_t (as void*), launches on that stream, allocates
 * nothing, never synchronises, and returns 0 or a negative lq_status.
 */
#ifndef LQ_ATTN_H
#define LQ_ATTN_H

#include "lq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Raised with every change of a structure's layout or an entry point's arguments, as LQ_ABI_VERSION of lq.h. */
#define LQ_ATTN_ABI_VERSION 1
int lq_attn_abi_version(void);

/* A layer's cache: NP pages of `page` tokens.  Element (page p, token t, head h, d) of k and v at p * page_ld + t * row_ld +
 * h * head_ld + d: bf16, or, int8 = 1, codes whose values are code * scale with k_scale, v_scale at p * s_page_ld + t * s_row_ld +
 * h * s_head_ld.  k and v are 16-byte aligned with strides divisible by 16 bytes; a page's elements lie within 2^29 of
 * its first. */
typedef struct lq_pages {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  long long page_ld, row_ld, head_ld, s_page_ld, s_row_ld, s_head_ld;
  int NP, page;            /* page % 16 == 0 */
  int HK, D;               /* D = 64, 128 or 256 */
  int int8;
} lq_pages;

/* A ragged batch: sequence n holds the packed new tokens loc[n] .. loc[n + 1] - 1 of T, the last ones of its lens[n] cached tokens.
 * Token t of a sequence (its position, from 0) is at t % page in page table[n * table_ld + t / page].  The kernels hold
 * every offset to 0 <= loc[n] <= loc[n + 1] <= T and lens[n] to 0 .. width * page; a new token before position 0 (as all of a
 * padding sequence with lens[n] <= 0) sees and writes nothing, its outputs are zero whatever its inputs hold.  Rows of outputs
 * that no sequence holds are not written. */
typedef struct lq_batch {
  const int* loc;         /* [N + 1] */
  const int* lens;        /* [N] */
  const int* table;       /* [N] rows of `width` entries, table_ld apart */
  long long table_ld;
  int width;              /* width * page < 2^31 (lq_attend: 2^31 - 4096), width * page * page < 2^40 */
  int N, T;
} lq_batch;

/* Rows of heads: element (token, h, d) at token * ld + h * hd + d, bf16, 16-byte aligned with strides divisible by 8. */
typedef struct lq_rows {
  void* p;
  long long ld, hd;
} lq_rows;

/* x rsqrt(mean(x^2) + eps) (offset + weight) over each head of q and k, then its first `rot` elements turned in pairs by position *
 * inv_freq: (i, i + rot / 2), or interleaved (2i, 2i + 1).  q goes to out, which may be q, k and v to the new tokens' places in the
 * pages (8 bits: code = rint(x / scale), scale = max|x| / 127 of a token's head, NaN where the head holds one, 0 where max|x| <= 1e-30; a
 * scale of 0, or not finite, has codes of 0).
 * A token whose table entry is outside 0 .. NP - 1 is not written.  Places that two new tokens of a call share hold either's. */
typedef struct lq_rope {
  lq_rows q, k, v, out;
  const void* q_weight;   /* [D], fp32 or bf16 (weight_bf16 bit 0) */
  const void* k_weight;   /* [D], fp32 or bf16 (weight_bf16 bit 1) */
  const void* inv_freq;   /* [rot / 2], fp32 or fp64 (freq64): radians a position */
  int HQ, rot;            /* rot % 16 == 0, 0 <= rot <= D */
  int weight_bf16, freq64, interleaved;
  float eps, offset;
} lq_rope;
int lq_rope_norm(const lq_rope* r, const lq_pages* p, const lq_batch* b, void* stream);

/* out = sum_j softmax_j(scale q . k_j) v_j over the cached tokens j that a new token at position t sees, t - window < j <= t (window
 * 0: all up to t), times sigmoid(gate) where gate.p is set.  Head h of q reads head h / (HQ / HK) of the cache.  A table entry
 * outside 0 .. NP - 1 reads page 0.  What a token does not see does not reach its output, infinities and NaN among it.  out may
 * be q.  `longest`: new tokens of the longest sequence where the host knows them, 0 where not; it decides on speed only.  `work`:
 * lq_attend_workspace(..) bytes of device memory, 16-byte aligned, whose contents do not matter before and after the call. */
typedef struct lq_attention {
  lq_rows q, gate, out;
  int HQ;
  int window;
  float scale;            /* positive, below 2^127 */
} lq_attention;
int lq_attend(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest, void* work, long long work_bytes,
              void* stream);
/* Bytes of `work`, 0 or more, or a negative lq_status for arguments that lq_attend refuses. */
long long lq_attend_workspace(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest);

#ifdef __cplusplus
}
#endif
#endif /* LQ_ATTN_H */
