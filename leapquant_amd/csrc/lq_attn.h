// Shared helpers of liblq_attn: argument checks, places of tokens in a paged cache.
#pragma once
#include "../../include/lq_attn.h"
#include "lq_common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__attribute__((visibility("hidden"))) int lq_attn_cus();      // compute units of the current GPU

// ---- checks (host) --------------------------------------------------------------------------------------------------
static inline bool rows_ok(const lq_rows& r) { return ((uintptr_t)r.p & 15) == 0 && r.ld % 8 == 0 && r.hd % 8 == 0; }

// no two of T x H vectors of D elements share a place
static inline bool rows_apart(const lq_rows& r, int T, int H, int D) {
  if (T > 1 && r.ld < D) return false;
  if (H > 1 && r.hd < D) return false;
  if (T < 2 || H < 2) return true;
  return r.ld >= r.hd ? r.ld >= (H - 1) * r.hd + D : r.hd >= (T - 1) * r.ld + D;
}

static inline bool pages_ok(const lq_pages* p) {
  if (!p || !p->k || !p->v || p->NP <= 0 || p->page <= 0 || p->page % 16 || p->HK <= 0) return false;
  if (p->D != 64 && p->D != 128 && p->D != 256) return false;
  if (p->int8 != 0 && p->int8 != 1) return false;
  const int unit = p->int8 ? 16 : 8;               // elements of 16 bytes
  if (((uintptr_t)p->k | (uintptr_t)p->v) & 15) return false;
  if (p->page_ld < 0 || p->row_ld < 0 || p->head_ld < 0) return false;
  if (p->page_ld % unit || p->row_ld % unit || p->head_ld % unit) return false;
  const long long far = 1ll << 29;                 // 32-bit byte offsets within a page
  if (p->row_ld >= far || p->head_ld >= far || p->page_ld >= 1ll << 31) return false;
  if ((p->page - 1) * p->row_ld + (p->HK - 1) * p->head_ld + p->D > far) return false;
  if (p->int8) {
    if (!p->k_scale || !p->v_scale || p->s_page_ld < 0 || p->s_row_ld < 0 || p->s_head_ld < 0) return false;
    if (p->s_row_ld >= far || p->s_head_ld >= far) return false;
    if ((p->page - 1) * p->s_row_ld + (p->HK - 1) * p->s_head_ld >= far) return false;
  }
  return true;
}

static inline bool batch_ok(const lq_batch* b, const lq_pages* p) {
  if (!b || b->N < 0 || b->T < 0 || b->width < 0 || (b->N > 0 && (!b->loc || !b->lens))) return false;
  if (b->N > 0 && b->width > 0 && !b->table) return false;
  if (b->N > 1 && b->table_ld < 0) return false;
  return (long long)b->width * p->page < 0x7fffffffll &&
         (unsigned long long)b->width * p->page * (unsigned long long)p->page < (1ull << 40);
}

// ---- a batch (device) -------------------------------------------------------------------------------------------------
// Start of sequence n, held to the packed tokens whatever loc says.
__device__ __forceinline__ int batch_at(const lq_batch& b, int n) { return min(max(b.loc[n], 0), b.T); }
// cached tokens of sequence n, held to what its row of the table has
__device__ __forceinline__ int batch_len(const lq_batch& b, const lq_pages& p, int n) {
  return min(max(b.lens[n], 0), b.width * p.page);
}

// t / page for t < width * page: with t16 = t / 16 and p16 = page / 16, t16 * mul >> 32 is exact where t16 * p16 < 2^32
struct PageDiv {
  uint32_t mul;           // ceil(2^32 / p16), 0: p16 = 1
  uint32_t p16;
};
static inline PageDiv page_div(int page) {
  const uint32_t p16 = (uint32_t)page / 16;
  return {p16 == 1 ? 0u : (uint32_t)((0x100000000ull + p16 - 1) / p16), p16};
}
__device__ __forceinline__ int page_of(const PageDiv& d, int t) {
  const uint32_t t16 = (uint32_t)t >> 4;
  return (int)(d.mul ? __umulhi(t16, d.mul) : t16);
}
