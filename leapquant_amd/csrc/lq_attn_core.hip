// Attention of a ragged batch's new tokens over a paged cache (lq_attend).
//
//   o_r = sum_j e^{s_rj - m_r} v_j / sum_j e^{s_rj - m_r},   s_rj = scale q_r . k_j,   t_r - window < j <= t_r
//
// A row r is a new token and one of the G = HQ / HK heads that read the same head of the cache, numbered token by token, so that
// a key or value is read once for all of them.  One pass over the keys in tiles, with the running maximum m and sum of a row.
//
// A wave forms S^T = K Q^T, keys by rows: a lane then holds scores of one row, its maximum takes one or two lane exchanges, and the weights
// are already laid out as the right operand of O^T = V^T P^T, keys in an order that the transposing reads of V from LDS follow.  m
// moves only when a row's maximum has grown by 2^8 or more: sums and outputs stay in fp32, so that only their common factor
// changes.  Weights are rounded to bf16 for the second product, and their sum is of what was rounded (weigh2).
//
// Two kinds of workgroups: "few" for sequences of up to 16 rows, bound by memory, "many" for tiles of 128 rows, bound by the matrix
// cores and the clock; where a call has both kinds, in one launch.  Keys are split into pieces where the rows do not fill the chip,
// and a second launch joins them.  Tiles go from the pages straight into LDS in places that spread every read over all 64 banks (bank conflicts
// of a prompt of 8192: 7.1e7 -> 3.9e6 cycles).
#include <algorithm>
#include <atomic>

#include "lq_attn.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lds_t;
typedef const __attribute__((address_space(4))) int const_int;     // what no kernel of the call writes: scalar loads

// What a call launches, from what the host knows.
struct Plan {
  int few;                 // rows up to which a sequence is not taken as many
  int few_splits, many_splits;           // pieces of its keys at most
  int tiles;               // row tiles of the sequences of many rows, at most
  int few_blocks, many_blocks;
  int G;
  PageDiv div;
  float *few_work, *many_work;
};

constexpr float GROWN = 8.f;
constexpr float LOG2E = 1.44269504f;

// a value where it is computed: not moved to its use
template <typename T> __device__ __forceinline__ void stay(T& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ u32x4 lds_read16(const char* p) { return *(const u32x4*)p; }
__device__ __forceinline__ u32x2 lds_read_tr(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_t*)p));
}
__device__ __forceinline__ u32x2 lds_read_tr8(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(lds_t*)p));
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 (4) bytes a lane from base + off into LDS at lds + 16 lane (4 lane); the caller waits before it reads them.  The compiler does not see
// what these wait for: M0, written by the scalar unit, one instruction on, and a base that v_readlane wrote, five on.
__device__ __forceinline__ void load16(const char* base, uint32_t off, const char* lds) {
  const unsigned to = (unsigned)(size_t)(const lds_t*)lds;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(to) : "memory", "m0");
}
// N of them, the j-th with an immediate of 1024 j bytes on both its address and its place
template <int N> __device__ __forceinline__ void load16s(const char* base, const uint32_t (&off)[N], const char* lds) {
  static_assert(N == 2 || N == 4, "loads of a wave");          // an immediate has 12 bits
  const unsigned to = (unsigned)(size_t)(const lds_t*)lds;
  if constexpr (N == 2)
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %2, %0\n\tglobal_load_lds_dwordx4 %3, %0 offset:1024"
                 :: "s"(base), "s"(to), "v"(off[0]), "v"(off[1]) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %2, %0\n\tglobal_load_lds_dwordx4 %3, %0 offset:1024\n\t"
                 "global_load_lds_dwordx4 %4, %0 offset:2048\n\tglobal_load_lds_dwordx4 %5, %0 offset:%6"
                 :: "s"(base), "s"(to), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "n"(3 * 1024) : "memory", "m0");
}
__device__ __forceinline__ void load4(const float* from, const char* lds) {
  const unsigned to = (unsigned)(size_t)(const lds_t*)lds;
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(from), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int LEFT> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(LEFT) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// four codes of 8 bits as bf16
__device__ __forceinline__ u32x2 codes(uint32_t w) {
  return u32x2{pk_bf16((float)(int8_t)w, (float)(int8_t)(w >> 8)), pk_bf16((float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24))};
}

// ---- sequences, keys, pieces --------------------------------------------------------------------------------------------
struct Seq {
  int lo, rows, pos0, len;  // first packed token, rows (tokens x G), position of the first new token, cached tokens
};
__device__ __forceinline__ Seq sequence(const lq_batch& b, const lq_pages& p, int G, int n) {
  Seq s;
  s.lo = batch_at(b, n);
  const int nq = max(batch_at(b, n + 1) - s.lo, 0);
  s.len = batch_len(b, p, n);
  s.rows = nq * G;
  s.pos0 = s.len - nq;
  return s;
}

// the first key that position pos sees; pos may lie before 0, and a window be as long as an int
__device__ __forceinline__ int first_key(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }
// keys [lo, hi) that rows [r0, r1) see
struct Keys { int lo, hi; };
__device__ __forceinline__ Keys keys_of(const Seq& s, int G, int r0, int r1, int window) {
  Keys k;
  const int first = s.pos0 + r0 / G, last = s.pos0 + (r1 - 1) / G;
  k.hi = max(last + 1, 0);
  k.lo = first_key(first, window);
  if (k.lo > k.hi) k.lo = k.hi;
  return k;
}
// tiles of KT keys [t0, t1) that piece `split` of a row tile's keys holds, and how many pieces there are
struct Piece { int t0, t1, pieces; };
template <class S> __device__ __forceinline__ Piece piece_of(const Keys& k, int splits, int split) {
  const int a = k.lo / S::KT, b = (k.hi + S::KT - 1) / S::KT, tiles = max(b - a, 0);
  Piece p;
  p.pieces = max(min(splits, tiles / S::LEAST), 1);
  const int per = (tiles + p.pieces - 1) / p.pieces;
  p.pieces = max((tiles + per - 1) / max(per, 1), 1);          // none is empty
  p.t0 = a + split * per;
  p.t1 = min(p.t0 + per, b);
  return p;
}

// ---- 32 keys and the rows of a wave -----------------------------------------------------------------------------------
// R = 32: 32 x 32 x 16 products, R = 16: 16 x 16 x 32.  A lane (group g = lane / R) holds E of 32 scores of the row lane % R: the
// i-th is of key STEP (i / 4) + 4 g + i % 4.  Eight in a row are a right operand of the second product (F of them).
template <int R> struct Rows;
template <> struct Rows<32> {
  typedef f32x16 acc;
  static constexpr int STEP = 8, AN = 16, DM = 32;             // scores of an accumulator, channels of an output
  static __device__ __forceinline__ acc mfma(const u32x4& a, const u32x4& b, const acc& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float max_over(float x) { return xor32_max(x); }
  static __device__ __forceinline__ float sum_over(float x) { return xor32_sum(x); }
};
template <> struct Rows<16> {
  typedef f32x4 acc;
  static constexpr int STEP = 16, AN = 4, DM = 16;
  static __device__ __forceinline__ acc mfma(const u32x4& a, const u32x4& b, const acc& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float max_over(float x) { return xor32_max(xor16_max(x)); }
  static __device__ __forceinline__ float sum_over(float x) { return xor32_sum(xor16_sum(x)); }
};

// What a wave carries along its keys: outputs O^T, a row's running maximum m (of q . k, not scaled) and sum l.
template <int R, int D> struct Run {
  typedef Rows<R> W;
  static constexpr int MB = D / W::DM, AN = W::AN;
  typename W::acc o[MB];
  float m, l, ref;
  bool huge;
  __device__ __forceinline__ void start() {
    m = -INFINITY;
    l = ref = 0.f;
    huge = false;
#pragma unroll
    for (int i = 0; i < MB; ++i) o[i] = typename W::acc(0.f);
  }
  // the largest of some keys' scores
  template <int A> static __device__ __forceinline__ float largest(const typename W::acc (&s)[A]) {
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < A * AN; ++i) mx = fmaxf(mx, s[i / AN][i % AN]);
    return mx;
  }
  // m follows scores whose largest is mx, by steps of 2^GROWN or more
  template <int A> __device__ __forceinline__ void follow(typename W::acc (&s)[A], float mx, float c) {
    mx = W::max_over(mx);
    if (__any((mx - m) * c > GROWN)) {
      const float to = fmaxf(m, mx), alpha = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - to) * c);
      m = to;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        o[i] *= alpha;
        __builtin_amdgcn_sched_barrier(0);                     // few at a time outside the accumulators' registers
      }
      // s c - ref is rounded once, but ref = m c itself is off by half its last place, which 2^ref would be too much for beyond 2^24
      huge = __any(fabsf(m * c) > 0x1p24f && m != -INFINITY);
      ref = huge || m == -INFINITY ? 0.f : m * c;
    }
    if (huge) {
      const float raw = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < A * AN; ++i) s[i / AN][i % AN] -= raw;
    }
  }
  // Of one accumulator, whose i-th score is of key STEP (i / 4) + i % 4: keys lo .. hi are seen, the others' become `none`.
  static __device__ __forceinline__ void mask(typename W::acc& s, int lo, int hi, float none) {
    asm volatile("" : "+v"(lo), "+v"(hi));                     // a branch of its own, not selects for every tile
#pragma unroll
    for (int i = 0; i < AN; ++i) {
      const int j = W::STEP * (i >> 2) + (i & 3);
      s[i] = j >= lo && j <= hi ? s[i] : none;
    }
  }
  // times the scales of its keys
  static __device__ __forceinline__ void times(typename W::acc& s, const float* scale) {
#pragma unroll
    for (int i = 0; i < AN; i += 4) {
      const f32x4 x = *(const f32x4*)(scale + W::STEP * (i >> 2));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i + e] *= x[e];
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Two weights as bf16 for the second product, codes' with the scales vs of their values.  Their sum l is of what was rounded: a key that
// outweighs the others then has no error left, two alike half of it (against 64 bits, 64 sequences up to 8192 from codes: 0.0024 -> 0.0017,
// which is the outputs' own rounding).  With scales, a rounded product is taken back through 1 / vs, `by`; where the scale is zero, not
// finite or far from one, so that a product or 1 / vs could leave the range of fp32, the weight itself counts (`by` 0).  Products below
// the smallest number are weights below 1e-19 then, of sums of 2^-8 or more.
__device__ __forceinline__ float inverse(float vs) { return fabsf(vs) > 1e-18f && fabsf(vs) < 1e18f ? __builtin_amdgcn_rcpf(vs) : 0.f; }
template <bool I8> __device__ __forceinline__ uint32_t weigh2(float a, float b, float va, float vb, float bya, float byb, float& l) {
  if constexpr (I8) {
    const uint32_t w = pk_bf16(a * va, b * vb);
    const float wa = bf_lo(w), wb = bf_hi(w);
    l += bya != 0.f ? wa * bya : a;
    l += byb != 0.f ? wb * byb : b;
    return w;
  } else {
    const uint32_t w = pk_bf16(a, b);
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2, w), s16x2{0x3f80, 0x3f80}, l, false);
    return w;
  }
}

// whether 32 rows of D bf16 in LDS hold an infinity or NaN
template <int D> __device__ __forceinline__ bool tile_not_finite(const char* tile) {
  const int lane = threadIdx.x & 63;
  uint32_t hit = 0;
#pragma unroll 2
  for (int i = 0; i < D / 16; ++i) {
    const u32x4 w = lds_read16(tile + (lane & 31) * 2 * D + 16 * ((lane >> 5) + 2 * i));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = (w[e] & 0x7f807f80u) ^ 0x7f807f80u;   // a half of zero: an exponent of ones
      hit |= (x - 0x00010001u) & ~x & 0x80008000u;
    }
  }
  return __any(hit != 0);
}

__device__ __forceinline__ bool scales_not_finite(const float* scale) {
  return __any(!(fabsf(scale[threadIdx.x & 31]) < INFINITY));
}

// Rows [ra, rb) of a sequence again, key by key: for a wave that met values (or scales of them) which are not finite in a tile that not
// all of its rows see.  The products give a key that a row does not see a probability of zero, and zero times an infinity or NaN is
// not zero.  Keys are those of the wave, 32 u .. 32 u + 31 for u = u0, u0 + step .. < u1.  sink(row, m, l, y): channels D / 64
// lane .. of a row.
template <int D, bool I8, class F>
__device__ __forceinline__ void rows_again(const lq_attention& a, const lq_pages& pg, const lq_batch& b, const Plan& pl, int n, int hk,
                                           const Seq& sq, int ra, int rb, int u0, int u1, int step, const F& sink) {
  constexpr int C = D / 64;
  const int lane = threadIdx.x & 63, tend = max(sq.len - 1, 0);
  const float c = a.scale * LOG2E;
  for (int r = ra; r < rb; ++r) {
    const int tok = r / pl.G, pos = sq.pos0 + tok, from = first_key(pos, a.window);
    const bf16_t* q = (const bf16_t*)a.q.p + (long long)(sq.lo + tok) * a.q.ld + (long long)(hk * pl.G + r - tok * pl.G) * a.q.hd;
    float m = -INFINITY, l = 0.f, y[C] = {};
#pragma unroll 1
    for (int u = u0; u < u1; u += step) {
      if (32 * u > pos || 32 * u + 31 < from) continue;
      const int key = 32 * u + (lane & 31), kk = min(key, tend), pi = page_of(pl.div, kk);
      const bool sees = lane < 32 && key >= from && key <= pos;
      int page = b.table[(long long)n * b.table_ld + pi];
      page = page >= 0 && page < pg.NP ? page : 0;
      const long long at = (long long)page * pg.page_ld + (long long)(kk - pi * pg.page) * pg.row_ld + (long long)hk * pg.head_ld;
      float s = 0.f;
#pragma unroll 1
      for (int i = 0; i < D; i += 8) {
        const u32x4 x = *(const u32x4*)(q + i);
        u32x4 k;
        if constexpr (I8) {
          const u32x2 w = *(const u32x2*)((const int8_t*)pg.k + at + i), k0 = codes(w[0]), k1 = codes(w[1]);
          k = u32x4{k0[0], k0[1], k1[0], k1[1]};
        } else {
          k = *(const u32x4*)((const bf16_t*)pg.k + at + i);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fmaf(bf_hi(x[e]), bf_hi(k[e]), fmaf(bf_lo(x[e]), bf_lo(k[e]), s));
      }
      float vs = 1.f;
      if constexpr (I8) {
        const long long x = (long long)page * pg.s_page_ld + (long long)(kk - pi * pg.page) * pg.s_row_ld + (long long)hk * pg.s_head_ld;
        s *= pg.k_scale[x];
        vs = pg.v_scale[x];
      }
      if (!sees) s = -INFINITY;
      const float to = fmaxf(m, max64(s)), raw = to == -INFINITY ? 0.f : to;
      const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - raw) * c);
      const float p = sees ? __builtin_amdgcn_exp2f((s - raw) * c) : 0.f;
      m = to;
      l = fmaf(l, alpha, sum64(p));
#pragma unroll
      for (int e = 0; e < C; ++e) y[e] *= alpha;
#pragma unroll 1
      for (int j = 0; j < 32; ++j) {
        if (32 * u + j < from || 32 * u + j > pos) continue;
        const float pj = __shfl(p, j) * __shfl(vs, j);
        const long long vj = __shfl(at, j);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const long long x = vj + C * lane + e;
          y[e] = fmaf(pj, I8 ? (float)((const int8_t*)pg.v)[x] : bf2f(((const bf16_t*)pg.v)[x]), y[e]);
        }
      }
    }
    sink(r, m, l, y);
  }
}

// ---- outputs ----------------------------------------------------------------------------------------------------------------
// sigmoid(gate) of 4 neighbours
__device__ __forceinline__ f32x4 gate4(const lq_rows& gate, long long token, int head, int d) {
  const u32x2 w = *(const u32x2*)((const bf16_t*)gate.p + token * gate.ld + (long long)head * gate.hd + d);
  const f32x4 z = {bf_lo(w[0]), bf_hi(w[0]), bf_lo(w[1]), bf_hi(w[1])};
  f32x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = __builtin_amdgcn_rcpf(1.0f + __expf(-z[e]));
  return y;
}
// An output at position pos.  Before 0 the row sees nothing: y is zero, and stays so whatever the gate of such a row holds.
__device__ __forceinline__ void store4(const lq_attention& a, long long token, int pos, int head, int d, f32x4 y) {
  if (a.gate.p && pos >= 0) y *= gate4(a.gate, token, head, d);
  *(u32x2*)((bf16_t*)a.out.p + token * a.out.ld + (long long)head * a.out.hd + d) = u32x2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
}

__device__ __forceinline__ void store1(const lq_attention& a, long long token, int pos, int head, int d, float y) {
  if (a.gate.p && pos >= 0) y *= __builtin_amdgcn_rcpf(1.0f + __expf(-bf2f(((const bf16_t*)a.gate.p)[token * a.gate.ld + (long long)head * a.gate.hd + d])));
  ((bf16_t*)a.out.p)[token * a.out.ld + (long long)head * a.out.hd + d] = f2bf(y);
}

// ---- few rows -----------------------------------------------------------------------------------------------------------------
// Up to 16 rows of a sequence (a token's heads): a wave takes all of them, the KW waves of a workgroup every KW-th tile of 32 keys,
// each by itself: K and V of a tile have a place in LDS each, and the next tile's are asked for as soon as this one's are used, so
// that 32 D .. 64 D elements a wave are on their way at any time.  Codes stay codes in LDS.
//
// Measured (MI355X): 64 sequences up to 8192 of 8 heads of 128 256 us, 5.2 TB/s, a large copy's rate (reads alone reach 6.3 by plain
// loads, 7.2 by nontemporal ones); from codes 168 us, 4.1 TB/s, beside the conversion of the codes.  One sequence of 8192, 2 heads of
// 256: 10 us and 5 for the join, chains of loads.  Workgroups of 32 or 64 rows of this kind lose to tiles of many rows (32 sequences of up to 64 rows, 2 heads of 256,
// 75 us against 58; one of 48 rows over 16384, 8 heads of 128, 44 against 23): their queries no longer fit beside the outputs, and one wave a SIMD shows every wait.
template <int D_, int KW_, bool I8_> struct Few {
  static constexpr int D = D_, KW = KW_, R = 16, ROWS = 16, KT = 32, LEAST = KW, THREADS = 64 * KW;
  static constexpr bool I8 = I8_;
  static constexpr int ES = I8 ? 1 : 2, RB = D * ES, CPR = RB / 16, RPL = 64 / CPR;  // bytes and chunks of a row, rows of a load
  static constexpr int UNIT = KT * RB, LOADS = UNIT / 1024, SC = I8 ? 1 : 0;
  static constexpr int WAVE = 2 * UNIT + SC * 512;             // K, V, the scales of two tiles
  static constexpr int JOIN = KW * ROWS * ((D + 4) * 4 + 8);
  static constexpr int LDS = KW * WAVE > JOIN ? KW * WAVE : JOIN;
  static constexpr int PART = ROWS * (D + 2);                  // floats of a workgroup's part of split keys
  // A chunk's place in its row, so that 256 bytes of the reads below go over all banks: 16 keys by a chunk of K; 8 keys by two chunks
  // of V, or, codes, 16 keys (of which 8 neighbours and those 16 on) by one.
  static constexpr int SPAN = CPR >= 16 ? 1 : 16 / CPR;        // rows of 256 bytes
  static __device__ __forceinline__ int place_k(int key) { return key / SPAN & (16 / SPAN - 1); }
  static __device__ __forceinline__ int place_v(int key) {
    return I8 ? ((key & 7) | (key >> 4 & 1) << 3) / SPAN : ((key & 7) / SPAN) << 1;
  }
};

template <class S>
__device__ __forceinline__ void few_rows(const lq_attention& a, const lq_pages& pg, const lq_batch& b, const Plan& pl, char* lds, int n,
                                         int hk, int split, int splits, int r0, const Seq& sq, float* part) {
  constexpr int D = S::D, KW = S::KW, MB = D / 16, KS = D / 32;
  const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int G = pl.G, rows = min(S::ROWS, sq.rows - r0);
  const Piece piece = piece_of<S>(keys_of(sq, G, r0, r0 + rows, a.window), splits, split);
  if (split >= piece.pieces) return;
  const int rc = r0 + min(col, rows - 1), tok = rc / G, pos = sq.pos0 + tok;
  const int from = first_key(pos, a.window);              // keys from .. pos are seen
  const int first = sq.pos0 + r0 / G, last = sq.pos0 + (r0 + rows - 1) / G;    // all rows see full .. first
  const int full = first_key(last, a.window);

  char* const mine = lds + kw * S::WAVE;
  const int* tab = b.table + (long long)n * b.table_ld;
  const int tend = max(sq.len - 1, 0);
  const char *at[2], *vat = (const char*)((const char*)pg.v - (const char*)pg.k);
  int most[2], pages[2], in[2];
  auto places = [&](int t) {                                   // where the two halves of tile t lie
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int kg = min(t * 32 + 16 * i, tend & ~15), pi = __builtin_amdgcn_readfirstlane(page_of(pl.div, kg));
      int page = ((const_int*)tab)[pi];
      page = page >= 0 && page < pg.NP ? page : 0;
      pages[i] = page;
      in[i] = kg - pi * pg.page;
      at[i] = (const char*)pg.k + ((long long)page * pg.page_ld + (long long)in[i] * pg.row_ld + (long long)hk * pg.head_ld) * S::ES;
      most[i] = tend - kg;
    }
  };
  const uint32_t row_bytes = (uint32_t)pg.row_ld * S::ES;
  auto ask = [&](bool values) {                                // for K or V of the tile that places() found
#pragma unroll
    for (int j = 0; j < S::LOADS; ++j) {
      const int key = S::RPL * j + lane / S::CPR, i = 2 * j / S::LOADS;
      const uint32_t off = (uint32_t)min(key - 16 * i, most[i]) * row_bytes + 16 * ((lane % S::CPR) ^ (values ? S::place_v(key) : S::place_k(key)));
      load16(at[i] + (values ? (size_t)vat : 0), off, mine + (values ? S::UNIT : 0) + 1024 * j);
    }
  };
  auto ask_scales = [&](int odd) {                             // lanes 0 .. 31: of the keys, 32 .. 63: of the values
    if constexpr (S::I8) {
      const int p0 = pages[0], p1 = pages[1], i0 = in[0], i1 = in[1], m0 = most[0], m1 = most[1];
      const bool far = lane & 16;
      const int row = (far ? i1 : i0) + min(lane & 15, far ? m1 : m0);
      const long long x = (long long)(far ? p1 : p0) * pg.s_page_ld + (long long)row * pg.s_row_ld + (long long)hk * pg.s_head_ld;
      load4((lane < 32 ? pg.k_scale : pg.v_scale) + x, mine + 2 * S::UNIT + 256 * odd);
    }
  };

  const float c = a.scale * LOG2E;
  Run<16, D> run;
  run.start();
  bool poisoned = false;
  int t = piece.t0 + kw;
  if (t < piece.t1) {
    u32x4 q[KS];
    {
      const bf16_t* p = (const bf16_t*)a.q.p + (long long)(sq.lo + tok) * a.q.ld + (long long)(hk * G + rc - tok * G) * a.q.hd + 8 * g;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = *(const u32x4*)(p + 32 * s);
    }
    places(t);
    ask_scales(0);
    ask(false);
    ask(true);
#pragma unroll
    for (int s = 0; s < KS; ++s) stay(q[s]);                   // here now: the loop must not wait for them, nor for what it asks for
    // this lane's reads: 8 channels of two keys; 4 (8) keys by 16 channels a group of 16 lanes
    const int kread = col * S::RB + (S::I8 ? ((g >> 1) ^ S::place_k(col)) * 16 + 8 * (g & 1) : (g ^ S::place_k(col)) * 16);
    const int vkey = S::I8 ? 4 * g + ((lane & 15) >> 1 & 3) + 16 * ((lane & 15) >> 3) : 4 * g + ((lane & 15) >> 2);
    const int vread = vkey * S::RB + (S::I8 ? S::place_v(vkey) * 16 + 8 * (lane & 1) : (((lane & 3) >> 1) ^ S::place_v(vkey)) * 16 + 8 * (lane & 1));
    for (int odd = 0; t < piece.t1; t += KW, odd ^= 1) {
      const bool more = t + KW < piece.t1;
      const float* sc = (const float*)(mine + 2 * S::UNIT + 256 * odd) + 4 * g;
      if (more) places(t + KW);
      wait_loads<S::LOADS>();                                  // K is here, V may be on its way
      f32x4 s[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[x] = f32x4(0.f);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          u32x4 k;
          if constexpr (S::I8) {
            const u32x2 w = *(const u32x2*)(mine + 16 * x * S::RB + (kread ^ (32 * i)));
            const u32x2 y = codes(w[0]), z = codes(w[1]);
            k = u32x4{y[0], y[1], z[0], z[1]};
          } else {
            k = lds_read16(mine + 16 * x * S::RB + (kread ^ (64 * i)));
          }
          s[x] = Rows<16>::mfma(k, q[i], s[x]);
        }
      }
      if constexpr (S::I8) {
#pragma unroll
        for (int x = 0; x < 2; ++x) run.times(s[x], sc + 16 * x);
      }
      if (more) {
        wait_lds();
        ask_scales(odd ^ 1);
        ask(false);
      }
      const int k0 = 32 * t;
      const bool masked = k0 + 31 > first || k0 < full;
      if (masked) {
#pragma unroll
        for (int x = 0; x < 2; ++x) run.mask(s[x], from - k0 - 16 * x - 4 * g, pos - k0 - 16 * x - 4 * g, -INFINITY);
      }
      run.follow(s, run.largest(s), c);
      u32x4 p;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[x][e] = __builtin_amdgcn_exp2f(fmaf(s[x][e], c, -run.ref));
        }
        f32x4 vs = f32x4(1.f), by = f32x4(1.f);
        if constexpr (S::I8) {
          vs = *(const f32x4*)(sc + 32 + 16 * x);
#pragma unroll
          for (int e = 0; e < 4; ++e) by[e] = inverse(vs[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2) p[2 * x + e / 2] = weigh2<S::I8>(s[x][e], s[x][e + 1], vs[e], vs[e + 1], by[e], by[e + 1], run.l);
      }
      if (more) wait_loads<S::LOADS + S::SC>();                // V is here
      else wait_loads<0>();
      const char* V = mine + S::UNIT;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        u32x4 v;
        if constexpr (S::I8) {
          const u32x2 w = lds_read_tr8(V + (vread ^ (16 * i)));
          const u32x2 y = codes(w[0]), z = codes(w[1]);
          v = u32x4{y[0], y[1], z[0], z[1]};
        } else {
          const u32x2 x = lds_read_tr(V + (vread ^ (32 * i))), y = lds_read_tr(V + 16 * S::RB + (vread ^ (32 * i)));
          v = u32x4{x[0], x[1], y[0], y[1]};
        }
        run.o[i] = Rows<16>::mfma(v, p, run.o[i]);
      }
      if (masked) poisoned |= S::I8 ? scales_not_finite(sc - 4 * g + 32) : tile_not_finite<D>(V);
      if (more) {
        wait_lds();
        ask(true);
      }
    }
    run.l = Rows<16>::sum_over(run.l);
  }

  // the waves' parts of a row, joined through LDS
  float* jo = (float*)lds;                                     // [KW][ROWS][D + 4]
  float* jm = jo + KW * S::ROWS * (D + 4);                     // [KW][ROWS] maxima, then sums
  __syncthreads();
  if (!poisoned) {
    float* to = jo + (kw * S::ROWS + col) * (D + 4) + 4 * g;
#pragma unroll
    for (int i = 0; i < MB; ++i) *(f32x4*)(to + 16 * i) = run.o[i];
    if (g == 0) { jm[kw * S::ROWS + col] = run.m; jm[(KW + kw) * S::ROWS + col] = run.l; }
  } else {
    rows_again<D, S::I8>(a, pg, b, pl, n, hk, sq, r0, r0 + rows, piece.t0 + kw, piece.t1, KW, [&](int r, float m, float l, const float* y) {
      constexpr int C = D / 64;
#pragma unroll
      for (int e = 0; e < C; ++e) jo[(kw * S::ROWS + r - r0) * (D + 4) + C * lane + e] = y[e];
      if (lane == 0) { jm[kw * S::ROWS + r - r0] = m; jm[(KW + kw) * S::ROWS + r - r0] = l; }
    });
  }
  __syncthreads();
  for (int x = threadIdx.x; x < rows * (D / 4); x += S::THREADS) {
    const int rr = x / (D / 4), d = 4 * (x % (D / 4));
    float M = -INFINITY, L = 0.f;
    f32x4 y = f32x4(0.f);
#pragma unroll
    for (int k = 0; k < KW; ++k) M = fmaxf(M, jm[k * S::ROWS + rr]);
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const float mk = jm[k * S::ROWS + rr], w = mk == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mk - M) * c);
      L = fmaf(w, jm[(KW + k) * S::ROWS + rr], L);             // a wave without a maximum: zeros, or NaN
      y += w * *(const f32x4*)(jo + (k * S::ROWS + rr) * (D + 4) + d);
    }
    if (piece.pieces > 1) {
      *(f32x4*)(part + rr * D + d) = y;
      if (d == 0) { part[S::ROWS * D + rr] = M; part[S::ROWS * (D + 1) + rr] = L; }
      continue;
    }
    const int tk = (r0 + rr) / G;
    store4(a, sq.lo + tk, sq.pos0 + tk, hk * G + (r0 + rr - tk * G), d, y * (L == 0.f ? 0.f : 1.f / L));
  }
}

// workgroup `block` = (split, sequence, head)
template <class S>
__device__ __forceinline__ void few_block(const lq_attention& a, const lq_pages& pg, const lq_batch& b, const Plan& pl, char* lds, int block) {
  const int items = b.N * pg.HK, item = block % items, split = block / items, n = item / pg.HK, hk = item % pg.HK;
  const Seq sq = sequence(b, pg, pl.G, n);
  if (sq.rows <= 0 || (pl.many_blocks && sq.rows > S::ROWS)) return;
  // more rows than a tile has, where nobody else takes them: one workgroup all of them, a tile after the other
  const int splits = sq.rows > S::ROWS ? 1 : pl.few_splits;
  for (int r0 = 0; r0 < sq.rows; r0 += S::ROWS) {
    few_rows<S>(a, pg, b, pl, lds, n, hk, split, splits, r0, sq, pl.few_work + (long long)block * S::PART);
    __syncthreads();
  }
}
template <class S>
__global__ __launch_bounds__(S::THREADS) void few_kernel(lq_attention a, lq_pages pg, lq_batch b, Plan pl) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  few_block<S>(a, pg, b, pl, lds, blockIdx.x);
}

// ---- many rows ------------------------------------------------------------------------------------------------------------
// RW waves of 32 rows each share tiles of KT keys, K and V twice in LDS, K a tile ahead of V.  A wave forms the scores of a tile while it
// takes the exponentials of the one before, and looks for their maximum while that one meets its values, so that its vector
// instructions go in the shadow of its matrix instructions.  What bounds it then is the number of a wave's instructions.
// Codes go through registers and into LDS as bf16, which holds them exactly; scales enter S and P in fp32.
//
// Measured (MI355X): a prompt of 8192, 32 / 8 heads of 128, 520 .. 535 us, 1.03 .. 1.06 PFLOP/s (a large product by the library 1.31): its clock falls to
// 1.5 .. 1.95 GHz; a piece of 2048 over 32768, 16 / 2 heads of 256, 1095 .. 1120 us, 0.95 .. 0.97 PFLOP/s, one wave a SIMD; 4096 tokens of 32 / 8
// of 128 145 us, from codes 257.  Without the order of instructions below 584 and 2184; without queries waited for before the loop 573 and 1344.
template <int D_, int RW_, int KT_, int EU_, bool I8_> struct Many {
  static constexpr int D = D_, RW = RW_, EU = EU_, KT = KT_, X = KT / 32, LEAST = 512 / KT, R = 32, ROWS = 32 * RW, THREADS = 64 * RW;
  static constexpr bool I8 = I8_;
  static constexpr int RB = 2 * D, TILE = KT * RB;             // bytes in LDS
  static constexpr int K0 = 0, V0 = 2 * TILE, SCALES = 4 * TILE, LDS = SCALES + (I8 ? 6 * KT * 4 : 0);          // scales of K and of V twice, the inverses of V's
  static constexpr int PART = ROWS * (D + 2);
  static constexpr int AHEAD = D == 256 ? 6 : 4;               // operands on their way: registers
  static constexpr int OWN = KT / RW;                          // keys of a tile that a wave loads, all of one page
  static_assert(OWN <= 16, "keys of one page");
  // as Few's: 16 keys by a chunk of K, 4 keys by four chunks of V
  static constexpr int SPAN = D == 64 ? 2 : 1;
  static __device__ __forceinline__ int place_k(int key) { return key / SPAN & (16 / SPAN - 1); }
  static __device__ __forceinline__ int place_v(int key) { return (key & 3) / SPAN << 2; }
};

// A wave's keys of the tiles, one tile after the other: where they lie, and on their way into LDS.
template <class S> struct Tiles {
  static constexpr int D = S::D, KT = S::KT, OWN = S::OWN, ES = S::I8 ? 1 : 2, CPR = D * ES / 16, RPL = 64 / CPR;
  static constexpr int LOADS = OWN / RPL > 0 ? OWN / RPL : 1;
  static_assert(S::I8 || OWN % RPL == 0, "a load of a whole wave");
  // The j-th load's immediate, 1024 j, moves its place in LDS and its address: the offsets are that much less, and, so that none is
  // below 0, the bases 4096 less.
  static constexpr int LESS = S::I8 ? 0 : 4096;
  const_int* tab;
  const char* kbase;
  long long vfar;
  uint32_t row_bytes, page_bytes;
  int rw, lane, hk, tend, end, whole, rest;
  uint32_t koff[LOADS], voff[LOADS];                           // where this lane's chunks come from, so that they lie swizzled
  int key, entry, in;                                          // the next tile's: in `entry` of the table's row, at place `in` of its page
  struct From { const char* k; int most, page, in; };          // addresses, and the last cached token, of a tile
  u32x4 kreg[S::I8 ? LOADS : 1], vreg[S::I8 ? LOADS : 1];
  float ksc, vsc;

  __device__ __forceinline__ void at(const lq_pages& pg, const PageDiv& div, int k) {
    key = min(k, end);
    entry = __builtin_amdgcn_readfirstlane(page_of(div, key));
    in = key - entry * pg.page;
  }
  __device__ __forceinline__ void start(const lq_pages& pg, const lq_batch& b, const PageDiv& div, int n, int hk_, int rw_, int last, int t0) {
    rw = rw_;
    hk = hk_;
    lane = threadIdx.x & 63;
    tab = (const_int*)(b.table + (long long)n * b.table_ld);
    tend = last;
    end = last & ~(OWN - 1);
    whole = KT / pg.page;
    rest = KT - whole * pg.page;
    kbase = (const char*)pg.k + (long long)hk * pg.head_ld * ES - LESS;
    vfar = (const char*)pg.v - (const char*)pg.k;
    row_bytes = (uint32_t)pg.row_ld * ES;
    page_bytes = (uint32_t)pg.page_ld * ES;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int k = min(RPL * j + lane / CPR, OWN - 1), tk = rw * OWN + k;
      const uint32_t off = (uint32_t)k * row_bytes + LESS - (S::I8 ? 0 : 1024 * j);
      koff[j] = off + 16 * (S::I8 ? lane % CPR : (lane % CPR) ^ S::place_k(tk));
      voff[j] = off + 16 * (S::I8 ? lane % CPR : (lane % CPR) ^ S::place_v(tk));
    }
    at(pg, div, t0 * KT + rw * OWN);
  }
  __device__ __forceinline__ void step(const lq_pages& pg, const PageDiv& div) {
    if (key + KT > end) {                                      // the last cached tokens, once and again
      at(pg, div, end);
    } else {
      key += KT;
      entry += whole;
      in += rest;
      if (in >= pg.page) { in -= pg.page; ++entry; }
    }
  }
  __device__ __forceinline__ int page() const { return tab[entry]; }
  __device__ __forceinline__ From where(const lq_pages& pg, int page) const {
    page = (unsigned)page < (unsigned)pg.NP ? page : 0;
    return {kbase + (unsigned long long)(uint32_t)page * page_bytes + (uint32_t)in * row_bytes, tend - key, page, in};
  }
  __device__ __forceinline__ void ask(const lq_pages& pg, const From& f, bool values, char* to) {
    uint32_t off[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) off[j] = values ? voff[j] : koff[j];
    if (f.most < OWN - 1) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int k = min(RPL * j + lane / CPR, OWN - 1);
        off[j] -= (uint32_t)(k - min(k, f.most)) * row_bytes;
      }
    }
    const char* from = values ? f.k + vfar : f.k;
    if constexpr (S::I8) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) (values ? vreg : kreg)[j] = *(const u32x4*)(from + off[j]);
      const long long x = (long long)f.page * pg.s_page_ld + (long long)(f.in + min(min(lane, OWN - 1), f.most)) * pg.s_row_ld + (long long)hk * pg.s_head_ld;
      if (values) vsc = pg.v_scale[x];
      else ksc = pg.k_scale[x];
    } else {
      load16s<LOADS>(from, off, to + rw * OWN * S::RB);
    }
  }
  // codes in registers -> bf16 in LDS
  __device__ __forceinline__ void settle(bool values, char* to, float* scale) const {
    if constexpr (S::I8) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int k = RPL * j + lane / CPR, tk = rw * OWN + k, ch = 2 * (lane % CPR), place = values ? S::place_v(tk) : S::place_k(tk);
        if (k < OWN) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const u32x4& w = (values ? vreg : kreg)[j];
            const u32x2 c0 = codes(w[2 * y]), c1 = codes(w[2 * y + 1]);
            *(u32x4*)(to + tk * S::RB + 16 * ((ch + y) ^ place)) = u32x4{c0[0], c0[1], c1[0], c1[1]};
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      if (lane < OWN) scale[rw * OWN + lane] = values ? vsc : ksc;
      if (values && lane < OWN) scale[2 * KT + rw * OWN + lane] = inverse(vsc);
    }
  }
};

template <class S>
__device__ __forceinline__ void many_rows(const lq_attention& a, const lq_pages& pg, const lq_batch& b, const Plan& pl, char* lds, int n,
                                          int hk, int split, int r0, const Seq& sq, float* part) {
  constexpr int D = S::D, KT = S::KT, X = S::X, KS = D / 16, MB = D / 32;
  const int rw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
  const int G = pl.G, rows = min(S::ROWS, sq.rows - r0);
  const Piece piece = piece_of<S>(keys_of(sq, G, r0, r0 + rows, a.window), pl.many_splits, split);
  if (split >= piece.pieces) return;
  const int row = r0 + 32 * rw + col, rc = min(row, r0 + rows - 1), tok = rc / G, pos = sq.pos0 + tok, head = hk * G + rc - tok * G;
  const bool busy = 32 * rw < rows;                            // the wave has rows
  const int first = sq.pos0 + min(r0 + 32 * rw, r0 + rows - 1) / G, last = sq.pos0 + (min(r0 + 32 * rw + 32, r0 + rows) - 1) / G;
  const int from = first_key(pos, a.window);               // keys from .. pos are seen
  const int full = first_key(last, a.window);              // all rows of the wave see full .. first
  u32x4 q[KS];
  {
    const bf16_t* p = (const bf16_t*)a.q.p + (long long)(sq.lo + tok) * a.q.ld + (long long)head * a.q.hd + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = *(const u32x4*)(p + 16 * s);
  }
  const float c = a.scale * LOG2E;
  typedef Run<32, D> Carry;
  Carry run;
  run.start();
  bool poisoned = false;

  // this lane's reads: a row of K; 4 keys by 16 channels a group of 16 lanes of V
  const int kread = col * S::RB + 16 * (g ^ S::place_k(col));
  const int vkey = 4 * g + ((lane & 15) >> 2);
  const int vread = vkey * S::RB + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ S::place_v(vkey)) + 8 * (lane & 1);
  const char *kat[KS], *vat[MB];
#pragma unroll
  for (int j = 0; j < KS; ++j) kat[j] = lds + S::K0 + (kread ^ (32 * j));
#pragma unroll
  for (int j = 0; j < MB; ++j) vat[j] = lds + S::V0 + (vread ^ (64 * j));
  constexpr int NK = X * KS, NV = 2 * X * MB;                      // operands of a tile: the j-th of
  auto keys = [&](int buf, int j) { return lds_read16(kat[j % KS] + buf * S::TILE + j / KS * 32 * S::RB); };   // 32 keys by 16 channels
  auto values = [&](int buf, int j) {                                                                       // 32 channels by 16 keys
    const char* at = vat[j % MB] + buf * S::TILE + j / MB * 16 * S::RB;
    const u32x2 y = lds_read_tr(at), z = lds_read_tr(at + 8 * S::RB);
    return u32x4{y[0], y[1], z[0], z[1]};
  };
  auto scale_at = [&](bool values, int buf) { return (const float*)(lds + S::SCALES) + KT * (2 * values + buf) + 4 * g; };
  auto masked = [&](int t) { return t * KT + KT - 1 > first || t * KT < full; };
  auto adjust = [&](int t, int buf, f32x16 (&s)[X]) {          // scores of tile t
#pragma unroll
    for (int x = 0; x < X; ++x) {
      if constexpr (S::I8) Carry::times(s[x], scale_at(false, buf) + 32 * x);
      if (masked(t)) Carry::mask(s[x], from - t * KT - 32 * x - 4 * g, pos - t * KT - 32 * x - 4 * g, -INFINITY);
    }
  };

  // The order of what follows is kept as written (nothing moves over a sched_barrier): a matrix instruction with its share of vector
  // instructions, and the operand of the one AHEAD of it.  Weights go in pairs: the product in the exponent of one beside
  // the exponentials of the one before, and the rounding and the sum (of what was rounded) of the one before that.
  constexpr int PAIRS = 8 * X, EARLY = X == 1 ? 5 : 4 * X;      // of a tile; those beside the next scores, with all four of the first operand
  float ex[2], old[2], vs[2], by[2];
  uint32_t w[PAIRS];
  auto exponent = [&](const f32x16 (&s)[X], int i) {
#pragma unroll
    for (int e = 0; e < 2; ++e) { ex[e] = fmaf(s[i >> 3][2 * (i & 7) + e], c, -run.ref); stay(ex[e]); }
  };
  auto finish = [&](int i) {
    if constexpr (S::I8) w[i] = weigh2<true>(old[0], old[1], vs[0], vs[1], by[0], by[1], run.l);
    else w[i] = weigh2<false>(old[0], old[1], 1.f, 1.f, 1.f, 1.f, run.l);
    stay(w[i]);
  };
  auto weigh = [&](const f32x16 (&s)[X], int buf, int lo, int hi) {            // pairs lo .. hi - 1; exponents of lo are there
#pragma unroll
    for (int i = lo; i < hi; ++i) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) { f[e] = __builtin_amdgcn_exp2f(ex[e]); stay(f[e]); }
      if (i + 1 < PAIRS) exponent(s, i + 1);
      if (i > 0) finish(i - 1);
#pragma unroll
      for (int e = 0; e < 2; ++e) old[e] = f[e];
      if constexpr (S::I8) {
        const f32x2 x = *(const f32x2*)(scale_at(true, buf) + 32 * (i >> 3) + 8 * ((i & 7) >> 1) + 2 * (i & 1));
        const f32x2 y = *(const f32x2*)(scale_at(true, buf) + 2 * KT + 32 * (i >> 3) + 8 * ((i & 7) >> 1) + 2 * (i & 1));
#pragma unroll
        for (int e = 0; e < 2; ++e) { vs[e] = x[e]; by[e] = y[e]; }
      }
    }
  };
  auto scores_and_weigh = [&](int kbuf, int vbuf, f32x16 (&next)[X], const f32x16 (&s)[X]) {
    u32x4 k[NK];
#pragma unroll
    for (int j = 0; j < S::AHEAD; ++j) k[j] = keys(kbuf, j);
    exponent(s, 0);
#pragma unroll
    for (int x = 0; x < X; ++x) next[x] = f32x16(0.f);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      if (j + S::AHEAD < NK) k[j + S::AHEAD] = keys(kbuf, j + S::AHEAD);
      next[j / KS] = Rows<32>::mfma(k[j], q[j % KS], next[j / KS]);
      weigh(s, vbuf, EARLY * j / NK, EARLY * (j + 1) / NK);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto meet_and_largest = [&](int vbuf, const f32x16 (&s)[X], const f32x16 (&next)[X]) {
    u32x4 v[NV];
    float mx = next[0][0];
#pragma unroll
    for (int j = 0; j < S::AHEAD; ++j) v[j] = values(vbuf, j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j + S::AHEAD < NV) v[j + S::AHEAD] = values(vbuf, j + S::AHEAD);
      // the weights of the 16 keys j / MB are there: the last pairs by the middle of the values, and a pair behind
      const u32x4 p = {w[4 * (j / MB)], w[4 * (j / MB) + 1], w[4 * (j / MB) + 2], w[4 * (j / MB) + 3]};
      run.o[j % MB] = Rows<32>::mfma(v[j], p, run.o[j % MB]);
      constexpr int H = NV / 2;
      if (j < H) {
        weigh(s, vbuf, EARLY + (PAIRS - EARLY) * j / H, EARLY + (PAIRS - EARLY) * (j + 1) / H);
        if (j == H - 1) finish(PAIRS - 1);
      } else {
#pragma unroll
        for (int e = 16 * X * (j - H) / H; e < 16 * X * (j + 1 - H) / H; ++e) mx = fmaxf(mx, next[e >> 4][e & 15]);
        stay(mx);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return mx;
  };

  const int tiles = piece.t1 - piece.t0;
  if (tiles > 0) {
    Tiles<S> tl;
    tl.start(pg, b, pl.div, n, hk, rw, max(sq.len - 1, 0), piece.t0);
    auto kplace = [&](int buf) { return lds + S::K0 + buf * S::TILE; };
    auto vplace = [&](int buf) { return lds + S::V0 + buf * S::TILE; };
    auto scale_to = [&](bool values, int buf) { return (float*)(lds + S::SCALES) + KT * (2 * values + buf); };
    typename Tiles<S>::From vfrom = tl.where(pg, tl.page());
    tl.ask(pg, vfrom, false, kplace(0));
    tl.ask(pg, vfrom, true, vplace(0));
    tl.settle(false, kplace(0), scale_to(false, 0));
    tl.settle(true, vplace(0), scale_to(true, 0));
    tl.step(pg, pl.div);
    if (tiles > 1) {
      vfrom = tl.where(pg, tl.page());
      tl.ask(pg, vfrom, false, kplace(1));
      tl.settle(false, kplace(1), scale_to(false, 1));
    }
    tl.step(pg, pl.div);
    int page = tl.page();
#pragma unroll
    for (int j = 0; j < KS; ++j) stay(q[j]);                   // here now: the loop must not wait for them, nor for what it asks for
    if constexpr (!S::I8) wait_loads<0>();
    __syncthreads();
    f32x16 one[X], two[X];                                     // scores of a tile and of the next, in turn
    if (busy) {
#pragma unroll
      for (int x = 0; x < X; ++x) one[x] = f32x16(0.f);
#pragma unroll
      for (int j = 0; j < NK; ++j) one[j / KS] = Rows<32>::mfma(keys(0, j), q[j % KS], one[j / KS]);
      adjust(piece.t0, 0, one);
      run.follow(one, Carry::largest(one), c);
    }
    // Every wave has used up the first keys and their scales before any asks for, or settles, the third tile's over them: the loop's first
    // barrier comes only after that, and a wave without rows is there at once.  In the loop a barrier lies between: what is asked for goes where
    // the turn before read, after this turn's barrier; codes settle before it, where two turns before read.
    __syncthreads();
    auto tile = [&](int i, int buf, f32x16 (&s)[X], f32x16 (&next)[X]) {       // buf: i & 1
      const bool more = i + 1 < tiles;
      const int t = piece.t0 + i;
      if (i > 0) {
        // this tile's V and the next one's K are here; the K of this one and the V before it are used up
        if constexpr (S::I8) {
          if (more) tl.settle(false, kplace(buf ^ 1), scale_to(false, buf ^ 1));
          tl.settle(true, vplace(buf), scale_to(true, buf));
        } else {
          wait_loads<0>();
        }
        __syncthreads();
      }
      if (more) tl.ask(pg, vfrom, true, vplace(buf ^ 1));
      if (i + 2 < tiles) {
        vfrom = tl.where(pg, page);
        tl.ask(pg, vfrom, false, kplace(buf));
        tl.step(pg, pl.div);
        page = tl.page();
      }
      if (!busy) return;
      scores_and_weigh(buf ^ 1, buf, next, s);                 // after the last tile: of what lies there, for nothing
      if (more) adjust(t + 1, buf ^ 1, next);
      const float mx = meet_and_largest(buf, s, next);
      if (masked(t)) {
#pragma unroll
        for (int x = 0; x < X; ++x)
          poisoned |= S::I8 ? scales_not_finite(scale_to(true, buf) + 32 * x) : tile_not_finite<D>(vplace(buf) + 32 * x * S::RB);
      }
      if (more) run.follow(next, mx, c);
    };
    for (int i = 0;;) {
      tile(i, 0, one, two);
      if (++i >= tiles) break;
      tile(i, 1, two, one);
      if (++i >= tiles) break;
    }
  }
  if (__builtin_amdgcn_readfirstlane(poisoned)) {
    rows_again<D, S::I8>(a, pg, b, pl, n, hk, sq, r0 + 32 * rw, min(r0 + 32 * rw + 32, r0 + rows), piece.t0 * (KT / 32), piece.t1 * (KT / 32), 1,
                  [&](int r, float m, float l, const float* y) {
      constexpr int C = D / 64;
      const int tk = r / G;
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const int d = C * lane + e;
        if (piece.pieces > 1) part[(r - r0) * D + d] = y[e];
        else store1(a, sq.lo + tk, sq.pos0 + tk, hk * G + r - tk * G, d, y[e] * inv);
      }
      if (piece.pieces > 1 && lane == 0) { part[S::ROWS * D + r - r0] = m; part[S::ROWS * (D + 1) + r - r0] = l; }
    });
    return;
  }
  run.l = xor32_sum(run.l);
  if (row >= r0 + rows) return;
  if (piece.pieces > 1) {
    float* to = part + (32 * rw + col) * D + 4 * g;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) *(f32x4*)(to + 32 * i + 8 * e) = f32x4{run.o[i][4 * e], run.o[i][4 * e + 1], run.o[i][4 * e + 2], run.o[i][4 * e + 3]};
    if (g == 0) { part[S::ROWS * D + 32 * rw + col] = run.m; part[S::ROWS * (D + 1) + 32 * rw + col] = run.l; }
    return;
  }
  const float inv = run.l == 0.f ? 0.f : 1.f / run.l;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      store4(a, sq.lo + tok, pos, head, 32 * i + 8 * e + 4 * g, f32x4{run.o[i][4 * e], run.o[i][4 * e + 1], run.o[i][4 * e + 2], run.o[i][4 * e + 3]} * inv);
      __builtin_amdgcn_sched_barrier(0);                       // not all gates at once: their registers
    }
}

// Row tiles are numbered without a scan over the batch: tile j of sequence n has the number loc[n] G / ROWS + n + j; numbers
// left over find a tile past the end.
struct RowTile { int n, r0; };
template <int ROWS> __device__ __forceinline__ RowTile row_tile(const lq_batch& b, int G, int number) {
  const int lane = threadIdx.x & 63;
  int a = 0, len = b.N;
  while (len > 1) {
    const int step = (len + 63) >> 6, m = a + lane * step;
    const bool below = lane * step < len && batch_at(b, m) * G / ROWS + m <= number;
    const int at = max((int)__popcll(__ballot(below)) - 1, 0) * step;
    a += at;
    len = min(step, len - at);
  }
  RowTile r;
  r.n = __builtin_amdgcn_readfirstlane(a);
  const int j = number - (batch_at(b, r.n) * G / ROWS + r.n);
  r.r0 = __builtin_amdgcn_readfirstlane(j < 0 ? 0x7fffffff : j * ROWS);
  return r;
}

// Workgroups go to the XCDs in turn: a head of the cache stays on one of them (or on 8 / HK), whose L2 then holds its tiles.
// The last row tiles, which see the most keys, come first.
template <class S>
__device__ __forceinline__ void many_block(const lq_attention& a, const lq_pages& pg, const lq_batch& b, const Plan& pl, char* lds, int block) {
  const int per = pl.tiles * pg.HK, split = block / per, x = block % per;
  int hk, number;
  if (pg.HK < 8 && 8 % pg.HK == 0 && per % 8 == 0) {
    const int share = 8 / pg.HK;
    hk = (x & 7) / share;
    number = (x >> 3) * share + (x & 7) % share;
  } else {
    hk = x % pg.HK;
    number = x / pg.HK;
  }
  number = pl.tiles - 1 - number;
  const RowTile rt = row_tile<S::ROWS>(b, pl.G, number);
  const Seq sq = sequence(b, pg, pl.G, rt.n);
  if (rt.r0 >= sq.rows || sq.rows <= pl.few) return;
  many_rows<S>(a, pg, b, pl, lds, rt.n, hk, split, rt.r0, sq, pl.many_work + ((long long)split * per + (long long)number * pg.HK + hk) * S::PART);
}
template <class S>
__global__ __launch_bounds__(S::THREADS) __attribute__((amdgpu_waves_per_eu(S::EU, S::EU)))
void many_kernel(lq_attention a, lq_pages pg, lq_batch b, Plan pl) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  many_block<S>(a, pg, b, pl, lds, blockIdx.x);
}

// Both kinds of sequences in one launch, eight workgroups of one kind and eight of the other in turn while both last: those of few
// rows, which wait for memory, beside those of many, which compute.
template <class F, class M>
__global__ __launch_bounds__(M::THREADS) __attribute__((amdgpu_waves_per_eu(M::EU, M::EU)))
void both_kernel(lq_attention a, lq_pages pg, lq_batch b, Plan pl) {
  static_assert(F::THREADS == M::THREADS);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int x = blockIdx.x, turns = 8 * (min(pl.few_blocks, pl.many_blocks) / 8);
  const bool many = x < 2 * turns ? !(x & 8) : pl.many_blocks > turns && x - turns < pl.many_blocks;
  const int block = x < 2 * turns ? (x >> 4) * 8 + (x & 7) : many ? x - turns : x - (pl.many_blocks > turns ? pl.many_blocks : turns);
  if (many) many_block<M>(a, pg, b, pl, lds, block);
  else few_block<F>(a, pg, b, pl, lds, block);
}

// ---- the pieces of split keys, joined -----------------------------------------------------------------------------------
// A row's D / 4 threads take 4 channels each; P of them share out the pieces of a row.
template <class S, bool FEW, int P>
__device__ __forceinline__ void join_block(const lq_attention& a, const lq_pages& pg, const lq_batch& b, const Plan& pl, float* lds, int block) {
  constexpr int D = S::D, ROWS = S::ROWS, C = D / 4, PER = 256 / (C * P);      // rows of a workgroup
  static_assert(PER >= 1 && ROWS % PER == 0, "rows of a workgroup");
  const int item = block / (ROWS / PER), rr = (block % (ROWS / PER)) * PER + threadIdx.x / (C * P);
  const int hk = item % pg.HK, number = item / pg.HK;
  RowTile rt = {number, 0};
  if (!FEW) rt = row_tile<ROWS>(b, pl.G, number);
  const Seq sq = sequence(b, pg, pl.G, rt.n);
  if (FEW ? sq.rows <= 0 || sq.rows > ROWS : rt.r0 >= sq.rows || sq.rows <= pl.few) return;
  const int rows = min(ROWS, sq.rows - rt.r0);
  if ((block % (ROWS / PER)) * PER >= rows) return;
  const int splits = FEW ? pl.few_splits : pl.many_splits;
  const Piece piece = piece_of<S>(keys_of(sq, pl.G, rt.r0, rt.r0 + rows, a.window), splits, 0);
  if (piece.pieces == 1) return;
  const int which = (threadIdx.x / C) % P, d = 4 * (threadIdx.x % C);
  const long long step = (long long)(FEW ? b.N : pl.tiles) * pg.HK * S::PART;
  const float* part = (FEW ? pl.few_work : pl.many_work) + (long long)item * S::PART;
  const float c = a.scale * LOG2E;
  float M = -INFINITY, L = 0.f;
  f32x4 y = f32x4(0.f);
  constexpr int U = 8;                                         // pieces on their way at once
  for (int k0 = which; k0 < piece.pieces; k0 += U * P) {
    float mk[U], lk[U];
    f32x4 yk[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* p = part + min(k0 + u * P, piece.pieces - 1) * step;
      mk[u] = p[ROWS * D + rr];
      lk[u] = p[ROWS * (D + 1) + rr];
      yk[u] = *(const f32x4*)(p + rr * D + d);
    }
    float to = M;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u * P < piece.pieces) to = fmaxf(to, mk[u]);
    const float w = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((M - to) * c);
    L *= w;
    y *= w;
    M = to;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u * P < piece.pieces) {
        const float w = mk[u] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mk[u] - M) * c);    // none: zeros, or NaN
        L = fmaf(w, lk[u], L);
        y += w * yk[u];
      }
  }
  if constexpr (P > 1) {
    float* jm = lds + 256 * 4;                                 // [PER][P] maxima, then sums
    *(f32x4*)(lds + 4 * threadIdx.x) = y;
    if (d == 0) { jm[threadIdx.x / C] = M; jm[PER * P + threadIdx.x / C] = L; }
    __syncthreads();
    if (which > 0) return;
    const int at = threadIdx.x / C;
    M = -INFINITY; L = 0.f; y = f32x4(0.f);
#pragma unroll
    for (int k = 0; k < P; ++k) M = fmaxf(M, jm[at + k]);
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const float w = jm[at + k] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((jm[at + k] - M) * c);
      L = fmaf(w, jm[PER * P + at + k], L);
      y += w * *(const f32x4*)(lds + 4 * (threadIdx.x + C * k));
    }
  }
  if (rr >= rows) return;
  const int tk = (rt.r0 + rr) / pl.G;
  store4(a, sq.lo + tk, sq.pos0 + tk, hk * pl.G + (rt.r0 + rr - tk * pl.G), d, y * (L == 0.f ? 0.f : 1.f / L));
}

template <class F, class M, int P>
__global__ __launch_bounds__(256) void join_kernel(lq_attention a, lq_pages pg, lq_batch b, Plan pl, int few_blocks) {
  __shared__ float lds[P > 1 ? 256 * 4 + 2 * 256 / (F::D / 4) : 1];
  if ((int)blockIdx.x < few_blocks) join_block<F, true, P>(a, pg, b, pl, lds, blockIdx.x);
  else join_block<M, false, P>(a, pg, b, pl, lds, blockIdx.x - few_blocks);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <int D, bool I8> struct Shapes {
  typedef Few<D, 4, I8> F;
  // Tiles of 64 keys, or 32 where 64 do not fit the registers: heads of 256 and codes (prompt of
  // 8192 of heads of 128 573 -> 563 us by 64; 4096 from codes 666, spilled, -> 257 by 32).  Heads of 256 hold 32 rows of outputs in half the registers of
  // a SIMD: one wave there.
  typedef Many<D, 4, !I8 && D <= 128 ? 64 : 32, D == 256 ? 1 : 2, I8> M;
};

// LDS beyond what a kernel has unasked: asked for once on each device, and again where that failed.
template <auto* KERNEL, int LDS> bool lds_asked() {
  static std::atomic<bool> had[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const bool known = dev >= 0 && dev < 64;
  if (known && had[dev].load(std::memory_order_relaxed)) return true;
  if (hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return false;
  if (known) had[dev].store(true, std::memory_order_relaxed);
  return true;
}

// Sizes and the longest sequence's tokens, where the caller says them, settle what a call launches and how the keys are split.
template <int D, bool I8> Plan plan_of(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest) {
  typedef typename Shapes<D, I8>::F F;
  typedef typename Shapes<D, I8>::M M;
  Plan c = {};
  c.G = a->HQ / p->HK;
  c.div = page_div(p->page);
  const long long cus = lq_attn_cus(), most = longest > 0 && longest < b->T ? longest : b->T, rows = most * c.G;
  // Which kernels, by rows: a sequence of up to 16 (a token's heads) reads its keys by waves of its own, which 64 of them at contexts up
  // to 8192 do at 5.2 TB/s.  Beside longer ones that is worth a second kind of workgroup only if the others are short by the mean (us,
  // with it / without): 32 sequences of up to 8 tokens, 8 heads a key head of 256 95 / 65, 5 of up to 777 under a window 19.5 / 19.4.
  // A piece of 449 tokens beside 15 of one token, 4 heads a key head: 86 with it; without, a tile of 128 rows for 4.
  // Without the hint any sequence may be the long one: both kinds are launched, the few one with the other's registers and fewer pieces (us,
  // said / not said: 64 single tokens up to 8192 of 8 heads of 128 257 / 345, from codes 169 / 273, 32 of up to 8 tokens up to 4099 of 2
  // of 256 58 / 87).
  const bool hint = longest > 0 && longest < b->T, many = rows > F::ROWS;
  const bool few = !many || (b->N > 1 && (!hint || (b->T - most) * c.G <= (long long)F::ROWS * (b->N - 1)));
  c.few = few ? F::ROWS : 0;
  c.tiles = many ? (int)((long long)b->T * c.G / M::ROWS + b->N) : 0;
  // keys that a row tile sees at most, by the table's width; under a window of its rows' tokens.  Short contexts under a wide table get a
  // join with nothing to join (us, as wide as needed / 4096 pages: 64 single tokens at 200 of 8 heads of 128 10.6 / 15.8, at 1000 39 / 47).
  auto reach = [&](int tile) {
    const long long all = (long long)b->width * p->page, near = (long long)a->window + (tile - 1) / c.G + 1;
    return a->window > 0 && near < all ? near : all;
  };
  // Pieces of the keys, so that workgroups are as many as the chip holds at once.  A workgroup costs as much before its first and after
  // its last key as some 500 keys, and a part is written and read again; four times as many where pieces still have 1024 keys (us, as
  // many as held / twice / four times): 64 sequences up to 8192 of 8 heads of 128 267 / 266 / 255, 64 up to 4099 of 2 of 256 78 / 78 / 85 and from
  // codes 61 / 68 / 89, 8 up to 4099 of 8 of 128 24 / 26 / 31, 2 up to 1024 9.5 / 12; tiles of many rows: 32 sequences up to 4099 of
  // 2 of 256 58 / 65 / 65, a piece of 449 over 4096 of 8 of 128 beside 15 of one token 86 / 86 / 85.
  constexpr int HELD = F::LDS > 81920 ? 1 : D == 64 ? 4 : 2;   // workgroups of few rows on a CU
  auto pieces = [&](long long target, long long items, long long keys, int least) {
    const long long by = (target + items - 1) / items, cap = keys / least;
    return (int)(by < 1 || cap < 2 ? 1 : by < cap ? (by < 256 ? by : 256) : (cap < 256 ? cap : 256));
  };
  const long long fi = (long long)b->N * p->HK, mi = (long long)c.tiles * p->HK;
  c.few_splits = few ? std::max(pieces(HELD * cus, fi, reach(F::ROWS), F::LEAST * F::KT),
                                many ? 1 : pieces(4 * HELD * cus, fi, reach(F::ROWS), 1024)) : 1;
  c.many_splits = many && mi < M::EU * cus ? pieces(M::EU * cus, mi, reach(M::ROWS), M::LEAST * M::KT) : 1;
  c.few_blocks = few ? (int)(fi * c.few_splits) : 0;
  c.many_blocks = (int)(mi * c.many_splits);
  return c;
}
template <int D, bool I8> long long few_floats(const Plan& c) {
  return c.few_splits > 1 ? (long long)c.few_blocks * Shapes<D, I8>::F::PART : 0;
}
template <int D, bool I8> long long many_floats(const Plan& c) {
  return c.many_splits > 1 ? (long long)c.many_blocks * Shapes<D, I8>::M::PART : 0;
}

template <int D, bool I8>
int go(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest, float* work, hipStream_t s) {
  typedef typename Shapes<D, I8>::F F;
  typedef typename Shapes<D, I8>::M M;
  Plan pl = plan_of<D, I8>(a, p, b, longest);
  pl.few_work = work;
  pl.many_work = work + few_floats<D, I8>(pl);
  const unsigned blocks = (unsigned)pl.few_blocks + (unsigned)pl.many_blocks;
  if (!pl.many_blocks) {
    if (!lds_asked<few_kernel<F>, F::LDS>()) return LQ_ERR_HIP;
    few_kernel<F><<<blocks, F::THREADS, F::LDS, s>>>(*a, *p, *b, pl);
  } else if (!pl.few_blocks) {
    if (!lds_asked<many_kernel<M>, M::LDS>()) return LQ_ERR_HIP;
    many_kernel<M><<<blocks, M::THREADS, M::LDS, s>>>(*a, *p, *b, pl);
  } else {
    constexpr int LDS = F::LDS > M::LDS ? F::LDS : M::LDS;
    if (!lds_asked<both_kernel<F, M>, LDS>()) return LQ_ERR_HIP;
    both_kernel<F, M><<<blocks, M::THREADS, LDS, s>>>(*a, *p, *b, pl);
  }
  if (hipGetLastError() != hipSuccess) return LQ_ERR_HIP;
  if (pl.few_splits == 1 && pl.many_splits == 1) return LQ_OK;
  // four groups of threads a row where there are pieces enough for them
  const int P = pl.few_splits > 8 || pl.many_splits > 8 ? 4 : 1, per = 256 / (D / 4 * P);
  const int few_join = pl.few_splits > 1 ? b->N * p->HK * (F::ROWS / per) : 0;
  const int many_join = pl.many_splits > 1 ? pl.tiles * p->HK * (M::ROWS / per) : 0;
  const unsigned joins = (unsigned)few_join + (unsigned)many_join;
  if (P == 4) join_kernel<F, M, 4><<<joins, 256, 0, s>>>(*a, *p, *b, pl, few_join);
  else join_kernel<F, M, 1><<<joins, 256, 0, s>>>(*a, *p, *b, pl, few_join);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
}

template <typename F> auto by_shape(const lq_pages* p, F f) {
  if (p->D == 64) return p->int8 ? f(std::integral_constant<int, 64>(), std::true_type()) : f(std::integral_constant<int, 64>(), std::false_type());
  if (p->D == 128) return p->int8 ? f(std::integral_constant<int, 128>(), std::true_type()) : f(std::integral_constant<int, 128>(), std::false_type());
  return p->int8 ? f(std::integral_constant<int, 256>(), std::true_type()) : f(std::integral_constant<int, 256>(), std::false_type());
}

int check(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest) {
  if (!a || !pages_ok(p) || !batch_ok(b, p) || longest < 0) return LQ_ERR_ARG;
  if (a->HQ <= 0 || a->HQ % p->HK || a->window < 0 || !(a->scale > 0.f) || a->scale >= 0x1p127f) return LQ_ERR_ARG;      // times log2(e) in fp32
  if (b->N == 0 || b->T == 0) return LQ_OK;
  if (!rows_ok(a->q) || !rows_ok(a->gate) || !rows_ok(a->out) || !a->q.p || !a->out.p) return LQ_ERR_ARG;
  if (!rows_apart(a->out, b->T, a->HQ, p->D)) return LQ_ERR_ARG;
  const long long G = a->HQ / p->HK;
  // places of a tile past the last key, rows, row tiles and workgroups in 32 bits
  if ((long long)b->width * p->page > 0x7fffffffll - 4096) return LQ_ERR_ARG;
  if (((long long)b->T + 64) * G > 0x3fffffffll || ((long long)b->T * G / 64 + b->N + 8) * p->HK > 0x7fffffffll / 256) return LQ_ERR_ARG;
  return LQ_OK;
}

}  // namespace

extern "C" long long lq_attend_workspace(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest) {
  if (int rc = check(a, p, b, longest)) return rc;
  if (b->N == 0 || b->T == 0) return 0;
  return by_shape(p, [&](auto d, auto i8) {
    constexpr int D = decltype(d)::value;
    constexpr bool I8 = decltype(i8)::value;
    const Plan c = plan_of<D, I8>(a, p, b, longest);
    return 4 * (few_floats<D, I8>(c) + many_floats<D, I8>(c));
  });
}

extern "C" int lq_attend(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest, void* work, long long work_bytes,
                         void* stream) {
  const long long need = lq_attend_workspace(a, p, b, longest);
  if (need < 0) return (int)need;
  if (b->N == 0 || b->T == 0) return LQ_OK;
  if (need > 0 && (!work || ((uintptr_t)work & 15) || work_bytes < need)) return LQ_ERR_ARG;
  return by_shape(p, [&](auto d, auto i8) {
    return go<decltype(d)::value, decltype(i8)::value>(a, p, b, longest, (float*)work, (hipStream_t)stream);
  });
}

__attribute__((visibility("hidden"))) int lq_attn_cus() {
  static std::atomic<int> cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cus[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
    cus[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
extern "C" int lq_attn_abi_version(void) { return LQ_ATTN_ABI_VERSION; }
