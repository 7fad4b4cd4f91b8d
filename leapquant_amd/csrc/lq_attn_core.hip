// Attention of a ragged batch's new tokens over a paged cache (lq_attend).
//
//   o_r = sum_j e^{s_rj - m_r} v_j / sum_j e^{s_rj - m_r},   s_rj = scale q_r . k_j,   t_r - window < j <= t_r
//
// A row r is a new token and one of the G = HQ / HK heads that read the same head of the cache, numbered token by token, so that
// a key or value is read once for all of them.  One pass over the keys in tiles, with the running maximum m and sum of a row.
//
// A wave owns 32 rows.  It forms S^T = K Q^T with 32 x 32 matrix instructions: a lane then holds 16 of 32 keys of one row, its
// maximum takes one exchange with lane ^ 32, and the probabilities are already laid out as the right operand of O^T = V^T P^T,
// keys in an order that the transposing reads of V from LDS follow.  m moves only when a row's maximum has grown by 2^8 or more:
// sums and outputs stay in fp32, so that only their common factor changes.  Probabilities are rounded to bf16 for the second
// product (2^-9 each, of random sign), their sum is not.
//
// Tiles go from the pages straight into LDS, a tile ahead, in swizzled places: both kinds of reads then spread over all banks.
// Codes of 8 bits go through registers and into LDS as bf16, which holds them exactly; their scales enter S and P in fp32.
#include <atomic>

#include "lq_attn.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lds_t;
typedef const __attribute__((address_space(4))) int const_int;     // what no kernel of the call writes: scalar loads

// The launches of a call: the few rows of a decode or draft (kernel A: a sequence's rows in one wave, waves share out the
// keys) and the many of a prompt (kernel B: waves share out the rows of a tile, tiles numbered over the batch).
struct Plan {
  int few, splits;         // rows up to which a sequence is the other kernel's (A: none); pieces of the keys at most
  int G;
  uint32_t g_mul;          // x / G = x * g_mul >> 32 for x < 2^16.., see rows_div
  PageDiv div;
  float* work;
};

constexpr float GROWN = 8.f;
constexpr float LOG2E = 1.44269504f;

__device__ __forceinline__ f32x16 mfma(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ u32x4 lds_read16(const char* p) { return *(const u32x4*)p; }
__device__ __forceinline__ u32x2 lds_read_tr(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_t*)p));
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes a lane from base + off into LDS at lds + 16 lane; the caller waits before it reads them
__device__ __forceinline__ void tile_load16(const char* base, uint32_t off, const char* lds) {
  const unsigned to = (unsigned)(size_t)(const lds_t*)lds;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// a sequence's rows and keys, as a workgroup finds them
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

// keys [lo, hi) that rows [r0, r1) see
struct Keys { int lo, hi; };
__device__ __forceinline__ Keys keys_of(const Seq& s, int G, int r0, int r1, int window) {
  Keys k;
  const int first = s.pos0 + r0 / G, last = s.pos0 + (r1 - 1) / G;
  k.hi = max(last + 1, 0);
  k.lo = window > 0 ? max(first - window + 1, 0) : 0;
  if (k.lo > k.hi) k.lo = k.hi;
  return k;
}
// tiles of KT keys [t0, t1) that piece `split` of a row tile's keys holds, and how many pieces there are
struct Piece { int t0, t1, pieces; };
template <int KT, int LEAST> __device__ __forceinline__ Piece piece_of(const Keys& k, int splits, int split) {
  const int a = k.lo / KT, b = (k.hi + KT - 1) / KT, tiles = max(b - a, 0);
  Piece p;
  p.pieces = max(min(splits, tiles / LEAST), 1);
  const int per = (tiles + p.pieces - 1) / p.pieces;
  p.pieces = max((tiles + per - 1) / max(per, 1), 1);          // none is empty
  p.t0 = a + split * per;
  p.t1 = min(p.t0 + per, b);
  return p;
}

// Rows of a row tile: D is the head's size; RW waves of 32 rows share a tile of keys, KW of them (or groups of RW) each take
// tiles of their own.
template <int D_, int RW_, int KW_, int KT_, int LEAST_, bool I8_> struct Shape {
  static constexpr int D = D_, RW = RW_, KW = KW_, KT = KT_, LEAST = LEAST_;
  static constexpr bool I8 = I8_;
  static constexpr int WAVES = RW * KW, THREADS = 64 * WAVES, ROWS = 32 * RW;
  static constexpr int TILE = KT * D * 2;                      // bytes of a tile of K or V in LDS
  static constexpr int STAGE = 2 * KW * TILE;
  static constexpr int SCALES = I8 ? 2 * KW * 2 * KT * 4 : 0;
  static constexpr int JOIN = KW > 1 ? KW * ROWS * (D + 4) * 4 + KW * ROWS * 8 : 0;
  static constexpr int LDS0 = 2 * STAGE + SCALES;
  static constexpr int LDS = LDS0 > JOIN ? LDS0 : JOIN;
  static constexpr int PART = ROWS * (D + 2);                  // floats of a workgroup's part of split keys
};

template <class S> __device__ __forceinline__ int swizzle_k(int key) { return key & 7; }
template <class S> __device__ __forceinline__ int swizzle_v(int key) { return S::D == 64 ? (key & 3) << 1 : (key & 7) << 1; }

// The work of a workgroup: rows [r0, r0 + ROWS) of a sequence and head hk of the cache, piece `split` of the keys.
template <class S>
__device__ __forceinline__ void attend(const lq_attention& a, const lq_pages& pg, const lq_batch& b, const Plan& pl, char* lds,
                                       int n, int hk, int split, int splits, int r0, const Seq& sq, float* part) {
  constexpr int D = S::D, RW = S::RW, KW = S::KW, KT = S::KT, TILE = S::TILE, KB = KT / 32, MB = D / 32, KS = D / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW, kw = wave / RW;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int G = pl.G, rows = min(S::ROWS, sq.rows - r0);
  const Keys keys = keys_of(sq, G, r0, r0 + rows, a.window);
  const Piece piece = piece_of<KT, S::LEAST>(keys, splits, split);
  if (split >= piece.pieces) return;

  // this lane's row
  const int row = r0 + 32 * rw + col, rc = min(row, r0 + rows - 1);
  const int tok = rc / G, g = rc - tok * G, pos = sq.pos0 + tok, head = hk * G + g;
  const bool busy = 32 * rw < rows;                            // the wave has rows
  const int first = sq.pos0 + min(r0 + 32 * rw, r0 + rows - 1) / G, last = sq.pos0 + (min(r0 + 32 * rw + 32, r0 + rows) - 1) / G;
  const int from = a.window > 0 ? max(pos - a.window + 1, 0) : 0;               // keys from .. pos are seen
  const int wave_from = a.window > 0 ? max(first - a.window + 1, 0) : 0;        // the wave's first and last key
  const int wave_full = a.window > 0 ? max(last - a.window + 1, 0) : 0;         // all rows see wave_full .. first
  u32x4 q[KS];
  {
    const bf16_t* p = (const bf16_t*)a.q.p + (long long)(sq.lo + tok) * a.q.ld + (long long)head * a.q.hd + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = *(const u32x4*)(p + 16 * s);
  }

  // ---- tiles: this wave loads KT / RW keys of its group's tile -----------------------------------------------------------
  constexpr int OWN = KT / RW, GROUPS = OWN > 16 ? OWN / 16 : 1, GK = OWN / GROUPS;    // keys a wave loads, in groups of one page
  const int* tab = b.table + (long long)n * b.table_ld;
  const char* kbase = (const char*)pg.k + (long long)hk * pg.head_ld * (S::I8 ? 1 : 2);
  const char* vbase = (const char*)pg.v + (long long)hk * pg.head_ld * (S::I8 ? 1 : 2);
  constexpr int PER = S::I8 ? 16 : 8;                          // elements of a 16-byte load
  constexpr int CPR = D / PER, LOADS = GK * CPR / 64 > 0 ? GK * CPR / 64 : 1;
  static_assert(GK * CPR >= 64 || S::I8, "a load of a whole wave");
  u32x4 kreg[S::I8 ? GROUPS * LOADS : 1], vreg[S::I8 ? GROUPS * LOADS : 1];
  float ksc = 0.f, vsc = 0.f;
  const int tend = max(sq.len - 1, 0);
  auto stage = [&](int t, int buf) {                           // t: the tile
    const int k0 = t * KT + rw * OWN;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const int kg = min(k0 + 16 * i, OWN >= 16 ? tend & ~15 : (tend & ~(OWN - 1)));
      const int pi = __builtin_amdgcn_readfirstlane(page_of(pl.div, kg));
      int page = __builtin_amdgcn_readfirstlane(((const_int*)tab)[pi]);
      page = page >= 0 && page < pg.NP ? page : 0;
      const int in = kg - pi * pg.page;
      const long long base = (long long)page * pg.page_ld + (long long)in * pg.row_ld;
      const int most = tend - kg;                              // places of the group's last cached token
      const char *kp = kbase + base * (S::I8 ? 1 : 2), *vp = vbase + base * (S::I8 ? 1 : 2);
      if constexpr (!S::I8) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          const int c = 64 * j + lane, key = c / CPR, tk = rw * OWN + 16 * i + key;
          const uint32_t off = (uint32_t)min(key, most) * (uint32_t)(2 * pg.row_ld);
          char* to = lds + buf * S::STAGE + (2 * kw) * TILE + (rw * OWN + 16 * i) * D * 2 + 1024 * j;
          tile_load16(kp, off + 16 * ((c % CPR) ^ swizzle_k<S>(tk)), to);
          tile_load16(vp, off + 16 * ((c % CPR) ^ swizzle_v<S>(tk)), to + TILE);
        }
      } else {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          const int c = 64 * j + lane, key = min(c / CPR, GK - 1);
          const uint32_t off = (uint32_t)min(key, most) * (uint32_t)pg.row_ld + 16 * (c % CPR);
          kreg[i * LOADS + j] = *(const u32x4*)(kp + off);
          vreg[i * LOADS + j] = *(const u32x4*)(vp + off);
        }
      }
    }
    if constexpr (S::I8) {                                     // lane's scale: key `lane` of the wave's (at most 64)
      const int kk = min(k0 + min(lane, OWN - 1), tend);
      const int pi = page_of(pl.div, kk);
      int page = tab[pi];
      page = page >= 0 && page < pg.NP ? page : 0;
      const long long at = (long long)page * pg.s_page_ld + (kk - pi * pg.page) * pg.s_row_ld + hk * pg.s_head_ld;
      ksc = pg.k_scale[at];
      vsc = pg.v_scale[at];
    }
  };
  auto settle = [&](int buf) {                                 // codes in registers -> bf16 in LDS
    if constexpr (S::I8) {
#pragma unroll
      for (int i = 0; i < GROUPS; ++i)
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          const int c = 64 * j + lane, key = c / CPR, tk = rw * OWN + 16 * i + key, ch = 2 * (c % CPR);
          if (key < GK) {
            char* to = lds + buf * S::STAGE + (2 * kw) * TILE + tk * D * 2;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const u32x4 w = x ? vreg[i * LOADS + j] : kreg[i * LOADS + j];
              const int sw = x ? swizzle_v<S>(tk) : swizzle_k<S>(tk);
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                u32x4 o;
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  const int two = (int)w[2 * y + (z >> 1)] >> (16 * (z & 1));
                  o[z] = pk_bf16((float)(int8_t)two, (float)(int8_t)(two >> 8));
                }
                *(u32x4*)(to + x * TILE + 16 * ((ch + y) ^ sw)) = o;
              }
            }
          }
        }
      float* sc = (float*)(lds + 2 * S::STAGE) + (buf * KW + kw) * 2 * KT + rw * OWN;
      if (lane < OWN) { sc[lane] = ksc; sc[KT + lane] = vsc; }
    }
  };

  const float c = a.scale * LOG2E;
  float m = -INFINITY, l = 0.f;
  f32x16 o[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) o[i] = f32x16(0.f);
  // this lane's reads: a row of K; V by 4 keys x 16 channels a group of 16 lanes
  const int kread = col * D * 2 + 16 * (half ^ swizzle_k<S>(col));
  const int vkey = 4 * half + ((lane & 15) >> 2);
  const int vread = vkey * D * 2 + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swizzle_v<S>(vkey)) + 8 * (lane & 1);

  auto tile = [&](int t, int buf) {
    const char* K = lds + buf * S::STAGE + (2 * kw) * TILE;
    const char* V = K + TILE;
    const int k0 = t * KT;
    if (!busy || k0 > last || k0 + KT <= wave_from) return;
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      s[kb] = f32x16(0.f);
#pragma unroll
      for (int i = 0; i < KS; ++i) s[kb] = mfma(lds_read16(K + kb * 32 * D * 2 + (kread ^ (32 * i))), q[i], s[kb]);
    }
    if constexpr (S::I8) {
      const float* sc = (const float*)(lds + 2 * S::STAGE) + (buf * KW + kw) * 2 * KT + 4 * half;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = *(const f32x4*)(sc + 32 * kb + 8 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[kb][4 * i + e] *= x[e];
        }
    }
    const bool masked = k0 + KT - 1 > first || k0 < wave_full;
    if (masked) {
      const int lo = from - k0 - 4 * half, hi = pos - k0 - 4 * half;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 32 * kb + 8 * (i >> 2) + (i & 3);
          s[kb][i] = j >= lo && j <= hi ? s[kb][i] : -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = xor32_max(mx);
    if (__any((mx - m) * c > GROWN)) {
      const float to = fmaxf(m, mx), alpha = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - to) * c);
      m = to;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < MB; ++i) o[i] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m * c;
    // s c - ref is rounded once, but ref itself is off by half its last place, which 2^ref would be too much for beyond 2^24
    if (__any(fabsf(ref) > 0x1p24f)) {
      const float raw = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f((s[kb][i] - raw) * c);
    } else {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], c, -ref));
    }
    u32x4 pr[2 * KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) l += s[kb][i];
      if constexpr (S::I8) {
        const float* sc = (const float*)(lds + 2 * S::STAGE) + (buf * KW + kw) * 2 * KT + KT + 4 * half;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = *(const f32x4*)(sc + 32 * kb + 8 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = 32 * kb + 8 * i + e + 4 * half + k0;
            const float y = s[kb][4 * i + e] * x[e];
            s[kb][4 * i + e] = !masked || (j >= from && j <= pos) ? y : 0.f;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) pr[2 * kb + (i >> 2)][i & 3] = pk_bf16(s[kb][2 * i], s[kb][2 * i + 1]);
    }
    uint32_t bad[KB] = {};                                     // keys of a masked tile whose values are not finite
    bool some = false;
    if (!S::I8 && masked) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        uint32_t hit = 0;
        for (int i = 0; i < D / 16; ++i) {
          const u32x4 w = lds_read16(V + (kb * 32 + col) * D * 2 + 16 * (half + 2 * i));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = (w[e] & 0x7f807f80u) ^ 0x7f807f80u;
            hit |= (x - 0x00010001u) & ~x & 0x80008000u;
          }
        }
        const unsigned long long any = __ballot(hit != 0);
        bad[kb] = (uint32_t)any | (uint32_t)(any >> 32);
        some |= bad[kb] != 0;
      }
    }
    if (!some) {
#pragma unroll
      for (int t2 = 0; t2 < 2 * KB; ++t2)
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const char* at = V + t2 * 16 * D * 2 + (vread ^ (64 * i));
          const u32x2 x = lds_read_tr(at), y = lds_read_tr(at + 8 * D * 2);
          o[i] = mfma(u32x4{x[0], x[1], y[0], y[1]}, pr[t2], o[i]);
        }
    } else {
      // The finite keys at once, then each of the others by itself, into the rows that see it alone: a zero probability times
      // an infinity or NaN is not zero.
#pragma unroll
      for (int t2 = 0; t2 < 2 * KB; ++t2) {
        const uint32_t b16 = bad[t2 >> 1] >> (16 * (t2 & 1)) & 0xffffu;
        for (int pass = -1; pass < 16; ++pass) {
          if (pass >= 0 && !(b16 >> pass & 1)) continue;
          const uint32_t take = pass < 0 ? ~b16 : 1u << pass;  // keys of the 16
          const uint32_t mine = take >> (4 * half);            // this half's: 0 .. 3 and 8 .. 11
          u32x4 keep;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t two = mine >> (8 * (e >> 1) + 2 * (e & 1));
            keep[e] = (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
          }
          const int j = k0 + 16 * t2 + pass;
          const bool sees = pass < 0 || (j >= from && j <= pos);
#pragma unroll
          for (int i = 0; i < MB; ++i) {
            const char* at = V + t2 * 16 * D * 2 + (vread ^ (64 * i));
            const u32x2 x = lds_read_tr(at), y = lds_read_tr(at + 8 * D * 2);
            const f32x16 d = mfma(u32x4{x[0], x[1], y[0], y[1]} & keep, pr[t2], f32x16(0.f));
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] += sees ? d[e] : 0.f;
            __builtin_amdgcn_sched_barrier(0);                 // one product's registers at a time
          }
        }
      }
    }
  };

  // ---- the walk over the piece's tiles -----------------------------------------------------------------------------------
  const int stages = (piece.t1 - piece.t0 + KW - 1) / KW;
  if (stages > 0) {
    stage(min(piece.t0 + kw, piece.t1 - 1), 0);
    if constexpr (S::I8) settle(0);
    for (int i = 0; i < stages; ++i) {
      if constexpr (!S::I8) wait_loads();
      if constexpr (S::WAVES > 1 || S::I8) __syncthreads();
      const int t = piece.t0 + i * KW + kw, buf = i & 1;
      if (i + 1 < stages) stage(min(t + KW, piece.t1 - 1), buf ^ 1);
      if (t < piece.t1) tile(t, buf);
      if constexpr (S::I8) {
        if (i + 1 < stages) settle(buf ^ 1);
      }
    }
  }
  l = xor32_sum(l);

  // ---- outputs ---------------------------------------------------------------------------------------------------------------
  const bool whole = piece.pieces == 1;
  if constexpr (KW == 1) {
    if (row >= r0 + rows) return;
    if (!whole) {
      float* to = part + (32 * rw + col) * D;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) *(f32x4*)(to + 32 * i + 8 * e + 4 * half) = f32x4{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]};
      if (half == 0) { part[S::ROWS * D + 32 * rw + col] = m; part[S::ROWS * (D + 1) + 32 * rw + col] = l; }
      return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bf16_t* to = (bf16_t*)a.out.p + (long long)(sq.lo + tok) * a.out.ld + (long long)head * a.out.hd + 4 * half;
    const bf16_t* gate = a.gate.p ? (const bf16_t*)a.gate.p + (long long)(sq.lo + tok) * a.gate.ld + (long long)head * a.gate.hd + 4 * half : nullptr;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] = o[i][4 * e + x] * inv;
        if (gate) {
          const u32x2 w = *(const u32x2*)(gate + 32 * i + 8 * e);
          const float z[4] = {bf_lo(w[0]), bf_hi(w[0]), bf_lo(w[1]), bf_hi(w[1])};
#pragma unroll
          for (int x = 0; x < 4; ++x) y[x] *= __builtin_amdgcn_rcpf(1.0f + __expf(-z[x]));
        }
        *(u32x2*)(to + 32 * i + 8 * e) = u32x2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
      }
  } else {
    // the groups' parts of a row, joined through LDS
    float* jo = (float*)lds;                                   // [KW][ROWS][D + 4]
    float* jm = jo + KW * S::ROWS * (D + 4);                   // [KW][ROWS] maxima, then sums
    __syncthreads();
    {
      float* to = jo + (kw * S::ROWS + 32 * rw + col) * (D + 4);
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) *(f32x4*)(to + 32 * i + 8 * e + 4 * half) = f32x4{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]};
      if (half == 0) { jm[kw * S::ROWS + 32 * rw + col] = m; jm[(KW + kw) * S::ROWS + 32 * rw + col] = l; }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < rows * (D / 8); x += S::THREADS) {
      const int rr = x / (D / 8), d = 8 * (x % (D / 8));
      float M = -INFINITY, L = 0.f, y[8] = {};
#pragma unroll
      for (int k = 0; k < KW; ++k) M = fmaxf(M, jm[k * S::ROWS + rr]);
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const float mk = jm[k * S::ROWS + rr], w = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mk - M) * c);
        const float* z = jo + (k * S::ROWS + rr) * (D + 4) + d;
        const float lk = jm[(KW + k) * S::ROWS + rr];
        L += mk == -INFINITY ? lk : w * lk;                    // NaN scores: no maximum, a sum of NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = mk == -INFINITY ? y[e] + z[e] : fmaf(w, z[e], y[e]);
      }
      if (!whole) {
        *(f32x4*)(part + rr * D + d) = f32x4{y[0], y[1], y[2], y[3]};
        *(f32x4*)(part + rr * D + d + 4) = f32x4{y[4], y[5], y[6], y[7]};
        if (d == 0) { part[S::ROWS * D + rr] = M; part[S::ROWS * (D + 1) + rr] = L; }
        continue;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const int tk = (r0 + rr) / G, hd = hk * G + (r0 + rr - tk * G);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= inv;
      if (a.gate.p) {
        const u32x4 w = *(const u32x4*)((const bf16_t*)a.gate.p + (long long)(sq.lo + tk) * a.gate.ld + (long long)hd * a.gate.hd + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= __builtin_amdgcn_rcpf(1.0f + __expf(-(e & 1 ? bf_hi(w[e >> 1]) : bf_lo(w[e >> 1]))));
      }
      *(u32x4*)((bf16_t*)a.out.p + (long long)(sq.lo + tk) * a.out.ld + (long long)hd * a.out.hd + d) =
          u32x4{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3]), pk_bf16(y[4], y[5]), pk_bf16(y[6], y[7])};
    }
  }
}

// ---- A: sequences of few rows -------------------------------------------------------------------------------------------
// workgroup (split, sequence, head)
template <class S>
__global__ __launch_bounds__(S::THREADS) void few_kernel(lq_attention a, lq_pages pg, lq_batch b, Plan pl) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int item = blockIdx.x % (b.N * pg.HK), split = blockIdx.x / (b.N * pg.HK), n = item / pg.HK, hk = item % pg.HK;
  const Seq sq = sequence(b, pg, pl.G, n);
  if (sq.rows <= 0 || (pl.few && sq.rows > pl.few)) return;
  // more rows than a tile has, where no other launch takes them: one workgroup all of them, a tile after the other
  const int splits = sq.rows > S::ROWS ? 1 : pl.splits;
  for (int r0 = 0; r0 < sq.rows; r0 += S::ROWS) {
    attend<S>(a, pg, b, pl, lds, n, hk, split, splits, r0, sq, pl.work + (long long)blockIdx.x * S::PART);
    __syncthreads();
  }
}

// ---- B: sequences of many rows -----------------------------------------------------------------------------------------
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
__global__ __launch_bounds__(S::THREADS) void many_kernel(lq_attention a, lq_pages pg, lq_batch b, Plan pl, int tiles) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int per = tiles * pg.HK, split = blockIdx.x / per, x = blockIdx.x % per;
  int hk, number;
  if (pg.HK < 8 && 8 % pg.HK == 0 && per % 8 == 0) {
    const int share = 8 / pg.HK;
    hk = (x & 7) / share;
    number = (x >> 3) * share + (x & 7) % share;
  } else {
    hk = x % pg.HK;
    number = x / pg.HK;
  }
  const RowTile rt = row_tile<S::ROWS>(b, pl.G, tiles - 1 - number);
  const Seq sq = sequence(b, pg, pl.G, rt.n);
  if (rt.r0 >= sq.rows || sq.rows <= pl.few) return;
  attend<S>(a, pg, b, pl, lds, rt.n, hk, split, pl.splits, rt.r0, sq,
            pl.work + ((long long)split * per + (long long)(tiles - 1 - number) * pg.HK + hk) * S::PART);
}

// ---- the pieces of split keys, joined -----------------------------------------------------------------------------------
// A workgroup for each row tile and head; a thread for 4 channels of a row.
template <class S, bool FEW>
__global__ __launch_bounds__(256) void join_kernel(lq_attention a, lq_pages pg, lq_batch b, Plan pl, int tiles) {
  constexpr int D = S::D, ROWS = S::ROWS;
  const int item = blockIdx.x, hk = item % pg.HK, number = item / pg.HK;
  RowTile rt = {number, 0};
  if (!FEW) rt = row_tile<ROWS>(b, pl.G, number);
  const Seq sq = sequence(b, pg, pl.G, rt.n);
  if (FEW ? sq.rows <= 0 || sq.rows > ROWS : rt.r0 >= sq.rows || sq.rows <= pl.few) return;
  const int rows = min(ROWS, sq.rows - rt.r0);
  const Piece piece = piece_of<S::KT, S::LEAST>(keys_of(sq, pl.G, rt.r0, rt.r0 + rows, a.window), pl.splits, 0);
  if (piece.pieces == 1) return;
  const long long step = (long long)tiles * pg.HK * S::PART;
  const float* part = pl.work + (long long)item * S::PART;
  const float c = a.scale * LOG2E;
  for (int x = blockIdx.y * 256 + threadIdx.x; x < rows * (D / 4); x += 256 * gridDim.y) {
    const int rr = x / (D / 4), d = 4 * (x % (D / 4));
    float M = -INFINITY, L = 0.f;
    for (int k = 0; k < piece.pieces; ++k) M = fmaxf(M, part[k * step + ROWS * D + rr]);
    f32x4 y = f32x4(0.f);
    for (int k = 0; k < piece.pieces; ++k) {
      const float* p = part + k * step;
      const float mk = p[ROWS * D + rr], w = mk == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mk - M) * c);
      L = fmaf(w, p[ROWS * (D + 1) + rr], L);                  // a piece without a maximum: zeros, or NaN
      y += w * *(const f32x4*)(p + rr * D + d);
    }
    y *= L == 0.f ? 0.f : 1.f / L;
    const int tk = (rt.r0 + rr) / pl.G, hd = hk * pl.G + (rt.r0 + rr - tk * pl.G);
    if (a.gate.p) {
      const u32x2 w = *(const u32x2*)((const bf16_t*)a.gate.p + (long long)(sq.lo + tk) * a.gate.ld + (long long)hd * a.gate.hd + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] *= __builtin_amdgcn_rcpf(1.0f + __expf(-(e & 1 ? bf_hi(w[e >> 1]) : bf_lo(w[e >> 1]))));
    }
    *(u32x2*)((bf16_t*)a.out.p + (long long)(sq.lo + tk) * a.out.ld + (long long)hd * a.out.hd + d) = u32x2{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
  }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <int D, bool I8> struct Shapes;
template <bool I8> struct Shapes<64, I8> {
  typedef Shape<64, 1, 4, 32, 8, I8> Few;
  typedef Shape<64, 4, 1, 64, 8, I8> Many;
};
template <bool I8> struct Shapes<128, I8> {
  typedef Shape<128, 1, 4, 32, 8, I8> Few;
  typedef Shape<128, 4, 1, 64, 8, I8> Many;
};
template <bool I8> struct Shapes<256, I8> {
  typedef Shape<256, 1, 2, 32, 8, I8> Few;
  typedef Shape<256, 4, 1, 32, 16, I8> Many;
};

// LDS beyond what a kernel has unasked: asked for once on each device, and again where that failed.
template <class S, bool FEW> bool lds_asked() {
  static std::atomic<bool> had[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const bool known = dev >= 0 && dev < 64;
  if (known && had[dev].load(std::memory_order_relaxed)) return true;
  const void* f;
  if constexpr (FEW) f = (const void*)few_kernel<S>;
  else f = (const void*)many_kernel<S>;
  if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess) return false;
  if (known) had[dev].store(true, std::memory_order_relaxed);
  return true;
}

// What a call launches, from what the host knows: sizes, and the longest sequence's tokens where the caller says.
struct Calls {
  bool few, many;          // which kernels
  int few_splits, many_splits, tiles;
  long long few_work, many_work;     // floats
};
template <int D, bool I8> Calls calls(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest) {
  typedef typename Shapes<D, I8>::Few F;
  typedef typename Shapes<D, I8>::Many M;
  const long long G = a->HQ / p->HK, cus = lq_attn_cus();
  const long long most = longest > 0 && longest < b->T ? longest : b->T;
  Calls c = {};
  c.few = most * G <= F::ROWS || b->N > 1;
  c.many = most * G > F::ROWS;
  c.tiles = (int)((long long)b->T * G / M::ROWS + b->N);
  const long long reach = (long long)b->width * p->page;       // the longest context
  auto pieces = [&](long long target, long long items, int least) {
    const long long by = (target + items - 1) / items, cap = reach / least;
    return (int)(by < 1 || cap < 2 ? 1 : by < cap ? (by < 256 ? by : 256) : (cap < 256 ? cap : 256));
  };
  const long long fi = (long long)b->N * p->HK, mi = (long long)c.tiles * p->HK;
  c.few_splits = c.few ? pieces(4 * cus, fi, F::LEAST * F::KT) : 1;
  c.many_splits = c.many && mi < 2 * cus ? pieces(2 * cus, mi, M::LEAST * M::KT) : 1;
  c.few_work = c.few_splits > 1 ? c.few_splits * fi * F::PART : 0;
  c.many_work = c.many_splits > 1 ? c.many_splits * mi * M::PART : 0;
  return c;
}

template <int D, bool I8>
int go(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest, float* work, hipStream_t s) {
  typedef typename Shapes<D, I8>::Few F;
  typedef typename Shapes<D, I8>::Many M;
  const Calls c = calls<D, I8>(a, p, b, longest);
  Plan pl = {};
  pl.G = a->HQ / p->HK;
  pl.div = page_div(p->page);
  const int fi = b->N * p->HK, mi = c.tiles * p->HK;
  if (c.few) {
    if (!lds_asked<F, true>()) return LQ_ERR_HIP;
    pl.few = c.many ? F::ROWS : 0;
    pl.splits = c.few_splits;
    pl.work = work;
    few_kernel<F><<<(unsigned)(fi * c.few_splits), F::THREADS, F::LDS, s>>>(*a, *p, *b, pl);
    if (hipGetLastError() != hipSuccess) return LQ_ERR_HIP;
    if (c.few_splits > 1) {
      join_kernel<F, true><<<(unsigned)fi, 256, 0, s>>>(*a, *p, *b, pl, b->N);
      if (hipGetLastError() != hipSuccess) return LQ_ERR_HIP;
    }
  }
  if (c.many) {
    if (!lds_asked<M, false>()) return LQ_ERR_HIP;
    pl.few = c.few ? F::ROWS : 0;
    pl.splits = c.many_splits;
    pl.work = work + c.few_work;
    many_kernel<M><<<(unsigned)(mi * c.many_splits), M::THREADS, M::LDS, s>>>(*a, *p, *b, pl, c.tiles);
    if (hipGetLastError() != hipSuccess) return LQ_ERR_HIP;
    if (c.many_splits > 1) {
      join_kernel<M, false><<<dim3((unsigned)mi, 4), 256, 0, s>>>(*a, *p, *b, pl, c.tiles);
      if (hipGetLastError() != hipSuccess) return LQ_ERR_HIP;
    }
  }
  return LQ_OK;
}

template <typename F> auto by_shape(const lq_pages* p, F f) {
  if (p->D == 64) return p->int8 ? f(std::integral_constant<int, 64>(), std::true_type()) : f(std::integral_constant<int, 64>(), std::false_type());
  if (p->D == 128) return p->int8 ? f(std::integral_constant<int, 128>(), std::true_type()) : f(std::integral_constant<int, 128>(), std::false_type());
  return p->int8 ? f(std::integral_constant<int, 256>(), std::true_type()) : f(std::integral_constant<int, 256>(), std::false_type());
}

int check(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest) {
  if (!a || !pages_ok(p) || !batch_ok(b, p) || longest < 0) return LQ_ERR_ARG;
  if (a->HQ <= 0 || a->HQ % p->HK || a->window < 0 || !(a->scale > 0.f) || a->scale > 3.4e38f) return LQ_ERR_ARG;
  if (b->N == 0 || b->T == 0) return LQ_OK;
  if (!rows_ok(a->q) || !rows_ok(a->gate) || !rows_ok(a->out) || !a->q.p || !a->out.p) return LQ_ERR_ARG;
  if (!rows_apart(a->out, b->T, a->HQ, p->D)) return LQ_ERR_ARG;
  const long long G = a->HQ / p->HK;
  // rows, row tiles and workgroups in 32 bits
  if (((long long)b->T + 64) * G > 0x3fffffffll || ((long long)b->T * G / 64 + b->N + 8) * p->HK > 0x7fffffffll / 256) return LQ_ERR_ARG;
  return LQ_OK;
}

}  // namespace

extern "C" long long lq_attend_workspace(const lq_attention* a, const lq_pages* p, const lq_batch* b, int longest) {
  if (int rc = check(a, p, b, longest)) return rc;
  if (b->N == 0 || b->T == 0) return 0;
  return by_shape(p, [&](auto d, auto i8) {
    const Calls c = calls<decltype(d)::value, decltype(i8)::value>(a, p, b, longest);
    return 4 * (c.few_work + c.many_work);
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
