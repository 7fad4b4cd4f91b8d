// The gated delta rule over prompts, in chunks of C = 32 tokens on the matrix cores (lq_delta_prefill).
//
// With G_i the sum of the log-gates of a chunk's tokens up to i, k and q normalised, and S0 the state before the chunk,
//
//   A_ij = beta_i e^{G_i - G_j} k_i.k_j  (i > j),    T = (I + A)^-1 diag(beta)
//   R = V - diag(e^G) K S0^T,    U = T R                              the values the recurrence would append
//   O = diag(e^G) Q S0^T + P U,    P_ij = e^{G_i - G_j} q_i.k_j  (i >= j)
//   S = e^{G_C} S0 + U^T diag(e^{G_C - G}) K
//
// so that with T' = diag(e^{G_C - G} / |k|) T and W = P T, which do not depend on the state, a chunk is O = .. + W R and
// S = e^{G_C} S0 + (T' R)^T K.  A first kernel forms T' and W of all chunks at once; a second walks each sequence's chunks.
// Rows of S (value channels) do not meet, so a head's rows are spread over waves, 16 a wave.
//
// The walk's chain of dependent products is shortened by K_c S_c = e^{G_C} K_c S_{c-1} + X_c (T' R)_{c-1} with
// X_c = K_c K_{c-1}^T: the product with the state is a chunk old when it is needed, and a second wave keeps the state.
//
// Rounding.  The raw keys, queries and values are bf16 and enter the products as they are; their norms, decays and beta are
// fp32 factors of rows and columns of fp32 sums, never folded into an operand.  fp32 operands are carried in bf16 parts, each
// 2.8e-6 (two parts) or 5e-9 (three) of the operand short in the mean.  What is appended to the state and leads to it (T', R,
// T' R, X) has three: errors of its terms do not cancel where the terms do, as with equal keys in a chunk.  The state ends
// within 8e-7 of its norm, 2e-7 in the median (fp32 sums: 2e-7); with two parts within 6e-6, and 2e-5 where appended values
// cancel, for 12% less time.  What is read of the state (S in K S and Q S), W, and R where it meets W have two: a third in K S
// takes 12% more time for the rest of the difference, and the outputs are bf16 (1.7e-3; their fp32 values are off by a few 1e-6
// of their terms, which rounds one in a few thousand the other way than fp32 sums would); single bf16 operands would lose
// digits where their terms cancel (a query nearly orthogonal to the state, equal keys).  Norms, decays, gates and beta come
// from the hardware's reciprocal square root, exp2, log and reciprocal, 1 ulp each.
//
// Measured (both kernels, heads of 128 x 128, 16 key and 32 value heads, a call among others): one prompt of 8192 tokens
// 203 us (201 MB of tokens and outputs; the first kernel 32, then 256 steps of 0.67 us), 13 prompts of 32768 tokens 473 us (850
// MB: 1.8 TB/s; the first kernel 120; with two parts everywhere, 414 us, matrix instructions were busy 42% of the walk's
// cycles, vector ones 50%, LDS 45%, at the 1.7 GHz that this mix leaves of the clock).  A profiler has more for the same
// kernels, 36 + 212 and 131 + 412; where forms of one kernel are compared below, the times are its.
#include <atomic>
#include <type_traits>

#include "lq_seq.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int C = 32;                  // tokens of a chunk

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mf(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mf(const bf16x4& a, const bf16x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ bf16x4 first4(const bf16x8& a) { return __builtin_shufflevector(a, a, 0, 1, 2, 3); }
// four or eight fp32 values as two or three bf16 parts
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pk_bf16_kept(x, y);
  lo = pk_bf16_kept(x - bf_lo(hi), y - bf_hi(hi));
}
__device__ __forceinline__ uint32_t third2(float x, float y, uint32_t hi, uint32_t lo) {
  return pk_bf16(x - bf_lo(hi) - bf_lo(lo), y - bf_hi(hi) - bf_hi(lo));
}
__device__ __forceinline__ void split4(const f32x4& x, bf16x4& hi, bf16x4& lo, bf16x4* third = nullptr) {
  u32x2 h, l, t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t a, b;
    split2(x[2 * i], x[2 * i + 1], a, b);
    h[i] = a; l[i] = b;
    if (third) t[i] = third2(x[2 * i], x[2 * i + 1], a, b);
  }
  hi = __builtin_bit_cast(bf16x4, h);
  lo = __builtin_bit_cast(bf16x4, l);
  if (third) *third = __builtin_bit_cast(bf16x4, t);
}
__device__ __forceinline__ void split8(const f32x4& x, const f32x4& y, bf16x8& hi, bf16x8& lo, bf16x8* third = nullptr) {
  const float f[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  u32x4 h, l, t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a, b;
    split2(f[2 * i], f[2 * i + 1], a, b);
    h[i] = a; l[i] = b;
    if (third) t[i] = third2(f[2 * i], f[2 * i + 1], a, b);
  }
  hi = __builtin_bit_cast(bf16x8, h);
  lo = __builtin_bit_cast(bf16x8, l);
  if (third) *third = __builtin_bit_cast(bf16x8, t);
}

// What the first kernel leaves for a chunk of a value head.  The matrices are operands as a lane takes them: lane l of a row
// tile holds row l % 16 at the columns 4 g .. 4 g + 3 and 16 + 4 g .. (g = l / 16), the order in which a lane of a product's
// result holds its rows, so that results are the next product's operands without moving between lanes.  The first row tile's
// columns 16 .. are zero and left out.  T' in three parts, W in two.
struct alignas(16) Coef {
  bf16x4 t0[3][64], w0[2][64];
  bf16x8 t1[3][64], w1[2][64];
  float c[C];                          // e^G / |k|: of the rows of K S
  float d[C];                          // scale e^G / |q|: of the rows of Q S
  float last[4];                       // e^{G_C}
};
static_assert(sizeof(Coef) % 16 == 0, "moved by 16-byte words");

struct alignas(16) Scratch {           // a 32 x 32 matrix row by row, and the tokens' factors
  float m[C][C + 4];
  float ghi[C], glo[C], bet[C], rk[C], rq[C];
};

// a block of row r sits at its place xor the row, so that 16 rows' blocks of one column meet different banks
__device__ __forceinline__ int swz(int r, int blocks) { return (r / (16 / blocks)) & (blocks - 1); }

// 16 bytes a lane from base + off straight to LDS, lane l's at lds + 16 l
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds(const void* base, unsigned off, unsigned lds) {
  const unsigned at = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(at) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int SHR> __device__ __forceinline__ double from_below(double x) {      // of lane l - SHR of the same 16, else 0
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = __builtin_amdgcn_mov_dpp((int)(unsigned)b, 0x110 + SHR, 0xf, 0xf, true);
  const unsigned hi = __builtin_amdgcn_mov_dpp((int)(unsigned)(b >> 32), 0x110 + SHR, 0xf, 0xf, true);
  return join_d(lo, hi);
}
typedef __attribute__((address_space(3))) char* lds_t;
__device__ __forceinline__ bf16x8 at16(lds_t p) { return *(__attribute__((address_space(3))) bf16x8*)p; }
// four columns of four rows a lane, by the transposing read: lane (n, g) points at columns 4 (n % 4) .. of row 4 g + n / 4 and
// gets column n of the rows 4 g ..
__device__ __forceinline__ s16x4 quad(lds_t p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}
// LDS written by this wave's other lanes may be read
__device__ __forceinline__ void wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// the step ends: this wave's LDS accesses are done, and every other wave's
__device__ __forceinline__ void end_step() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Which of `items` groups of M workgroups a workgroup belongs to, and its number in it.  The M of a group read the same keys
// and queries: consecutive workgroups go to the eight XCDs in turn, each with an L2 of its own, so those of a group are eight
// apart.  Fewer groups than XCDs are spread over all of them instead.
struct Place { int item, m; };
__device__ __forceinline__ Place place_of(int b, int items, int M) {
  if (items < 8) return {b / M, b % M};
  const int q = b / (8 * M), r = b - q * 8 * M;
  return {8 * q + (r & 7), r >> 3};
}
inline long long place_grid(long long items, int M) { return (items < 8 ? items : (items + 7) / 8 * 8) * M; }

// T' or W of a chunk, in N parts, times R, onto y: the products that reach the N-th part's digits
template <int N> struct Operand { bf16x4 m0[N]; bf16x8 m1[N]; };
template <int N> __device__ __forceinline__ Operand<N> operand(const bf16x4 (&m0)[N][64], const bf16x8 (&m1)[N][64], int l) {
  Operand<N> m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m.m0[i] = m0[i][l];
    m.m1[i] = m1[i][l];
  }
  return m;
}
template <int N>
__device__ __forceinline__ void chunk_product(const Operand<N>& m, const bf16x8 (&r)[N], f32x4 (&y)[2]) {
#pragma unroll
  for (int a = 0; a < N; ++a)
#pragma unroll
    for (int b = 0; a + b < N; ++b) {
      y[0] = mf(m.m0[a], first4(r[b]), y[0]);
      y[1] = mf(m.m1[a], r[b], y[1]);
    }
}
// a result's rows, tokens, that there are: this lane's offsets from the chunk's first token, and their stores
__device__ __forceinline__ void store_places(unsigned (&at)[8], unsigned old, int n, int g) {
#pragma unroll
  for (int i = 0; i < 8; ++i) at[i] = (16 * (i >> 2) + 4 * g + (i & 3)) * old + 2u * n;
}
__device__ __forceinline__ void store_chunk(char* out, const unsigned (&at)[8], const f32x4 (&o)[2], int g, int left) {
  uint32_t two[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) two[i] = pk_bf16_kept(o[i >> 1][2 * (i & 1)], o[i >> 1][2 * (i & 1) + 1]);
  if (left >= C) {
#pragma unroll
    for (int i = 0; i < 8; ++i) *(bf16_t*)(out + at[i]) = (bf16_t)(i & 1 ? two[i >> 1] >> 16 : two[i >> 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (16 * (i >> 2) + 4 * g + (i & 3) < left) *(bf16_t*)(out + at[i]) = (bf16_t)(i & 1 ? two[i >> 1] >> 16 : two[i >> 1]);
  }
}

// ---- T' and W of every chunk ---------------------------------------------------------------------------------------------
// 32 us for 8192 tokens (256 chunks, 32 heads), 120 us for 32768: 530 MB of keys, queries and results, 4.4 TB/s, and 53% of the
// vector units' cycles.  One wave a chunk and value head.  (I + A)^-1 by forward substitution in its two diagonal blocks of 16
// (a column a lane) and -T11 A10 T00 below them by fp32 matrix instructions: substitution stays accurate where powers of A
// would not (equal keys without decay make them grow like binomials).
//
// Tokens past a sequence's end are copies of its last one, so that nothing foreign enters a product: their beta and log-gate
// are zero, so their columns of T' and W are, their rows of T' R come out zero, and their outputs are not stored.
//
// The last workgroup sorts the sequences by length, for the walk to begin with the longest: a CU takes several sequences, and
// those that come last should be short ones (more than SORTED sequences even out by themselves, and go in order).
constexpr int SORTED = 256;
__device__ __forceinline__ void sort_by_length(const lq_seqs& s, int* order, int* len) {
  for (int n = threadIdx.x; n < s.N; n += 64) {
    if (s.N > SORTED) order[n] = n;
    else len[n] = seq_at(s, n + 1) - seq_at(s, n);
  }
  if (s.N > SORTED) return;
  wave_sync();
  for (int n = threadIdx.x; n < s.N; n += 64) {
    int rank = 0;
    for (int m = 0; m < s.N; ++m) rank += len[m] > len[n] || (len[m] == len[n] && m < n);
    order[rank] = n;
  }
}
constexpr int CHUNKS = 4;              // waves of a workgroup: heads of a chunk side by side, which share its keys and queries
template <int K>
__global__ __launch_bounds__(64 * CHUNKS) __attribute__((amdgpu_waves_per_eu(4)))
void chunk_kernel(lq_delta p, lq_seqs s, Coef* __restrict__ work, int* __restrict__ order) {
  constexpr int KS = K / 32;
  __shared__ Scratch all[CHUNKS];
  static_assert(sizeof(all) >= SORTED * sizeof(int), "lengths in scratch");
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x + 1 == gridDim.x) {
    if (w == 0) sort_by_length(s, order, (int*)all);
    return;
  }
  Scratch& my = all[w];
  const int item = blockIdx.x * CHUNKS + w, number = item / p.HV, hv = item - number * p.HV, hk = hv / (p.HV / p.H);
  if (number >= s.T / C + s.N) return;
  const SeqRun run = seq_run<C>(s, number);
  const int t0 = run.lo + run.j * C, nv = min(C, run.hi - t0);
  if (nv <= 0) return;
  const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  bf16x8 kf[2][KS], qf[2][KS];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bf16_t* row = (const bf16_t*)p.mixed + (t0 + min(16 * i + n, nv - 1)) * p.mixed_ld + hk * K + 8 * g;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      qf[i][x] = *(const bf16x8*)(row + 32 * x);
      kf[i][x] = *(const bf16x8*)(row + 32 * x + p.H * K);
    }
  }
  {
      // token l % 32 of each half wave; the sum over the chunk in fp64, kept as two floats, so that the difference of two
      // large sums is as good as the gates between them.  A gate under -128 has the same exponential as -128: zero.
      const int t = l & 31;
      const bool live = t < nv;
      const long long row = t0 + min(t, nv - 1);
      const float ea = expf(gate_param(p.A_log, p.gate_bf16 & 1, hv));
      float gate = -ea * softplus_f(bf2f(((const bf16_t*)p.a)[row * p.a_ld + hv]) + gate_param(p.dt_bias, p.gate_bf16 & 2, hv));
      gate = live ? (gate < -128.f ? -128.f : gate) : 0.f;
      const float beta = live ? __builtin_amdgcn_rcpf(1.0f + exp_f(-bf2f(((const bf16_t*)p.b)[row * p.b_ld + hv]))) : 0.f;
      double sum = gate;
      sum += from_below<1>(sum);
      sum += from_below<2>(sum);
      sum += from_below<4>(sum);
      sum += from_below<8>(sum);
      {
        const unsigned long long bits = __builtin_bit_cast(unsigned long long, sum);
        const double first = join_d(__builtin_amdgcn_readlane((int)(unsigned)bits, 15),
                                    __builtin_amdgcn_readlane((int)(unsigned)(bits >> 32), 15));
        sum += t & 16 ? first : 0.0;
      }
      if (l < 32) {
        my.ghi[t] = (float)sum;
        my.glo[t] = (float)(sum - (double)(float)sum);
        my.bet[t] = beta;
      }
    }
    f32x4 kk[3] = {}, qk[3] = {}, qq[2] = {};    // tiles (0, 0), (1, 0), (1, 1)
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      kk[0] = mf(kf[0][x], kf[0][x], kk[0]); kk[1] = mf(kf[1][x], kf[0][x], kk[1]); kk[2] = mf(kf[1][x], kf[1][x], kk[2]);
      qk[0] = mf(qf[0][x], kf[0][x], qk[0]); qk[1] = mf(qf[1][x], kf[0][x], qk[1]); qk[2] = mf(qf[1][x], kf[1][x], qk[2]);
      qq[0] = mf(qf[0][x], qf[0][x], qq[0]); qq[1] = mf(qf[1][x], qf[1][x], qq[1]);
    }
    // the diagonals, squared norms of row 4 g + i: lane n = 4 g + i has its own
    {
      float k0 = kk[0][0], k1 = kk[2][0], q0 = qq[0][0], q1 = qq[1][0];
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        const bool me = (n & 3) == i;
        k0 = me ? kk[0][i] : k0; k1 = me ? kk[2][i] : k1; q0 = me ? qq[0][i] : q0; q1 = me ? qq[1][i] : q1;
      }
      if (n >> 2 == g) {
        my.rk[n] = __builtin_amdgcn_rsqf(k0 + 1e-6f); my.rk[16 + n] = __builtin_amdgcn_rsqf(k1 + 1e-6f);
        my.rq[n] = __builtin_amdgcn_rsqf(q0 + 1e-6f); my.rq[16 + n] = __builtin_amdgcn_rsqf(q1 + 1e-6f);
      }
    }
    wave_sync();
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      const int ri = 16 * (x > 0) + 4 * g, cj = 16 * (x > 1) + n;
      const float hj = my.ghi[cj], lj = my.glo[cj], kj = my.rk[cj];
      const f32x4 hi = *(const f32x4*)&my.ghi[ri], li = *(const f32x4*)&my.glo[ri];
      const f32x4 ai = *(const f32x4*)&my.bet[ri] * *(const f32x4*)&my.rk[ri], pi = *(const f32x4*)&my.rq[ri] * p.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // above the diagonal e^0 and a factor of zero, without a branch
        const float dec = exp_f(fminf((hi[i] - hj) + (li[i] - lj), 0.f)) * kj;
        const bool below = x == 1 || 4 * g + i > n, upto = x == 1 || 4 * g + i >= n;
        my.m[ri + i][cj] = (below ? ai[i] : 0.f) * dec * kk[x][i];
        qk[x][i] *= (upto ? pi[i] : 0.f) * dec;                    // P from here on
      }
    }
    wave_sync();
    {
      const int blk = 16 * (g & 1);              // inverses of the diagonal blocks: lane (block, column), rows top down
      float x[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {              // four rows of A at a time (all of them at once would take 160 registers)
        f32x4 a[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i4 = 0; i4 <= q; ++i4) a[r][i4] = *(const f32x4*)&my.m[blk + 4 * q + r][blk + 4 * i4];
#pragma unroll
        for (int r = 4 * q; r < 4 * q + 4; ++r) {
          float acc = r == n ? 1.f : 0.f;
#pragma unroll
          for (int i = 0; i < r; ++i) acc = fmaf(-a[r & 3][i >> 2][i & 3], x[i], acc);
          x[r] = acc;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      wave_sync();
#pragma unroll
      for (int r = 0; r < 16; ++r) my.m[blk + r][blk + n] = x[r];          // the wave's halves write the same
    }
    wave_sync();
    f32x4 y = {}, t10 = {}, t00, t11;            // results: column n, rows 4 g + i
    {
      const f32x4 a10 = *(const f32x4*)&my.m[16 + n][4 * g], r11 = *(const f32x4*)&my.m[16 + n][16 + 4 * g];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t00[i] = my.m[4 * g + i][n];
        t11[i] = my.m[16 + 4 * g + i][16 + n];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) y = __builtin_amdgcn_mfma_f32_16x16x4f32(a10[i], t00[i], y, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) t10 = __builtin_amdgcn_mfma_f32_16x16x4f32(-r11[i], y[i], t10, 0, 0, 0);
    }
    // three tiles, (0, 0), (1, 0), (1, 1), out of the results' layout into rows
    auto spread = [&](const f32x4& a00, const f32x4& a10, const f32x4& a11) {
      wave_sync();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        my.m[4 * g + i][n] = a00[i];
        my.m[16 + 4 * g + i][n] = a10[i];
        my.m[16 + 4 * g + i][16 + n] = a11[i];
      }
      wave_sync();
    };
    spread(qk[0], qk[1], qk[2]);
    f32x4 ww[3] = {};                             // W before its columns' beta
    {
      const f32x4 p00 = *(const f32x4*)&my.m[n][4 * g], p10 = *(const f32x4*)&my.m[16 + n][4 * g];
      const f32x4 p11 = *(const f32x4*)&my.m[16 + n][16 + 4 * g];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ww[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(p00[i], t00[i], ww[0], 0, 0, 0);
        ww[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(p11[i], t11[i], ww[2], 0, 0, 0);
        ww[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(p10[i], t00[i], ww[1], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) ww[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(p11[i], t10[i], ww[1], 0, 0, 0);
    }
    spread(t00, t10, t11);
    Coef& out = work[(long long)number * p.HV + hv];
    const float gh = my.ghi[C - 1], gl = my.glo[C - 1];
    const f32x4 b0 = *(const f32x4*)&my.bet[4 * g], b1 = *(const f32x4*)&my.bet[16 + 4 * g];
    const float e0 = exp_f((gh - my.ghi[n]) + (gl - my.glo[n])) * my.rk[n];
    const float e1 = exp_f((gh - my.ghi[16 + n]) + (gl - my.glo[16 + n])) * my.rk[16 + n];
    bf16x8 hi, lo;
    split4(*(const f32x4*)&my.m[n][4 * g] * b0 * e0, out.t0[0][l], out.t0[1][l], &out.t0[2][l]);
    split8(*(const f32x4*)&my.m[16 + n][4 * g] * b0 * e1,
           *(const f32x4*)&my.m[16 + n][16 + 4 * g] * b1 * e1, hi, lo, &out.t1[2][l]);
    out.t1[0][l] = hi; out.t1[1][l] = lo;
    spread(ww[0], ww[1], ww[2]);
    split4(*(const f32x4*)&my.m[n][4 * g] * b0, out.w0[0][l], out.w0[1][l]);
    split8(*(const f32x4*)&my.m[16 + n][4 * g] * b0, *(const f32x4*)&my.m[16 + n][16 + 4 * g] * b1, hi, lo);
    out.w1[0][l] = hi; out.w1[1][l] = lo;
    if (l < C) {
      const float e = exp_f(my.ghi[l] + my.glo[l]);
      out.c[l] = e * my.rk[l];
      out.d[l] = e * my.rq[l] * p.scale;
      if (l < 4) out.last[l] = exp_f(gh + gl);
    }
}

// ---- the walk over a sequence's chunks -----------------------------------------------------------------------------------
// Chunk c is requested in step c - 1 - AHEAD, has landed when step c - 1 begins, and meets the waves in the steps c - 1 (K in
// K_c S_{c-1} and X), c (Q, V, T', c, ..) and c + 1 (K^T in the state's update, W, d, e^{G_C}).
//
// A step ends when the slowest wave has done its part.  8192 tokens take 171 us.  With two parts everywhere, by the profiler
// (which has 202 to 212 for three), it was 173: of a step's 1500 cycles the state's waves worked 1390, the chain 1110, the others
// 820 to 1190, and LDS moved 125 KB, 970 cycles' worth.  X by way of LDS to its operand's layout took 12 us more.  Not kept (of
// 173): X from the first kernel (166, but 8 more there), X by one wave (183), 32 channels a state wave (218: LDS), a step's tiles
// read into registers a step ahead (177 to 189: the reads then stand before the step's end).
constexpr int AHEAD = 2;               // chunks requested before the step that first needs one
constexpr int SERVICE = 4;             // service waves of a workgroup
constexpr int ROLES = 4;               // waves of 16 rows of the state: chain, two halves of the channels, outputs
struct Pass {                          // between the waves of 16 rows, of one step
  f32x4 kp[2][2][64], qs[2][2][64];    // K S, Q S of a half of the channels: row tile
  bf16x8 r[2][64], u[3][64];           // R, T' R in parts, the highest first
};
constexpr int PASS = (int)sizeof(Pass) / 16;

template <int K>
struct Tiles {                         // places in LDS, in 16-byte blocks
  static constexpr int RB = K / 8, TU = C * RB;                    // blocks of a row of K, of a tile
  static constexpr int VB = 2, VU = C * VB;                        // the same of the workgroup's columns of V
  static constexpr int CU = (int)sizeof(Coef) / 16, CN = 8;
  static constexpr int KN = AHEAD + 3, QN = AHEAD + 2, VN = AHEAD + 2;
  static constexpr int QAT = KN * TU, VAT = QAT + QN * TU, CAT = VAT + VN * VU, XAT = CAT + KN * CN * 64;
  static constexpr int PAT = XAT + 2 * 6 * 64, END = PAT + 2 * PASS, BYTES = 16 * END;      // PAT: what the waves pass on
  // loads of a service wave for a chunk, the same for each (all four load V), so that one count says what is still on its way
  static constexpr int LOADS = 2 * TU / 64 / SERVICE + CN / SERVICE + 1;
  static_assert(VU == 64 && CN * 64 >= CU && CN % SERVICE == 0, "loads of a chunk");
  static_assert(BYTES <= 160 * 1024, "LDS of a CU");
  static_assert(LOADS < 64, "what a wave may have outstanding");
};

template <int K, int V>
struct Walk {
  typedef Tiles<K> B;
  static constexpr int KS = K / 32, RB = B::RB, TU = B::TU, VB = B::VB;
  const lq_delta& p;
  u32x4* lds;
  int lo, len, nc, hv, part;

  // the tiles of K and the Coefs go round KN places: a chunk's place, the next one's, the one's before
  static __device__ __forceinline__ int after(int at) { return at == B::KN - 1 ? 0 : at + 1; }
  static __device__ __forceinline__ int before(int at) { return at == 0 ? B::KN - 1 : at - 1; }
  __device__ __forceinline__ const u32x4* ktile(int at) const { return lds + at * TU; }
  __device__ __forceinline__ const Coef& coef(int at) const { return *(const Coef*)(lds + B::CAT + at * B::CN * 64); }
  __device__ __forceinline__ bf16x8* xtile(int c) const { return (bf16x8*)(lds + B::XAT + (c & 1) * 384); }
  __device__ __forceinline__ Pass& pass(int c) const { return ((Pass*)(lds + B::PAT))[c & 1]; }

  // the order of what comes before: N matrix instructions with M vector ones under each, and LDS reads among the first
  template <int N, int M> static __device__ __forceinline__ void under() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      if (i < 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x2, M, 0);
    }
  }

  // ---- a service wave: a part of the tiles to come, and a 16 x 16 tile of X ----
  __device__ __forceinline__ void service(int k, const Coef* work) const {
    const int l = threadIdx.x & 63, n = l & 15, g = l >> 4, hk = hv / (p.HV / p.H);
    const unsigned ld = 2u * (unsigned)p.mixed_ld, lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)(char*)lds;
    const char* rows = (const char*)p.mixed + (long long)lo * ld;
    const char *kb = rows + 2u * (p.H + hk) * K, *qb = rows + 2u * hk * K;
    const char* vb = rows + 2u * (2 * p.H * K + hv * V + part * 16);
    const char* cb = (const char*)work;
    const int xi = k >> 1, xe = k & 1;           // rows of this chunk, of the one before
    constexpr int TL = TU / 64 / SERVICE, CL = B::CN / SERVICE;
    unsigned toff[TL], coff[CL], voff;               // this lane's offsets from a chunk's first row, past its last row that row's
    auto place = [&](int count) {
#pragma unroll
      for (int i = 0; i < TL; ++i) {
        const int u = l + 64 * (SERVICE * i + k), r = u / RB;
        toff[i] = (unsigned)min(r, count - 1) * ld + 16u * ((u % RB) ^ swz(r, RB));
      }
      voff = (unsigned)min(l / VB, count - 1) * ld + 16u * ((l % VB) ^ swz(l / VB, VB));
    };
#pragma unroll
    for (int i = 0; i < CL; ++i) coff[i] = 16u * min(l + 64 * (CL * k + i), B::CU - 1);
    place(C);
    int jk = 0, sk = B::KN - 1 - AHEAD;          // places of the chunks j and s
    for (int s = -1 - AHEAD; s <= nc; ++s) {
      const int j = s + 1 + AHEAD;
      if (j < nc) {                              // request chunk j
        if (len - j * C < C) place(len - j * C);
        const unsigned ka = lds0 + 16u * jk * TU + 1024u * k, qa = lds0 + 16u * (B::QAT + (unsigned)j % B::QN * TU) + 1024u * k;
        const unsigned va = lds0 + 16u * (B::VAT + (unsigned)j % B::VN * B::VU);
        const unsigned ca = lds0 + 16u * (B::CAT + jk * B::CN * 64) + 1024u * CL * k;
#pragma unroll
        for (int i = 0; i < TL; ++i) {
          to_lds(kb, toff[i], ka + 1024u * SERVICE * i);
          to_lds(qb, toff[i], qa + 1024u * SERVICE * i);
        }
#pragma unroll
        for (int i = 0; i < CL; ++i) to_lds(cb, coff[i], ca + 1024u * i);
        to_lds(vb, voff, va);
        kb += (long long)C * ld; qb += (long long)C * ld; vb += (long long)C * ld;
        cb += (long long)p.HV * sizeof(Coef);
      }
      if (s >= 0 && s + 1 < nc) {                // X of chunk s + 1
        const u32x4 *kt = ktile(after(sk)) + (16 * xi + n) * RB, *ko = ktile(sk) + (16 * xe + n) * RB;
        f32x4 xx = {};
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          const int at = (4 * x + g) ^ swz(n, RB);
          xx = mf(__builtin_bit_cast(bf16x8, ko[at]), __builtin_bit_cast(bf16x8, kt[at]), xx);
        }
        // X's transpose as a result: a lane has row n of X at the columns 4 g .., as the chain takes it
        bf16x4* out = (bf16x4*)(xtile(s + 1) + 192 * xi + l) + xe;
        split4(xx, out[0], out[128], &out[256]);
      }
      // what the next step needs has landed; this step's request may still be on its way
      if (j < nc) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(B::LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (s < nc) end_step();
      jk = after(jk);
      sk = after(sk);
    }
  }

  // ---- a wave that keeps 16 rows of the state, half of their channels ----
  // S as result tiles of K^T U: lane (n, g) the row v = n, channels 32 x + 8 g .. + 7 in the registers (x, 0), (x, 1), which
  // are also the operand of K S and Q S.
  __device__ __forceinline__ void state(int half, int src, int dst) const {
    constexpr int KH = KS / 2;
    const int l = threadIdx.x & 63, n = l & 15, g = l >> 4, qrow = 4 * g + (n >> 2);
    const long long head = (long long)hv * V * K + (long long)(part * 16 + n) * K + 32 * KH * half + 8 * g;
    f32x4 S[KH][2] = {};
    if (src != 0) {
#pragma unroll
      for (int x = 0; x < KH; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) S[x][h] = *(const f32x4*)(p.S + src * p.slot_stride + head + 32 * x + 4 * h);
    }
    // This lane's places in a tile: a row of K and Q (row 16 + n: 16 RB blocks on), and what it reads of K^T.
    unsigned row_at[KH], col_at[KH];
#pragma unroll
    for (int x = 0; x < KH; ++x) {
      row_at[x] = 16u * (n * RB + ((4 * (KH * half + x) + g) ^ swz(n, RB)));
      col_at[x] = 16u * (qrow * RB + ((4 * (KH * half + x) + (n & 3)) ^ swz(qrow, RB)));
    }
    const lds_t base = (lds_t)(char*)lds;
    // step t: S_t, then K_{t+1} S_t and Q_t S_t (of whatever is in LDS where there is no such chunk: nobody reads that), and
    // S_t e^{G_C} for the next step.  In the order in which it is to issue: 32 channels' halves are formed and scaled between
    // the matrix instructions of the 32 before, behind the update of the 32 after.
    int tk = B::KN - 1;                          // place of chunk t
    auto step = [&](int t, bool update) {
      const lds_t ko = base + 16u * before(tk) * TU, kn = base + 16u * after(tk) * TU;
      const lds_t qt = base + 16u * (B::QAT + (unsigned)(t + B::QN) % B::QN * TU);
      const Pass& in = pass(t + 1);
      Pass& out = pass(t);
      const float next = t < 0 || t == nc ? 1.f : coef(tk).last[0];
      tk = after(tk);
      bf16x8 u[3], kf[2][2], qf[2][2], sh[2], sl[2];
      auto fetch = [&](int x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          kf[x & 1][i] = at16(kn + row_at[x] + 256u * i * RB);
          qf[x & 1][i] = at16(qt + row_at[x] + 256u * i * RB);
        }
      };
      s16x4 k2[KH][2][2];                        // channels 32 x + 8 q + 4 h ..; row 16 + .. has the same column place
      if (update) {
#pragma unroll
        for (int i = 0; i < 3; ++i) u[i] = in.u[i][l];
#pragma unroll
        for (int x = 0; x < KH; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              k2[x][h][i] = quad(ko + col_at[x] + 256u * i * RB + 8u * h);
      }
      fetch(0);
      __builtin_amdgcn_sched_barrier(0);
      auto advance = [&](int x) {
        bf16x8 kT[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          kT[h] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(k2[x][h][0], k2[x][h][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) S[x][h] = mf(kT[h], u[i], S[x][h]);
      };
      f32x4 kp[2] = {}, qs[2] = {};
      auto products = [&](int x) {
        const int b = x & 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          kp[i] = mf(kf[b][i], sh[b], kp[i]);
          qs[i] = mf(qf[b][i], sh[b], qs[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          kp[i] = mf(kf[b][i], sl[b], kp[i]);
          qs[i] = mf(qf[b][i], sl[b], qs[i]);
        }
      };
      if (update) {
        advance(0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int x = 0; x < KH; ++x) {
        if (update && x + 1 < KH) advance(x + 1);
        if (x > 0) products(x - 1);
        if (x + 1 < KH) fetch(x + 1);
        split8(S[x][0], S[x][1], sh[x & 1], sl[x & 1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) S[x][h] *= next;
        if (update && x + 1 < KH) under<4, 8>();
        else if (update && x > 0) under<8, 4>();
        __builtin_amdgcn_sched_barrier(0);
      }
      products(KH - 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        out.kp[half][i][l] = kp[i];
        out.qs[half][i][l] = qs[i];
      }
    };
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) end_step();
    step(-1, false);
    end_step();
    step(0, false);
    end_step();
    for (int t = 1; t < nc; ++t) {
      step(t, true);
      end_step();
    }
    step(nc, true);
#pragma unroll
    for (int x = 0; x < KH; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) *(f32x4*)(p.S + dst * p.slot_stride + head + 32 * x + 4 * h) = S[x][h];
  }

  // ---- the wave that walks the chain R -> T' R -> R of these rows ----
  __device__ __forceinline__ void chain() const {
    const int l = threadIdx.x & 63, n = l & 15, g = l >> 4, qrow = 4 * g + (n >> 2);
    bf16x8 u[3] = {};
    int tk = 0;                                  // place of chunk t
    auto step = [&](int t, bool first) {
      const Coef& ck = coef(tk);
      const Pass& in = pass(t + 1);
      Pass& out = pass(t);
      f32x4 ks[2], r[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) ks[i] = in.kp[0][i][l] + in.kp[1][i][l];
      if (!first) {
        const bf16x8* xt = xtile(t);
        const float last = coef(before(tk)).last[0];
#pragma unroll
        for (int i = 0; i < 2; ++i) ks[i] *= last;
#pragma unroll
        for (int a = 0; a < 3; ++a)
#pragma unroll
          for (int b = 0; a + b < 3; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) ks[i] = mf(xt[192 * i + 64 * a + l], u[b], ks[i]);
      }
      const lds_t vt = (lds_t)(char*)lds + 16u * (B::VAT + (unsigned)t % B::VN * B::VU);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const s16x4 q = quad(vt + 16u * ((16 * i + qrow) * VB + (((n & 3) >> 1) ^ swz(16 * i + qrow, VB))) + 8u * (n & 1));
        const f32x4 cc = *(const f32x4*)&ck.c[16 * i + 4 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[i][e] = fmaf(-cc[e], ks[i][e], bf2f((bf16_t)q[e]));
      }
      bf16x8 rp[3];
      split8(r[0], r[1], rp[0], rp[1], &rp[2]);
      f32x4 U[2] = {};
      chunk_product(operand(ck.t0, ck.t1, l), rp, U);
      out.r[0][l] = rp[0];
      out.r[1][l] = rp[1];
      split8(U[0], U[1], u[0], u[1], &u[2]);
#pragma unroll
      for (int i = 0; i < 3; ++i) out.u[i][l] = u[i];
      tk = after(tk);
    };
#pragma unroll
    for (int s = 0; s < AHEAD + 1; ++s) end_step();
    step(0, true);
    end_step();
    for (int t = 1; t < nc; ++t) {
      step(t, false);
      end_step();
    }
  }

  // ---- the wave that forms their outputs, a step after the chain ----
  __device__ __forceinline__ void outputs() const {
    const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
    const unsigned old = 2u * p.HV * V;          // bytes from token to token
    char* out = (char*)p.out + (long long)lo * old + 2u * (hv * V + part * 16);
    unsigned at[8];
    store_places(at, old, n, g);
#pragma unroll
    for (int s = 0; s < AHEAD + 2; ++s) end_step();
    for (int t = 0, tk = 0; t < nc; ++t, tk = after(tk)) {
      const Coef& ck = coef(tk);
      const Pass& in = pass(t);
      f32x4 o[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) o[i] = (in.qs[0][i][l] + in.qs[1][i][l]) * *(const f32x4*)&ck.d[16 * i + 4 * g];
      const bf16x8 rp[2] = {in.r[0][l], in.r[1][l]};
      chunk_product(operand(ck.w0, ck.w1, l), rp, o);
      store_chunk(out, at, o, g, len - t * C);
      out += (long long)C * old;
      if (t + 1 < nc) end_step();
    }
  }
};

template <int K, int V>
__global__ __launch_bounds__(64 * (ROLES + SERVICE)) __attribute__((amdgpu_waves_per_eu(2)))
void walk_kernel(lq_delta p, lq_seqs s, const Coef* __restrict__ work, const int* __restrict__ order) {
  // the size at launch: the compiler would take LDS as a bound of the waves on a SIMD, and hand out more registers than
  // a wave can use without moves between their two halves
  extern __shared__ u32x4 lds[];
  constexpr int COLS = 16, PARTS = V / COLS;
  const int M = p.HV / p.H * PARTS;
  const Place at = place_of(blockIdx.x, s.N * p.H, M);
  if (at.item >= s.N * p.H) return;
  const int rank = at.item / p.H, sn = order[rank], hk = at.item - rank * p.H;
  const int part = at.m % PARTS, hv = hk * (p.HV / p.H) + at.m / PARTS;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo = seq_at(s, sn), len = max(0, seq_at(s, sn + 1) - lo);
  const int dst = seq_dst(s, sn, p.NS), src = seq_src(s, sn, p.NS);
  if (dst == 0) {                                // a padding sequence
    const long long old = (long long)p.HV * V;
    bf16_t* out = (bf16_t*)p.out + lo * old + (long long)hv * V + part * COLS;
    for (long long i = threadIdx.x; i < (long long)len * COLS; i += 64 * (ROLES + SERVICE)) out[i / COLS * old + i % COLS] = 0;
    return;
  }
  if (len == 0) {                                // no tokens: the state moves on
    const long long rows = (long long)hv * V * K + (long long)part * COLS * K;
    for (int i = 4 * threadIdx.x; i < COLS * K; i += 4 * 64 * (ROLES + SERVICE)) {
      f32x4 x = {};
      if (src != 0) x = *(const f32x4*)(p.S + src * p.slot_stride + rows + i);
      *(f32x4*)(p.S + dst * p.slot_stride + rows + i) = x;
    }
    return;
  }
  const Walk<K, V> walk = {p, lds, lo, len, (len + C - 1) / C, hv, part};
  if (w == 0) walk.chain();
  else if (w < 3) walk.state(w - 1, src, dst);
  else if (w == 3) walk.outputs();
  else walk.service(w - ROLES, work + ((long long)(lo / C + sn) * p.HV + hv));
}

// ---- the walk with a wave alone for 16 rows --------------------------------------------------------------------------------
// All of a chunk in one wave, R = V - c K S straight from the state: fewer instructions in all (74 matrix ones a chunk), and LDS
// for two chunks only, so that two workgroups share a CU and fill each other's waits.  13 sequences of 32768 tokens: 350 us.
// With two parts everywhere (by the profiler 348, against 406 to 412 with three): a third workgroup a CU gained 2%, 32 columns a
// wave lost 18% (registers).
template <int K, int NW>
struct Pair {                          // places in LDS of the two chunks, in 16-byte blocks
  static constexpr int RB = K / 8, TU = C * RB, VB = 2 * NW, VU = C * VB;
  static constexpr int CU = (int)sizeof(Coef) / 16, TH = 64 * NW;
  static constexpr int VAT = 2 * TU, CAT = VAT + VU, BUF = CAT + CU, BYTES = 2 * 16 * BUF;
};
template <int K, int V, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(3)))
void lone_kernel(lq_delta p, lq_seqs s, const Coef* __restrict__ work, const int* __restrict__ order) {
  typedef Pair<K, NW> B;
  extern __shared__ u32x4 lds[];
  constexpr int KS = K / 32, COLS = 16 * NW, PARTS = V / COLS, RB = B::RB, TU = B::TU, VB = B::VB, TH = B::TH;
  const int M = p.HV / p.H * PARTS;
  const Place at = place_of(blockIdx.x, s.N * p.H, M);
  if (at.item >= s.N * p.H) return;
  const int rank = at.item / p.H, sn = order[rank], hk = at.item - rank * p.H;
  const int part = at.m % PARTS, hv = hk * (p.HV / p.H) + at.m / PARTS;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, n = l & 15, g = l >> 4;
  const int qrow = 4 * g + (n >> 2);
  const int lo = seq_at(s, sn), len = max(0, seq_at(s, sn + 1) - lo), nc = (len + C - 1) / C;
  const int dst = seq_dst(s, sn, p.NS), src = seq_src(s, sn, p.NS);
  const unsigned old = 2u * p.HV * V, ld = 2u * (unsigned)p.mixed_ld;        // bytes from token to token
  const int v0 = part * COLS + 16 * w + n;
  char* out = (char*)p.out + (long long)lo * old + 2u * (hv * V + v0);       // of the chunk
  if (dst == 0) {                                // a padding sequence
    for (int t = g; t < len; t += 4) *(bf16_t*)(out + (long long)t * old) = 0;
    return;
  }
  f32x4 S[KS][2] = {};
  const long long head = (long long)hv * V * K + (long long)v0 * K + 8 * g;
  if (src != 0) {
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) S[x][h] = *(const f32x4*)(p.S + src * p.slot_stride + head + 32 * x + 4 * h);
  }
  const lds_t base = (lds_t)(char*)lds;
  const unsigned lds0 = (unsigned)(size_t)base + 1024u * w;
  const char* rows = (const char*)p.mixed + (long long)lo * ld;              // of the chunk that is requested next
  const char* chunk = (const char*)(work + ((long long)(lo / C + sn) * p.HV + hv));
  auto request = [&](int nv, int buf) {          // rows past the end: the last one again
    const unsigned at = lds0 + 16u * B::BUF * buf;
    const char *kb = rows + 2u * (p.H + hk) * K, *qb = rows + 2u * hk * K, *vb = rows + 2u * (2 * p.H * K + hv * V + part * COLS);
#pragma unroll
    for (int i = 0; i < TU / TH; ++i) {
      const int u = tid + i * TH, r = u / RB, b = (u % RB) ^ swz(r, RB);
      const unsigned off = (unsigned)min(r, nv - 1) * ld + 16u * b;
      to_lds(kb, off, at + 16u * i * TH);
      to_lds(qb, off, at + 16u * (TU + i * TH));
    }
    {
      const int r = tid / VB, b = (tid % VB) ^ swz(r, VB);
      to_lds(vb, (unsigned)min(r, nv - 1) * ld + 16u * b, at + 16u * B::VAT);
    }
#pragma unroll
    for (int i = 0; i * TH < B::CU; ++i)
      if (tid + i * TH < B::CU) to_lds(chunk, 16u * (tid + i * TH), at + 16u * (B::CAT + i * TH));
    rows += (long long)C * ld;
    chunk += (long long)p.HV * sizeof(Coef);
  };
  unsigned row_at[KS], col_at[KS];               // this lane's places in a tile, as in Walk::state
#pragma unroll
  for (int x = 0; x < KS; ++x) {
    row_at[x] = 16u * (n * RB + ((4 * x + g) ^ swz(n, RB)));
    col_at[x] = 16u * (qrow * RB + ((4 * x + (n & 3)) ^ swz(qrow, RB)));
  }
  if (nc > 0) request(min(C, len), 0);
  auto step = [&](int c, auto half) {             // the buffer a constant: every place in LDS is a register and an offset
    constexpr int BUF = decltype(half)::value;
    const int left = len - c * C;
    // chunk c has landed: after its loads came the stores of the chunk before
    if (c > 0) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    end_step();
    if (left > C) request(min(C, left - C), 1 - BUF);
    const lds_t kt = base + 16u * B::BUF * BUF, qt = kt + 16u * TU;
    const Coef& ck = *(const Coef*)(lds + B::BUF * BUF + B::CAT);
    f32x4 ks[2] = {}, qs[2] = {};
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      bf16x8 kf[2], qf[2], sh, sl;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kf[i] = at16(kt + row_at[x] + 256u * i * RB);
        qf[i] = at16(qt + row_at[x] + 256u * i * RB);
      }
      split8(S[x][0], S[x][1], sh, sl);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = mf(kf[i], sh, ks[i]);
        qs[i] = mf(qf[i], sh, qs[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = mf(kf[i], sl, ks[i]);
        qs[i] = mf(qf[i], sl, qs[i]);
      }
    }
    bf16x8 u[3];
    {
      f32x4 r[2], U[2] = {};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 16 * i + qrow;
        const s16x4 q = quad(kt + 16u * (B::VAT + row * VB + ((2 * w + ((n & 3) >> 1)) ^ swz(row, VB))) + 8u * (n & 1));
        const f32x4 cc = *(const f32x4*)&ck.c[16 * i + 4 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[i][e] = fmaf(-cc[e], ks[i][e], bf2f((bf16_t)q[e]));
        qs[i] *= *(const f32x4*)&ck.d[16 * i + 4 * g];
      }
      bf16x8 rp[3];
      split8(r[0], r[1], rp[0], rp[1], &rp[2]);
      chunk_product(operand(ck.t0, ck.t1, l), rp, U);
      split8(U[0], U[1], u[0], u[1], &u[2]);
      const bf16x8 rw[2] = {rp[0], rp[1]};
      chunk_product(operand(ck.w0, ck.w1, l), rw, qs);
    }
    const float last = ck.last[0];
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const s16x4 k0 = quad(kt + col_at[x] + 8u * h), k1 = quad(kt + col_at[x] + 256u * RB + 8u * h);
        const bf16x8 kT = __builtin_bit_cast(bf16x8, __builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7));
        S[x][h] *= last;
#pragma unroll
        for (int i = 0; i < 3; ++i) S[x][h] = mf(kT, u[i], S[x][h]);
      }
    if (left > C) {                              // eight stores, which the next step's wait counts
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = pk_bf16_kept(qs[i >> 1][2 * (i & 1)], qs[i >> 1][2 * (i & 1) + 1]);
        bf16_t* to = (bf16_t*)(out + (16 * (i >> 1) + 4 * g + 2 * (i & 1)) * old);
        to[0] = (bf16_t)two;
        *(bf16_t*)((char*)to + old) = (bf16_t)(two >> 16);
      }
    } else {
      unsigned at[8];
      store_places(at, old, 0, g);
      store_chunk(out, at, qs, g, left);
    }
    out += (long long)C * old;
  };
  for (int c = 0; c < nc; c += 2) {
    step(c, std::integral_constant<int, 0>());
    if (c + 1 < nc) step(c + 1, std::integral_constant<int, 1>());
  }
#pragma unroll
  for (int x = 0; x < KS; ++x)
#pragma unroll
    for (int h = 0; h < 2; ++h) *(f32x4*)(p.S + dst * p.slot_stride + head + 32 * x + 4 * h) = S[x][h];
}

// The walk's LDS is more than a kernel may have unasked: asked for once on each device, and again where that failed.
template <int K, int V> bool walk_lds() {
  static std::atomic<bool> had[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const bool known = dev >= 0 && dev < 64;
  if (known && had[dev].load(std::memory_order_relaxed)) return true;
  if (hipFuncSetAttribute((const void*)walk_kernel<K, V>, hipFuncAttributeMaxDynamicSharedMemorySize,
                          Tiles<K>::BYTES) != hipSuccess)
    return false;
  if (known) had[dev].store(true, std::memory_order_relaxed);
  return true;
}

template <int K, int V>
int prefill(const lq_delta* d, const lq_seqs* s, Coef* work, hipStream_t st) {
  typedef Tiles<K> T;
  typedef Pair<K, 4> P;
  if (!walk_lds<K, V>()) return LQ_ERR_HIP;
  int* order = (int*)(work + seq_runs<C>(s) * d->HV);
  chunk_kernel<K><<<(unsigned)((seq_runs<C>(s) * d->HV + CHUNKS - 1) / CHUNKS) + 1, 64 * CHUNKS, 0, st>>>(*d, *s, work, order);
  if (hipGetLastError() != hipSuccess) return LQ_ERR_HIP;
  auto grid = [&](int parts) { return (unsigned)place_grid((long long)s->N * d->H, d->HV / d->H * parts); };
  // Up to half a CU for every 16 rows the walk spreads each over eight waves (0.67 us a chunk, one workgroup a CU); with more
  // of them, one (1.2 to 2.3 us, several a CU).  Eight | one, both kernels, 2048 tokens a sequence in the mean, 128 x 128 (random
  // cuts: the mean of two draws):
  //   times 16 rows   256 (1 x 32 heads)  384 (6 x 8)  512 (2 x 32)  512 (8 x 8)  640 (10 x 8)  768 (3 x 32)  1024 (4 x 32)
  //   equal lengths        70 | 106        112 | 110    118 | 115     114 | 111    162 | 116     167 | 127     213 | 144 us
  //   random cuts          66 | 105        179 | 328    115 | 164     126 | 204    172 | 294     165 | 222     218 | 264
  // 16 heads of 64 x 64: 512 (8 sequences) 113 | 94, 121 | 160; 768 160 | 105, 177 | 198; 1024 212 | 127, 230 | 217.
  // Lengths are known on the device only.  Up to twice the CUs eight waves lose little at equal lengths (3%; 64 x 64: 20%) and
  // gain more at others.  Above, where a CU takes a third workgroup in turn, neither is right for all: equal lengths lose 31 to
  // 67% by eight waves, random cuts up to 70% by one.  One it is there: what it loses, the CUs that wait for the longest
  // sequences, shrinks with more of them (71% at 640, 15 to 21% at 1024).
  if ((long long)s->N * d->HV * (V / 16) <= 2 * lq_seq_cus())
    walk_kernel<K, V><<<grid(V / 16), 64 * (ROLES + SERVICE), T::BYTES, st>>>(*d, *s, work, order);
  else
    lone_kernel<K, V, 4><<<grid(V / 64), 256, P::BYTES, st>>>(*d, *s, work, order);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
}

}  // namespace

__attribute__((visibility("hidden"))) bool lq_prefill_fits(const lq_delta* d, const lq_seqs* s) {
  return (seq_runs<C>(s) + 8) * d->HV <= 0x7fffffffll && ((long long)s->N * d->HV + 8) * 8 <= 0x7fffffffll &&
         d->mixed_ld <= (1 << 24);
}

extern "C" long long lq_delta_workspace(const lq_delta* d, const lq_seqs* s) {
  if (lq_delta_check(d, s, 1) || s->N == 0) return 0;
  return seq_runs<C>(s) * d->HV * (long long)sizeof(Coef) + 4ll * s->N;
}

extern "C" int lq_delta_prefill(const lq_delta* d, const lq_seqs* s, void* work, long long work_bytes, void* stream) {
  if (int rc = lq_delta_check(d, s, 1)) return rc;
  if (s->N == 0) return LQ_OK;
  const long long need = lq_delta_workspace(d, s);
  if (need > 0 && (!work || ((uintptr_t)work & 15) || work_bytes < need)) return LQ_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (d->K == 128) return prefill<128, 128>(d, s, (Coef*)work, st);
  if (d->V == 128) return prefill<64, 128>(d, s, (Coef*)work, st);
  return prefill<64, 64>(d, s, (Coef*)work, st);
}
