// The gated delta rule over prompts, in chunks of C = 32 tokens on the matrix cores (lq_delta_prefill).
//
// With G_i the sum of the log-gates of a chunk's tokens up to i, k and q normalised, and S0 the state before the chunk,
//
//   A_ij = beta_i e^{G_i - G_j} k_i.k_j  (i > j),    T = (I + A)^-1 diag(beta)
//   U = T (V - diag(e^G) K S0^T)                                      the values the recurrence would append
//   O = diag(e^G) Q S0^T + P U,    P_ij = e^{G_i - G_j} q_i.k_j  (i >= j)
//   S = e^{G_C} S0 + U^T diag(e^{G_C - G}) K
//
// T and P do not depend on the state: a first kernel forms them for all chunks at once, and a second walks each sequence's
// chunks with the state in registers.  Rows of S (value channels) do not meet, so a head's rows are spread over waves.
//
// Rounding.  The raw keys, queries and values are bf16 and enter the products as they are; their norms, decays and beta are
// fp32 factors of rows and columns of fp32 sums, never folded into an operand.  fp32 operands (S, V - ..., T, P, U) are
// carried as two bf16 halves (hi + lo, 2^-17 of an element is lost), their products as the two or three significant ones: the
// state is accurate to a few 1e-6, where single bf16 operands would leave 3e-3, and the outputs keep their digits where
// their terms cancel (a query nearly orthogonal to the state, equal keys in a chunk).
#include "lq_seq.h"

__attribute__((visibility("hidden"))) int lq_check_delta(const lq_delta* d, const lq_seqs* s);

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int C = 32;                  // tokens of a chunk

// What the first kernel leaves for a chunk of a value head.  The matrices are operands as a lane takes them: lane l of a row
// tile holds row l % 16 at the columns 4 g .. 4 g + 3 and 16 + 4 g .. (g = l / 16), the order in which a lane of a product's
// result holds its rows, so that results are the next product's operands without moving between lanes.
struct alignas(16) Chunk {
  bf16x8 t[2][2][64];                  // T: row tile, high and low half
  bf16x8 p[2][2][64];                  // P, likewise
  float c[C];                          // e^G / |k|: of the rows of K S
  float d[C];                          // scale e^G / |q|: of the rows of Q S
  float e[C];                          // e^{G_C - G} / |k|: of the rows of U for the state
  float last[4];                       // e^{G_C}
};
static_assert(sizeof(Chunk) % 16 == 0, "moved by 16-byte words");

__device__ __forceinline__ f32x4 mf(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// eight fp32 values as two bf16 halves
__device__ __forceinline__ void split8(const f32x4& x, const f32x4& y, bf16x8& hi, bf16x8& lo) {
  const float f[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = pk_bf16_kept(f[2 * i], f[2 * i + 1]);
    l[i] = pk_bf16(f[2 * i] - bf_lo(h[i]), f[2 * i + 1] - bf_hi(h[i]));
  }
  hi = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
  lo = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
}

// ---- T and P of every chunk --------------------------------------------------------------------------------------------
// One wave a chunk and value head.  (I + A)^-1 by forward substitution in its two diagonal blocks of 16 (a column a lane) and
// -T11 A10 T00 below them by fp32 matrix instructions: substitution stays accurate where powers of A would not (equal keys
// without decay make them grow like binomials).
template <int K>
__global__ __launch_bounds__(64) void chunk_kernel(lq_delta p, lq_seqs s, Chunk* __restrict__ work) {
  constexpr int KS = K / 32, LD = C + 4;
  __shared__ float m[C][LD];                     // a 32 x 32 matrix, row by row
  __shared__ float glo[C], ghi[C], bet[C], rk[C], rq[C];
  const int hv = blockIdx.x % p.HV;
  const SeqRun r = seq_run<C>(s, blockIdx.x / p.HV);
  const int t0 = r.lo + r.j * C, nv = min(C, r.hi - t0);
  if (nv <= 0 || seq_dst(s, r.n, p.NS) == 0) return;
  const int l = threadIdx.x, n = l & 15, g = l >> 4, hk = hv / (p.HV / p.H);
  bf16x8 kf[2][KS], qf[2][KS];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = 16 * i + n;
    const uint4* row = (const uint4*)((const bf16_t*)p.mixed + (t0 + min(t, nv - 1)) * p.mixed_ld + hk * K) + g;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      qf[i][x] = __builtin_bit_cast(bf16x8, keep4(row[4 * x], t < nv));
      kf[i][x] = __builtin_bit_cast(bf16x8, keep4(row[4 * x + p.H * K / 8], t < nv));
    }
  }
  // gates: token l % 32 of each half wave; the sum over the chunk in fp64, kept as two floats, so that the difference of
  // two large sums is as good as the gates between them.  A gate under -128 has the same exponential as -128: zero.
  {
    const int t = l & 31;
    const bool live = t < nv;
    const long long row = t0 + min(t, nv - 1);
    const float x = bf2f(((const bf16_t*)p.a)[row * p.a_ld + hv]) + gate_param(p.dt_bias, p.gate_bf16 & 2, hv);
    float gate = -expf(gate_param(p.A_log, p.gate_bf16 & 1, hv)) * softplus20f(x);
    gate = live ? (gate < -128.f ? -128.f : gate) : 0.f;
    const float b = bf2f(((const bf16_t*)p.b)[row * p.b_ld + hv]);
    double sum = gate;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up(sum, o, 32);
      if (t >= o) sum += y;
    }
    if (l < 32) {
      ghi[t] = (float)sum;
      glo[t] = (float)(sum - (double)(float)sum);
      bet[t] = live ? 1.0f / (1.0f + expf(-b)) : 0.f;
    }
  }
  // Gram matrices: tiles (0, 0), (1, 0), (1, 1)
  f32x4 kk[3] = {}, qk[3] = {}, qq[2] = {};
#pragma unroll
  for (int x = 0; x < KS; ++x) {
    kk[0] = mf(kf[0][x], kf[0][x], kk[0]); kk[1] = mf(kf[1][x], kf[0][x], kk[1]); kk[2] = mf(kf[1][x], kf[1][x], kk[2]);
    qk[0] = mf(qf[0][x], kf[0][x], qk[0]); qk[1] = mf(qf[1][x], kf[0][x], qk[1]); qk[2] = mf(qf[1][x], kf[1][x], qk[2]);
    qq[0] = mf(qf[0][x], qf[0][x], qq[0]); qq[1] = mf(qf[1][x], qf[1][x], qq[1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)                    // the diagonals: squared norms of row 4 g + i
    if (n == 4 * g + i) {
      rk[n] = rsqrtf_rn(kk[0][i] + 1e-6f); rk[16 + n] = rsqrtf_rn(kk[2][i] + 1e-6f);
      rq[n] = rsqrtf_rn(qq[0][i] + 1e-6f); rq[16 + n] = rsqrtf_rn(qq[1][i] + 1e-6f);
    }
  __syncthreads();
  // A into LDS, P kept
#pragma unroll
  for (int x = 0; x < 3; ++x) {
    const int ri = 16 * (x > 0), cj = 16 * (x > 1) + n;
    const float hj = ghi[cj], lj = glo[cj], kj = rk[cj];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = ri + 4 * g + i;
      const float dec = __expf((ghi[row] - hj) + (glo[row] - lj)) * kj;
      const bool below = x == 1 || 4 * g + i > n, diag = x != 1 && 4 * g + i == n;
      m[row][cj] = below ? bet[row] * rk[row] * dec * kk[x][i] : 0.f;
      qk[x][i] = below || diag ? rq[row] * p.scale * dec * qk[x][i] : 0.f;
    }
  }
  __syncthreads();
  // inverses of the diagonal blocks: lane (block, column), rows top down
  {
    const int blk = 16 * (g & 1);
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float acc = j == n ? 1.f : 0.f;
#pragma unroll
      for (int i4 = 0; i4 < (j + 3) / 4; ++i4) {
        const float4 a = *(const float4*)&m[blk + j][blk + 4 * i4];
        const float av[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * i4 + i < j) acc = fmaf(-av[i], x[4 * i4 + i], acc);
      }
      x[j] = acc;
    }
    __syncthreads();
    if (l < 32) {
#pragma unroll
      for (int j = 0; j < 16; ++j) m[blk + j][blk + n] = x[j];
    }
  }
  __syncthreads();
  f32x4 y = {}, z = {};
  {
    const f32x4 a10 = *(const f32x4*)&m[16 + n][4 * g], t11 = *(const f32x4*)&m[16 + n][16 + 4 * g];
#pragma unroll
    for (int i = 0; i < 4; ++i) y = __builtin_amdgcn_mfma_f32_16x16x4f32(a10[i], m[4 * g + i][n], y, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) z = __builtin_amdgcn_mfma_f32_16x16x4f32(-t11[i], y[i], z, 0, 0, 0);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) m[16 + 4 * g + i][n] = z[i];
  __syncthreads();
  Chunk& out = work[blockIdx.x];
  const f32x4 zero = {};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f32x4 a = *(const f32x4*)&m[16 * i + n][4 * g], b = i ? *(const f32x4*)&m[16 + n][16 + 4 * g] : zero;
    a *= *(const f32x4*)&bet[4 * g];
    b *= *(const f32x4*)&bet[16 + 4 * g];
    split8(a, b, out.t[i][0][l], out.t[i][1][l]);
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 3; ++x)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[16 * (x > 0) + 4 * g + i][16 * (x > 1) + n] = qk[x][i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x4 a = *(const f32x4*)&m[16 * i + n][4 * g], b = i ? *(const f32x4*)&m[16 + n][16 + 4 * g] : zero;
    split8(a, b, out.p[i][0][l], out.p[i][1][l]);
  }
  if (l < C) {
    const float e = __expf(ghi[l] + glo[l]);
    out.c[l] = e * rk[l];
    out.d[l] = e * rq[l] * p.scale;
    out.e[l] = __expf((ghi[C - 1] - ghi[l]) + (glo[C - 1] - glo[l])) * rk[l];
    if (l < 4) out.last[l] = __expf(ghi[C - 1] + glo[C - 1]);
  }
}

// ---- the walk over a sequence's chunks -----------------------------------------------------------------------------------
// A wave holds 16 NT rows of S as result tiles of K U: lane (n, g) the rows v = n, channels 32 x + 8 g .. + 7 in its register
// pairs (x, 0), (x, 1).  The same registers are the operand of K S and Q S, and K S's and T R's results that of the next
// product, so the chain S -> R -> U -> S stays in the lane's registers; only K, Q, T and P come from LDS, where the waves
// of the workgroup share them.  K^T is read by the transposing LDS read.  The next chunk's tiles are requested before the
// current chunk's products and written to the other half of LDS after them.
template <int K, int V, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void walk_kernel(lq_delta p, lq_seqs s, const Chunk* __restrict__ work) {
  constexpr int KS = K / 32, TH = 64 * NW, PARTS = V / (16 * NT * NW);
  constexpr int RB = K / 8, TU = C * RB;         // 16-byte blocks of a row of K, of a tile
  constexpr int WU = sizeof(Chunk) / 16;
  constexpr int NK = TU / TH, NWK = (WU + TH - 1) / TH;
  static_assert(TU % TH == 0, "whole tiles by the workgroup");
  __shared__ u32x4 lds[2][2 * TU + WU];
  const int part = blockIdx.x % PARTS, hn = blockIdx.x / PARTS, sn = hn / p.HV, hv = hn - sn * p.HV;
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, n = l & 15, g = l >> 4, hk = hv / (p.HV / p.H);
  const int lo = seq_at(s, sn), hi = max(lo, seq_at(s, sn + 1)), len = hi - lo;
  const int dst = seq_dst(s, sn, p.NS), src = seq_src(s, sn, p.NS);
  const int v0 = (part * NW + w) * 16 * NT + n;
  const long long old = (long long)p.HV * V;
  bf16_t* out = (bf16_t*)p.out + lo * old + (long long)hv * V + v0;
  if (dst == 0) {
    for (int t = g; t < len; t += 4)
#pragma unroll
      for (int y = 0; y < NT; ++y) out[t * old + 16 * y] = 0;
    return;
  }
  f32x4 S[KS][2][NT] = {};
  const long long head = (long long)hv * V * K + (long long)v0 * K + 8 * g;
  if (src != 0) {
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int y = 0; y < NT; ++y)
          S[x][h][y] = *(const f32x4*)(p.S + src * p.slot_stride + head + 16 * y * K + 32 * x + 4 * h);
  }
  // a block of row r sits at its place xor the row, so that 16 rows' blocks of one column meet different banks
  auto place = [](int r, int b) { return r * RB + (b ^ (RB == 16 ? (r & 15) : ((r >> 1) & 7))); };

  const bf16_t* rows = (const bf16_t*)p.mixed + lo * p.mixed_ld;
  const Chunk* wrk = work + ((long long)(lo / C + sn) * p.HV + hv);
  u32x4 kq[2][NK], wk[NWK];
  bf16_t vn[NT][8];
  auto request = [&](int c) {
    const int nv = min(C, len - c * C);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int u = tid + i * TH, r = u / RB, b = u % RB;
      const bf16_t* q = rows + (c * C + min(r, nv - 1)) * p.mixed_ld + hk * K + 8 * b;
      const unsigned mask = r < nv ? 0xffffffffu : 0u;
      kq[0][i] = *(const u32x4*)(q + p.H * K) & mask;
      kq[1][i] = *(const u32x4*)q & mask;
    }
    const u32x4* f = (const u32x4*)(wrk + (long long)c * p.HV);
#pragma unroll
    for (int i = 0; i < NWK; ++i)
      wk[i] = f[min(tid + i * TH, WU - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = 16 * (i >> 2) + 4 * g + (i & 3);
      const bf16_t* q = rows + (c * C + min(t, nv - 1)) * p.mixed_ld + 2 * p.H * K + hv * V + v0;
#pragma unroll
      for (int y = 0; y < NT; ++y) vn[y][i] = t < nv ? q[16 * y] : (bf16_t)0;
    }
  };
  auto deliver = [&](int buf) {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int u = tid + i * TH;
      lds[buf][place(u / RB, u % RB)] = kq[0][i];
      lds[buf][TU + place(u / RB, u % RB)] = kq[1][i];
    }
#pragma unroll
    for (int i = 0; i < NWK; ++i)
      if (tid + i * TH < WU) lds[buf][2 * TU + tid + i * TH] = wk[i];
  };
  const int nc = (len + C - 1) / C;
  if (nc > 0) {
    request(0);
    deliver(0);
    __syncthreads();
  }
  for (int c = 0; c < nc; ++c) {
    const int buf = c & 1;
    f32x4 val[2][NT];
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
      for (int i = 0; i < 8; ++i) val[i >> 2][y][i & 3] = bf2f(vn[y][i]);
    if (c + 1 < nc) request(c + 1);
    const u32x4* kt = lds[buf];
    const Chunk& ck = *(const Chunk*)(lds[buf] + 2 * TU);
    f32x4 ks[2][NT] = {}, qs[2][NT] = {};
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      bf16x8 kf[2], qf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kf[i] = __builtin_bit_cast(bf16x8, kt[place(16 * i + n, 4 * x + g)]);
        qf[i] = __builtin_bit_cast(bf16x8, kt[TU + place(16 * i + n, 4 * x + g)]);
      }
#pragma unroll
      for (int y = 0; y < NT; ++y) {
        bf16x8 sh, sl;
        split8(S[x][0][y], S[x][1][y], sh, sl);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ks[i][y] = mf(kf[i], sh, ks[i][y]);
          qs[i][y] = mf(qf[i], sh, qs[i][y]);
          ks[i][y] = mf(kf[i], sl, ks[i][y]);
          qs[i][y] = mf(qf[i], sl, qs[i][y]);
        }
      }
    }
    f32x4 U[2][NT];
#pragma unroll
    for (int y = 0; y < NT; ++y) {
#pragma unroll
      for (int i = 0; i < 2; ++i) val[i][y] -= *(const f32x4*)&ck.c[16 * i + 4 * g] * ks[i][y];
      bf16x8 rh, rl;
      split8(val[0][y], val[1][y], rh, rl);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4 u = {};
        u = mf(ck.t[i][0][l], rh, u);
        u = mf(ck.t[i][0][l], rl, u);
        U[i][y] = mf(ck.t[i][1][l], rh, u);
      }
    }
#pragma unroll
    for (int y = 0; y < NT; ++y) {
      bf16x8 uh, ul;
      split8(U[0][y], U[1][y], uh, ul);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4 o = *(const f32x4*)&ck.d[16 * i + 4 * g] * qs[i][y];
        o = mf(ck.p[i][0][l], uh, o);
        o = mf(ck.p[i][0][l], ul, o);
        o = mf(ck.p[i][1][l], uh, o);
        const int t = c * C + 16 * i + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t + e < len) out[(t + e) * old + 16 * y] = f2bf(o[e]);
      }
    }
    const float last = ck.last[0];
    bf16x8 uh[NT], ul[NT];
#pragma unroll
    for (int y = 0; y < NT; ++y)
      split8(U[0][y] * *(const f32x4*)&ck.e[4 * g], U[1][y] * *(const f32x4*)&ck.e[16 + 4 * g], uh[y], ul[y]);
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s16x4 k2[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {            // channels 32 x + 8 q + 4 h .. of row 4 g + n / 4, q = n % 4
          const int row = 16 * i + 4 * g + (n >> 2);
          const char* at = (const char*)(kt + place(row, 4 * x + (n & 3))) + 8 * h;
          k2[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        }
        const bf16x8 kT = __builtin_bit_cast(bf16x8, __builtin_shufflevector(k2[0], k2[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int y = 0; y < NT; ++y) {
          f32x4 a = S[x][h][y] * last;
          a = mf(kT, uh[y], a);
          S[x][h][y] = mf(kT, ul[y], a);
        }
      }
    if (c + 1 < nc) deliver(buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < KS; ++x)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int y = 0; y < NT; ++y)
        *(f32x4*)(p.S + dst * p.slot_stride + head + 16 * y * K + 32 * x + 4 * h) = S[x][h][y];
}

int num_cus() {
  static int cache[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cache[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

template <int K, int V, int NT, int NW>
void launch_walk(const lq_delta* d, const lq_seqs* s, const Chunk* work, hipStream_t st) {
  const unsigned grid = (unsigned)s->N * d->HV * (V / (16 * NT * NW));
  walk_kernel<K, V, NT, NW><<<grid, 64 * NW, 0, st>>>(*d, *s, work);
}

template <int K, int V>
int prefill(const lq_delta* d, const lq_seqs* s, Chunk* work, hipStream_t st) {
  if (s->T > 0) {
    chunk_kernel<K><<<(unsigned)(seq_runs<C>(s) * d->HV), 64, 0, st>>>(*d, *s, work);
    if (hipGetLastError() != hipSuccess) return LQ_ERR_HIP;
  }
  const long long heads = (long long)s->N * d->HV;
  if (heads * (V / 16) <= 4ll * num_cus()) launch_walk<K, V, 1, 1>(d, s, work, st);
  else launch_walk<K, V, 2, V / 32>(d, s, work, st);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
}

}  // namespace

extern "C" long long lq_delta_workspace(const lq_delta* d, const lq_seqs* s) {
  if (!d || d->kda || lq_check_delta(d, s) || s->N == 0 || s->T == 0) return 0;
  return seq_runs<C>(s) * d->HV * (long long)sizeof(Chunk);
}

extern "C" int lq_delta_prefill(const lq_delta* d, const lq_seqs* s, void* work, long long work_bytes, void* stream) {
  if (int rc = lq_check_delta(d, s)) return rc;
  if (d->kda) return LQ_ERR_ARG;
  if (s->N == 0) return LQ_OK;
  if (seq_runs<C>(s) * d->HV > 0x7fffffffll || (long long)s->N * d->HV * 8 > 0x7fffffffll) return LQ_ERR_ARG;
  const long long need = lq_delta_workspace(d, s);
  if (need > 0 && (!work || ((uintptr_t)work & 15) || work_bytes < need)) return LQ_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (d->K == 128) return prefill<128, 128>(d, s, (Chunk*)work, st);
  if (d->V == 128) return prefill<64, 128>(d, s, (Chunk*)work, st);
  return prefill<64, 64>(d, s, (Chunk*)work, st);
}
