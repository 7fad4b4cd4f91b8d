// The norms around a block: the gated norm after it and the residual add with the norm before the next (lq_gated_norm,
// lq_add_norm).  One pass: a row's elements stay in registers between the sum of squares (fp32) and the scaled result, so
// every input is read once and every output written once; both are bound by memory.
//
// A row is held by LANES threads (8 to 256), CH groups of VEC elements each, groups of one thread LANES * VEC apart so that a
// load instruction covers consecutive bytes.  LANES <= 64 reduces by lane exchanges, above that through LDS.
//
// Measured: gated, 32768 rows of 32 heads of 128, 140 us (805 MB: 5.7 TB/s); add, 16385 rows of 2048, 46.6 us (268 MB:
// 5.8 TB/s), both past a large copy's 4.9; the hints that calls larger than the shared cache give (ONCE) are 2 and 6% of
// that.  64 rows take 2.9 us, a launch and a load.  Not at that rate: rows of 513 to 1024 elements, where half the threads
// of a row have none (16384 rows of 1024: 3.8 and 4.6 TB/s), and 2-byte loads (of 2049: 1.9 and 2.2).
#include "lq_seq.h"

namespace {

constexpr int TH = 256;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ONCE: by the hint that nothing here or soon reads these bytes again
template <int VEC, bool ONCE> __device__ __forceinline__ void load_elems(const bf16_t* p, float* f) {
  if constexpr (VEC == 8) {
    u32x4 w;
    if (ONCE) w = __builtin_nontemporal_load((const u32x4*)p);
    else w = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = bf_lo(w[i]); f[2 * i + 1] = bf_hi(w[i]); }
  } else {
    f[0] = bf2f(*p);
  }
}
template <int VEC, bool ONCE> __device__ __forceinline__ void store_elems(bf16_t* p, const float* f) {
  if constexpr (VEC == 8) {
    const u32x4 w = {pk_bf16(f[0], f[1]), pk_bf16(f[2], f[3]), pk_bf16(f[4], f[5]), pk_bf16(f[6], f[7])};
    if (ONCE) __builtin_nontemporal_store(w, (u32x4*)p);
    else *(u32x4*)p = w;
  } else {
    *p = f2bf(f[0]);
  }
}

// sum over the LANES threads of a row; every thread of the workgroup calls it
template <int LANES> __device__ __forceinline__ float row_sum(float x, float* lds) {
  x = sum8(x);
  if (LANES >= 16) x += dpp<DPP_MIRROR>(x);
  if (LANES >= 32) x = xor16_sum(x);
  if (LANES >= 64) x = xor32_sum(x);
  if (LANES > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0] + lds[1] + lds[2] + lds[3];
  }
  return x;
}

template <int VEC, int LANES, int CH, bool ADD, bool ONCE>
__global__ __launch_bounds__(TH) void norm_kernel(lq_norm p) {
  __shared__ float lds[TH / 64];
  const long long v = (long long)blockIdx.x * (TH / LANES) + threadIdx.x / LANES;     // vector: row * heads + head
  const bool live = v < (long long)p.rows * p.heads;
  const long long row = live ? v / p.heads : 0, hd = live ? v - row * p.heads : 0;
  const int lane = threadIdx.x & (LANES - 1);
  const bf16_t* x = (const bf16_t*)p.x + row * p.x_ld + hd * p.x_hd;
  const bf16_t* z = (const bf16_t*)p.z + row * p.z_ld + hd * p.z_hd;
  const long long o = row * p.o_ld + hd * p.o_hd;
  float f[CH][VEC], g[CH][VEC], sum = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int d = (i * LANES + lane) * VEC;
    if (live && d < p.D) {
      load_elems<VEC, ONCE>(x + d, f[i]);
      load_elems<VEC, ONCE>(z + d, g[i]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[i][e] = g[i][e] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (ADD) f[i][e] = fmaf(p.scale, g[i][e], f[i][e]);
      sum = fmaf(f[i][e], f[i][e], sum);
    }
  sum = row_sum<LANES>(sum, lds);
  const float inv = rsqrtf_rn(sum / (float)p.D + p.eps);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int d = (i * LANES + lane) * VEC;
    if (d >= p.D) break;
    float w[VEC], y[VEC];
    if (p.weight_bf16) {
      load_elems<VEC, false>((const bf16_t*)p.weight + d, w);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = ((const float*)p.weight)[d + e];
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      y[e] = f[i][e] * inv * (p.offset + w[e]);
      if (!ADD) y[e] *= p.act ? fast_sigmoid(g[i][e]) : g[i][e] * fast_sigmoid(g[i][e]);
    }
    if (ADD) store_elems<VEC, ONCE>((bf16_t*)p.res + o + d, f[i]);
    store_elems<VEC, ONCE>((bf16_t*)p.out + o + d, y);
  }
}

template <int VEC, int LANES, int CH, bool ADD, bool ONCE>
int launch(const lq_norm* p, hipStream_t s) {
  const long long vecs = (long long)p->rows * p->heads, per = TH / LANES, grid = (vecs + per - 1) / per;
  if (grid > 0x7fffffffll) return LQ_ERR_ARG;
  norm_kernel<VEC, LANES, CH, ADD, ONCE><<<(unsigned)grid, TH, 0, s>>>(*p);
  return hipGetLastError() == hipSuccess ? LQ_OK : LQ_ERR_HIP;
}

constexpr long long CACHED = 256ll << 20;        // of the cache that all XCDs share

template <bool ADD, bool ONCE>
int rows_of_8(const lq_norm* p, hipStream_t s) {
  const int D = p->D;
  if (D <= 64) return launch<8, 8, 1, ADD, ONCE>(p, s);
  if (D <= 128) return launch<8, 16, 1, ADD, ONCE>(p, s);
  if (D <= 256) return launch<8, 32, 1, ADD, ONCE>(p, s);
  if (D <= 512) return launch<8, 64, 1, ADD, ONCE>(p, s);
  if (D <= 2048) return launch<8, 256, 1, ADD, ONCE>(p, s);
  if (D <= 4096) return launch<8, 256, 2, ADD, ONCE>(p, s);
  if (D <= 8192) return launch<8, 256, 4, ADD, ONCE>(p, s);
  return launch<8, 256, 8, ADD, ONCE>(p, s);
}

template <bool ADD>
int norm(const lq_norm* p, hipStream_t s) {
  if (!p || p->rows < 0 || p->heads <= 0 || p->D <= 0 || p->D > 16384) return LQ_ERR_ARG;
  if ((p->act != 0 && p->act != 1) || (p->weight_bf16 != 0 && p->weight_bf16 != 1) || !(p->eps >= 0.f)) return LQ_ERR_ARG;
  if (p->rows == 0) return LQ_OK;
  if ((p->rows > 1 && p->o_ld < p->D) || (p->heads > 1 && p->o_hd < p->D)) return LQ_ERR_ARG;     // vectors of out overlap
  if (!p->x || !p->z || !p->weight || !p->out || (ADD && !p->res)) return LQ_ERR_ARG;
  const long long ld = p->x_ld | p->x_hd | p->z_ld | p->z_hd | p->o_ld | p->o_hd;
  const uintptr_t at = (uintptr_t)p->x | (uintptr_t)p->z | (uintptr_t)p->out | (uintptr_t)(ADD ? p->res : nullptr) |
                       (uintptr_t)(p->weight_bf16 ? p->weight : nullptr);
  const int D = p->D;
  if (D % 8 == 0 && ld % 8 == 0 && (at & 15) == 0) {     // 16-byte loads
    const long long bytes = 2ll * p->rows * p->heads * D * (ADD ? 4 : 3);
    return bytes > CACHED ? rows_of_8<ADD, true>(p, s) : rows_of_8<ADD, false>(p, s);
  }
  if (D <= 64) return launch<1, 16, 4, ADD, false>(p, s);
  if (D <= 256) return launch<1, 64, 4, ADD, false>(p, s);
  if (D <= 1024) return launch<1, 256, 4, ADD, false>(p, s);
  if (D <= 4096) return launch<1, 256, 16, ADD, false>(p, s);
  return launch<1, 256, 64, ADD, false>(p, s);
}

}  // namespace

extern "C" int lq_gated_norm(const lq_norm* p, void* stream) { return norm<false>(p, (hipStream_t)stream); }
extern "C" int lq_add_norm(const lq_norm* p, void* stream) { return norm<true>(p, (hipStream_t)stream); }
