// Appending to and reading from the paged 8-bit cache (interface in gb_paged.h).
//
// A page of a head is one block's: it sees all numbers that share a scale, and nobody else writes to the page, so nothing here needs an atomic or a second pass over
// memory.  The block also rotates the query heads of its key head, which reads every row of the input once and looks positions up where they are known.
#include <algorithm>

#include "paged_util.cuh"

namespace gb {

// Smallest power of two s with 127 * s >= amax, at least 2^-120.  amax = 1.f * 2^x: s = 2^(x-6) where 1.f <= 127/64, which is a fraction of at most 63/64.
__device__ __forceinline__ float pg_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 127 - 120) << 23);
}
// 1 / s of a power of two between 2^-120 and 2^122
__device__ __forceinline__ float pg_inv(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

constexpr int PA_THREADS = 256;

// Blocks: (sequence, page of its new tokens, key head).  HD / 16 lanes take a row: each the 8 pairs 8c ... 8c + 7 that a rotation turns, as two vectors of 8 numbers.
template <typename T, int HD, int ROPE>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const __grid_constant__ gb_paged a, const T* __restrict__ qkv, long long ld, int H,
                                                                  T* __restrict__ q_out, long long ld_q, const float* __restrict__ qw,
                                                                  const float* __restrict__ kw, float eps, const float* __restrict__ cs, int positions) {
  constexpr int LPR = HD / 16, RPP = PA_THREADS / LPR, PASSES = (PG + RPP - 1) / RPP, LDV = PG + 8;
  __shared__ __align__(16) signed char sv[HD * LDV];
  __shared__ float red[2][PA_THREADS / 32];
  pdl_wait();
  const int b = blockIdx.z, g = blockIdx.y, G = H / a.KV;
  const PgSeq s = pg_seq(a, b);
  const int p = s.start / PG + (int)blockIdx.x;
  const int lo = max(s.start, p * PG), hi = min(s.start + s.n, (p + 1) * PG);      // positions of this block
  if (lo >= hi) return;
  if (hi > positions) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, ST_BAD_ARGUMENT);
    return;
  }
  const int id = pg_page(a, b, p);
  const int n = hi - lo, off = lo - p * PG;
  const long long row0 = s.first + (lo - s.start);
  const int c = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  const int o0 = ROPE == 0 ? 16 * c : 8 * c, o1 = ROPE == 0 ? 16 * c + 8 : HD / 2 + 8 * c;

  // x: the two vectors of a row; normed and turned
  auto turn = [&](float* x, const float* w, int pos) {
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      float inv = rsqrtf(ss / (float)HD + eps);
      if (!isfinite(inv)) inv = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) { x[i] *= inv * w[o0 + i]; x[8 + i] *= inv * w[o1 + i]; }
    }
    const float4* cp = reinterpret_cast<const float4*>(cs + (long long)pos * HD + 8 * c);
    const float4* sp = reinterpret_cast<const float4*>(cs + (long long)pos * HD + HD / 2 + 8 * c);
    const float4 ca = cp[0], cb = cp[1], sa = sp[0], sb = sp[1];
    const float co[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w}, si[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {                         // products and differences rounded one by one, as the definition has them
      const int i0 = ROPE == 0 ? 2 * i : i, i1 = ROPE == 0 ? 2 * i + 1 : 8 + i;
      const float u = x[i0], v = x[i1];
      x[i0] = __fsub_rn(__fmul_rn(u, co[i]), __fmul_rn(v, si[i]));
      x[i1] = __fadd_rn(__fmul_rn(u, si[i]), __fmul_rn(v, co[i]));
    }
  };

  float ky[PASSES][16], vy[PASSES][16], km = 0.f, vm = 0.f;
  bool bad = false;
#pragma unroll
  for (int ps = 0; ps < PASSES; ++ps) {
    const int r = ps * RPP + r0;
    const bool on = r < n;
    const T* src = qkv + (row0 + (on ? r : 0)) * ld;
    const T *kp = src + (long long)(H + g) * HD, *vp = src + (long long)(H + a.KV + g) * HD;
    pg_load8(kp + o0, ky[ps]);
    pg_load8(kp + o1, ky[ps] + 8);
    pg_load8(vp + o0, vy[ps]);
    pg_load8(vp + o1, vy[ps] + 8);
    turn(ky[ps], kw, lo + (on ? r : 0));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (!(fabsf(ky[ps][i]) <= 3.402823466e38f)) { ky[ps][i] = 0.f; bad |= on; }
      if (!(fabsf(vy[ps][i]) <= 3.402823466e38f)) { vy[ps][i] = 0.f; bad |= on; }
      if (on) { km = fmaxf(km, fabsf(ky[ps][i])); vm = fmaxf(vm, fabsf(vy[ps][i])); }
    }
  }
  if (bad) atomicCAS(a.status, 0, ST_NOT_FINITE);
  km = warp_max(km);
  vm = warp_max(vm);
  if ((threadIdx.x & 31) == 0) { red[0][threadIdx.x >> 5] = km; red[1][threadIdx.x >> 5] = vm; }

  // the query heads while the maxima meet
  for (int i = r0; i < n * G; i += RPP) {
    const int t = i / G, h = g * G + i - t * G;
    float x[16];
    const T* src = qkv + (row0 + t) * ld + (long long)h * HD;
    pg_load8(src + o0, x);
    pg_load8(src + o1, x + 8);
    if (qw) {                                            // a row's lanes norm together: those past the end went home, so the mask is theirs
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) ss += x[k] * x[k];
      const unsigned mine = ((1u << LPR) - 1u) << ((threadIdx.x & 31) / LPR * LPR);
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(mine, ss, o);
      float inv = rsqrtf(ss / (float)HD + eps);
      if (!isfinite(inv)) inv = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) { x[k] *= inv * qw[o0 + k]; x[8 + k] *= inv * qw[o1 + k]; }
    }
    turn(x, nullptr, lo + t);
    T* dst = q_out + (row0 + t) * ld_q + (long long)h * HD;
    pg_store8(dst + o0, x);
    pg_store8(dst + o1, x + 8);
  }
  __syncthreads();
  if (id < 0) return;
  km = vm = 0.f;
#pragma unroll
  for (int w = 0; w < PA_THREADS / 32; ++w) { km = fmaxf(km, red[0][w]); vm = fmaxf(vm, red[1][w]); }
  const long long at = (long long)id * a.KV + g;
  signed char *kc = a.k + at * PG * HD, *vc = a.v + at * PG * HD;
  float ks = pg_scale(km), vs = pg_scale(vm);
  if (off > 0) {                                         // tokens of earlier calls share the page
    const float ko = a.ks[at], vo = a.vs[at];
    ks = fmaxf(ks, ko);
    vs = fmaxf(vs, vo);
    if (ks > ko) {
      const float r = ko * pg_inv(ks);
      for (int i = threadIdx.x; i < off * HD; i += PA_THREADS) kc[i] = (signed char)__float2int_rn((float)kc[i] * r);
    }
    if (vs > vo) {
      const float r = vo * pg_inv(vs);
      for (int i = threadIdx.x; i < off * HD; i += PA_THREADS) {
        signed char* q = vc + (i / off) * PG + i % off;
        *q = (signed char)__float2int_rn((float)*q * r);
      }
    }
    __syncthreads();                                     // the old scales are read
  }
  if (threadIdx.x == 0) { a.ks[at] = ks; a.vs[at] = vs; }
  const float ki = pg_inv(ks), vi = pg_inv(vs);
#pragma unroll
  for (int ps = 0; ps < PASSES; ++ps) {
    const int r = ps * RPP + r0;
    if (r >= n) continue;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i >> 2] |= (uint32_t)(__float2int_rn(ky[ps][i] * ki) & 255) << (8 * (i & 3));
    signed char* kr = kc + (off + r) * HD;
    *reinterpret_cast<uint2*>(kr + o0) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(kr + o1) = make_uint2(w[2], w[3]);
#pragma unroll
    for (int i = 0; i < 16; ++i) sv[((i < 8 ? o0 : o1 - 8) + i) * LDV + off + r] = (signed char)__float2int_rn(vy[ps][i] * vi);
  }
  __syncthreads();
  // columns off ... off + n - 1 of every dimension: whole groups of 8 tokens at once, the edges one by one
  const int g0 = off / 8, ng = (off + n + 7) / 8 - g0;
  for (int i = threadIdx.x; i < HD * ng; i += PA_THREADS) {
    const int d = i / ng, c0 = (g0 + i - d * ng) * 8;
    const signed char* src = sv + d * LDV + c0;
    signed char* dst = vc + d * PG + c0;
    if (c0 >= off && c0 + 8 <= off + n) {
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
    } else {
      for (int j = max(c0, off) - c0; j < min(c0 + 8, off + n) - c0; ++j) dst[j] = src[j];
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(PA_THREADS) paged_read_kernel(const __grid_constant__ gb_paged a, T* __restrict__ k_out, long long ld_k,
                                                                T* __restrict__ v_out, long long ld_v) {
  constexpr int CH = HD / 16, LDV = PG + 16;
  __shared__ __align__(16) signed char sv[HD * LDV];
  pdl_wait();
  const int b = blockIdx.z, g = blockIdx.y;
  const PgSeq s = pg_seq(a, b);
  const int p = s.start / PG + (int)blockIdx.x;
  const int lo = max(s.start, p * PG), hi = min(s.start + s.n, (p + 1) * PG);
  if (lo >= hi) return;
  const int id = pg_page(a, b, p);
  if (id < 0) return;
  const int n = hi - lo, off = lo - p * PG;
  const long long row0 = s.first + (lo - s.start), at = (long long)id * a.KV + g;
  const signed char *kc = a.k + at * PG * HD, *vc = a.v + at * PG * HD;
  const float ks = a.ks[at], vs = a.vs[at];
  constexpr float top = PgTop<T>::value;
  for (int i = threadIdx.x; i < HD * 4; i += PA_THREADS)
    *reinterpret_cast<uint4*>(sv + (i >> 2) * LDV + (i & 3) * 16) = *reinterpret_cast<const uint4*>(vc + i * 16);
  __syncthreads();
  for (int i = threadIdx.x; i < n * CH; i += PA_THREADS) {
    const int t = i / CH, d0 = (i - t * CH) * 16;
    const uint4 u = *reinterpret_cast<const uint4*>(kc + (off + t) * HD + d0);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = fminf(fmaxf((float)(signed char)(w[j >> 2] >> (8 * (j & 3))) * ks, -top), top);
    T* dk = k_out + (row0 + t) * ld_k + (long long)g * HD + d0;
    pg_store8(dk, x);
    pg_store8(dk + 8, x + 8);
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = fminf(fmaxf((float)sv[(d0 + j) * LDV + off + t] * vs, -top), top);
    T* dv = v_out + (row0 + t) * ld_v + (long long)g * HD + d0;
    pg_store8(dv, x);
    pg_store8(dv + 8, x + 8);
  }
}

}  // namespace gb

using namespace gb;

static bool gb_paged_rows_ok(const void* p, long long ld, long long width) {
  return p && !(reinterpret_cast<uintptr_t>(p) & 15) && ld % 8 == 0 && ld >= width;
}

#define GB_PAGED_TYPES(hd, bf, CALL)                                                                                      \
  do {                                                                                                                    \
    if (bf) { if (hd == 32) { CALL(__nv_bfloat16, 32); } else if (hd == 64) { CALL(__nv_bfloat16, 64); } else { CALL(__nv_bfloat16, 128); } } \
    else { if (hd == 32) { CALL(__half, 32); } else if (hd == 64) { CALL(__half, 64); } else { CALL(__half, 128); } }     \
  } while (0)

// Blocks along x: pages that max_new tokens can touch, wherever in a page they begin.
static int gb_paged_grid(const gb_paged* a, dim3* grid) {
  const int px = (int)std::min<long long>(((long long)a->max_new + 2 * GB_PAGE - 2) / GB_PAGE, a->W);
  if (a->KV > 65535 || a->B > 65535) return -3;
  *grid = dim3(px, a->KV, a->B);
  return 0;
}

extern "C" int gb_paged_append(const gb_paged* a, const void* qkv, long long ld_qkv, int H, void* q_out, long long ld_q, const float* qw,
                               const float* kw, float eps, const float* cos_sin, int positions, int rope_type, cudaStream_t st) {
  if (const int rc = gb_paged_check(a)) return rc;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  if (H <= 0 || H % a->KV || !cos_sin || (reinterpret_cast<uintptr_t>(cos_sin) & 15) || positions <= 0 || (rope_type != 0 && rope_type != 1)) return -1;
  if (!gb_paged_rows_ok(qkv, ld_qkv, (long long)(H + 2 * a->KV) * a->hd) || !gb_paged_rows_ok(q_out, ld_q, (long long)H * a->hd)) return -4;
  dim3 grid;
  if (const int rc = gb_paged_grid(a, &grid)) return rc;
#define CALL(T, HD) \
  GB_PDL_LAUNCH((paged_append_kernel<T, HD, ROPE>), grid, dim3(PA_THREADS), st, *a, (const T*)qkv, ld_qkv, H, (T*)q_out, ld_q, qw, kw, eps, cos_sin, positions)
  if (rope_type == 0) {
    constexpr int ROPE = 0;
    GB_PAGED_TYPES(a->hd, a->is_bf16, CALL);
  } else {
    constexpr int ROPE = 1;
    GB_PAGED_TYPES(a->hd, a->is_bf16, CALL);
  }
#undef CALL
  return gb_launch_rc();
}

extern "C" int gb_paged_read(const gb_paged* a, void* k_out, long long ld_k, void* v_out, long long ld_v, cudaStream_t st) {
  if (const int rc = gb_paged_check(a)) return rc;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  const long long width = (long long)a->KV * a->hd;
  if (!gb_paged_rows_ok(k_out, ld_k, width) || !gb_paged_rows_ok(v_out, ld_v, width)) return -4;
  dim3 grid;
  if (const int rc = gb_paged_grid(a, &grid)) return rc;
#define CALL(T, HD) GB_PDL_LAUNCH((paged_read_kernel<T, HD>), grid, dim3(PA_THREADS), st, *a, (T*)k_out, ld_k, (T*)v_out, ld_v)
  GB_PAGED_TYPES(a->hd, a->is_bf16, CALL);
#undef CALL
  return gb_launch_rc();
}
