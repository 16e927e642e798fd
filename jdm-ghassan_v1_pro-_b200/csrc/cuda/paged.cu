// Appending to and reading from the paged 8-bit cache (interface in gb_paged.h).
//
// A page of a head is one block's: it sees all numbers that share a scale, and nobody else writes to the page, so nothing here needs an atomic or a second pass over
// memory.  A page's rows of a query head are another block's, so that all of a block's loads are on their way before it waits for any: with the query heads in the loop of
// their key head's block, a page at a time, six prompts of 7.7 thousand tokens (32/8 heads of 128) took twice as long.
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

constexpr int PA_THREADS = 256, PA_FEW = 64;             // threads of a block; with few new tokens a sequence

// Blocks: (page of the new tokens, key head or, from KV on, query head, sequence).  HD / 16 lanes take a row: each the 8 pairs 8c ... 8c + 7 that a rotation turns, as two
// vectors of 8 numbers.  NT threads take ROWS rows, all of a page's or, with PA_FEW, at most PA_FEW * 16 / HD.
template <typename T, int HD, int ROPE, int NT>
__global__ void __launch_bounds__(NT) paged_append_kernel(const __grid_constant__ gb_paged a, const T* __restrict__ qkv, long long ld, int H,
                                                          T* __restrict__ q_out, long long ld_q, const float* __restrict__ qw,
                                                          const float* __restrict__ kw, float eps, const float* __restrict__ cs, int positions) {
  constexpr int LPR = HD / 16, RPP = NT / LPR, ROWS = NT == PA_FEW && RPP < PG ? RPP : PG, PASSES = (ROWS + RPP - 1) / RPP, LDV = PG + 8;
  __shared__ __align__(16) signed char sv[HD * LDV];
  __shared__ float red[2][NT / 32];
  pdl_wait();
  const int b = blockIdx.z, g = blockIdx.y;
  const PgSeq s = pg_seq(a, b);
  const int p = s.start / PG + (int)blockIdx.x;
  const int lo = max(s.start, p * PG), hi = min(s.start + s.n, (p + 1) * PG);      // positions of this block
  if (lo >= hi) return;
  if (hi > positions) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, ST_BAD_ARGUMENT);
    return;
  }
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

  if (g >= a.KV) {                                       // a query head
    const int h = g - a.KV;
    float x[PASSES][16];
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const T* src = qkv + (row0 + min(ps * RPP + r0, n - 1)) * ld + (long long)h * HD;
      pg_load8(src + o0, x[ps]);
      pg_load8(src + o1, x[ps] + 8);
    }
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int r = ps * RPP + r0;
      turn(x[ps], qw, lo + min(r, n - 1));
      if (r >= n) continue;
      T* dst = q_out + (row0 + r) * ld_q + (long long)h * HD;
      pg_store8(dst + o0, x[ps]);
      pg_store8(dst + o1, x[ps] + 8);
    }
    return;
  }

  const int id = pg_page(a, b, p);
  float ky[PASSES][16], vy[PASSES][16], km = 0.f, vm = 0.f;
  bool bad = false;
#pragma unroll
  for (int ps = 0; ps < PASSES; ++ps) {
    const int r = ps * RPP + r0;
    const T* src = qkv + (row0 + min(r, n - 1)) * ld;
    const T *kp = src + (long long)(H + g) * HD, *vp = src + (long long)(H + a.KV + g) * HD;
    pg_load8(kp + o0, ky[ps]);
    pg_load8(kp + o1, ky[ps] + 8);
    pg_load8(vp + o0, vy[ps]);
    pg_load8(vp + o1, vy[ps] + 8);
  }
#pragma unroll
  for (int ps = 0; ps < PASSES; ++ps) {
    const int r = ps * RPP + r0;
    const bool on = r < n;
    turn(ky[ps], kw, lo + min(r, n - 1));
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

  __syncthreads();
  if (id < 0) return;
  km = vm = 0.f;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) { km = fmaxf(km, red[0][w]); vm = fmaxf(vm, red[1][w]); }
  const long long at = (long long)id * a.KV + g;
  signed char *kc = a.k + at * PG * HD, *vc = a.v + at * PG * HD;
  float ks = pg_scale(km), vs = pg_scale(vm);
  if (off > 0) {                                         // tokens of earlier calls share the page
    const float ko = a.ks[at], vo = a.vs[at];
    ks = fmaxf(ks, ko);
    vs = fmaxf(vs, vo);
    if (ks > ko) {
      const float r = ko * pg_inv(ks);
      for (int i = threadIdx.x; i < off * HD; i += NT) kc[i] = (signed char)__float2int_rn((float)kc[i] * r);
    }
    if (vs > vo) {
      const float r = vo * pg_inv(vs);
      for (int i = threadIdx.x; i < off * HD; i += NT) {
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
  for (int i = threadIdx.x; i < HD * ng; i += NT) {
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

// 4 codes as numbers: the byte, raised by 128, under the exponent of 2^23.  (Conversions of integers run at a quarter of this rate.)
__device__ __forceinline__ void pg_numbers(uint32_t w, float scale, float* x) {
  const uint32_t u = w ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)) - 8388736.f) * scale;
}

// A block has a page of a head.  No shared memory: keys are rows already; of the values a thread takes 4 tokens of HD / 8 dimensions, a word each, and turns them byte by
// byte, and neighbours fetch the rest of the sectors.
constexpr int PR_THREADS = 128;
template <typename T, int HD>
__global__ void __launch_bounds__(PR_THREADS) paged_read_kernel(const __grid_constant__ gb_paged a, T* __restrict__ k_out, long long ld_k,
                                                                T* __restrict__ v_out, long long ld_v) {
  constexpr int CH = HD / 16, NK = PG * CH / PR_THREADS, UD = HD / 8;
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
  uint4 kw[NK];
  uint32_t vw[UD];
  const int d0 = (threadIdx.x & 7) * UD, t0 = (threadIdx.x >> 3) * 4;
#pragma unroll
  for (int j = 0; j < NK; ++j) kw[j] = reinterpret_cast<const uint4*>(kc)[j * PR_THREADS + threadIdx.x];
#pragma unroll
  for (int j = 0; j < UD; ++j) vw[j] = *reinterpret_cast<const uint32_t*>(vc + (d0 + j) * PG + t0);
  const float ks = a.ks[at], vs = a.vs[at];
  const float top = PgTop<T>::value;
  const bool clip = !(127.f * fmaxf(ks, vs) <= top);
  auto put = [&](T* dst, float (&x)[8], int n8) {
    if (clip) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -top), top);
    }
    if (n8 == 8) pg_store8(dst, x);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(Cvt<T>::pack2(x[0], x[1]), Cvt<T>::pack2(x[2], x[3]));
  };
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    const int i = j * PR_THREADS + threadIdx.x, t = i / CH, r = t - off;
    if (r < 0 || r >= n) continue;
    T* dk = k_out + (row0 + r) * ld_k + (long long)g * HD + (i - t * CH) * 16;
    float x[8], y[8];
    pg_numbers(kw[j].x, ks, x);
    pg_numbers(kw[j].y, ks, x + 4);
    pg_numbers(kw[j].z, ks, y);
    pg_numbers(kw[j].w, ks, y + 4);
    put(dk, x, 8);
    put(dk + 8, y, 8);
  }
  // word j: dimension d0 + j of tokens t0 ... t0 + 3; turned: word q of a token: its dimensions d0 + 4q ... d0 + 4q + 3
  uint32_t tw[4][UD / 4];
#pragma unroll
  for (int q = 0; q < UD / 4; ++q) {
    const uint32_t a0 = __byte_perm(vw[4 * q], vw[4 * q + 1], 0x5140), a1 = __byte_perm(vw[4 * q], vw[4 * q + 1], 0x7362);
    const uint32_t b0 = __byte_perm(vw[4 * q + 2], vw[4 * q + 3], 0x5140), b1 = __byte_perm(vw[4 * q + 2], vw[4 * q + 3], 0x7362);
    tw[0][q] = __byte_perm(a0, b0, 0x5410);
    tw[1][q] = __byte_perm(a0, b0, 0x7632);
    tw[2][q] = __byte_perm(a1, b1, 0x5410);
    tw[3][q] = __byte_perm(a1, b1, 0x7632);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = t0 + k - off;
    if (r < 0 || r >= n) continue;
    T* dv = v_out + (row0 + r) * ld_v + (long long)g * HD + d0;
    float x[8];
    if constexpr (UD == 4) {
      pg_numbers(tw[k][0], vs, x);
#pragma unroll
      for (int i = 4; i < 8; ++i) x[i] = 0.f;
      put(dv, x, 4);
    } else {
#pragma unroll
      for (int q = 0; q < UD / 8; ++q) {
        pg_numbers(tw[k][2 * q], vs, x);
        pg_numbers(tw[k][2 * q + 1], vs, x + 4);
        put(dv + 8 * q, x, 8);
      }
    }
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
  grid.y += H;
  if (grid.y > 65535) return -3;
  const bool few = a->max_new <= PA_FEW * 16 / a->hd;
#define CALL(T, HD)                                                                                                                                                 \
  do {                                                                                                                                                              \
    if (few) GB_PDL_LAUNCH((paged_append_kernel<T, HD, ROPE, PA_FEW>), grid, dim3(PA_FEW), st, *a, (const T*)qkv, ld_qkv, H, (T*)q_out, ld_q, qw, kw, eps, cos_sin, positions); \
    else GB_PDL_LAUNCH((paged_append_kernel<T, HD, ROPE, PA_THREADS>), grid, dim3(PA_THREADS), st, *a, (const T*)qkv, ld_qkv, H, (T*)q_out, ld_q, qw, kw, eps, cos_sin, positions); \
  } while (0)
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
#define CALL(T, HD) GB_PDL_LAUNCH((paged_read_kernel<T, HD>), grid, dim3(PR_THREADS), st, *a, (T*)k_out, ld_k, (T*)v_out, ld_v)
  GB_PAGED_TYPES(a->hd, a->is_bf16, CALL);
#undef CALL
  return gb_launch_rc();
}
