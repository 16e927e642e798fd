// Appending to and reading from the paged 8-bit cache (interface in gb_paged.h).
//
// A page of a head is one block's: it sees all numbers that share a scale, and nobody else writes to the page, so nothing here needs an atomic or a second pass over
// memory.  A page's rows of a query head are another block's, so that all of a block's loads are on their way before it waits for any: with the query heads in the loop of
// their key head's block, a page at a time, appending six prompts of 7.7 thousand tokens (32/8 heads of 128) and reading them back took 76.9 us instead of 71.8.
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

// 4 codes as numbers: the byte, raised by 128, under the exponent of 2^23.  (Conversions of integers run at a quarter of this rate.)
__device__ __forceinline__ void pg_numbers(uint32_t w, float scale, float* x) {
  const uint32_t u = w ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)) - 8388736.f) * scale;
}

// 4 numbers of at most 127 as codes, rounded to the nearest (even) integer: that is what is left in the low byte of x + 1.5 * 2^23.
__device__ __forceinline__ uint32_t pg_codes(const float* x, float inv) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(fmaf(x[i], inv, 12582912.f));
  return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
}

// Threads of a block with few new tokens a sequence, PA_FEW * 16 / HD at most: more such blocks are on an SM.  us of appending and reading back, these blocks against 4 HD threads:
// 12/4 heads of 64, 1 and 16 tokens, one sequence 4.1 and 4.2 against 4.5 and 5.2, 512 of them 14.8 and 22.3 against 26.7 and 42.3; 32/8 heads of 128, 1 and 8 tokens, 256
// sequences 23.9 and 34.0 against 63.7 and 87.9.
constexpr int PA_FEW = 64;

// Blocks: (key head, behind them two query heads each; page of the new tokens; sequence): neighbours read neighbouring parts of the same rows.  HD / 16 lanes take a row:
// each the 8 pairs 8c ... 8c + 7 that a rotation turns, as two vectors of 8 numbers.  4 HD threads have a page's 64 tokens at once, which 64 registers
// allow; half the threads with two rows each took 114, two blocks an SM.  Bound by instructions issued as much as by memory: codes are rounded by an addition
// and not by conversions, a page's values are turned in registers, four tokens to a word, not stored byte by byte.  Six prompts of 7.7 thousand tokens (32/8 heads of 128,
// 98 MB read, 40 written): 39 us, memory 43 % and issue slots 53 % busy.
template <typename T, int HD, int ROPE, int NT>
__global__ void __launch_bounds__(NT, NT == PA_FEW ? 8 : 1024 / NT) paged_append_kernel(const __grid_constant__ gb_paged a, int page0, const T* __restrict__ qkv, long long ld, int H,
                                                          T* __restrict__ q_out, long long ld_q, const float* __restrict__ qw,
                                                          const float* __restrict__ kw, float eps, const float* __restrict__ cs, int positions) {
  constexpr bool FEW = NT != 4 * HD;
  constexpr int LPR = HD / 16, LDV = PG + 4;
  __shared__ __align__(16) uint32_t sv[FEW ? 1 : HD * LDV / 4];
  __shared__ uint32_t red[2][NT / 32];
  pdl_wait();
  const int b = blockIdx.z, g = blockIdx.x;
  const PgSeq s = pg_seq(a, b);
  const int p = s.start / PG + page0 + (int)blockIdx.y;
  if ((unsigned)p >= (unsigned)a.W) return;
  const int lo = max(s.start, p * PG), hi = min(s.start + s.n, (p + 1) * PG);      // positions of this block
  if (lo >= hi) return;
  if (hi > positions) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, ST_BAD_ARGUMENT);
    return;
  }
  const int n = hi - lo, off = lo - p * PG, c = threadIdx.x % LPR;
  const int r = (int)threadIdx.x / LPR - (FEW ? 0 : off), slot = off + r;            // this thread's row of the block's n (if it is one), and its place in the page
  const bool on = r >= 0 && r < n;
  const int rr = min(max(r, 0), n - 1);
  const long long row = s.first + (lo - s.start) + rr;
  const int o0 = ROPE == 0 ? 16 * c : 8 * c, o1 = ROPE == 0 ? 16 * c + 8 : HD / 2 + 8 * c;
  const T* src = qkv + row * ld;

  float co[8], si[8];
  auto angles = [&]() {                                    // asked for with the row
    const float4* cp = reinterpret_cast<const float4*>(cs + (long long)(lo + rr) * HD + 8 * c);
    const float4 ca = cp[0], cb = cp[1], sa = cp[HD / 8], sb = cp[HD / 8 + 1];
    co[0] = ca.x; co[1] = ca.y; co[2] = ca.z; co[3] = ca.w; co[4] = cb.x; co[5] = cb.y; co[6] = cb.z; co[7] = cb.w;
    si[0] = sa.x; si[1] = sa.y; si[2] = sa.z; si[3] = sa.w; si[4] = sb.x; si[5] = sb.y; si[6] = sb.z; si[7] = sb.w;
  };
  // x: the two vectors of a row; normed and turned
  auto turn = [&](float* x, const float* w) {
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {                         // products and differences rounded one by one, as the definition has them
      const int i0 = ROPE == 0 ? 2 * i : i, i1 = ROPE == 0 ? 2 * i + 1 : 8 + i;
      const float u = x[i0], v = x[i1];
      x[i0] = __fsub_rn(__fmul_rn(u, co[i]), __fmul_rn(v, si[i]));
      x[i1] = __fadd_rn(__fmul_rn(u, si[i]), __fmul_rn(v, co[i]));
    }
  };

  if (g >= a.KV) {                                       // query heads h, h + 1
    const int h = 2 * (g - a.KV);
    const bool two = h + 1 < H;
    float x[16], y[16];
    pg_load8(src + (long long)h * HD + o0, x);
    pg_load8(src + (long long)h * HD + o1, x + 8);
    pg_load8(src + (long long)(h + two) * HD + o0, y);
    pg_load8(src + (long long)(h + two) * HD + o1, y + 8);
    angles();
    turn(x, qw);
    turn(y, qw);
    if (!on) return;
    T* dst = q_out + row * ld_q + (long long)h * HD;
    pg_store8(dst + o0, x);
    pg_store8(dst + o1, x + 8);
    if (two) {
      pg_store8(dst + HD + o0, y);
      pg_store8(dst + HD + o1, y + 8);
    }
    return;
  }

  const int id = pg_page(a, b, p);
  float ky[16], vy[16];
  const T *kp = src + (long long)(H + g) * HD, *vp = src + (long long)(H + a.KV + g) * HD;
  pg_load8(kp + o0, ky);
  pg_load8(kp + o1, ky + 8);
  pg_load8(vp + o0, vy);
  pg_load8(vp + o1, vy + 8);
  angles();
  turn(ky, kw);
  uint32_t km = 0, vm = 0;                               // largest sizes, as bits: what is not finite is larger than all that is
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    km = max(km, __float_as_uint(ky[i]) & 0x7fffffffu);
    vm = max(vm, __float_as_uint(vy[i]) & 0x7fffffffu);
  }
  if (max(km, vm) >= 0x7f800000u) {
    if (on) atomicCAS(a.status, 0, ST_NOT_FINITE);
    km = vm = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t ku = __float_as_uint(ky[i]) & 0x7fffffffu, vu = __float_as_uint(vy[i]) & 0x7fffffffu;
      if (ku >= 0x7f800000u) ky[i] = 0.f; else km = max(km, ku);
      if (vu >= 0x7f800000u) vy[i] = 0.f; else vm = max(vm, vu);
    }
  }
  km = __reduce_max_sync(0xffffffffu, on ? km : 0u);
  vm = __reduce_max_sync(0xffffffffu, on ? vm : 0u);
  if ((threadIdx.x & 31) == 0) { red[0][threadIdx.x >> 5] = km; red[1][threadIdx.x >> 5] = vm; }
  __syncthreads();
  if (id < 0) return;
  km = vm = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) { km = max(km, red[0][w]); vm = max(vm, red[1][w]); }
  const long long at = (long long)id * a.KV + g;
  signed char *kc = a.k + at * PG * HD, *vc = a.v + at * PG * HD;
  float ks = pg_scale(__uint_as_float(km)), vs = pg_scale(__uint_as_float(vm));
  if (off > 0) {                                         // tokens of earlier calls share the page
    const float ko = a.ks[at], vo = a.vs[at];
    ks = fmaxf(ks, ko);
    vs = fmaxf(vs, vo);
    if (ks > ko) {
      const float f = ko * pg_inv(ks);
      uint32_t* w = reinterpret_cast<uint32_t*>(kc);
      for (int i = threadIdx.x; i < off * (HD / 4); i += NT) {
        float x[4];
        pg_numbers(w[i], f, x);
        w[i] = pg_codes(x, 1.f);
      }
    }
    if (vs > vo) {
      const float f = vo * pg_inv(vs);
      uint32_t* w = reinterpret_cast<uint32_t*>(vc);
      for (int i = threadIdx.x; i < HD * (PG / 4); i += NT) {
        const int t = (i & 15) * 4;                      // this word's tokens: those from `off` on are the next call's, or nobody's
        if (t >= off) continue;
        float x[4];
        pg_numbers(w[i], f, x);
        const uint32_t mine = off - t >= 4 ? 0xffffffffu : (1u << (8 * (off - t))) - 1u;
        w[i] = (pg_codes(x, 1.f) & mine) | (w[i] & ~mine);
      }
    }
    __syncthreads();                                     // the old scales are read, the old codes written
  }
  if (threadIdx.x == 0) { a.ks[at] = ks; a.vs[at] = vs; }
  const float ki = pg_inv(ks), vi = pg_inv(vs);
  if (on) {
    signed char* kr = kc + slot * HD;
    *reinterpret_cast<uint2*>(kr + o0) = make_uint2(pg_codes(ky, ki), pg_codes(ky + 4, ki));
    *reinterpret_cast<uint2*>(kr + o1) = make_uint2(pg_codes(ky + 8, ki), pg_codes(ky + 12, ki));
  }
  if constexpr (FEW) {
    if (on) {
#pragma unroll
      for (int i = 0; i < 16; ++i) vc[((i < 8 ? o0 : o1 - 8) + i) * PG + slot] = (signed char)__float_as_uint(fmaf(vy[i], vi, 12582912.f));
    }
  } else {
    // word j of a lane: 4 dimensions of its token; the lanes of 4 tokens turn them, so that lane k has dimension k of the four and all tokens
    const int k = (threadIdx.x / LPR) & 3, t4 = (int)threadIdx.x / LPR / 4;
    const uint32_t one = k & 1 ? 0x3715u : 0x6240u, other = k & 2 ? 0x3276u : 0x5410u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w = pg_codes(vy + 4 * j, vi);
      w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, LPR), one);
      w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 2 * LPR), other);
      sv[((j < 2 ? o0 + 4 * j : o1 + 4 * j - 8) + k) * (LDV / 4) + t4] = w;
    }
    __syncthreads();
    // 16 tokens of a dimension a thread
    const int d = threadIdx.x >> 2, t = (threadIdx.x & 3) * 16;
    const uint32_t* from = sv + d * (LDV / 4) + t / 4;
    const uint32_t w[4] = {from[0], from[1], from[2], from[3]};
    signed char* dst = vc + d * PG + t;
    if (t >= off && t + 16 <= off + n) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (t + j >= off && t + j < off + n) dst[j] = (signed char)(w[j >> 2] >> (8 * (j & 3)));
    }
  }
}

// A block has a page of a head.  No shared memory: keys are rows already; of the values a thread takes 4 tokens of HD / 8 dimensions, a word each, and turns them byte by
// byte, and neighbours fetch the rest of the sectors.
constexpr int PR_THREADS = 128;
template <typename T, int HD>
__global__ void __launch_bounds__(PR_THREADS) paged_read_kernel(const __grid_constant__ gb_paged a, int page0, T* __restrict__ k_out, long long ld_k,
                                                                T* __restrict__ v_out, long long ld_v) {
  constexpr int CH = HD / 16, NK = PG * CH / PR_THREADS, UD = HD / 8;
  pdl_wait();
  const int b = blockIdx.z, g = blockIdx.x;
  const PgSeq s = pg_seq(a, b);
  const int p = s.start / PG + page0 + (int)blockIdx.y;
  if ((unsigned)p >= (unsigned)a.W) return;
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

// Launches over all pages that max_new tokens can touch, wherever in a page they begin, and all sequences: as many launches as it takes, since a grid has at most 65535 blocks along y
// and z.  launch(part, b0, page0, grid): `part` has the sequences from b0 on, their pages count from page0.
template <typename F>
static int gb_paged_launches(const gb_paged* a, int grid_x, F&& launch) {
  constexpr int MOST = 65535;
  const int pages = (int)std::min<long long>(((long long)a->max_new + 2 * GB_PAGE - 2) / GB_PAGE, a->W);
  for (int b0 = 0; b0 < a->B; b0 += MOST) {
    gb_paged part = *a;
    part.B = std::min(MOST, a->B - b0);
    part.table += (long long)b0 * a->W;
    part.start += b0;
    if (a->count) {
      part.first += b0;
      part.count += b0;
    } else {
      part.rows = std::max(0ll, a->rows - b0);              // rows are counted from a launch's first sequence
    }
    for (int page0 = 0; page0 < pages; page0 += MOST) {
      launch(part, a->count ? 0 : b0, page0, dim3(grid_x, std::min(MOST, pages - page0), part.B));
      if (const int rc = gb_launch_rc()) return rc;
    }
  }
  return 0;
}

extern "C" int gb_paged_append(const gb_paged* a, const void* qkv, long long ld_qkv, int H, void* q_out, long long ld_q, const float* qw,
                               const float* kw, float eps, const float* cos_sin, int positions, int rope_type, cudaStream_t st) {
  if (const int rc = gb_paged_check(a)) return rc;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  if (H <= 0 || H % a->KV || !cos_sin || (reinterpret_cast<uintptr_t>(cos_sin) & 15) || positions <= 0 || (rope_type != 0 && rope_type != 1)) return -1;
  if (!gb_paged_rows_ok(qkv, ld_qkv, (long long)(H + 2 * a->KV) * a->hd) || !gb_paged_rows_ok(q_out, ld_q, (long long)H * a->hd)) return -4;
  const bool few = a->max_new <= PA_FEW * 16 / a->hd;
  return gb_paged_launches(a, a->KV + (H + 1) / 2, [&](const gb_paged& part, int row0, int page0, dim3 grid) {
#define CALL(T, HD)                                                                                                                                                  \
  do {                                                                                                                                                               \
    const T* in = (const T*)qkv + row0 * ld_qkv;                                                                                                                     \
    T* out = (T*)q_out + row0 * ld_q;                                                                                                                                \
    if (few) GB_PDL_LAUNCH((paged_append_kernel<T, HD, ROPE, PA_FEW>), grid, dim3(PA_FEW), st, part, page0, in, ld_qkv, H, out, ld_q, qw, kw, eps, cos_sin, positions); \
    else GB_PDL_LAUNCH((paged_append_kernel<T, HD, ROPE, 4 * HD>), grid, dim3(4 * HD), st, part, page0, in, ld_qkv, H, out, ld_q, qw, kw, eps, cos_sin, positions);  \
  } while (0)
    if (rope_type == 0) {
      constexpr int ROPE = 0;
      GB_PAGED_TYPES(a->hd, a->is_bf16, CALL);
    } else {
      constexpr int ROPE = 1;
      GB_PAGED_TYPES(a->hd, a->is_bf16, CALL);
    }
#undef CALL
  });
}

extern "C" int gb_paged_read(const gb_paged* a, void* k_out, long long ld_k, void* v_out, long long ld_v, cudaStream_t st) {
  if (const int rc = gb_paged_check(a)) return rc;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  const long long width = (long long)a->KV * a->hd;
  if (!gb_paged_rows_ok(k_out, ld_k, width) || !gb_paged_rows_ok(v_out, ld_v, width)) return -4;
  return gb_paged_launches(a, a->KV, [&](const gb_paged& part, int row0, int page0, dim3 grid) {
#define CALL(T, HD) GB_PDL_LAUNCH((paged_read_kernel<T, HD>), grid, dim3(PR_THREADS), st, part, page0, (T*)k_out + row0 * ld_k, ld_k, (T*)v_out + row0 * ld_v, ld_v)
    GB_PAGED_TYPES(a->hd, a->is_bf16, CALL);
#undef CALL
  });
}
