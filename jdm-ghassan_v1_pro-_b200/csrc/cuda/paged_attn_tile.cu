// Attention over the paged 8-bit cache for many query rows a key head (interface in gb_paged.h, choice in paged_attn.cu): prompts and portions of them.
//
// Rows are (token, query head of the group) pairs of a key head, 256 of them an item, so any group size fills the tiles and a key is expanded once for all its
// query heads.  Bound by the exponentials at hd 64 (one a score, 16 a cycle and SM, against 8192 tensor operations of 256 a score), by them and the products about equally at 128.
//
// One block an SM: two warpgroups of soft-max threads, a row each, take turns with the tensor cores (while one finds its weights, the products of the other run); four warps expand the
// pages, a tile of 128 keys at a time, from codes in global memory to float16 integers in the swizzled layout of the MMAs (integers up to 127 are exact, the scales go into the
// soft-max: a key scale into the score's factor, a value scale into the weight's exponent, as in paged_attn_token.cu); a warp for each warpgroup issues (one for both was busy
// issuing and asking barriers all the time).  Scores and weights share tensor memory:
// weights of a chunk of 32 columns go where scores that have been read were, and are the A operand of the second product from there.
//
// The work is dealt in key tiles: all (sequence, key head, item, key tile) in a row are cut into equal runs, one a block.  Items that a cut goes through leave records
// that a second kernel joins.  A causal prompt's items differ in length by a factor of its tiles; dealt whole, the last round of items would leave most SMs idle.
#include <algorithm>

#include "paged_attn.cuh"
#include "tc_tiles.cuh"

namespace gb {

constexpr int TL_ROWS = 256, TL_THREADS = 512;
constexpr float TL_OFF = 7.f, TL_LAZY = 8.f;   // weights are held as 2^7 of themselves and may grow 2^8 before the sums are rescaled

template <int HD>
struct Tl {
  // Tensor memory has 512 columns.  At hd 128 the results take 256: scores come in tiles of 64 keys, two buffers a warpgroup, and weights go over the scores; the products of a
  // tile run while the soft-max is at work on the next (2048 tokens behind 14000, 32/8 heads, 558 us; tiles of 128 keys with one buffer, whose products a
  // warpgroup waits for, 571).  Else tiles have 128 keys and one buffer, which is free once the scores are in registers, and weights have places of their own.
  static constexpr bool OVER = HD == 128;
  static constexpr int KEYS = OVER ? 64 : 128, PP = KEYS / PG, BUFS = OVER && KEYS == 64 ? 2 : 1;
  static constexpr int P0 = OVER ? 0 : 256, O0 = OVER ? 256 : 384;
  static constexpr int PANELS = HD <= 64 ? 1 : 2;             // 64 dimensions each
  static constexpr int Q = 128 * 128 * PANELS, K = KEYS * 128 * PANELS, V = PP * HD * 128, STAGE = K + V;
  static constexpr int STAGES = OVER ? 256 / KEYS : 3, AHEAD = 128 / KEYS;
  // registers a thread: soft-max, expanding, issuing; launched with 128, so 2 x 128 x S + 128 x (E + I) is at most 65536
  static constexpr int REGS_S = OVER && KEYS == 128 ? 176 : 184, REGS_E = OVER && KEYS == 128 ? 104 : 88, REGS_I = 56;
  static constexpr int REC = TL_ROWS * (HD + 2);              // floats of a record: [HD / 4][256] four results, then [256] pairs (maximum, sum)
};

// What a record is of: places of its item, and which it is.  f1 == 0: nothing.
struct TlDesc { int f0, f1, b, g, qt, quota, pad0, pad1; };

// Bounded waits: false once the block has given up.  The first polls are all that a phase takes that is over already.  (The rest is no call: there are 128 scores in registers.)
__device__ __forceinline__ bool tl_wait(uint64_t* bar, uint32_t parity, int* status, int code, volatile int* abort_flag) {
  return mbar_try_wait_some(bar, parity) || at_wait(bar, parity, status, code, abort_flag);
}

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 tl_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 tl_add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}

struct TlItem { int lo, n; };                                 // first key tile, number of them
template <int KEYS>
__device__ __forceinline__ TlItem tl_item(const PgAttn& p, const PgSeq& s, int G, int qt) {
  const int r1 = min(s.n * G, (qt + 1) * TL_ROWS) - 1;
  const int p0 = s.start + qt * TL_ROWS / G, p1 = s.start + r1 / G;
  const int lo = p.window > 0 ? max(0, p0 - p.window + 1) / KEYS : 0;
  return {lo, p1 / KEYS - lo + 1};
}

// A block's walk over its run: places f ... end, one piece of an item after the other.  An item has a place for each key tile and, ahead of them, AHEAD for its start and end: loading queries,
// filling and emptying the pipelines take as long as a tile of 128 keys.
template <int AHEAD>
struct TlWalk {
  int f, end, b, g, qt, k;                                    // k: places of the item that come before place f
  PgSeq s;
  int tiles;
  __device__ __forceinline__ void load(const PgAttn& p, int G) {
    s = pg_seq(p.a, b);
    tiles = (s.n * G + TL_ROWS - 1) / TL_ROWS;
  }
  // the run's part of this item: key tiles k0 ... k1 - 1
  __device__ __forceinline__ void part(const TlItem& item, int& k0, int& k1) const {
    k0 = max(0, k - AHEAD);
    k1 = max(0, min(item.n + AHEAD, k + end - f) - AHEAD);
  }
  __device__ __forceinline__ void next(const PgAttn& p, int G, const int* cum, const TlItem& item) {
    const int taken = min(item.n + AHEAD - k, end - f);
    f += taken;
    k += taken;
    if (k < item.n + AHEAD || f >= end) return;
    k = 0;
    if (++qt < tiles) return;
    qt = 0;
    if (++g < p.a.KV) return;
    g = 0;
    do ++b; while (cum[b + 1] == cum[b]);
    load(p, G);
  }
};

template <typename T, int HD>
__global__ void __launch_bounds__(TL_THREADS, 1) paged_tile_kernel(const __grid_constant__ PgAttn p) {
  using L = Tl<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sKV = smem + 2 * L::Q;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + L::STAGES * L::STAGE);
  uint64_t *k_full = bars, *k_empty = k_full + L::STAGES, *v_full = k_empty + L::STAGES, *v_empty = v_full + L::STAGES;
  uint64_t *s_full = v_empty + L::STAGES, *p_ready = s_full + 4, *o_full = s_full + 8, *q_full = s_full + 10, *s_free = s_full + 12, *turn = s_full + 14;   // s_full, p_ready: [2 wg + buffer]
  float4* scales = reinterpret_cast<float4*>(turn + 2);                       // of eight key tiles (they outlive a stage): key scales of the two pages, value scales; a negative
                                                                              // key scale: no page
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scales + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* cum = reinterpret_cast<int*>(tmem_slot + 2);                           // key tiles (of one head) of the sequences before
  const gb_paged& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.H / a.KV;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) { mbar_init(&k_full[s], 4); mbar_init(&k_empty[s], 2); mbar_init(&v_full[s], 4); mbar_init(&v_empty[s], 2); }
    for (int w = 0; w < 4; ++w) { mbar_init(&s_full[w], 2); mbar_init(&p_ready[w], 4); }
    for (int w = 0; w < 2; ++w) { mbar_init(&o_full[w], 1); mbar_init(&q_full[w], 4); mbar_init(&s_free[w], 4); mbar_init(&turn[w], 4); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 12) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  pdl_wait();
  for (int b = warp; b < a.B; b += TL_THREADS / 32) {
    const PgSeq s = pg_seq(a, b);
    const int tiles = (s.n * G + TL_ROWS - 1) / TL_ROWS;
    int n = 0;
    for (int qt = lane; qt < tiles; qt += 32) n += tl_item<L::KEYS>(p, s, G, qt).n + L::AHEAD;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) cum[b + 1] = n;
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp == 0) {
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      int v = b0 + lane < a.B ? cum[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (b0 + lane < a.B) cum[b0 + lane + 1] = before + v;
      before += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) cum[0] = 0;
  }
  __syncthreads();
  const int total = a.KV * cum[a.B], quota = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  TlWalk<L::AHEAD> start;
  start.f = min(total, (int)blockIdx.x * quota);
  start.end = min(total, start.f + quota);
  TlDesc* desc = reinterpret_cast<TlDesc*>(p.part);
  float* records = p.part + (size_t)2 * gridDim.x * (sizeof(TlDesc) / 4);
  if (threadIdx.x == 0) desc[2 * blockIdx.x].f1 = desc[2 * blockIdx.x + 1].f1 = 0;
  if (start.f < start.end) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] * a.KV <= start.f) lo = mid; else hi = mid;
    }
    start.b = lo;
    const int w = cum[lo + 1] - cum[lo], local = start.f - cum[lo] * a.KV;
    start.g = local / w;
    int rem = local - start.g * w;
    start.load(p, G);
    start.qt = 0;
    start.k = 0;
    for (int q0 = 0; q0 < start.tiles; q0 += 32) {            // the item that holds place f: a warp looks through 32 at a time
      const int n = q0 + lane < start.tiles ? tl_item<L::KEYS>(p, start.s, G, q0 + lane).n + L::AHEAD : 0;
      int v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      const unsigned past = __ballot_sync(0xffffffffu, v > rem);
      if (past) {
        const int at = __ffs(past) - 1;
        start.qt = q0 + at;
        start.k = rem - __shfl_sync(0xffffffffu, v - n, at);
        break;
      }
      rem -= __shfl_sync(0xffffffffu, v, 31);
    }

    if (warp < 8) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::REGS_S));
      // ------------------------------------------------------------------------------------------ soft-max: a thread a row
      const int wg = warp >> 2, r = threadIdx.x & 127;
      const uint32_t row = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t tO = tmem + L::O0 + wg * HD + row;
      uint8_t* q_at = sQ + wg * L::Q;
      uint32_t kv_it = 0, it = 0, turns = 0;                   // key tiles so far; those of this warpgroup; its turns at the exponentials
      bool ok = true;
      TlWalk<L::AHEAD> w = start;
      while (w.f < w.end && ok) {
        const TlItem item = tl_item<L::KEYS>(p, w.s, G, w.qt);
        const int rows = w.s.n * G, first = w.qt * TL_ROWS + wg * 128;
        int k0, k1;
        w.part(item, k0, k1);
        if (first < rows && k0 < k1) {
          const bool both = w.qt * TL_ROWS + 128 < rows;       // the other warpgroup has rows too
          const int rr = first + r, i = rr / G, pos = w.s.start + i;
          const bool row_ok = rr < rows;
          const int pos_a = w.s.start + first / G, pos_z = w.s.start + (min(rows, first + 128) - 1) / G;
          float qs;
          {                                                    // this row's query, scaled to float16's middle
            const T* src = reinterpret_cast<const T*>(p.q) + (long long)(w.s.first + (row_ok ? i : 0)) * p.ld_q + (long long)(w.g * G + (row_ok ? rr - i * G : 0)) * HD;
            uint32_t top = 0;
            uint4 raw[HD / 8];
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) raw[c] = row_ok ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
              const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 v = Cvt<T>::unpack2(u[e]);
                top = max(top, max(__float_as_uint(fabsf(v.x)), __float_as_uint(fabsf(v.y))));
              }
            }
            const int e = top == 0 ? 127 : min(max(254 + 14 - (int)(top >> 23), 1), 253);
            const float mul = __uint_as_float((uint32_t)e << 23), inv = __uint_as_float((uint32_t)(254 - e) << 23);
            qs = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : inv * p.scale2;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
              const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
              uint32_t h[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 v = Cvt<T>::unpack2(u[j]);
                h[j] = Cvt<__half>::pack2(v.x * mul, v.y * mul);
              }
              *reinterpret_cast<uint4*>(q_at + (c >> 3) * (128 * 128) + sw128_off(r, (c & 7) * 8)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[wg]);
          float m2 = -1e30f, l = 0.f;
          int E = -1000;
          for (int t = k0; t < k1; ++t, ++it, ++kv_it) {
            const uint32_t buf = L::BUFS == 2 ? it & 1u : 0u, phase = (L::BUFS == 2 ? it >> 1 : it) & 1u;
            const uint32_t tS = tmem + wg * 128 + buf * 64 + row, tP = L::OVER ? tS : tmem + L::P0 + wg * 64 + row;
            if (!tl_wait(&s_full[2 * wg + buf], phase, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag)) { ok = false; break; }
            tc_fence_after();
            const float4 sc = scales[kv_it & 7];
            float x[L::KEYS];
            {
              uint32_t(*rg)[32] = reinterpret_cast<uint32_t(*)[32]>(x);
#pragma unroll
              for (int c = 0; c < L::KEYS / 32; ++c) tmem_ld_32x32(tS + c * 32, rg[c]);
              tmem_ld_wait();
            }
            if constexpr (!L::OVER) {                          // the next scores may come
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s_free[wg]);
            }
            const int base = (item.lo + t) * L::KEYS;
            if (base + L::KEYS - 1 > pos_a || (p.window > 0 && pos_z - p.window + 1 > base) || sc.x < 0.f || (L::PP > 1 && sc.y < 0.f)) {
              // a bit a column, so that a column costs a test and a choice: three comparisons each were a third of the loop's code, and its fetching showed
              const int hi = pos - base, lo = p.window > 0 ? pos - p.window + 1 - base : 0;
#pragma unroll
              for (int w = 0; w < L::KEYS / 32; ++w) {
                const int h = hi - 32 * w, l0 = lo - 32 * w;              // columns l0 ... h of this word
                uint32_t see = (h >= 31 ? 0xffffffffu : h < 0 ? 0u : (2u << h) - 1u) & (l0 <= 0 ? 0xffffffffu : l0 > 31 ? 0u : 0xffffffffu << l0);
                if ((w < 2 ? sc.x : sc.y) < 0.f) see = 0u;
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (!(see & (1u << k))) x[32 * w + k] = -INFINITY;
              }
            }
            // a factor that is too small for fp32 must not make nothing of a hidden score
            float f[2] = {qs * fabsf(sc.x), qs * fabsf(sc.y)};
#pragma unroll
            for (int h = 0; h < 2; ++h) f[h] = f[h] == 0.f ? 1e-37f : f[h];
            float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int h = 0; h < L::PP; ++h) {
              float mr[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) mr[c] = fmaxf(x[h * 64 + c], x[h * 64 + 4 + c]);
#pragma unroll
              for (int k = 8; k < 64; k += 8)
#pragma unroll
                for (int c = 0; c < 4; ++c) mr[c] = fmaxf(fmaxf(mr[c], x[h * 64 + k + c]), x[h * 64 + k + 4 + c]);
              mt[h] = fmaxf(fmaxf(mr[0], mr[1]), fmaxf(mr[2], mr[3])) * f[h];
            }
            const float top = fmaxf(mt[0], mt[1]);
            const int e0 = (int)(__float_as_uint(sc.z) >> 23) - 127, e1 = L::PP > 1 ? (int)(__float_as_uint(sc.w) >> 23) - 127 : e0, En = max(E, max(e0, e1));
            // the last second product is done: its weights' places are free, its sums can be rescaled
            const bool grow = __any_sync(0xffffffffu, top > m2 + TL_LAZY || En != E);
            if (t > k0 && (!L::OVER || grow)) {
              if (!tl_wait(&o_full[wg], (it - 1u) & 1u, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag)) { ok = false; break; }
              tc_fence_after();
            }
            if (grow) {
              const float mn = fmaxf(m2, top), corr = pg_ex2(m2 - mn);
              l *= corr;
              m2 = mn;
              if (t > k0) {
                const float c2 = corr * exp2f((float)(E - En));
#pragma unroll 1
                for (int c = 0; c < HD / 16; ++c) {
                  uint32_t rg[16];
                  tmem_ld_32x16(tO + c * 16, rg);
                  tmem_ld_wait();
#pragma unroll
                  for (int k = 0; k < 16; ++k) rg[k] = __float_as_uint(__uint_as_float(rg[k]) * c2);
                  tmem_st_32x16(tO + c * 16, rg);
                }
              }
              E = En;
            }
            // exponentials in turn: while one warpgroup has the unit that makes them, the other loads and looks for maxima
            if (both) {
              if (!tl_wait(&turn[wg], (turns & 1u) ^ (wg == 0 ? 1u : 0u), a.status, ST_TIMEOUT_EMPTY, abort_flag)) { ok = false; break; }
              ++turns;
            }
            const float de[2] = {fmaxf((float)(e0 - En), -60.f), fmaxf((float)(e1 - En), -60.f)};
#pragma unroll
            for (int h = 0; h < L::PP; ++h) {
              const float2 ff = make_float2(f[h], f[h]), bias = make_float2(TL_OFF + de[h] - m2, TL_OFF + de[h] - m2);
              float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                uint32_t pk[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  const int j = h * 64 + c * 32 + 2 * k;
                  float2 e = tl_fma2(make_float2(x[j], x[j + 1]), ff, bias);
                  e.x = pg_ex2(e.x);
                  e.y = pg_ex2(e.y);
                  ls[k & 1] = tl_add2(ls[k & 1], e);
                  pk[k] = Cvt<__half>::pack2(e.x, e.y);
                }
                tmem_st_32x16(tP + (2 * h + c) * 16, pk);
              }
              l = fmaf((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y), exp2f(-de[h]), l);
            }
            if (both && lane == 0) mbar_arrive(&turn[wg ^ 1]);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[2 * wg + buf]);
          }
          if (!ok) break;
          if (!tl_wait(&o_full[wg], (it - 1u) & 1u, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const bool whole = k0 == 0 && k1 == item.n;
          const int f0 = w.f - w.k + L::AHEAD, slot = 2 * blockIdx.x + (f0 > start.f ? 1 : 0);
          float* rec = records + (size_t)slot * L::REC;
          const float fac = l == 0.f ? 0.f : __uint_as_float((uint32_t)(E + 127) << 23) / l;
          T* dst = reinterpret_cast<T*>(p.out) + (long long)(w.s.first + i) * p.ld_o + (long long)(w.g * G + rr - i * G) * HD;
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t rg[32];
            tmem_ld_32x32(tO + c * 32, rg);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(rg[k]) * fac;
            if (whole) {
              if (row_ok) {
#pragma unroll
                for (int k = 0; k < 4; ++k) pg_store8(dst + c * 32 + 8 * k, v + 8 * k);
              }
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                reinterpret_cast<float4*>(rec)[(c * 8 + k) * TL_ROWS + wg * 128 + r] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            }
          }
          if (!whole) {
            reinterpret_cast<float2*>(rec + TL_ROWS * HD)[wg * 128 + r] = make_float2(m2, l);
            if (threadIdx.x == 0) desc[slot] = {f0, f0 + item.n, w.b, w.g, w.qt, quota, 0, 0};
          }
          tc_fence_before();
        } else {
          kv_it += k1 - k0;
        }
        w.next(p, G, cum, item);
      }
    } else if (warp < 12) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_E));
      // ------------------------------------------------------------------------------------------ pages to float16
      const int tid = threadIdx.x - 256;
      constexpr int NK = HD * L::KEYS / 2048, NP = NK / L::PP;                            // chunks of 16 codes a thread has of a tile's keys, and of its values
      uint32_t kv_it = 0;
      bool ok = true;
      TlWalk<L::AHEAD> w = start;
      while (w.f < w.end && ok) {
        const TlItem item = tl_item<L::KEYS>(p, w.s, G, w.qt);
        // pages that the item's rows see: ahead of them there may be none any more (a window), although the first tile begins there
        const int last = (w.s.start + w.s.n - 1) / PG, low = p.window > 0 ? max(0, w.s.start + w.qt * TL_ROWS / G - p.window + 1) / PG : 0;
        int k0, k1;
        w.part(item, k0, k1);
        uint4 rk[NK], rv[NK];
        int id[L::PP], after[L::PP];                                   // pages of the tile whose codes are on their way; what the table has for the one behind it
        float sc = 0.f;
        auto look = [&](int t) {                               // nothing waits for the answer here
#pragma unroll
          for (int h = 0; h < L::PP; ++h) {
            const int pg = L::PP * (item.lo + t) + h;
            after[h] = t < k1 && pg >= low && pg <= last ? a.table[(long long)w.b * a.W + pg] : -2;
          }
        };
        // codes of a tile's keys or values, chunk c of a page (HD * 64 codes) in the order of memory
        auto fetch = [&](uint4 (&r)[NK], const signed char* from) {
#pragma unroll
          for (int c = 0; c < NK; ++c) {
            const int h = c / NP, ch = (c % NP) * 128 + tid;
            const long long at = ((long long)max(id[h], 0) * a.KV + w.g) * (PG * HD);
            r[c] = id[h] < 0 ? make_uint4(0, 0, 0, 0) : reinterpret_cast<const uint4*>(from + at)[ch];
          }
        };
        auto fetch_keys = [&](int t) {                         // and the scales of tile t, the pages' numbers of tile t + 1
#pragma unroll
          for (int h = 0; h < L::PP; ++h) {
            id[h] = after[h];
            if ((unsigned)id[h] >= (unsigned)a.pages) {
              const int pg = L::PP * (item.lo + t) + h;
              if (pg >= low && pg <= last) atomicCAS(a.status, 0, ST_BAD_ARGUMENT);
              id[h] = -1;
            }
          }
          fetch(rk, a.k);
          if (tid < 4) {
            const int page = id[L::PP > 1 ? tid & 1 : 0];
            sc = page >= 0 ? (tid < 2 ? a.ks : a.vs)[(long long)page * a.KV + w.g] : tid < 2 ? -1.f : PG_LEAST;
          }
          look(t + 1);
        };
        if (k0 < k1) {
          look(k0);
          fetch_keys(k0);
          fetch(rv, a.v);
        }
        for (int t = k0; t < k1; ++t, ++kv_it) {
          const int st = kv_it % L::STAGES;
          const uint32_t free = ((kv_it / L::STAGES) & 1u) ^ 1u;
          uint8_t *sk = sKV + st * L::STAGE, *sv = sk + L::K;
          if (!tl_wait(&k_empty[st], free, a.status, ST_TIMEOUT_EMPTY, abort_flag)) { ok = false; break; }
#pragma unroll
          for (int c = 0; c < NK; ++c) {
            const int ch = (c % NP) * 128 + tid, key = c / NP * 64 + ch / (HD / 16), d = (ch % (HD / 16)) * 16;      // 16 dimensions of a key
            uint32_t x[8];
            pg_halves(rk[c].x, x[0], x[1]);
            pg_halves(rk[c].y, x[2], x[3]);
            pg_halves(rk[c].z, x[4], x[5]);
            pg_halves(rk[c].w, x[6], x[7]);
            uint8_t* kp = sk + (d >> 6) * (L::KEYS * 128);
            *reinterpret_cast<uint4*>(kp + sw128_off(key, d & 63)) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(kp + sw128_off(key, (d & 63) + 8)) = make_uint4(x[4], x[5], x[6], x[7]);
          }
          if (tid < 4) reinterpret_cast<float*>(&scales[kv_it & 7])[tid] = sc;
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&k_full[st]);
          if (t + 1 < k1) fetch_keys(t + 1);
          if (!tl_wait(&v_empty[st], free, a.status, ST_TIMEOUT_EMPTY, abort_flag)) { ok = false; break; }
#pragma unroll
          for (int c = 0; c < NK; ++c) {
            const int ch = (c % NP) * 128 + tid, vd = ch >> 2, vt = (ch & 3) * 16;                                          // 16 tokens of a dimension
            uint32_t x[8];
            pg_halves(rv[c].x, x[0], x[1]);
            pg_halves(rv[c].y, x[2], x[3]);
            pg_halves(rv[c].z, x[4], x[5]);
            pg_halves(rv[c].w, x[6], x[7]);
            uint8_t* vp = sv + c / NP * (HD * 128);
            *reinterpret_cast<uint4*>(vp + sw128_off(vd, vt)) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(vp + sw128_off(vd, vt + 8)) = make_uint4(x[4], x[5], x[6], x[7]);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[st]);
          if (t + 1 < k1) fetch(rv, a.v);
        }
        if (!ok) break;
        w.next(p, G, cum, item);
      }
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_I));
      if (warp < 14) {
      // ------------------------------------------------------------------------------------------ MMAs
      const uint32_t on = elect_one();
      const uint32_t id_s = make_idesc_f16(0, 0, 0, 128, L::KEYS), id_o = make_idesc_f16(0, 0, 0, 128, HD);
      // What the loops go by is handed around by lane 0, which is how the compiler learns that it is the same for all: counters, descriptors and addresses then stay in
      // uniform registers, where these instructions want them (descriptors found lane by lane made issuing a tile's products take 1400 cycles a warpgroup).
      const int wg = warp - 12;
      uint32_t kv_it = 0, q_it = 0, it = 0, s_it = 0;          // key tiles; this warpgroup's pieces, tiles summed, tiles scored
      TlWalk<L::AHEAD> w = start;
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), tS = tm + __shfl_sync(0xffffffffu, wg, 0) * 128;
      const uint32_t tO = tm + L::O0 + __shfl_sync(0xffffffffu, wg, 0) * HD, tP = L::OVER ? tS : tm + L::P0 + __shfl_sync(0xffffffffu, wg, 0) * 64;
      const uint64_t dq = make_smem_desc_sw128(smem_u32(sQ) + __shfl_sync(0xffffffffu, wg, 0) * L::Q, 16, 1024), dkv = make_smem_desc_sw128(smem_u32(sKV), 16, 1024);
      auto full = [&](uint64_t* bar, uint32_t at) {
        wait_or_report(&bar[at % L::STAGES], (at / L::STAGES) & 1u, a.status, ST_TIMEOUT_FULL, abort_flag);
        tc_fence_after();
      };
      bool more = w.f < w.end;
      while (__shfl_sync(0xffffffffu, (int)more, 0)) {
        const TlItem item = tl_item<L::KEYS>(p, w.s, G, w.qt);
        int k0, k1;
        w.part(item, k0, k1);
        const bool two = __shfl_sync(0xffffffffu, (int)(w.qt * TL_ROWS + 128 < w.s.n * G), 0) != 0;
        const int all = __shfl_sync(0xffffffffu, k1 - k0, 0), n = wg == 1 && !two ? 0 : all;
        auto scores = [&](uint32_t at) {
          const uint32_t buf = L::BUFS == 2 ? s_it & 1u : 0u;
          ++s_it;
          const uint64_t db = dkv + (at % L::STAGES) * (L::STAGE >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            umma_f16_on(on, tS + buf * 64, dq + (((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4), db + (((kk >> 2) * (L::KEYS * 128) + (kk & 3) * 32) >> 4), id_s, kk > 0 ? 1u : 0u);
          if (on) mbar_arrive(&s_full[2 * wg + buf]);          // hands on what k_full brought: the scales, which no MMA touches
          umma_commit_on(on, &s_full[2 * wg + buf]);
          umma_commit_on(on, &k_empty[at % L::STAGES]);
        };
#pragma unroll
        for (int j = 0; j < L::BUFS; ++j) {
          if (j >= n) continue;
          full(k_full, kv_it + j);
          if (j == 0) {
            wait_or_report(&q_full[wg], q_it & 1u, a.status, ST_TIMEOUT_FULL, abort_flag);
            ++q_it;
            tc_fence_after();
          }
          scores(kv_it + j);
        }
        for (int t = 0; t < n; ++t) {
          const uint32_t at = kv_it + t, buf = L::BUFS == 2 ? it & 1u : 0u, phase = (L::BUFS == 2 ? it >> 1 : it) & 1u;
          if (!L::OVER && t + 1 < n) {
            full(k_full, at + 1);
            wait_or_report(&s_free[wg], it & 1u, a.status, ST_TIMEOUT_TMEM_EMPTY, abort_flag);
            tc_fence_after();
            scores(at + 1);
          }
          full(v_full, at);
          const uint64_t dv = dkv + (((at % L::STAGES) * L::STAGE + L::K) >> 4);
          wait_or_report(&p_ready[2 * wg + buf], phase, a.status, ST_TIMEOUT_TMEM_EMPTY, abort_flag);
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < L::KEYS / 16; ++kk)
            umma_f16_ts_on(on, tO, tP + buf * 64 + kk * 8, dv + (((kk >> 2) * (HD * 128) + (kk & 3) * 32) >> 4), id_o, t > 0 || kk > 0 ? 1u : 0u);
          umma_commit_on(on, &o_full[wg]);
          umma_commit_on(on, &v_empty[at % L::STAGES]);
          if (L::OVER && t + L::BUFS < n) {
            // scores go where these weights are, and products of different accumulators need not run in the order of their issue
            full(k_full, at + L::BUFS);
            wait_or_report(&o_full[wg], it & 1u, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag);
            tc_fence_after();
            scores(at + L::BUFS);
          }
          ++it;
        }
        // Tiles that are the other warpgroup's alone are followed stage by stage all the same: a barrier's phase is known by its parity, so neither warp may be more than one ahead.
        for (int t = n; t < all; ++t) {
          full(k_full, kv_it + t);
          if (on) mbar_arrive(&k_empty[(kv_it + t) % L::STAGES]);
          full(v_full, kv_it + t);
          if (on) mbar_arrive(&v_empty[(kv_it + t) % L::STAGES]);
        }
        kv_it += all;
        w.next(p, G, cum, item);
        more = w.f < w.end;
      }
      __syncwarp();
      }
    }
  }
  __syncthreads();
  if (*abort_flag) {
    for (int k = 0; k < 64; ++k) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 12) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// Joins the pieces of the item that begins in block x's run and is cut by its end: 32 rows a block.
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_tile_join_kernel(const __grid_constant__ PgAttn p, int blocks) {
  using L = Tl<HD>;
  pdl_wait();
  const TlDesc* desc = reinterpret_cast<const TlDesc*>(p.part);
  const float* records = p.part + (size_t)2 * blocks * (sizeof(TlDesc) / 4);
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y * 32 + lane;
  for (int k = 0; k < 2; ++k) {
    const TlDesc d = desc[2 * c + k];
    if (d.f1 <= 0 || d.f0 < c * d.quota || d.f1 <= (c + 1) * d.quota) continue;
    const int G = p.H / p.a.KV, last = (d.f1 - 1) / d.quota;
    const PgSeq s = pg_seq(p.a, d.b);
    const int rr = d.qt * TL_ROWS + row, i = rr / G;
    if (rr >= s.n * G) continue;
    auto rec_of = [&](int x) { return records + (size_t)(x == c ? 2 * c + k : 2 * x) * L::REC; };
    float top = -1e30f, sum = 0.f;
    for (int x = c; x <= last; ++x) top = fmaxf(top, reinterpret_cast<const float2*>(rec_of(x) + TL_ROWS * HD)[row].x);
    float4 acc[HD / 32];
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = c; x <= last; ++x) {
      const float2 ml = reinterpret_cast<const float2*>(rec_of(x) + TL_ROWS * HD)[row];
      const float wt = ml.y == 0.f ? 0.f : ml.y * pg_ex2(ml.x - top);
      sum += wt;
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {
        const float4 v = reinterpret_cast<const float4*>(rec_of(x))[(warp * (HD / 32) + j) * TL_ROWS + row];
        acc[j].x = fmaf(wt, v.x, acc[j].x);
        acc[j].y = fmaf(wt, v.y, acc[j].y);
        acc[j].z = fmaf(wt, v.z, acc[j].z);
        acc[j].w = fmaf(wt, v.w, acc[j].w);
      }
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    T* dst = reinterpret_cast<T*>(p.out) + (long long)(s.first + i) * p.ld_o + (long long)(d.g * G + rr - i * G) * HD + warp * (HD / 8);
#pragma unroll
    for (int j = 0; j < HD / 32; ++j)
      *reinterpret_cast<uint2*>(dst + 4 * j) = make_uint2(Cvt<T>::pack2(acc[j].x * f, acc[j].y * f), Cvt<T>::pack2(acc[j].z * f, acc[j].w * f));
  }
}

template <typename T, int HD>
static int tl_go(const PgAttn& p, cudaStream_t st) {
  using L = Tl<HD>;
  // at least 120 KB, so that one block takes an SM with its tensor memory
  const size_t smem = std::max<size_t>(120 * 1024, 1024 + 2 * L::Q + L::STAGES * (L::STAGE + 32) + 16 * 8 + 128 + 16 + (size_t)(p.a.B + 1) * 4);
  const int blocks = pg_sms();
  GB_PDL_LAUNCH_SMEM((paged_tile_kernel<T, HD>), dim3(blocks), dim3(TL_THREADS), smem, st, p);
  const int rc = gb_launch_rc();
  if (rc) return rc;
  GB_PDL_LAUNCH((paged_tile_join_kernel<T, HD>), dim3(blocks, TL_ROWS / 32), dim3(256), st, p, blocks);
  return gb_launch_rc();
}

template <typename T>
static int tl_size(const PgAttn& p, cudaStream_t st) { return p.a.hd == 32 ? tl_go<T, 32>(p, st) : p.a.hd == 64 ? tl_go<T, 64>(p, st) : tl_go<T, 128>(p, st); }

long long pg_tile_ws(const PgAttn& p) { return 2ll * pg_sms() * (TL_ROWS * (p.a.hd + 2) + (long long)(sizeof(TlDesc) / 4)); }

int pg_tile_attn(const PgAttn& p, cudaStream_t st) { return p.a.is_bf16 ? tl_size<__nv_bfloat16>(p, st) : tl_size<__half>(p, st); }

}  // namespace gb
