// Attention over the paged 8-bit cache for many query rows a key head (interface in gb_paged.h, choice in paged_attn.cu): prompts and portions of them.
//
// Rows are (token, query head of the group) pairs of a key head, 256 of them an item, so any group size fills the tiles and a page is expanded once for all its query heads.
// What bounds it: the exponentials (one a score, 16 a cycle and SM) and, at hd 128, the products about as much; neither is reached, since a warpgroup's step on a page is a chain of
// scores, maxima, exponentials and products (2100 to 2200 cycles for both, of which the exponentials are 1024: special functions 49 % busy at hd 64, 47 % at hd 128).
//
// One block an SM: two warpgroups of soft-max threads, a row each; four warps expand the pages from codes in global memory to float16 integers in the swizzled layout of the MMAs
// (integers up to 127 are exact, the scales go into the soft-max: a key scale into the score's factor, a value scale into the weight's exponent, as in paged_attn_token.cu, but that a
// row's largest weight is held as 2^6 to 2^15, so that one is off by 2^-31 of the largest where that is more than half a step of 2^-11 of itself); a warp for each warpgroup issues (one for both was busy issuing and asking barriers all the time).  Scores and weights share tensor memory: weights go over scores that have been read,
// and are the A operand of the second product from there.
//
// The work is dealt in pages: all (sequence, key head, item, page) in a row are cut into equal runs, one a block.  Items that a cut goes through leave records
// that a second kernel joins.  A causal prompt's items differ in length by a factor of its tiles; dealt whole, the last round of items would leave most SMs idle.
#include <algorithm>

#include "paged_attn.cuh"
#include "tc_tiles.cuh"

namespace gb {

constexpr float TL_OFF = 7.f, TL_LAZY = 8.f;   // weights are held as 2^7 of themselves and may grow 2^8 before the sums are rescaled
constexpr float TL_NONE = -1000.f;             // less than any exponent of a value scale

template <int HD>
struct Tl {
  // Tensor memory has 512 columns; a warpgroup (128 rows) takes HD of them for results and 64 for a buffer of the scores of a page, which its weights go over.  That leaves room for two
  // buffers at hd 128 and three else, so that the products of a page run while the soft-max is at work on the next.  Measured beside it, with two places an item ahead of its pages (TlWalk): one buffer of 128 keys, 7 ragged prompts
  // (12/4 heads of 64) 188 us instead of 197, but 571 instead of 534 for 2048 tokens behind 14000 (32/8 heads of 128); four warpgroups with one buffer, scores
  // read twice for want of registers, 183, but 28.8 instead of 23.6 for a prompt of 1024.
  static constexpr int WGS = 2, BUFS = HD == 128 ? 2 : 3, ROWS = 128 * WGS, THREADS = 128 * (WGS + 2);
  static constexpr int E_WARP = 4 * WGS, I_WARP = E_WARP + 4;                // first warps that expand and that issue
  static constexpr int PANELS = HD <= 64 ? 1 : 2;             // 64 dimensions each
  static constexpr int Q = 128 * 128 * PANELS, K = PG * 128 * PANELS, V = HD * 128, STAGE = K + V, STAGES = HD == 128 ? 4 : 6;
  // registers a thread: soft-max, expanding, issuing; launched with 128, so 2 x 128 x S + 128 x (E + I) is at most 65536
  static constexpr int REGS_S = 184, REGS_E = 88, REGS_I = 56;
  static_assert(REGS_S >= 128 && REGS_E <= 128 && REGS_I <= 128 && 2 * 128 * REGS_S + 128 * (REGS_E + REGS_I) <= 65536 && THREADS == 512,
                "soft-max warps take registers, the others give them, and no more than the block has");
  static constexpr int O0 = 64 * BUFS * WGS, AHEAD = 4;       // first column of the results; places of an item ahead of its pages' (TlWalk)
  static constexpr int REC = ROWS * (HD + 2);                 // floats of a record: [HD / 4][ROWS] four results, then [ROWS] pairs (maximum, sum)
};

// What a record is of: places of its item, and which it is.  f1 == 0: nothing.
struct TlDesc { int f0, f1, b, g, qt, quota, pad0, pad1; };

// Bounded waits: false once the block has given up.  The first polls are all that a phase takes that is over already.  (The rest is no call: scores are in registers.)
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

struct TlItem { int lo, n; };                                 // first page that any of its rows sees, number of them
template <int ROWS>
__device__ __forceinline__ TlItem tl_item(const PgAttn& p, const PgSeq& s, int G, int qt) {
  const int r1 = min(s.n * G, (qt + 1) * ROWS) - 1;
  const int p0 = s.start + qt * ROWS / G, p1 = s.start + r1 / G;
  const int lo = p.window > 0 ? max(0, p0 - p.window + 1) / PG : 0;
  return {lo, p1 / PG - lo + 1};
}

// A block's walk over its run: places f ... end, one piece of an item after the other.  An item has a place for each page and, ahead of them, AHEAD for its start and end: loading queries,
// filling and emptying the pipelines, and the last pages' masks.  Four of them: 7 ragged prompts (12/4 heads of 64) 184 us, 2 of them 196, 3 of them 190, 6 of them 184; a prompt of 2048 tokens
// 32.8, 37.4, 33.3, 34.2.
template <int ROWS, int AHEAD>
struct TlWalk {
  int f, end, b, g, qt, k;                                    // k: places of the item that come before place f
  PgSeq s;
  int tiles;
  __device__ __forceinline__ void load(const PgAttn& p, int G) {
    s = pg_seq(p.a, b);
    tiles = (s.n * G + ROWS - 1) / ROWS;
  }
  // the run's part of this item: pages k0 ... k1 - 1
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
__global__ void __launch_bounds__(Tl<HD>::THREADS, 1) paged_tile_kernel(const __grid_constant__ PgAttn p) {
  using L = Tl<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sKV = smem + L::WGS * L::Q;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + L::STAGES * L::STAGE);
  uint64_t *k_full = bars, *k_empty = k_full + L::STAGES, *v_full = k_empty + L::STAGES, *v_empty = v_full + L::STAGES;
  uint64_t *s_full = v_empty + L::STAGES, *p_ready = s_full + 6, *o_full = s_full + 12, *q_full = s_full + 18;     // but for the last: [warpgroup][buffer], so that no
                                                                              // barrier can be two phases on
  float2* scales = reinterpret_cast<float2*>(s_full + 20);                    // of sixteen pages (they outlive a stage): key scale, value scale; a negative key scale: no page
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scales + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* cum = reinterpret_cast<int*>(tmem_slot + 2);                           // places (of one head) of the sequences before
  const gb_paged& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.H / a.KV;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) { mbar_init(&k_full[s], 4); mbar_init(&k_empty[s], L::WGS); mbar_init(&v_full[s], 4); mbar_init(&v_empty[s], L::WGS); }
    for (int w = 0; w < 6; ++w) { mbar_init(&s_full[w], 2); mbar_init(&p_ready[w], 4); mbar_init(&o_full[w], 1); }
    for (int w = 0; w < 2; ++w) mbar_init(&q_full[w], 4);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == L::I_WARP) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  pdl_wait();
  for (int b = warp; b < a.B; b += L::THREADS / 32) {
    const PgSeq s = pg_seq(a, b);
    const int tiles = (s.n * G + L::ROWS - 1) / L::ROWS;
    int n = 0;
    for (int qt = lane; qt < tiles; qt += 32) n += tl_item<L::ROWS>(p, s, G, qt).n + L::AHEAD;
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
  TlWalk<L::ROWS, L::AHEAD> start;
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
      const int n = q0 + lane < start.tiles ? tl_item<L::ROWS>(p, start.s, G, q0 + lane).n + L::AHEAD : 0;
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

    if (warp < L::E_WARP) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::REGS_S));
      // ------------------------------------------------------------------------------------------ soft-max: a thread a row
      const int wg = warp >> 2, r = threadIdx.x & 127;
      const uint32_t row = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t tO = tmem + L::O0 + wg * HD + row;
      uint8_t* q_at = sQ + wg * L::Q;
      uint32_t kv_it = 0, it = 0;                              // pages so far; those of this warpgroup
      bool ok = true;
      TlWalk<L::ROWS, L::AHEAD> w = start;
      while (w.f < w.end && ok) {
        const TlItem item = tl_item<L::ROWS>(p, w.s, G, w.qt);
        const int rows = w.s.n * G, first = w.qt * L::ROWS + wg * 128;
        int k0, k1;
        w.part(item, k0, k1);
        if (first < rows && k0 < k1) {
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
          // soft-max of 2^s: m2, the running maximum (or up to TL_LAZY less), to which l is the sum; m2 + rel, that of s + e, with e a value scale's exponent, to which the
          // weights and the results are (d, which is rel rounded up): what a row does not see, or gives no weight, does not move either
          float m2 = PG_START, rel = TL_NONE, l = 0.f;
          bool far = false;
          for (int t = k0; t < k1; ++t, ++it, ++kv_it) {
            const uint32_t buf = it % L::BUFS, phase = (it / L::BUFS) & 1u;
            const uint32_t tS = tmem + wg * (64 * L::BUFS) + buf * 64 + row;
            if (!tl_wait(&s_full[wg * L::BUFS + buf], phase, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag)) { ok = false; break; }
            tc_fence_after();
            const float2 sc = scales[kv_it & 15];
            const int base = (item.lo + t) * PG;
            const bool edge = base + PG - 1 > pos_a || (p.window > 0 && pos_z - p.window + 1 > base) || sc.x < 0.f;
            // a bit a column, so that a column costs a test and a choice: three comparisons each were a third of the loop's code, and its fetching showed
            uint32_t see[2] = {0xffffffffu, 0xffffffffu};
            if (edge) {
              const int hi = pos - base, lo = p.window > 0 ? pos - p.window + 1 - base : 0;
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                const int h = hi - 32 * w, l0 = lo - 32 * w;              // columns l0 ... h of this word
                see[w] = sc.x < 0.f ? 0u : (h >= 31 ? 0xffffffffu : h < 0 ? 0u : (2u << h) - 1u) & (l0 <= 0 ? 0xffffffffu : l0 > 31 ? 0u : 0xffffffffu << l0);
              }
            }
            float x[64];
            auto hide = [&](float* y, uint32_t bits) {
              if (edge) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (!(bits & (1u << k))) y[k] = -INFINITY;
              }
            };
            auto most = [&](const float* y) {
              float mr[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) mr[c] = fmaxf(y[c], y[4 + c]);
#pragma unroll
              for (int k = 8; k < 32; k += 8)
#pragma unroll
                for (int c = 0; c < 4; ++c) mr[c] = fmaxf(fmaxf(mr[c], y[k + c]), y[k + 4 + c]);
              return fmaxf(fmaxf(mr[0], mr[1]), fmaxf(mr[2], mr[3]));
            };
            {
              uint32_t(*rg)[32] = reinterpret_cast<uint32_t(*)[32]>(x);
              tmem_ld_32x32(tS, rg[0]);
              tmem_ld_32x32(tS + 32, rg[1]);
              tmem_ld_wait();
            }
            hide(x, see[0]);
            hide(x + 32, see[1]);
            float top = fmaxf(most(x), most(x + 32));
            // a factor that is too small for fp32 must not make nothing of a hidden score
            float f = qs * fabsf(sc.x);
            f = f == 0.f ? 1e-37f : f;
            top = __fmul_ru(top, f);                           // never less than the score that the weights are found from
            const float ev = (float)((int)(__float_as_uint(sc.y) >> 23) - 127);
            float d = ceilf(rel);
            if (__any_sync(0xffffffffu, fmaxf(top - m2, top - m2 + (ev - d)) > TL_LAZY)) {
              const float mn = fmaxf(m2, top), down = m2 - mn, was = d;
              l *= pg_ex2(down);
              m2 = mn;
              rel = fmaxf(rel + down, ev + (top - mn));                   // where all of the page is hidden top is -inf
              d = ceilf(rel);
              far = __any_sync(0xffffffffu, pg_far(m2));
              if (t > k0) {                                    // what the pages before added up to is rescaled, once it is there
                if (!tl_wait(&o_full[wg * L::BUFS + (it - 1u) % L::BUFS], ((it - 1u) / L::BUFS) & 1u, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const float c2 = pg_ex2(down + (was - d));
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
            }
            const float de = fmaxf(ev - d, -60.f);                        // no less, so that the row sum gets all weights: 2^-60 of the page's values is nothing
            float2 ff = make_float2(f, f), bias = make_float2(TL_OFF + de - m2, TL_OFF + de - m2);
            if (far) {                                           // scores less their maximum first: it would swallow the rest of the exponent
#pragma unroll
              for (int j = 0; j < 64; j += 2) {
                const float2 y = tl_fma2(make_float2(x[j], x[j + 1]), ff, make_float2(-m2, -m2));
                x[j] = y.x;
                x[j + 1] = y.y;
              }
              ff = make_float2(1.f, 1.f);
              bias = make_float2(TL_OFF + de, TL_OFF + de);
            }
            float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t pk[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const int j = 32 * c + 2 * k;
                float2 e = tl_fma2(make_float2(x[j], x[j + 1]), ff, bias);
                e.x = pg_ex2(e.x);
                e.y = pg_ex2(e.y);
                ls[k & 1] = tl_add2(ls[k & 1], e);
                pk[k] = Cvt<__half>::pack2(e.x, e.y);
              }
              tmem_st_32x16(tS + c * 16, pk);
            }
            l = fmaf((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y), pg_ex2(-de), l);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[wg * L::BUFS + buf]);
          }
          if (!ok) break;
          if (!tl_wait(&o_full[wg * L::BUFS + (it - 1u) % L::BUFS], ((it - 1u) / L::BUFS) & 1u, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const bool whole = k0 == 0 && k1 == item.n;
          const int f0 = w.f - w.k + L::AHEAD, slot = 2 * blockIdx.x + (f0 > start.f ? 1 : 0);
          float* rec = records + (size_t)slot * L::REC;
          const float inv = l == 0.f ? 0.f : 1.f / l, unit = pg_pow2(ceilf(rel));       // 2^d / l, in two steps: together they may be less than fp32 has
          T* dst = reinterpret_cast<T*>(p.out) + (long long)(w.s.first + i) * p.ld_o + (long long)(w.g * G + rr - i * G) * HD;
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t rg[32];
            tmem_ld_32x32(tO + c * 32, rg);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(rg[k]) * inv * unit;
            if (whole) {
              if (row_ok) {
#pragma unroll
                for (int k = 0; k < 4; ++k) pg_store8(dst + c * 32 + 8 * k, v + 8 * k);
              }
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                reinterpret_cast<float4*>(rec)[(c * 8 + k) * L::ROWS + wg * 128 + r] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            }
          }
          if (!whole) {
            reinterpret_cast<float2*>(rec + L::ROWS * HD)[wg * 128 + r] = make_float2(m2, l);
            if (threadIdx.x == 0) desc[slot] = {f0, f0 + item.n, w.b, w.g, w.qt, quota, 0, 0};
          }
          tc_fence_before();
        } else {
          kv_it += k1 - k0;
        }
        w.next(p, G, cum, item);
      }
    } else if (warp < L::I_WARP) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_E));
      // ------------------------------------------------------------------------------------------ pages to float16
      const int tid = threadIdx.x - 32 * L::E_WARP;
      constexpr int NK = HD / 32;                              // chunks of 16 codes a thread has of a page's keys, and of its values
      uint32_t kv_it = 0;
      bool ok = true;
      TlWalk<L::ROWS, L::AHEAD> w = start;
      while (w.f < w.end && ok) {
        const TlItem item = tl_item<L::ROWS>(p, w.s, G, w.qt);
        int k0, k1;
        w.part(item, k0, k1);
        uint4 rk[NK], rv[NK];
        int id = -1, after = -1;                               // the page whose codes are on their way; what the table has for the one behind it
        float sc = 0.f;
        auto look = [&](int t) {                               // nothing waits for the answer here
          if (t < k1) after = a.table[(long long)w.b * a.W + item.lo + t];
        };
        auto fetch = [&](uint4 (&r)[NK], const signed char* from) {
          const uint4* src = reinterpret_cast<const uint4*>(from + ((long long)max(id, 0) * a.KV + w.g) * (PG * HD)) + tid;
#pragma unroll
          for (int c = 0; c < NK; ++c) r[c] = id < 0 ? make_uint4(0, 0, 0, 0) : src[c * 128];
        };
        auto fetch_keys = [&](int t) {                         // and the scales of page t, the number of page t + 1
          id = after;
          if ((unsigned)id >= (unsigned)a.pages) {
            atomicCAS(a.status, 0, ST_BAD_ARGUMENT);
            id = -1;
          }
          fetch(rk, a.k);
          if (tid < 2) sc = id >= 0 ? (tid == 0 ? a.ks : a.vs)[(long long)id * a.KV + w.g] : tid == 0 ? -1.f : PG_LEAST;
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
            const int ch = c * 128 + tid, key = ch / (HD / 16), d = (ch % (HD / 16)) * 16;        // 16 dimensions of a key
            uint32_t x[8];
            pg_halves(rk[c].x, x[0], x[1]);
            pg_halves(rk[c].y, x[2], x[3]);
            pg_halves(rk[c].z, x[4], x[5]);
            pg_halves(rk[c].w, x[6], x[7]);
            uint8_t* kp = sk + (d >> 6) * (PG * 128);
            *reinterpret_cast<uint4*>(kp + sw128_off(key, d & 63)) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(kp + sw128_off(key, (d & 63) + 8)) = make_uint4(x[4], x[5], x[6], x[7]);
          }
          if (tid < 2) reinterpret_cast<float*>(&scales[kv_it & 15])[tid] = sc;
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&k_full[st]);
          if (t + 1 < k1) fetch_keys(t + 1);
          if (!tl_wait(&v_empty[st], free, a.status, ST_TIMEOUT_EMPTY, abort_flag)) { ok = false; break; }
#pragma unroll
          for (int c = 0; c < NK; ++c) {
            const int ch = c * 128 + tid, vd = ch >> 2, vt = (ch & 3) * 16;                       // 16 tokens of a dimension
            uint32_t x[8];
            pg_halves(rv[c].x, x[0], x[1]);
            pg_halves(rv[c].y, x[2], x[3]);
            pg_halves(rv[c].z, x[4], x[5]);
            pg_halves(rv[c].w, x[6], x[7]);
            *reinterpret_cast<uint4*>(sv + sw128_off(vd, vt)) = make_uint4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint4*>(sv + sw128_off(vd, vt + 8)) = make_uint4(x[4], x[5], x[6], x[7]);
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
      if (warp < L::I_WARP + L::WGS) {
      // ------------------------------------------------------------------------------------------ MMAs
      const uint32_t on = elect_one();
      const uint32_t id_s = make_idesc_f16(0, 0, 0, 128, PG), id_o = make_idesc_f16(0, 0, 0, 128, HD);
      // What the loops go by is handed around by lane 0, which is how the compiler learns that it is the same for all: counters, descriptors and addresses then stay in
      // uniform registers, where these instructions want them (descriptors found lane by lane made issuing a tile's products take 1400 cycles a warpgroup).
      const int wg = warp - L::I_WARP, wu = __shfl_sync(0xffffffffu, wg, 0);
      uint32_t kv_it = 0, q_it = 0, it = 0, s_it = 0;          // pages; this warpgroup's pieces, pages summed, pages scored
      TlWalk<L::ROWS, L::AHEAD> w = start;
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), tS = tm + wu * (64 * L::BUFS), tO = tm + L::O0 + wu * HD;
      const uint64_t dq = make_smem_desc_sw128(smem_u32(sQ) + wu * L::Q, 16, 1024), dkv = make_smem_desc_sw128(smem_u32(sKV), 16, 1024);
      auto full = [&](uint64_t* bar, uint32_t at) {
        wait_or_report(&bar[at % L::STAGES], (at / L::STAGES) & 1u, a.status, ST_TIMEOUT_FULL, abort_flag);
        tc_fence_after();
      };
      bool more = w.f < w.end;
      while (__shfl_sync(0xffffffffu, (int)more, 0)) {
        const TlItem item = tl_item<L::ROWS>(p, w.s, G, w.qt);
        int k0, k1;
        w.part(item, k0, k1);
        const int all = __shfl_sync(0xffffffffu, k1 - k0, 0), n = __shfl_sync(0xffffffffu, (int)(w.qt * L::ROWS + wg * 128 < w.s.n * G), 0) ? all : 0;
        auto scores = [&](uint32_t at) {
          const uint32_t buf = s_it % L::BUFS;
          ++s_it;
          const uint64_t db = dkv + (at % L::STAGES) * (L::STAGE >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            umma_f16_on(on, tS + buf * 64, dq + (((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4), db + (((kk >> 2) * (PG * 128) + (kk & 3) * 32) >> 4), id_s, kk > 0 ? 1u : 0u);
          if (on) mbar_arrive(&s_full[wg * L::BUFS + buf]);          // hands on what k_full brought: the scales, which no MMA touches
          umma_commit_on(on, &s_full[wg * L::BUFS + buf]);
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
          const uint32_t at = kv_it + t, buf = it % L::BUFS, phase = (it / L::BUFS) & 1u;
          full(v_full, at);
          const uint64_t dv = dkv + (((at % L::STAGES) * L::STAGE + L::K) >> 4);
          wait_or_report(&p_ready[wg * L::BUFS + buf], phase, a.status, ST_TIMEOUT_TMEM_EMPTY, abort_flag);
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < PG / 16; ++kk)
            umma_f16_ts_on(on, tO, tS + buf * 64 + kk * 8, dv + (kk * 32 >> 4), id_o, t > 0 || kk > 0 ? 1u : 0u);
          umma_commit_on(on, &o_full[wg * L::BUFS + buf]);
          umma_commit_on(on, &v_empty[at % L::STAGES]);
          if (t + L::BUFS < n) {
            // scores go where these weights are, and products of different accumulators need not run in the order of their issue
            full(k_full, at + L::BUFS);
            wait_or_report(&o_full[wg * L::BUFS + buf], phase, a.status, ST_TIMEOUT_TMEM_FULL, abort_flag);
            tc_fence_after();
            scores(at + L::BUFS);
          }
          ++it;
        }
        // Pages that are other warpgroups' alone are followed stage by stage all the same: a barrier's phase is known by its parity, so no warp may be more than one ahead.
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
  if (warp == L::I_WARP) { tc_fence_after(); tmem_dealloc(tmem, 512); }
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
    const int rr = d.qt * L::ROWS + row, i = rr / G;
    if (rr >= s.n * G) continue;
    auto rec_of = [&](int x) { return records + (size_t)(x == c ? 2 * c + k : 2 * x) * L::REC; };
    float top = PG_START, sum = 0.f;
    for (int x = c; x <= last; ++x) top = fmaxf(top, reinterpret_cast<const float2*>(rec_of(x) + L::ROWS * HD)[row].x);
    float4 acc[HD / 32];
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = c; x <= last; ++x) {
      const float2 ml = reinterpret_cast<const float2*>(rec_of(x) + L::ROWS * HD)[row];
      const float wt = ml.y == 0.f ? 0.f : ml.y * pg_ex2(ml.x - top);
      sum += wt;
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {
        const float4 v = reinterpret_cast<const float4*>(rec_of(x))[(warp * (HD / 32) + j) * L::ROWS + row];
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
  const size_t smem = std::max<size_t>(120 * 1024, 1024 + L::WGS * L::Q + L::STAGES * (L::STAGE + 32) + 20 * 8 + 128 + 16 + (size_t)(p.a.B + 1) * 4);
  const int blocks = pg_sms();
  GB_PDL_LAUNCH_SMEM((paged_tile_kernel<T, HD>), dim3(blocks), dim3(L::THREADS), smem, st, p);
  const int rc = gb_launch_rc();
  if (rc) return rc;
  GB_PDL_LAUNCH((paged_tile_join_kernel<T, HD>), dim3(blocks, L::ROWS / 32), dim3(256), st, p, blocks);
  return gb_launch_rc();
}

template <typename T>
static int tl_size(const PgAttn& p, cudaStream_t st) { return p.a.hd == 32 ? tl_go<T, 32>(p, st) : p.a.hd == 64 ? tl_go<T, 64>(p, st) : tl_go<T, 128>(p, st); }

long long pg_tile_ws(const PgAttn& p) {
  const int rec = p.a.hd == 32 ? Tl<32>::REC : p.a.hd == 64 ? Tl<64>::REC : Tl<128>::REC;
  return 2ll * pg_sms() * (rec + (long long)(sizeof(TlDesc) / 4));
}

int pg_tile_attn(const PgAttn& p, cudaStream_t st) { return p.a.is_bf16 ? tl_size<__nv_bfloat16>(p, st) : tl_size<__half>(p, st); }

}  // namespace gb
