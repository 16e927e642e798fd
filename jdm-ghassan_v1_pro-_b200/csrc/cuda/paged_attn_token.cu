// Attention over the paged 8-bit cache for few query rows a key head (interface in gb_paged.h, choice in paged_attn.cu): a token or some proposed ones a sequence.
//
// Bound by the bytes of the codes, so the work is cut by pages, not by sequences: all (sequence, key head, page) in a row are dealt to the GPU's warps in equal runs, whatever the
// lengths are (mode "balanced"; the lengths are on the device and so is the dealing).  A warp streams its run through a ring of its own in shared memory, a bulk copy a
// page of keys or values (4 KB at hd 64), and waits for nobody until its run is over: pieces of a (sequence, head) that lie in one warp are finished there, the others are joined
// first in the block, then, across blocks, by a second kernel.  Where all items have a block each and few pages, a block takes an item and nothing is left to join (mode "item").
// On the device: 192 sequences of 100 to 8000 tokens (8/2 heads of 64) 48.6 us, 4.1 TB/s of codes; one of 100001 (32/8 heads of 128) 44.1 us, 4.6 TB/s; 32 of 3 to 4095 (12/4 heads of
// 64) 16.4 us, 2.1 TB/s, of which about 2.3 us pass before the first page is there and 3 us in joining a block's warps.
//
// A page is two products on the legacy tensor path, with the codes as float16 integers (exact): keys x queries and values x weights, so that
// queries (8 columns) rather than keys are padded; 16 rows of queries would pad 3 of them to 16.  The order of the contracted dimensions is free as long as both operands have the
// same, so a lane takes 16 consecutive bytes of a key, or of a value's tokens, and these are its MMA fragments.  The page's key scale joins the score's factor and its value
// scale the exponent of the weights: w = 2^(s - m + 15 + e - d), with m the row's running maximum, e the value scale's exponent and m + d the running maximum of s + e, rounded up: what a
// row does not see, or gives no weight, does not move its d, however large its values are.  Rounded to float16 a weight is off by half a step of 2^-11 of itself, or by 2^-39 of the
// largest 2^(s + e - d) that the row sees, whichever is more; the row sum has the unrounded weights.  Queries are scaled by a power of two so that a
// row's largest is between 2^14 and 2^15: float16 then holds them as exactly as bfloat16 does.
#include <algorithm>

#include "paged_attn.cuh"

namespace gb {

constexpr int TK_WARPS = 8, TK_THREADS = 32 * TK_WARPS;
// Most pages a sequence may show in mode "item", which saves the second kernel and waits for a block's own pages only.  us, mode "item" against "balanced", 12/4 heads of 64, one
// token behind 4, 8, 16, 24, 32 and 64 pages: one sequence 5.0, 5.5, 7.1, 8.8, 10.5, 17.0 against 7.1, 7.0, 8.3, 8.6, 8.6, 9.3; 32 sequences as long as each other gain more
// (10.9 against 12.7 at 32 pages), but lengths are on the device and blocks of a ragged batch wait for the longest.
constexpr int TK_ITEM_PAGES = 16;
constexpr float TK_OFF = 15.f;               // the largest weight is held as 2^15 or (d is rounded up) a little less, the most float16 takes
constexpr float TK_NONE = -1000.f;           // less than any exponent of a value scale

__device__ __forceinline__ void tk_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tk_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void tk_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Row r of a key head's queries: token r / G, head r % G of its group.
struct TkRow { int token, head; };
// Where the row goes, for the sequence with rows from `first` on and key head g.
template <typename T, int HD>
__device__ __forceinline__ T* tk_out(const PgAttn& p, int first, int g, const TkRow& r) {
  return reinterpret_cast<T*>(p.out) + (long long)(first + r.token) * p.ld_o + (long long)(g * (p.H / p.a.KV) + r.head) * HD;
}

// Pages of sequence b that its queries see: from page `lo`, `n` of them.
struct TkPages { int lo, n; };
struct TkSeq { PgSeq s; int lo; };           // a sequence and its first visible page
__device__ __forceinline__ TkPages tk_pages(const PgAttn& p, const PgSeq& s) {
  if (s.n == 0) return {0, 0};
  const int lo = p.window > 0 ? max(0, s.start - p.window + 1) / PG : 0;
  return {lo, (s.start + s.n - 1) / PG - lo + 1};
}

// Whose piece a warp left in a record: the item, its places, its sequence's first row, its rows.
struct TkCut { int item, f0, f1, first, rows, quota, pad0, pad1; };
// In the workspace: two of these a block, item -1 where there is nothing, then the records of which blocks' pieces they are.
__device__ __forceinline__ TkCut* tk_cuts(const PgAttn& p) { return reinterpret_cast<TkCut*>(p.part); }
__device__ __forceinline__ float* tk_parts(const PgAttn& p, int blocks) { return p.part + (size_t)2 * blocks * (sizeof(TkCut) / 4); }
// A record: R x HD results, then R pairs (maximum, sum)
template <int HD> __host__ __device__ constexpr int tk_record(int R) { return R * (HD + 2); }

template <typename T, int HD, int NQ>
__global__ void __launch_bounds__(TK_THREADS, 1) paged_token_kernel(const __grid_constant__ PgAttn p, int R, int slots, int item_mode) {
  constexpr int SLOT = PG * HD, KK = HD / 16, VW = HD / 4 < 16 ? HD / 4 : 16, WPC = VW / 4;   // bytes of a lane's chunk of a key, words of it
  extern __shared__ __align__(128) uint8_t smem[];
  const gb_paged& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int rec_n = tk_record<HD>(R);
  uint8_t* ring = smem + (size_t)warp * slots * SLOT;
  float* heads = reinterpret_cast<float*>(smem + (size_t)TK_WARPS * slots * SLOT);            // records of the warps' first items
  uint64_t* bars = reinterpret_cast<uint64_t*>(heads + (TK_WARPS * rec_n + 1) / 2 * 2);
  TkCut* cut = reinterpret_cast<TkCut*>(bars + TK_WARPS * slots);                             // what the warps' records are of
  int* scan = reinterpret_cast<int*>(cut + 2 * TK_WARPS);                                     // sums of the warps
  volatile int* abort_flag = scan + TK_WARPS;
  int* cum = scan + TK_WARPS + 1;                                                             // pages of the sequences before
  TkRow* rows_of = reinterpret_cast<TkRow*>(cum + (item_mode ? 1 : p.a.B) + 1);
  TkSeq* seqs = reinterpret_cast<TkSeq*>(rows_of + 8 * NQ);
  uint64_t* bar = bars + warp * slots;

  const int G = p.H / a.KV;
  if (warp == 1 && lane < 8 * NQ) rows_of[lane] = {lane / G, lane % G};
  if (lane == 0) {
    for (int s = 0; s < slots; ++s) mbar_init(&bar[s], 1);
    cut[2 * warp].item = cut[2 * warp + 1].item = -1;
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  pdl_wait();
  // the run of this block: items [ib, ...) of `KVs` heads, pages [c_lo, c_hi) of them all, `quota` a warp
  const int KVs = item_mode ? 1 : a.KV, b_base = item_mode ? (int)blockIdx.x / a.KV : 0, g_base = item_mode ? (int)blockIdx.x % a.KV : 0;
  const int nb = item_mode ? 1 : a.B;
  if (item_mode) {
    if (threadIdx.x == 0) {
      cum[0] = 0;
      const PgSeq sq = pg_seq(a, b_base);
      const TkPages v = tk_pages(p, sq);
      cum[1] = v.n;
      seqs[0] = {sq, v.lo};
    }
    __syncthreads();
  } else {
    int before = 0;
    for (int b0 = 0; b0 < nb; b0 += TK_THREADS) {
      const int b = b0 + (int)threadIdx.x;
      int v = 0;
      if (b < nb) {
        const PgSeq sq = pg_seq(a, b);
        const TkPages seen = tk_pages(p, sq);
        v = seen.n;
        seqs[b] = {sq, seen.lo};
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) scan[warp] = v;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w < TK_WARPS; ++w) {
        if (w < warp) v += scan[w];
        all += scan[w];
      }
      if (b < nb) cum[b + 1] = before + v;
      before += all;
      __syncthreads();
    }
    if (threadIdx.x == 0) cum[0] = 0;
    __syncthreads();
  }
  if (!item_mode && threadIdx.x == 0) tk_cuts(p)[2 * blockIdx.x].item = tk_cuts(p)[2 * blockIdx.x + 1].item = -1;
  const int total = KVs * cum[nb];
  const int blocks = item_mode ? 1 : (int)gridDim.x, quota = max(1, (total + TK_WARPS * blocks - 1) / (TK_WARPS * blocks));
  const int c_lo = item_mode ? 0 : min(total, (int)blockIdx.x * TK_WARPS * quota), c_hi = min(total, c_lo + TK_WARPS * quota);
  const int w_lo = min(c_hi, c_lo + warp * quota), w_hi = min(c_hi, w_lo + quota);
  auto seq_of = [&](int f) {                  // the sequence whose pages hold place f
    int lo = 0, hi = nb;                      // cum[lo] * KVs <= f < cum[hi] * KVs
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] * KVs <= f) lo = mid; else hi = mid;
    }
    return lo;
  };

  uint32_t qf[NQ][KK][2];
  float qs[NQ][2], m[NQ][2], l[NQ][2], rel[NQ][2], o[NQ][KK][4];   // rel: the largest s + e so far, less m; d is rel rounded up
  int item = -1, pos0 = 0, n_new = 0, f_begin = 0, f_end = 0;
  PgSeq sq{0, 0, 0};
  bool far = false;                           // a maximum is large (pg_far)

  // A lane has HD / 4 numbers of its rows, where it has them of a key.  Those of the warp's first item are asked for ahead of all else.
  uint4 raw[NQ][HD / 32];
  auto fetch_queries = [&](const PgSeq& s, int g) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const TkRow r = rows_of[8 * q + gq];
      const bool on = r.token < s.n;
      const T* src = reinterpret_cast<const T*>(p.q) + (long long)(s.first + (on ? r.token : 0)) * p.ld_q + (long long)(g * G + r.head) * HD + tq * VW;
#pragma unroll
      for (int k = 0; k < HD / 32; ++k) raw[q][k] = on ? *reinterpret_cast<const uint4*>(src + (k * 8 / VW) * 64 + (k * 8) % VW) : make_uint4(0, 0, 0, 0);
    }
  };
  auto make_queries = [&]() {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      float x[HD / 4];
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < HD / 32; ++k) {
        const uint32_t w[4] = {raw[q][k].x, raw[q][k].y, raw[q][k].z, raw[q][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = Cvt<T>::unpack2(w[e]);
          x[8 * k + 2 * e] = v.x;
          x[8 * k + 2 * e + 1] = v.y;
          top = max(top, max(__float_as_uint(fabsf(v.x)), __float_as_uint(fabsf(v.y))));
        }
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^14 / (power of two of the largest), and its inverse; a row with a number that is not finite gives NaN
      const int e = top == 0 ? 127 : min(max(254 + 14 - (int)(top >> 23), 1), 253);
      const float mul = __uint_as_float((uint32_t)e << 23), inv = __uint_as_float((uint32_t)(254 - e) << 23);
      const float f = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : inv * p.scale2;
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        const float* y = x + k * 4;
        qf[q][k][0] = Cvt<__half>::pack2(y[0] * mul, y[1] * mul);
        qf[q][k][1] = Cvt<__half>::pack2(y[2] * mul, y[3] * mul);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {           // the factor where scores have it: lanes of queries 2t, 2t + 1
        qs[q][c] = __shfl_sync(0xffffffffu, f, (2 * tq + c) * 4);
        m[q][c] = PG_START;
        l[q][c] = 0.f;
        rel[q][c] = TK_NONE;
      }
#pragma unroll
      for (int k = 0; k < KK; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[q][k][c] = 0.f;
    }
    far = false;
  };

  // the piece at hand is over: to the output where it is the whole item, else into a record
  auto finish = [&]() {
    if (item < 0) return;
    const int rows = sq.n * G;
    const bool whole = f_begin >= w_lo && f_end <= w_hi, first = f_begin <= w_lo;
    float* rec = first ? heads + warp * rec_n : reinterpret_cast<float*>(ring);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s = l[q][c];
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        s += __shfl_xor_sync(0xffffffffu, s, 8);
        s += __shfl_xor_sync(0xffffffffu, s, 16);
        // 2^d / s, in two steps: together they may be less than fp32 has
        const float f = s == 0.f ? 0.f : __fdividef(1.f, s), unit = pg_pow2(ceilf(rel[q][c]));
        const int r = 8 * q + 2 * tq + c;
        if (r >= rows) continue;
        if (whole) {
          T* dst = tk_out<T, HD>(p, sq.first, g_base + item % KVs, rows_of[r]) + gq;
#pragma unroll
          for (int k = 0; k < KK; ++k) {
            dst[16 * k] = Cvt<T>::from_f(o[q][k][c] * f * unit);
            dst[16 * k + 8] = Cvt<T>::from_f(o[q][k][2 + c] * f * unit);
          }
        } else {
          float* dst = rec + r * HD + gq;
#pragma unroll
          for (int k = 0; k < KK; ++k) {
            dst[16 * k] = o[q][k][c] * f * unit;
            dst[16 * k + 8] = o[q][k][2 + c] * f * unit;
          }
          if (gq == 0) *reinterpret_cast<float2*>(rec + R * HD + 2 * r) = make_float2(m[q][c], s);
        }
      }
    }
    if (!whole && lane == 0) cut[2 * warp + (first ? 0 : 1)] = {item, f_begin, f_end, sq.first, rows, quota, 0, 0};
    __syncwarp();
  };

  int slot_in = 0, slot_out = 0;
  uint32_t parity = 0;
  if (w_lo < w_hi) {
    const int b = seq_of(w_lo);
    fetch_queries(seqs[b].s, g_base + (w_lo - cum[b] * KVs) / (cum[b + 1] - cum[b]));
  }
  for (int base = w_lo; base < w_hi; base += 32) {
    const int cnt = min(32, w_hi - base);
    // lane i looks up page i of the batch
    int u_b = 0, u_g = 0, u_p = 0, u_id = 0, u_f = 0, u_np = 1;
    float u_ks = 1.f, u_vs = 1.f;
    bool u_bad = false;
    if (lane < cnt) {
      const int f = base + lane;
      u_b = seq_of(f);
      u_np = cum[u_b + 1] - cum[u_b];
      const int local = f - cum[u_b] * KVs;
      u_g = local / u_np;
      u_f = cum[u_b] * KVs + u_g * u_np;      // where its item begins
      u_p = seqs[u_b].lo + local - u_g * u_np;
      u_id = pg_page(a, b_base + u_b, u_p);
      u_bad = u_id < 0;
      if (u_bad) u_id = 0;
      const long long at = (long long)u_id * a.KV + g_base + u_g;
      if (!u_bad) { u_ks = a.ks[at]; u_vs = a.vs[at]; }
    }
    const unsigned bad = __ballot_sync(0xffffffffu, u_bad);
    auto issue = [&](int h) {                 // half h of the batch: keys (even) or values of page h / 2
      const int id = __shfl_sync(0xffffffffu, u_id, h >> 1), g = g_base + __shfl_sync(0xffffffffu, u_g, h >> 1);
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar[slot_in], SLOT);
        tk_bulk(ring + slot_in * SLOT, ((h & 1) ? a.v : a.k) + ((long long)id * a.KV + g) * SLOT, SLOT, &bar[slot_in]);
      }
      slot_in = slot_in + 1 == slots ? 0 : slot_in + 1;
    };
    auto next = [&]() {
      if (++slot_out == slots) { slot_out = 0; parity ^= 1u; }
    };
    for (int h = 0; h < min(slots, 2 * cnt); ++h) issue(h);
    for (int i = 0; i < cnt; ++i) {
      const int f0 = __shfl_sync(0xffffffffu, u_f, i), pg = __shfl_sync(0xffffffffu, u_p, i);
      const int ub = __shfl_sync(0xffffffffu, u_b, i), ug = __shfl_sync(0xffffffffu, u_g, i), it = ub * KVs + ug;
      if (it != item) {
        finish();
        item = it;
        f_begin = f0;
        f_end = f0 + __shfl_sync(0xffffffffu, u_np, i);
        sq = seqs[ub].s;
        pos0 = sq.start;
        n_new = sq.n;
        if (base != w_lo || i != 0) fetch_queries(sq, g_base + ug);
        make_queries();
      }
      const float ks = __shfl_sync(0xffffffffu, u_ks, i), vs = __shfl_sync(0xffffffffu, u_vs, i);
      const bool all_bad = (bad >> i) & 1u;
      // ---- scores: s[q][j]: keys kA, kA + 2 of key tile j (16 keys), queries 2t, 2t + 1
      float s[NQ][4][4];
      wait_or_report(&bar[slot_out], parity, a.status, ST_TIMEOUT_FULL, abort_flag);
      const uint8_t* sk = ring + slot_out * SLOT + tq * VW;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int kA = 16 * (gq >> 1) + 4 * j + (gq & 1);
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[q][j][c] = 0.f;
#pragma unroll
        for (int ch = 0; ch < HD / 4 / VW; ++ch) {
          uint32_t ra[WPC], rb[WPC];
          if constexpr (WPC == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(sk + kA * HD + 64 * ch), y = *reinterpret_cast<const uint4*>(sk + (kA + 2) * HD + 64 * ch);
            ra[0] = x.x; ra[1] = x.y; ra[2] = x.z; ra[3] = x.w;
            rb[0] = y.x; rb[1] = y.y; rb[2] = y.z; rb[3] = y.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sk + kA * HD), y = *reinterpret_cast<const uint2*>(sk + (kA + 2) * HD);
            ra[0] = x.x; ra[1] = x.y;
            rb[0] = y.x; rb[1] = y.y;
          }
#pragma unroll
          for (int w = 0; w < WPC; ++w) {
            uint32_t a0, a1, a2, a3;
            pg_halves(ra[w], a0, a2);
            pg_halves(rb[w], a1, a3);
#pragma unroll
            for (int q = 0; q < NQ; ++q) tk_mma(s[q][j], a0, a1, a2, a3, qf[q][ch * WPC + w][0], qf[q][ch * WPC + w][1]);
          }
        }
      }
      __syncwarp();
      next();
      if (2 * i + slots < 2 * cnt) issue(2 * i + slots);
      // ---- weights
      const bool edge = all_bad || (pg + 1) * PG > pos0 + 1 || (p.window > 0 && pg * PG <= pos0 + n_new - 1 - p.window);
      float f[NQ][2];
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        f[q][0] = qs[q][0] * ks;
        f[q][1] = qs[q][1] * ks;
      }
      if (edge) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int pos = pos0 + rows_of[8 * q + 2 * tq + c].token;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = pg * PG + 16 * (gq >> 1) + 4 * j + (gq & 1) + 2 * e;
                const bool see = !all_bad && key <= pos && (p.window <= 0 || key > pos - p.window);
                s[q][j][2 * e + c] = see ? s[q][j][2 * e + c] : -INFINITY;
              }
            f[q][c] = f[q][c] == 0.f ? 1e-37f : f[q][c];       // a factor that is too small for fp32 must not make a number of a hidden score
          }
      }
      const float ev = (float)((int)(__float_as_uint(vs) >> 23) - 127);
      bool same = true;
      uint32_t pb[NQ][4][2];
      float corr[NQ][2], scale_o[NQ][2], de[NQ][2];
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(fmaxf(fmaxf(s[q][0][c], s[q][0][2 + c]), fmaxf(s[q][1][c], s[q][1][2 + c])),
                          fmaxf(fmaxf(s[q][2][c], s[q][2][2 + c]), fmaxf(s[q][3][c], s[q][3][2 + c])));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = __fmul_ru(x, f[q][c]);                                   // never less than the score that the weights are found from
          const float mn = fmaxf(m[q][c], x), was = ceilf(rel[q][c]), down = m[q][c] - mn;
          rel[q][c] = fmaxf(rel[q][c] + down, ev + (x - mn));          // where all of the page is hidden x is -inf
          const float d = ceilf(rel[q][c]);
          de[q][c] = fmaxf(ev - d, -60.f);                             // no less, so that the row sum gets all weights: 2^-60 of the page's values is nothing
          corr[q][c] = pg_ex2(down);
          scale_o[q][c] = pg_ex2(down + (was - d));
          same = same && down == 0.f && was == d;
          m[q][c] = mn;
        }
      }
      if (__any_sync(0xffffffffu, !same)) {
        bool some = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          some = some || pg_far(m[q][0]) || pg_far(m[q][1]);
#pragma unroll
          for (int k = 0; k < KK; ++k)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[q][k][c] *= scale_o[q][c & 1];
        }
        far = __any_sync(0xffffffffu, some);
      }
      float base[NQ][2];
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int c = 0; c < 2; ++c) base[q][c] = TK_OFF + de[q][c] - m[q][c];
      if (far) {                                                       // scores less their maximum first: it would swallow the rest of the exponent
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s[q][j][c] = fmaf(s[q][j][c], f[q][c], -m[q][c]);
              s[q][j][2 + c] = fmaf(s[q][j][2 + c], f[q][c], -m[q][c]);
            }
            f[q][c] = 1.f;
            base[q][c] = TK_OFF + de[q][c];
          }
      }
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float w0 = pg_ex2(fmaf(s[q][j][2 * e], f[q][0], base[q][0]));
            const float w1 = pg_ex2(fmaf(s[q][j][2 * e + 1], f[q][1], base[q][1]));
            sum[0] += w0;
            sum[1] += w1;
            pb[q][j][e] = tk_transpose(Cvt<__half>::pack2(w0, w1));
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) l[q][c] = fmaf(l[q][c], corr[q][c], sum[c] * pg_ex2(-de[q][c]));
      }
      // ---- values: o[q][k]: dimensions 16k + g, 16k + g + 8, queries 2t, 2t + 1
      wait_or_report(&bar[slot_out], parity, a.status, ST_TIMEOUT_FULL, abort_flag);
      const uint8_t* sv = ring + slot_out * SLOT + tq * 16;
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        const uint4 x = *reinterpret_cast<const uint4*>(sv + (16 * k + gq) * PG), y = *reinterpret_cast<const uint4*>(sv + (16 * k + gq + 8) * PG);
        const uint32_t ra[4] = {x.x, x.y, x.z, x.w}, rb[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a0, a1, a2, a3;
          pg_halves(ra[j], a0, a2);
          pg_halves(rb[j], a1, a3);
#pragma unroll
          for (int q = 0; q < NQ; ++q) tk_mma(o[q][k], a0, a1, a2, a3, pb[q][j][0], pb[q][j][1]);
        }
      }
      __syncwarp();
      next();
      if (2 * i + 1 + slots < 2 * cnt) issue(2 * i + 1 + slots);
    }
  }
  finish();
  __syncthreads();

  // ---- pieces of the block's warps; those of one item are joined, a warp a row.  A lane has a record's maximum and sum, so the weights need no shared memory and no further barrier
  // (they took 1200 cycles of the block's end); loads are unconditional and picked from afterwards, since behind branches each would wait for the one before.
  auto rec_of = [&](int k) { return reinterpret_cast<const float*>((k & 1) ? smem + (size_t)(k >> 1) * slots * SLOT : reinterpret_cast<const uint8_t*>(heads + (k >> 1) * rec_n)); };
  constexpr int RECS = 2 * TK_WARPS;
  const int my_item = lane < RECS ? cut[lane].item : -1;
  const float* my_rec = rec_of(min(lane, RECS - 1));
  unsigned left = __ballot_sync(0xffffffffu, my_item >= 0);
  for (int turn = 0; left;) {
    const int k0 = __ffs(left) - 1;
    const unsigned same = __ballot_sync(0xffffffffu, my_item == __shfl_sync(0xffffffffu, my_item, k0));
    left &= ~same;
    const TkCut c = cut[k0];
    const bool whole = c.f0 >= c_lo && c.f1 <= c_hi;
    const int g = g_base + c.item % KVs, place = 2 * blockIdx.x + (c.f0 > c_lo ? 1 : 0);
    float* part = tk_parts(p, blocks) + (size_t)place * rec_n;
    // an item's records: perhaps the last one of a warp (odd), then first ones of the warps behind it
    const int w0 = (k0 + 1) >> 1, w1 = (33 - __clz(same)) >> 1;
    if (!whole && threadIdx.x == 0) tk_cuts(p)[place] = c;
    for (int r = 0; r < c.rows; ++r, ++turn) {
      if (turn % TK_WARPS != warp) continue;
      const float2 at = *reinterpret_cast<const float2*>(my_rec + R * HD + 2 * r);
      const bool mine = my_item == c.item;
      const float top = warp_max(mine ? at.x : PG_START);
      const float weight = !mine || at.y == 0.f ? 0.f : at.y * pg_ex2(at.x - top), sum = warp_sum(weight);
      const float f = sum == 0.f ? 0.f : __fdividef(1.f, sum);
#pragma unroll
      for (int d0 = 0; d0 < HD; d0 += 64) {
        const int d = d0 + 2 * lane % HD;                             // (hd 32: the upper lanes do the lower ones' work again)
        float u = 0.f, v = 0.f;
        auto add = [&](int k, const float* rec) {                     // what weighs nothing adds nothing, whatever it holds
          const float w = __shfl_sync(0xffffffffu, weight, k);
          const float2 x = *reinterpret_cast<const float2*>(rec);
          u += w == 0.f ? 0.f : w * x.x;
          v += w == 0.f ? 0.f : w * x.y;
        };
        if (k0 & 1) add(k0, rec_of(k0) + r * HD + d);
        const float* rec = heads + w0 * rec_n + r * HD + d;
#pragma unroll 4
        for (int w = w0; w < w1; ++w, rec += rec_n) add(2 * w, rec);
        if (whole) *reinterpret_cast<uint32_t*>(tk_out<T, HD>(p, c.first, g, rows_of[r]) + d) = Cvt<T>::pack2(u * f, v * f);
        else *reinterpret_cast<float2*>(part + r * HD + d) = make_float2(u * f, v * f);
      }
      if (!whole && lane == 0) *reinterpret_cast<float2*>(part + R * HD + 2 * r) = make_float2(top, sum);
    }
  }
}

// Joins what blocks left of the item that begins in block x's run and is cut by its end: one block a row.
constexpr int TJ_THREADS = 128;
template <typename T, int HD>
__global__ void __launch_bounds__(TJ_THREADS) paged_join_kernel(const __grid_constant__ PgAttn p, int R, int blocks) {
  __shared__ float top_of[4], wt[PG_MOST_BLOCKS], sums[TJ_THREADS / 32], acc_of[TJ_THREADS];
  const int c0 = blockIdx.x, r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  // of the two, the later begins last
  const TkCut a0 = tk_cuts(p)[2 * c0], a1 = tk_cuts(p)[2 * c0 + 1];
  const int k = a1.item >= 0 ? 1 : 0;
  const TkCut c = k ? a1 : a0;
  const int span = TK_WARPS * c.quota;
  if (c.item < 0 || r >= c.rows || c.f0 < c0 * span || c.f1 <= (c0 + 1) * span) return;
  const int rec_n = tk_record<HD>(R), n = (c.f1 - 1) / span - c0 + 1;
  const float* parts = tk_parts(p, blocks);
  auto rec_of = [&](int j) { return parts + (size_t)(j == 0 ? 2 * c0 + k : 2 * (c0 + j)) * rec_n; };
  float2 ml[PG_MOST_BLOCKS / TJ_THREADS];
  float top = PG_START;
#pragma unroll
  for (int i = 0; i < PG_MOST_BLOCKS / TJ_THREADS; ++i) {
    const int j = i * TJ_THREADS + threadIdx.x;
    ml[i] = j < n ? *reinterpret_cast<const float2*>(rec_of(j) + R * HD + 2 * r) : make_float2(PG_START, 0.f);
    top = fmaxf(top, ml[i].x);
  }
  top = warp_max(top);
  if (lane == 0) top_of[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PG_MOST_BLOCKS / TJ_THREADS; ++i) {
    const float w = ml[i].y == 0.f ? 0.f : ml[i].y * pg_ex2(ml[i].x - top);
    wt[i * TJ_THREADS + threadIdx.x] = w;
    sum += w;
  }
  sum = warp_sum(sum);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  const int d = threadIdx.x % HD;
  float acc = 0.f;
#pragma unroll 8
  for (int j = threadIdx.x / HD; j < n; j += TJ_THREADS / HD) acc = fmaf(wt[j], rec_of(j)[r * HD + d], acc);
  acc_of[threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.x < HD) {
#pragma unroll
    for (int j = 1; j < TJ_THREADS / HD; ++j) acc += acc_of[threadIdx.x + j * HD];
    const int G = p.H / p.a.KV;
    tk_out<T, HD>(p, c.first, c.item % p.a.KV, {r / G, r % G})[d] = Cvt<T>::from_f(sum == 0.f ? 0.f : acc / sum);
  }
}

// Pages of a sequence that can be visible, at most
static int tk_most_pages(const PgAttn& p) {
  if (p.window <= 0) return p.a.W;
  return (int)std::min<long long>(p.a.W, ((long long)p.window + p.a.max_new + 2 * PG - 3) / PG);
}
static bool tk_item_mode(const PgAttn& p) { return (long long)p.a.B * p.a.KV <= pg_sms() && tk_most_pages(p) <= TK_ITEM_PAGES; }

constexpr size_t TK_SMEM = 227 * 1024;

template <typename T, int HD, int NQ>
static int tk_go(const PgAttn& p, int R, cudaStream_t st) {
  const int item = tk_item_mode(p), blocks = item ? p.a.B * p.a.KV : pg_sms();
  const size_t fixed = ((size_t)TK_WARPS * tk_record<HD>(R) * 4 + 15) / 16 * 16 + 2 * TK_WARPS * sizeof(TkCut) +
                       (TK_WARPS + 1 + 5 * (item ? 1 : p.a.B) + 1 + 2 * 8 * NQ) * 4;
  constexpr int most = HD == 32 ? 8 : HD == 64 ? 5 : 3;
  const int slots = (int)std::min<size_t>(most, (TK_SMEM - fixed) / (TK_WARPS * ((size_t)PG * HD + 8)));
  if (slots < 2) return -3;
  const size_t smem = fixed + (size_t)slots * TK_WARPS * (PG * HD + 8);
  GB_PDL_LAUNCH_SMEM((paged_token_kernel<T, HD, NQ>), dim3(blocks), dim3(TK_THREADS), smem, st, p, R, slots, item);
  const int rc = gb_launch_rc();
  if (rc || item) return rc;
  GB_PDL_LAUNCH((paged_join_kernel<T, HD>), dim3(blocks, R), dim3(TJ_THREADS), st, p, R, blocks);
  return gb_launch_rc();
}

template <typename T, int HD>
static int tk_rows(const PgAttn& p, int R, cudaStream_t st) { return R <= 8 ? tk_go<T, HD, 1>(p, R, st) : tk_go<T, HD, 2>(p, R, st); }
template <typename T>
static int tk_size(const PgAttn& p, int R, cudaStream_t st) {
  return p.a.hd == 32 ? tk_rows<T, 32>(p, R, st) : p.a.hd == 64 ? tk_rows<T, 64>(p, R, st) : tk_rows<T, 128>(p, R, st);
}

long long pg_token_ws(const PgAttn& p) {
  const int R = (int)(p.a.max_new * (p.H / p.a.KV));
  return tk_item_mode(p) ? 0 : 2ll * pg_sms() * (R * (p.a.hd + 2) + (long long)(sizeof(TkCut) / 4));
}

int pg_token_attn(const PgAttn& p, cudaStream_t st) {
  const int R = p.a.max_new * (p.H / p.a.KV);
  return p.a.is_bf16 ? tk_size<__nv_bfloat16>(p, R, st) : tk_size<__half>(p, R, st);
}

}  // namespace gb
