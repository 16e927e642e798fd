// Attention over the paged 8-bit cache (interface in gb_paged.h): one warp per query head, keys page by page.
#include <algorithm>
#include <atomic>

#include "paged_attn.cuh"

namespace gb {

// A lane scores two keys of a page, then sums its dimensions of the values over the page's 64 tokens.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_kernel(const __grid_constant__ gb_paged a, const T* __restrict__ q, long long ld_q, int H, float scale,
                                                         int window, T* __restrict__ out, long long ld_o) {
  __shared__ float sq[4][HD], sp[4][PG];
  pdl_wait();
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z, g = h / (H / a.KV);
  const PgSeq s = pg_seq(a, b);
  constexpr int DL = HD / 32;
  for (int i = blockIdx.x * 4 + wp; i < s.n; i += gridDim.x * 4) {
    const long long row = s.first + i;
    const int pos = s.start + i, from = window > 0 ? max(0, pos - window + 1) : 0;
    for (int d = lane; d < HD; d += 32) sq[wp][d] = Cvt<T>::to_f(q[row * ld_q + (long long)h * HD + d]);
    __syncwarp();
    float m = -1e30f, l = 0.f, o[DL] = {};
    for (int p = from / PG; p <= pos / PG; ++p) {
      const int id = pg_page(a, b, p);
      if (id < 0) continue;
      const long long at = (long long)id * a.KV + g;
      float x[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = lane + 32 * e, key = p * PG + t;
        float acc = 0.f;
        for (int d = 0; d < HD; ++d) acc += sq[wp][d] * (float)a.k[(at * PG + t) * HD + d];
        x[e] = key <= pos && key >= from ? acc * a.ks[at] * scale : -INFINITY;
      }
      const float mn = fmaxf(m, warp_max(fmaxf(x[0], x[1]))), corr = __expf(m - mn);
      float ps = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float w = __expf(x[e] - mn);
        sp[wp][lane + 32 * e] = w;
        ps += w;
      }
      l = l * corr + warp_sum(ps);
      m = mn;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < DL; ++k) {
        float acc = 0.f;
        for (int t = 0; t < PG; ++t) acc += sp[wp][t] * (float)a.v[(at * HD + lane + 32 * k) * PG + t];
        o[k] = o[k] * corr + acc * a.vs[at];
      }
      __syncwarp();
    }
#pragma unroll
    for (int k = 0; k < DL; ++k) out[row * ld_o + (long long)h * HD + lane + 32 * k] = Cvt<T>::from_f(l == 0.f ? 0.f : o[k] / l);
  }
}

int pg_sms() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { (void)cudaGetLastError(); return 148; }
  if ((n = known[dev].load(std::memory_order_relaxed))) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) { (void)cudaGetLastError(); return 148; }
  n = std::min(n, PG_MOST_BLOCKS);
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace gb

using namespace gb;

// The sequences from b0 on, at most PG_MOST_SEQS of them.
static PgAttn gb_paged_some(const PgAttn& p, int b0) {
  PgAttn s = p;
  s.a.B = std::min(PG_MOST_SEQS, p.a.B - b0);
  s.a.table += (long long)b0 * p.a.W;
  s.a.start += b0;
  if (s.a.count) {
    s.a.first += b0;
    s.a.count += b0;
  } else {                                                 // rows are counted from a launch's first sequence
    s.q = (const char*)p.q + 2ll * b0 * p.ld_q;
    s.out = (char*)p.out + 2ll * b0 * p.ld_o;
    s.a.rows = std::max(0ll, p.a.rows - b0);
  }
  return s;
}

static int gb_paged_attn_args(const gb_paged* a, int H, int window) {
  if (const int rc = gb_paged_check(a)) return rc;
  if (H <= 0 || H % a->KV || window < 0 || H > 65535) return -1;
  if ((long long)std::min(a->B, PG_MOST_SEQS) * a->W * a->KV > 0x7fffffffll) return -3;
  return 0;
}

extern "C" long long gb_paged_attn_ws(const gb_paged* a, int H, int window) {
  if (const int rc = gb_paged_attn_args(a, H, window)) return rc;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  PgAttn p = {*a, nullptr, 0, H, 0.f, window, nullptr, 0, nullptr};
  if ((long long)a->max_new * (H / a->KV) <= PG_TOKEN_ROWS) return pg_token_ws(gb_paged_some(p, 0));
  return 0;
}

extern "C" int gb_paged_attn(const gb_paged* a, const void* q, long long ld_q, int H, float scale, int window, void* out, long long ld_o,
                             float* ws, long long ws_floats, cudaStream_t st) {
  if (const int rc = gb_paged_attn_args(a, H, window)) return rc;
  if (!(scale > 0.f)) return -1;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  const long long width = (long long)H * a->hd;
  if (!q || !out || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) || ld_q % 8 || ld_o % 8 || ld_q < width || ld_o < width) return -4;
  const long long need = gb_paged_attn_ws(a, H, window);
  if (need > 0 && (!ws || ws_floats < need || (reinterpret_cast<uintptr_t>(ws) & 15))) return -5;
  const PgAttn p = {*a, q, ld_q, H, scale * 1.4426950408889634f, window, out, ld_o, ws};
  const bool few = (long long)a->max_new * (H / a->KV) <= PG_TOKEN_ROWS;
  for (int b0 = 0; b0 < a->B; b0 += PG_MOST_SEQS) {
    const PgAttn s = gb_paged_some(p, b0);
    int rc = 0;
    if (few) {
      rc = pg_token_attn(s, st);
    } else {
      const dim3 grid((a->max_new + 3) / 4, H, s.a.B);
#define CALL(T, HD) GB_PDL_LAUNCH((paged_attn_kernel<T, HD>), grid, dim3(128), st, s.a, (const T*)s.q, ld_q, H, scale, window, (T*)s.out, ld_o)
      if (a->is_bf16) {
        if (a->hd == 32) { CALL(__nv_bfloat16, 32); } else if (a->hd == 64) { CALL(__nv_bfloat16, 64); } else { CALL(__nv_bfloat16, 128); }
      } else {
        if (a->hd == 32) { CALL(__half, 32); } else if (a->hd == 64) { CALL(__half, 64); } else { CALL(__half, 128); }
      }
#undef CALL
      rc = gb_launch_rc();
    }
    if (rc) return rc;
  }
  return 0;
}
