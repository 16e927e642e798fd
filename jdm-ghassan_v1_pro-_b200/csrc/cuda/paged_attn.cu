// Attention over the paged 8-bit cache (interface in gb_paged.h): one warp per query head, keys page by page.
#include "paged_util.cuh"

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

}  // namespace gb

using namespace gb;

extern "C" int gb_paged_attn(const gb_paged* a, const void* q, long long ld_q, int H, float scale, int window, void* out, long long ld_o,
                             cudaStream_t st) {
  if (const int rc = gb_paged_check(a)) return rc;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  if (H <= 0 || H % a->KV || !(scale > 0.f) || window < 0) return -1;
  const long long width = (long long)H * a->hd;
  if (!q || !out || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) || ld_q % 8 || ld_o % 8 || ld_q < width || ld_o < width) return -4;
  if (H > 65535 || a->B > 65535) return -3;
  const dim3 grid((a->max_new + 3) / 4, H, a->B);
#define CALL(T, HD) GB_PDL_LAUNCH((paged_attn_kernel<T, HD>), grid, dim3(128), st, *a, (const T*)q, ld_q, H, scale, window, (T*)out, ld_o)
  if (a->is_bf16) {
    if (a->hd == 32) { CALL(__nv_bfloat16, 32); } else if (a->hd == 64) { CALL(__nv_bfloat16, 64); } else { CALL(__nv_bfloat16, 128); }
  } else {
    if (a->hd == 32) { CALL(__half, 32); } else if (a->hd == 64) { CALL(__half, 64); } else { CALL(__half, 128); }
  }
#undef CALL
  return gb_launch_rc();
}
