// Attention over the paged 8-bit cache (interface in gb_paged.h): checks of arguments, choice of the kernel.
#include <algorithm>
#include <atomic>

#include "paged_attn.cuh"

namespace gb {

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

// New tokens of a sequence, at most: max_new may be more than there are rows.
static long long gb_paged_most_new(const gb_paged* a) { return std::min<long long>(a->max_new, a->rows); }
// Sequences of a launch: work is dealt by places counted in 32 bits, a sequence's being at most its pages or, for every 256 query rows, its pages and four more.
static int gb_paged_most_seqs(const gb_paged* a, int H) {
  const long long items = (gb_paged_most_new(a) * (H / a->KV) + 255) / 256;
  const double places = (double)a->KV * items * (a->W + 4);
  return (int)std::min<double>(PG_MOST_SEQS, 2e9 / places);
}
// The sequences from b0 on, as many as fit.
static PgAttn gb_paged_some(const PgAttn& p, int b0) {
  PgAttn s = p;
  s.a.B = std::min(gb_paged_most_seqs(&p.a, p.H), p.a.B - b0);
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
  if (gb_paged_most_new(a) * H > 0x7fffffffll) return -3;
  if (gb_paged_most_new(a) > 0 && gb_paged_most_seqs(a, H) < 1) return -3;
  return 0;
}

extern "C" long long gb_paged_attn_ws(const gb_paged* a, int H, int window) {
  if (const int rc = gb_paged_attn_args(a, H, window)) return rc;
  if (a->B == 0 || a->max_new == 0 || a->rows == 0) return 0;
  PgAttn p = {*a, nullptr, 0, H, 0.f, window, nullptr, 0, nullptr};
  p = gb_paged_some(p, 0);
  return (long long)a->max_new * (H / a->KV) <= PG_TOKEN_ROWS ? pg_token_ws(p) : pg_tile_ws(p);
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
  for (int b0 = 0; b0 < a->B;) {
    const PgAttn s = gb_paged_some(p, b0);
    const int rc = few ? pg_token_attn(s, st) : pg_tile_attn(s, st);
    if (rc) return rc;
    b0 += s.a.B;
  }
  return 0;
}
