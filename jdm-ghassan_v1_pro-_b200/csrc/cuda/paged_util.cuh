// What the kernels of the paged 8-bit cache share (interface in gb_paged.h).
#pragma once
#include "gb_paged.h"
#include "sm100_common.cuh"

namespace gb {

constexpr int PG = GB_PAGE;
constexpr int ST_NOT_FINITE = 303;
constexpr float PG_LEAST = 7.52316385e-37f;       // 2^-120, the least scale

template <typename T> struct PgTop;               // largest finite number
template <> struct PgTop<__half> { static constexpr float value = 65504.f; };
template <> struct PgTop<__nv_bfloat16> { static constexpr float value = 3.3895313892515355e38f; };

struct PgSeq { int start, first, n; };

// Sequence b of a call; n == 0 where it has no new tokens or the call's numbers do not fit.
__device__ __forceinline__ PgSeq pg_seq(const gb_paged& a, int b) {
  PgSeq s;
  s.start = a.start[b];
  s.first = a.first ? a.first[b] : b;
  s.n = a.count ? a.count[b] : 1;
  if (s.n <= 0 || s.start < 0 || s.first < 0 || s.n > a.max_new || (long long)s.first + s.n > a.rows || (long long)s.start + s.n > (long long)a.W * PG) {
    if (s.n != 0) atomicCAS(a.status, 0, ST_BAD_ARGUMENT);
    s.n = 0;
  }
  return s;
}

// Page `p` of sequence b, or -1 where the table names none of the pool.
__device__ __forceinline__ int pg_page(const gb_paged& a, int b, int p) {
  const int id = a.table[(long long)b * a.W + p];
  if ((unsigned)id >= (unsigned)a.pages) {
    atomicCAS(a.status, 0, ST_BAD_ARGUMENT);
    return -1;
  }
  return id;
}

// 8 numbers of 16 bits at a 16-byte aligned place
template <typename T>
__device__ __forceinline__ void pg_load8(const T* p, float* v) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Cvt<T>::unpack2(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void pg_store8(T* p, const float* v) {
  uint4 u;
  u.x = Cvt<T>::pack2(v[0], v[1]);
  u.y = Cvt<T>::pack2(v[2], v[3]);
  u.z = Cvt<T>::pack2(v[4], v[5]);
  u.w = Cvt<T>::pack2(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = u;
}

}  // namespace gb

// 0, or why these arguments are refused (the codes of gb_paged.h's launchers)
static inline int gb_paged_check(const gb_paged* a) {
  if (!a || !a->k || !a->ks || !a->v || !a->vs || !a->status || (a->B > 0 && (!a->table || !a->start))) return -1;
  if (!a->first != !a->count) return -1;
  if (a->hd != 32 && a->hd != 64 && a->hd != 128) return -2;
  if (a->KV <= 0 || a->pages <= 0 || a->W <= 0 || a->B < 0 || a->max_new < 0 || a->rows < 0) return -3;
  if ((long long)a->W * GB_PAGE > 0x7fffffffll - 4096 || a->max_new > a->W * GB_PAGE || a->rows > 0x7fffffffll) return -3;
  if ((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15) return -4;
  return 0;
}
