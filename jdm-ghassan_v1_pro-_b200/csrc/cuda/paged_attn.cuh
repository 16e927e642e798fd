// What the attention kernels of the paged 8-bit cache share (paged_attn.cu, paged_attn_token.cu, paged_attn_tile.cu).
#pragma once
#include "paged_util.cuh"

namespace gb {

constexpr int PG_TOKEN_ROWS = 16;            // query rows a key head (tokens x heads of a group) up to which the token kernel runs
constexpr int PG_MOST_BLOCKS = 256;          // blocks that pieces are dealt to, at most
constexpr int PG_MOST_SEQS = 1024;           // sequences of one launch (their numbers are in shared memory); more are several launches

struct PgAttn {
  gb_paged a;
  const void* q; long long ld_q; int H;
  float scale2;                              // scale * log2(e): scores are in powers of two
  int window;
  void* out; long long ld_o;
  float* part;                               // records of pieces (pg_*_ws floats)
};

__device__ __forceinline__ float pg_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 4 codes (a little-endian word) as two pairs of float16: the bytes, raised by 128, under the exponent of 1024, which is 1024 + 128 + code
__device__ __forceinline__ void pg_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 off = __half2half2(__ushort_as_half(0x6480));           // 1152
  uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
  lo = *reinterpret_cast<uint32_t*>(&x);
  hi = *reinterpret_cast<uint32_t*>(&y);
}

int pg_sms();                                // of the current device, at most PG_MOST_BLOCKS
long long pg_token_ws(const PgAttn& p);
int pg_token_attn(const PgAttn& p, cudaStream_t st);
long long pg_tile_ws(const PgAttn& p);
int pg_tile_attn(const PgAttn& p, cudaStream_t st);

}  // namespace gb
