// What the attention kernels of the paged 8-bit cache share (paged_attn.cu, paged_attn_token.cu, paged_attn_tile.cu).
#pragma once
#include "paged_util.cuh"

namespace gb {

// Query rows a key head (tokens x heads of a group) up to which the token kernel runs: two columns of eight, which is all it has registers for.  The prompt kernel has 256
// rows in hand, most of them empty here.  us, 12/4 heads of 64, 3 and 15 rows, token kernel against prompt kernel: one sequence of 2000 tokens 8.7
// and 11.1 against 22.8 and 22.9, 32 of them 12.7 and 17.9 against 37.5 and 38.0, one of 30000 13.1 and 17.4 against 35.1 and 35.2; 16 rows, 32 of 2000, 8/2 heads: 14.9 against 24.8.
constexpr int PG_TOKEN_ROWS = 16;
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

constexpr float PG_START = -3.4028235e38f;   // a running maximum before its first score: no more than any
// A maximum that a weight's exponent (offset + value scale - maximum, a few hundred) is not added to in one step: an fp32 number past 2^8 has steps of 2^-15 and more.
__device__ __forceinline__ bool pg_far(float m) { return fabsf(m) > 256.f && m != PG_START; }

// 2^x of a whole number up to 127; 0 where that is no normal number
__device__ __forceinline__ float pg_pow2(float x) { return x < -126.f ? 0.f : __uint_as_float((uint32_t)((int)x + 127) << 23); }

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
