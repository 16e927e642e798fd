// What the attention kernels of the paged 8-bit cache share (paged_attn.cu, paged_attn_token.cu).
#pragma once
#include "paged_util.cuh"

namespace gb {

constexpr int PG_TOKEN_ROWS = 16;            // query rows a key head (tokens x heads of a group) up to which the token kernel runs
constexpr int PG_MOST_BLOCKS = 256;          // blocks that pieces are dealt to, at most
constexpr int PG_MOST_SEQS = 2048;           // sequences of one launch; more are several launches

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

int pg_sms();                                // of the current device, at most PG_MOST_BLOCKS
long long pg_token_ws(const PgAttn& p);
int pg_token_attn(const PgAttn& p, cudaStream_t st);

}  // namespace gb
