// Key/value cache in 8 bits, in pages of 64 tokens: appending with the position rotation, attention, reading back.
//
// A pool has `pages` pages.  Of a page, each key head has 64 x hd codes of keys, k[page][head][token][dim], and of values with the tokens
// innermost, v[page][head][dim][token], and one scale each, ks[page][head] and vs[page][head]: a code c (-127 ... 127) stands for c * scale.  A scale is a power
// of two, at least 2^-120: the smallest that takes the largest number of its 64 x hd ones to at most 127.  So a page that grows is rescaled
// by shifts, codes and scales multiply without rounding, and the attention kernels feed codes to 16-bit MMAs as they are.
//
// Every call names the sequences it works on in the same way: sequence b has start[b] tokens in the pages table[b][0 ...] before the call's own count[b] ones,
// which are the rows first[b] ... first[b] + count[b] - 1 of the call's tensors (first NULL: row b; count NULL: one row each).  Rows that belong to no sequence are
// neither read nor written, and no row is two sequences'.  A page that a sequence appends to is in no other's table, nor twice in its own (pages that are only read may be), and
// results do not lie over a call's inputs.  What does not fit (more new tokens than max_new, positions past the table's width, rows outside the tensors, a negative number)
// leaves the sequence out, a page number outside the pool leaves the page's tokens out; both set the status to 301.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GB_PAGE 64

typedef struct gb_paged {
  signed char* k; float* ks; signed char* v; float* vs;     // 16-byte aligned codes
  int pages, KV, hd;                                        // hd: 32, 64 or 128
  const int* table; int W;                                  // [B, W]
  int B; const int* start; const int* first; const int* count;
  int max_new;                                              // most new tokens of a sequence
  long long rows;                                           // rows of the call's tensors
  int is_bf16;                                              // their type: bfloat16, else float16
  int* status;                                              // 301 (above), 303: a key or value was not finite (append; held as zero)
} gb_paged;

// Rows qkv[row] = (H query heads, KV key heads, KV value heads) of hd numbers, 16-byte aligned.  Queries, and keys on their way into the pages, are normed
// (qw, kw not NULL: RMS norm over the head times the weight) and rotated by their position: cos_sin[position] holds hd / 2 cosines, then hd / 2 sines, for `positions`
// positions; rope_type 0: pairs (2i, 2i + 1), 1: pairs (i, i + hd / 2).  Queries go to q_out.
int gb_paged_append(const gb_paged* a, const void* qkv, long long ld_qkv, int H, void* q_out, long long ld_q, const float* qw, const float* kw,
                    float eps, const float* cos_sin, int positions, int rope_type, cudaStream_t st);

// The new tokens' rows of the pages: k_out[row], v_out[row] = KV * hd numbers, at most the type's largest finite one in size.
int gb_paged_read(const gb_paged* a, void* k_out, long long ld_k, void* v_out, long long ld_v, cudaStream_t st);

// out[row] = softmax(q K^T * scale) V for the H query heads of every new token over the tokens up to its own, which are in the pages; window > 0: over the last
// `window` of them.  Scores are fp32: what passes its range (3.4e38 after times log2 e) has no defined result.  scale > 0, H a multiple of KV.  ws: gb_paged_attn_ws floats (0 or more; negative: why the arguments are refused), 16-byte aligned, this call's own until it
// is done.
long long gb_paged_attn_ws(const gb_paged* a, int H, int window);
int gb_paged_attn(const gb_paged* a, const void* q, long long ld_q, int H, float scale, int window, void* out, long long ld_o, float* ws,
                  long long ws_floats, cudaStream_t st);

#ifdef __cplusplus
}
#endif
