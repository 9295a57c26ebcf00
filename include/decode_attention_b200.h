/* SPDX-License-Identifier: MIT
 *
 * decode_attention_b200.h -- C ABI of the operators between a decode layer's
 * products, in libdecode_gemm_b200.so (no counterpart in the reference, whose
 * path is the products alone):
 *
 *   dg_build_block_tables   a step's pages, slots and positions from request lengths
 *   dg_rotary               rotary positions with up to four axes, forward and inverse, and
 *                           the write of the step's keys and values into a paged cache
 *   dg_paged_attention      attention of one new token per request over that cache
 *
 * Conventions as in decode_gemm_b200.h: plain C, device pointers owned by the
 * caller, `stream` a cudaStream_t, cudaError_t results (1 = cudaErrorInvalidValue
 * for arguments that are refused before anything is launched), nothing
 * allocated, no host synchronisation (every call can be captured in a CUDA
 * graph).  What only the device can see (lengths, pages, slots, positions) is
 * checked there: the access is left out and `status` (a device int, 0 before
 * the launch, may be NULL) receives the first code.  pdl_attr launches with
 * programmatic stream serialization; every kernel waits for the kernels before
 * it on the stream before it reads or writes global memory.
 *
 * Strides are in elements.  The last dimension of every tensor is contiguous,
 * its address a multiple of its elements' size (refused otherwise).
 */
#ifndef DECODE_ATTENTION_B200_H_
#define DECODE_ATTENTION_B200_H_

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define DG_TYPE_BF16 0
#define DG_TYPE_FP16 1
#define DG_TYPE_FP32 2
#define DG_TYPE_E4M3 3

/* Device status codes of these operators (dg_status_string knows them). */
#define DG_ERR_LENGTH 0xA1     /* a request length is negative, or the sum passes 2^31 - 1         */
#define DG_ERR_POOL 0xA2       /* the free list has too few pages: entries and slots left at -1    */
#define DG_ERR_TABLE_WIDTH 0xA3/* a request needs more pages than its table row holds              */
#define DG_ERR_TOKENS 0xA4     /* the requests bring more tokens than the output arrays hold       */
#define DG_ERR_POSITION 0xB1   /* a position outside [0, max_position): the token's rows are NaN   */
#define DG_ERR_SLOT 0xB2       /* a slot past the cache's end: not written                         */
#define DG_ERR_PAGE 0xC1       /* a page of a live token outside [0, num_pages): token left out    */
#define DG_ERR_SEQ_LEN 0xC2    /* a length that is negative or longer than its table row: clamped  */

/* Paged cache bookkeeping of one step, from the requests' lengths.
   Request b has context_lens[b] = c tokens in the cache and brings
   new_lens[b] = n.  With P = page_size it owns ceil(c / P) pages already
   (block_table[b, 0 .. ceil(c/P)) ) and takes ceil((c+n)/P) - ceil(c/P) more,
   in request order, from free_pages[*cursor_in ...] (NULL: from 0):
     block_table[b, ceil(c/P) + j] = free_pages[cursor + pages taken before b + j]
   (other entries are left alone).  The new tokens stand request by request:
     query_start[b] = new tokens of the requests before b   (b = 0 .. batch)
     seq_lens[b]    = c + n
   and for token t of request b, at position p = c + t - query_start[b]:
     slots[t] = block_table[b, p / P] * P + p % P,  positions[t] = p,  requests[t] = b.
   Tokens past query_start[batch] (padding up to num_tokens) get slot -1,
   position 0, request -1.  cursor_out[0] = the free list's next page.
   The call can be repeated: it reads nothing that it writes. */
typedef struct dg_block_tables {
  int batch;                 /* 1 .. 16384                                                       */
  int page_size;             /* tokens a page, >= 1                                              */
  int table_width;           /* entries a row of block_table holds                               */
  int num_tokens;            /* length of slots, positions and requests                          */
  int free_count;            /* length of free_pages                                             */
  long long table_stride;    /* elements between rows of block_table, >= table_width             */
  const int* context_lens;   /* [batch]                                                          */
  const int* new_lens;       /* [batch]                                                          */
  const int* free_pages;     /* [free_count]; no part of block_table                             */
  const int* cursor_in;      /* [1], may be NULL                                                 */
  int* block_table;          /* [batch, table_width]                                             */
  int* seq_lens;             /* [batch]; not context_lens or new_lens                            */
  int* query_start;          /* [batch + 1]                                                      */
  long long* slots;          /* [num_tokens]                                                     */
  int* positions;            /* [num_tokens]                                                     */
  int* requests;             /* [num_tokens]                                                     */
  int* cursor_out;           /* [1]; not cursor_in                                               */
  int* status;
} dg_block_tables;

int dg_build_block_tables(const dg_block_tables* args, void* stream, int pdl_attr);

/* Rotary positions, and the write of keys and values into a paged cache.
   A head's first `rot` values turn in pairs i = 0 .. rot/2 - 1, (i, i + rot/2)
   (DG_PAIR_HALF) or (2i, 2i + 1) (DG_PAIR_ADJACENT); the rest passes:
     (x, y) -> (x cos - y sin, y cos + x sin),  inverse: the same with -sin
   with cos = cos_sin[p][i], sin = cos_sin[p][rot/2 + i] of the position p that
   token t has on the pair's axis: positions[axis * position_stride + t].  The
   inverse is the gradient (the transpose of a rotation).
   q [T, heads, head_dim] -> q_out; k [T, kv_heads, head_dim] -> k_out and/or
   k_cache; v [T, kv_heads, head_dim] -> v_cache.  Outputs may be the inputs
   themselves.  A cache row is slots[t] = page * page_size + offset, skipped
   below 0; with an e4m3 cache the stored value is e4m3(clamp(x / scale[head],
   +-448)) (a scale of NULL: 1).  k_cache and v_cache go together; without them
   slots is not read.  Computed in fp32, rounded once. */
#define DG_PAIR_HALF 0
#define DG_PAIR_ADJACENT 1
#define DG_MAX_ROT 512

typedef struct dg_rotary_args {
  int tokens;                /* T >= 1                                                           */
  int heads, kv_heads;       /* of q (0 without q) and of k and v (0 without k)                  */
  int head_dim;              /* 2 .. 2048                                                        */
  int rot;                   /* even, 2 .. min(head_dim, DG_MAX_ROT)                             */
  int type;                  /* of q, k, v and the outputs: bf16, fp16, fp32                     */
  int cache_type;            /* of the caches: `type` (not fp32) or e4m3                         */
  int pairing;               /* DG_PAIR_*                                                        */
  int inverse;               /* 1: rotate back                                                   */
  int position_64;           /* positions are 0: int32, 1: int64                                 */
  int max_position;          /* rows of cos_sin                                                  */
  int page_size, num_pages;  /* of the caches                                                    */
  const void *q, *k, *v;
  void *q_out, *k_out;
  void *k_cache, *v_cache;   /* [num_pages, page_size, kv_heads, head_dim]                       */
  long long q_stride[2], k_stride[2], v_stride[2];      /* token, head: 0 .. 2^31 - 1 bytes each */
  long long q_out_stride[2], k_out_stride[2];           /* the same                              */
  long long k_cache_stride[3], v_cache_stride[3];       /* page, offset in the page, head        */
  const void* positions;     /* [axes, T]                                                        */
  long long position_stride; /* between axes (0: every axis reads the same)                      */
  const long long* slots;    /* [T]                                                              */
  const float* cos_sin;      /* [max_position, rot]                                              */
  const float *k_scale, *v_scale;                       /* [kv_heads], may be NULL               */
  int* status;
  unsigned axis_of[DG_MAX_ROT / 32]; /* pair i's axis: bits 2*(i%16) of word i/16                */
} dg_rotary_args;

int dg_rotary(const dg_rotary_args* args, void* stream, int pdl_attr);

/* Attention of one new token per request over a paged cache (the new token's
   own key and value included: seq_lens counts it).  For request b and query
   head h of kv head j = h / (heads / kv_heads):
     s_t = scale * k_scale[j] * (q[b, h] . k[t, j])            (with softcap c > 0: c * tanh(s_t / c))
     out[b, h] = v_scale[j] * sum_t exp(s_t - m) v[t, j] / sum_t exp(s_t - m)
     lse[b, h] = log sum_t exp(s_t)
   over the live tokens t in [max(0, len - window), len), len = seq_lens[b]
   (window 0: all of them); token t lies at offset t % page_size of page
   block_table[b, t / page_size].  A request without live tokens gives 0 and
   lse -inf; so does one whose live tokens are all left out for bad pages
   (DG_ERR_PAGE).  Memory outside the live tokens is never read, whatever it
   holds.  A NaN among the live tokens makes out and lse NaN, for the heads that
   read it.
   Products of the stored values accumulate in fp32; probabilities enter the
   second product as two terms of the cache's 16-bit type (fp16 for e4m3): 16 to
   17 bits with a bf16 cache, 22 with the others, so that the rounding of the
   result is what shows; sums and maxima are fp32.  Capped scores are exact to
   2^-21 of themselves for any cap (beyond 2^-100 .. 2^100: as at those).
   q_out / q_scales (optional, bf16 out, head_dim a multiple of 128): the
   result also as e4m3 [batch, heads * head_dim] with fp32 scales [batch,
   heads * head_dim / 128], the bytes dg_quantize_act makes from `out`.
   workspace: dg_attention_workspace_bytes() bytes, 16-byte aligned, zeroed
   once; a launch leaves it ready for the next.  Launches that can overlap
   (other streams) need workspaces of their own.  Results do not depend on
   timing: work is cut and joined in an order that the lengths alone set. */
typedef struct dg_attention_args {
  int batch, heads, kv_heads;/* heads a multiple of kv_heads                                     */
  int head_dim;              /* a multiple of 8 (e4m3 cache: 16), at most 256                    */
  int page_size, num_pages;
  int table_width;
  int type;                  /* of q and out: bf16, fp16                                         */
  int cache_type;            /* `type` or e4m3                                                   */
  int window;                /* 0: none                                                          */
  float scale;
  float softcap;             /* 0: none                                                          */
  const void* q;             /* [batch, heads, head_dim], 4-byte aligned, even strides           */
  const void *k_cache, *v_cache; /* [num_pages, page_size, kv_heads, head_dim]: 16-byte aligned,
                                strides multiples of 16 bytes                                    */
  long long q_stride[2];                                /* request, head                         */
  long long k_cache_stride[3], v_cache_stride[3];       /* page, offset in the page, head        */
  const int* block_table;    /* [batch, table_width]                                             */
  long long table_stride;
  const int* seq_lens;       /* [batch]                                                          */
  const float *k_scale, *v_scale;                       /* [kv_heads], may be NULL; e4m3 only    */
  void* out;                 /* [batch, heads, head_dim]                                         */
  long long out_stride[2];   /* request, head                                                    */
  float* lse;                /* [batch, heads], may be NULL                                      */
  void* q_out;
  float* q_scales;
  void* workspace;
  unsigned long long workspace_bytes;
  int* status;
} dg_attention_args;

int dg_paged_attention(const dg_attention_args* args, void* stream, int pdl_attr);

/* Workspace of dg_paged_attention on the current device, for any arguments
   (0 where there is no device). */
unsigned long long dg_attention_workspace_bytes(void);

#ifdef __cplusplus
}
#endif

#endif /* DECODE_ATTENTION_B200_H_ */
