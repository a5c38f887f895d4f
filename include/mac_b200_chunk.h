/*
 * mac_b200_chunk.h -- C ABI of the paged chunk attention and the 8-bit K/V cache.
 *
 * Companion of mac_b200.h (same library, error codes, status word, stream and
 * device rules).  The operators here have no counterpart in the reference
 * project, which takes prompt attention from another library and keeps its
 * cache in bf16 only: chunk attention yields the states (output and LSE) that
 * mac_b200_prefill_downdate_update_cache turns into ring rows, and the 8-bit
 * pool is a second format for the rows that the paged K/V pool holds.
 *
 * The 8-bit row format.  A row is the 128 values x of one (token, KV head).
 * It is held as 128 e4m3 codes and one exponent byte e:
 *     s = 2^(e-127) = the smallest power of two >= 2^-124 with max|x| / s <= 448
 *     code = e4m3(x / s), round to nearest even; |code| <= 240 where s = 2^120
 * and stands for code * s.  (2^120 is the scale of rows that reach 1.75 * 2^127;
 * a code of 256 would stand for 2^128 there.)  e = 255 stands for NaN and marks a row that held an
 * infinity or a NaN (codes 0).  A power of two loses no relative precision
 * (the codes are floating point), and code * s is a bf16 number, so reading a
 * row back is exact.
 */
#ifndef MAC_B200_CHUNK_H_
#define MAC_B200_CHUNK_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Arguments of the chunk attention.  B requests; request b owns rows
 * offsets[b] .. offsets[b+1]-1 of q (n of them): the last n of the kv_lens[b]
 * tokens that its page-table row req_to_token[req_ids[b]] lists, already
 * written to the pool.  Row i sits at position p = kv_lens[b] - n + i and
 * attends the keys j of [max(0, p + 1 - window), p]:
 *     out = sum_j softmax_j(sm_scale * q.k_j) v_j,   lse = ln sum_j exp(sm_scale * q.k_j)
 * A row that attends nothing (p < 0, window 0) gets out = 0, lse = -inf.  A
 * value that a row does not attend does not reach it, whatever it holds.
 * Weights are summed before they are normalised, in fp32 and up to 2^8 each:
 * out may be infinite or NaN where |v| * attended keys * 2^8 passes the fp32 range.
 *
 * Rows of q outside [offsets[0], offsets[B]) reach nothing and are not written
 * in out / lse.  q and out must not share memory.  All lengths are read on the device; nothing about a call has to
 * change between replays of a captured graph but the contents of its tensors.
 *
 * What cannot be run sets MAC_B200_STATUS_BAD_REQUEST (mac_b200_query_status):
 * a request whose offsets are not inside [0, q_rows] or decrease is left out;
 * one whose req_id or length is outside the page table gets empty rows; a
 * page-table entry outside the pool counts as a row of zeros.  Waits inside the
 * kernel are bounded (about two seconds); one that runs out ends the call with
 * MAC_B200_STATUS_COPY_TIMEOUT, and its out and lse are not valid.
 */
typedef struct MacB200ChunkArgs {
  int32_t B;                   /* requests                                                  */
  int32_t Hq, Hkv;             /* heads; Hq / Hkv in 1..16                                  */
  int32_t D;                   /* head dim, must be 128                                     */
  int32_t q_rows;              /* rows of q, out and lse                                    */
  int32_t req_to_token_rows;
  int32_t req_to_token_stride; /* columns of req_to_token                                   */
  int32_t window;              /* tokens a row looks back on, itself included; < 0: all     */
  int64_t kv_tokens;           /* rows of the pool, < 2^31                                  */
  int64_t q_stride0;           /* elements from row to row of q, a multiple of 8            */
  int64_t workspace_bytes;
  float sm_scale;              /* > 0                                                       */
  int32_t reserved;            /* 0                                                         */
  const void* q;               /* [q_rows,Hq,128] bf16, heads contiguous, 16-byte aligned   */
  const void* k;               /* pool: [kv_tokens,Hkv,128] bf16 or e4m3, 16-byte aligned   */
  const void* v;
  const uint8_t* k_exp;        /* [kv_tokens,Hkv] exponent bytes (e4m3 pool), else NULL; read
                                  in aligned blocks of 16 bytes, nothing behind the end     */
  const uint8_t* v_exp;
  const int32_t* req_to_token; /* [rows,stride] logical position -> pool row                */
  const int32_t* req_ids;      /* [B]                                                       */
  const int32_t* offsets;      /* [B+1]                                                     */
  const int32_t* kv_lens;      /* [B] cached tokens, the chunk's own included               */
  void* out;                   /* [q_rows,Hq,128] bf16, 16-byte aligned                     */
  float* lse;                  /* [q_rows,Hq] f32 natural log, or NULL                      */
  void* workspace;             /* mac_b200_chunk_attention_workspace_bytes() bytes, 16-byte
                                  aligned, whatever it holds; calls that may run at the same
                                  time need one each                                        */
} MacB200ChunkArgs;

/* Chunk attention over a bf16 pool / over an e4m3 pool. */
int mac_b200_chunk_attention_bf16(const MacB200ChunkArgs* args, void* stream);
int mac_b200_chunk_attention_e4m3(const MacB200ChunkArgs* args, void* stream);

/* Bytes of a chunk attention workspace on the current device. */
int mac_b200_chunk_attention_workspace_bytes(int64_t* bytes);

/*
 * Writes rows into an e4m3 pool; with q != NULL the decode step's rotation goes
 * before it.  Without rotation: pool row cache_locs[n] <- held form of k[n], v[n].
 * With it: q_post[n] <- rotated q[n] (q stays as it is: the pre-RoPE query), and
 * pool row cache_locs[n] <- held form of the rotated k[n] (in fp32, not rounded
 * to bf16 before) and of v[n].  A rotated pair is x0*c - x1*s, x1*c + x0*s, each
 * product and sum rounded to fp32.
 *
 * Rows of cache_locs outside [0, kv_pool_tokens) are not written to the pool
 * (padding).  Entries inside have to be distinct: a pool row named twice holds
 * bytes of either.  q_post must not share memory with q, k or v.  A position outside [0, max_positions) sets
 * MAC_B200_STATUS_BAD_REQUEST; its token is neither rotated nor written.
 */
typedef struct MacB200QuantizeKvArgs {
  int64_t N;                   /* tokens                                                    */
  int32_t Hq, Hkv;             /* Hq only with q                                            */
  int32_t D;                   /* must be 128                                               */
  int32_t cache_locs_i64;      /* 0: int32, 1: int64                                        */
  int64_t k_stride0, v_stride0;/* elements from row to row                                  */
  int64_t kv_pool_tokens;
  const void* k;               /* [N, Hkv*128] bf16                                         */
  const void* v;               /* [N, Hkv*128] bf16                                         */
  void* k_pool;                /* [T,Hkv,128] e4m3, 16-byte aligned                         */
  void* v_pool;
  uint8_t* k_exp;              /* [T,Hkv]                                                   */
  uint8_t* v_exp;
  const void* cache_locs;      /* [>=N] int32|int64                                         */
  /* rotation; q = NULL: none, the rest is not read */
  const void* q;               /* [N, Hq*128] bf16                                          */
  void* q_post;                /* [>=N,Hq,128] bf16                                         */
  const float* cos_sin_cache;  /* [max_positions, rotary_dim] f32: cos | sin                */
  const void* positions;       /* [>=N] int32|int64                                         */
  int64_t q_stride0, cos_sin_stride0, max_positions;
  int32_t rotary_dim;          /* even, 2..128                                              */
  int32_t is_neox;             /* 1: pairs (d, d + rotary_dim/2); 0: pairs (2p, 2p+1)       */
  int32_t positions_i64;       /* 0: int32, 1: int64                                        */
  int32_t reserved;
} MacB200QuantizeKvArgs;

int mac_b200_quantize_kv_e4m3(const MacB200QuantizeKvArgs* args, void* stream);

/*
 * Reads rows of an e4m3 pool back into a bf16 pool: row dst_locs[i] (i without
 * dst_locs) of k_buffer / v_buffer <- code * s of pool row src_locs[i].  A pair
 * with either row outside its pool is left out (padding).  Entries of dst_locs
 * inside the pool have to be distinct.
 */
typedef struct MacB200DequantizeKvArgs {
  int64_t N;
  int32_t Hkv, D;              /* D must be 128                                             */
  int32_t src_locs_i64, dst_locs_i64;
  int64_t src_tokens, dst_tokens;
  const void* k_pool;          /* [src_tokens,Hkv,128] e4m3, 16-byte aligned                */
  const void* v_pool;
  const uint8_t* k_exp;        /* [src_tokens,Hkv]                                          */
  const uint8_t* v_exp;
  const void* src_locs;        /* [N] int32|int64                                           */
  void* k_buffer;              /* [dst_tokens,Hkv,128] bf16, 16-byte aligned                */
  void* v_buffer;
  const void* dst_locs;        /* [N] int32|int64, or NULL                                  */
} MacB200DequantizeKvArgs;

int mac_b200_dequantize_kv_e4m3(const MacB200DequantizeKvArgs* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MAC_B200_CHUNK_H_ */
