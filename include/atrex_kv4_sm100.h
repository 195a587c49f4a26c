/*
 * C ABI of the 4-bit KV cache on sm_100a (B200): the write that quantises a step's K / V rows into it and the
 * attention that reads it.  Lives in the same library as atrex_fa_sm100.h and keeps that header's rules: plain C
 * types, caller-owned memory, no allocation, no synchronisation, everything on the caller's stream, 0 = success and
 * otherwise a status of enum atrex_fa_status with its text in atrex_fa_sm100_last_error().
 *
 * The format.  A row (one token, one KV head) of head_dim values is head_dim / 2 bytes of E2M1 codes, element 2i in
 * the low and 2i + 1 in the high nibble of byte i, and head_dim / 16 E4M3 scales, one for every 16 consecutive
 * values.  A cached value is code * scale * factor with an FP32 factor per KV head (1 when none is given); the
 * attention call takes the factor as k_descale / v_descale.  The reference has no counterpart.
 */
#ifndef ATREX_KV4_SM100_H_
#define ATREX_KV4_SM100_H_

#include "atrex_fa_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ATREX_KV4_SM100_ABI_VERSION 1

/*
 * Quantising write.  Token t of key / value [num_tokens, num_kv_heads, head_dim] BF16 goes to page
 * slot_mapping[t] / page_size, row slot_mapping[t] % page_size; a slot that is negative or at or past
 * num_pages * page_size skips the token.  Per block of 16 values x with top = max |x| (a NaN does not count):
 *   scale = e4m3(min(top / 6 / factor, 448)), step = scale * factor, code = e2m1(x / step), 0 where step is 0,
 * every operation rounded to nearest even in FP32, a quotient beyond 6 saturated, a NaN stored as +6; the sign of a zero
 * is not kept.  A factor is positive, between 2^-100 and 2^100.  Slots are distinct: of tokens with one slot any mixture
 * may be kept.
 * key_out / value_out (NULL, or BF16 like key with strides of their own) receive the stored rows,
 * bf16(code * step); rows of skipped tokens are left as they were.  key_out may be key and value_out value (the same
 * address and strides); otherwise rows of key_out and value_out share no byte with key, value or another row of either
 * (ATREX_FA_INVALID_VALUE; tensors of unlike strides whose address ranges meet are taken to share one).
 * Strides are in elements of their tensor (bytes for the caches).  head_dim is a multiple of 16; key, value and the
 * out rows start on 32-byte boundaries (base and strides), code rows on 8-byte ones.
 */
typedef struct atrex_kv4_sm100_write_params {
  uint32_t struct_bytes, abi_version;
  const void* key;
  const void* value;
  void* key_cache;            /* uint8 [num_pages, page_size, num_kv_heads, head_dim / 2]  */
  void* value_cache;
  void* key_block_scale;      /* E4M3  [num_pages, page_size, num_kv_heads, head_dim / 16] */
  void* value_block_scale;
  void* key_out;
  void* value_out;
  const int64_t* slot_mapping;
  const float* k_factor;      /* device FP32, index head * stride; NULL: 1 */
  const float* v_factor;
  int64_t key_token_stride, key_head_stride, value_token_stride, value_head_stride;
  int64_t key_out_token_stride, key_out_head_stride, value_out_token_stride, value_out_head_stride;
  int64_t key_cache_page_stride, key_cache_row_stride, key_cache_head_stride;
  int64_t value_cache_page_stride, value_cache_row_stride, value_cache_head_stride;
  int64_t key_scale_page_stride, key_scale_row_stride, key_scale_head_stride;
  int64_t value_scale_page_stride, value_scale_row_stride, value_scale_head_stride;
  int64_t k_factor_stride, v_factor_stride;
  int32_t num_tokens, num_kv_heads, head_dim, page_size, num_pages, reserved;
} atrex_kv4_sm100_write_params;

/*
 * Attention over such a cache: the call of atrex_fa_sm100_forward with paged K / V in 4 bits.  `fa` is that
 * function's block with dtype ATREX_FA_BF16 (of q and out), k / v the code caches with strides in BYTES,
 * k_descale / v_descale the factors [batch, num_kv_heads]; softcap, q_descale and context parallelism are not
 * served, softmax_scale is positive.  Rows and pages that no query row sees may hold anything, NaN scales too.  The
 * route field is ATREX_FA_ROUTE_AUTO, _MMA or _UMMA.
 */
typedef struct atrex_kv4_sm100_params {
  uint32_t struct_bytes, abi_version;
  atrex_fa_sm100_params fa;
  const void* k_block_scale;
  const void* v_block_scale;
  int64_t k_scale_page_stride, k_scale_row_stride, k_scale_head_stride;
  int64_t v_scale_page_stride, v_scale_row_stride, v_scale_head_stride;
} atrex_kv4_sm100_params;

ATREX_FA_API int atrex_kv4_sm100_abi_version(void);
ATREX_FA_API size_t atrex_kv4_sm100_params_bytes(void);
ATREX_FA_API size_t atrex_kv4_sm100_write_params_bytes(void);
ATREX_FA_API int atrex_kv4_sm100_write(const atrex_kv4_sm100_write_params* p, void* stream);
/* Route, splits and scratch of an attention call, from graph-static sizes; launches nothing. */
ATREX_FA_API int atrex_kv4_sm100_plan(const atrex_kv4_sm100_params* p, atrex_fa_sm100_plan_info* plan);
/* `workspace`: plan.workspace_bytes of caller-owned device scratch, 256-byte aligned, contents irrelevant. */
ATREX_FA_API int atrex_kv4_sm100_forward(const atrex_kv4_sm100_params* p, void* workspace, uint64_t workspace_bytes,
                                         void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ATREX_KV4_SM100_H_ */
