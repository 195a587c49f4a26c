/*
 * C ABI of the page bookkeeping of paged KV caches on sm_100a (B200): forking, freeing and compacting the pages that
 * a batch of sequences holds, with the copies that this takes.  Lives in the same library as atrex_fa_sm100.h and
 * keeps that header's rules: plain C types, caller-owned memory, no allocation, no synchronisation, everything on
 * the caller's stream, 0 = success and otherwise a status of enum atrex_fa_status with its text in
 * atrex_fa_sm100_last_error().  The reference has no counterpart (its block tables are made by the caller).
 *
 * A sequence of seq_lens[b] tokens holds the pages block_table[b][0 .. ceil(seq_lens[b] / page_size)) (at most the
 * table's width); ref_counts[p] says how often page p is held, 0 = free.  All metadata is read on the device at every
 * launch.  Results go to arrays of their own; the caches are changed in place, in pages that were free.
 */
#ifndef ATREX_KVPAGES_SM100_H_
#define ATREX_KVPAGES_SM100_H_

#include "atrex_fa_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ATREX_KVPAGES_SM100_ABI_VERSION 1

/* Layout of one cache tensor [num_pages, page_size, heads, row_bytes], byte strides; a row is contiguous. */
typedef struct atrex_kvpages_sm100_cache {
  int64_t page_stride, row_stride, head_stride;
  int32_t heads, row_bytes;
} atrex_kvpages_sm100_cache;

typedef struct atrex_kvpages_sm100_params {
  uint32_t struct_bytes, abi_version;
  const int32_t* block_table;    /* [batch, width], row stride below      */
  const int32_t* seq_lens;       /* [batch]                               */
  const int32_t* ref_counts;     /* [num_pages]                           */
  const int32_t* parents;        /* [batch], reassign only                */
  int32_t* new_table;            /* [batch, width], dense                 */
  int32_t* new_lens;             /* [batch], reassign only                */
  int32_t* new_refs;             /* [num_pages]                           */
  int32_t* page_map;             /* [num_pages], compact only             */
  int32_t* count;                /* [1]: shortage (reassign), live pages (compact) */
  const atrex_kvpages_sm100_cache* caches;   /* HOST arrays of num_caches entries, read during the call: layouts */
  void* const* bases;                        /* and device addresses                                            */
  int64_t table_row_stride;
  int32_t batch, width, num_pages, page_size, num_caches;
  int32_t sm_count;              /* SMs that the grids are sized for, 0 or less: all; results do not depend on it */
} atrex_kvpages_sm100_params;

ATREX_FA_API int atrex_kvpages_sm100_abi_version(void);
ATREX_FA_API size_t atrex_kvpages_sm100_params_bytes(void);
ATREX_FA_API size_t atrex_kvpages_sm100_cache_bytes(void);
/* Scratch of either call below (256-byte aligned, contents irrelevant). */
ATREX_FA_API uint64_t atrex_kvpages_sm100_workspace_bytes(int32_t batch, int32_t num_pages);

/*
 * Row b continues the sequence of row parents[b]: b itself (unchanged), another row (a fork), or, with a parent
 * outside [0, batch), none (freed: length 0).  The finished pages of a sequence are shared by all rows that continue
 * it.  Its unfinished last page goes to one of them, the parent row if it continues itself and else the lowest one;
 * every other row gets the lowest free pages in row order, and the tokens of the unfinished page are copied there in
 * every cache.  Pages that this call frees are not used by it.  new_refs: every page's count less the rows that gave
 * it up, plus those that took it.  Entries of new_table past a sequence's last page are -1.
 * When fewer pages are free than are needed, *count says how many are missing and nothing else changes (the tables
 * and counts come back as they were); otherwise *count is 0.
 */
ATREX_FA_API int atrex_kvpages_sm100_reassign(const atrex_kvpages_sm100_params* p, void* workspace,
                                              uint64_t workspace_bytes, void* stream);

/*
 * Moves the live pages (ref_counts > 0) of a pool to its front: with n live pages, the i-th live page at or behind
 * page n goes to the i-th free page before it, in every cache.  page_map[p]: where page p is now, -1 for a free page;
 * *count = n.  Entries of new_table past a sequence's last page are -1.
 */
ATREX_FA_API int atrex_kvpages_sm100_compact(const atrex_kvpages_sm100_params* p, void* workspace,
                                             uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ATREX_KVPAGES_SM100_H_ */
