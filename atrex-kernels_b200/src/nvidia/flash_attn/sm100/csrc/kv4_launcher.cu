// C-ABI launcher of the 4-bit cache (declared in include/atrex_kv4_sm100.h): argument checks, the split policy from
// graph-static sizes, workspace carving and the launches.  Allocates nothing, reads no device memory.
#include <algorithm>
#include <cstring>
#include <initializer_list>

#include "atrex_kv4_sm100.h"
#include "kv4_kernels.cuh"

namespace atrex_sm100 {
namespace {

constexpr int kMaxSplits = 256;
// Packed query rows (per request and KV head) up to which the mma.sync kernel runs; it widens the cache once per 8 or
// 16 rows, the tcgen05 kernel once per 128.  Measured (us, mma.sync / tcgen05; 4 or 2 KV heads, head_dim 128 | 256):
//   64 requests x 4 096 keys: 16 rows 70 / 129 | 78 / 99, 24: 115 / 130 | 111 / 99, 32: 117 / 130 | 145 / 100,
//     48: 160 / 130 | 204 / 101;
//   8 requests: 16 rows 17 / 27 | 18 / 27, 24: 31 / 28 | 32 / 29, 64: 43 / 29 | 63 / 29;
//   1 request x 8 192 keys: 16 rows 17 / 19 | 19 / 33, 48: 21 / 21 | 23 / 35, 80: 23 / 21 | 32 / 37.
int max_decode_rows(int64_t heads, int head_dim, int sm_count) {
  if (heads <= 16) return 64;                                    // (request, KV head) pairs: few, the row tiles run side by side
  return head_dim == 128 && heads > sm_count ? 32 : 16;
}

bool aligned(const void* ptr, unsigned bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }
bool strides_ok(std::initializer_list<int64_t> strides, int64_t elem, int64_t bytes) {
  for (int64_t s : strides)
    if (s < 0 || (s * elem) % bytes != 0) return false;
  return true;
}

CacheStrides cache_strides(int64_t page, int64_t row, int64_t head) { return {(uint32_t)page, (uint32_t)row, (long long)head}; }
// Page and row strides below 4 GB: the kernels multiply 32-bit numbers.
bool strides_small(std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s >= (1ll << 32)) return false;
  return true;
}

// Rows of `bytes` bytes, tokens x heads of them, at byte strides.
struct Rows {
  const void* base;
  int64_t token, head;
};
bool same_rows(const Rows& a, const Rows& b) { return a.base == b.base && a.token == b.token && a.head == b.head; }
// Whether a row of `a` and a row of `b` share a byte; with `a` itself for `b`: two different rows of it.  Two sets of
// unlike strides that lie within each other's range count as sharing.
bool rows_meet(const Rows& a, const Rows& b, int64_t tokens, int64_t heads, int64_t bytes) {
  const bool self = same_rows(a, b);
  const int64_t first_a = (int64_t)reinterpret_cast<intptr_t>(a.base), first_b = (int64_t)reinterpret_cast<intptr_t>(b.base);
  const int64_t last_a = first_a + (tokens - 1) * a.token + (heads - 1) * a.head + bytes;
  const int64_t last_b = first_b + (tokens - 1) * b.token + (heads - 1) * b.head + bytes;
  if (last_a <= first_b || last_b <= first_a) return false;
  if (a.token != b.token || a.head != b.head) return true;
  // equal strides: some row of b is dt tokens and dh heads away and less than a row's bytes
  for (int64_t dh = 1 - heads; dh < heads; ++dh) {
    const int64_t apart = first_b - first_a + dh * a.head;
    if (a.token == 0) {
      if (apart < bytes && -apart < bytes && !(self && dh == 0 && tokens == 1)) return true;
      continue;
    }
    const int64_t floor = apart >= 0 ? apart / a.token : -((-apart + a.token - 1) / a.token);
    for (int64_t back = floor; back <= floor + 1; ++back) {         // the two nearest
      const int64_t dt = std::max(1 - tokens, std::min(tokens - 1, back));
      const int64_t gap = apart - dt * a.token;
      if (gap < bytes && -gap < bytes && !(self && dh == 0 && dt == 0)) return true;
    }
  }
  return false;
}

// The out rows are written while other CTAs still read key and value and write the other side's rows.
bool outs_alias(const atrex_kv4_sm100_write_params* p) {
  auto rows = [&](const void* base, int64_t token, int64_t head) -> Rows {      // strides of single tokens and heads say nothing
    return {base, p->num_tokens > 1 ? 2 * token : 0, p->num_kv_heads > 1 ? 2 * head : 0};
  };
  const Rows in[2] = {rows(p->key, p->key_token_stride, p->key_head_stride),
                      rows(p->value, p->value_token_stride, p->value_head_stride)};
  const Rows out[2] = {rows(p->key_out, p->key_out_token_stride, p->key_out_head_stride),
                       rows(p->value_out, p->value_out_token_stride, p->value_out_head_stride)};
  auto meet = [&](const Rows& a, const Rows& b) { return rows_meet(a, b, p->num_tokens, p->num_kv_heads, 2ll * p->head_dim); };
  for (int i = 0; i < 2; ++i) {
    if (out[i].base == nullptr) continue;
    if (meet(out[i], out[i])) return true;                          // of an expanded tensor, say
    if (!same_rows(out[i], in[i]) && meet(out[i], in[i])) return true;
    // a set of rows and itself have no two rows that meet, but here the two are written and read as one
    if (same_rows(out[i], in[1 - i]) || meet(out[i], in[1 - i])) return true;
  }
  return out[0].base != nullptr && out[1].base != nullptr && (same_rows(out[0], out[1]) || meet(out[0], out[1]));
}

int check_write(const atrex_kv4_sm100_write_params* p) {
  if (p == nullptr) return report_failure(ATREX_FA_INVALID_VALUE, "parameter block is NULL");
  if (p->struct_bytes != sizeof(*p) || p->abi_version != ATREX_KV4_SM100_ABI_VERSION)
    return report_failure(ATREX_FA_ABI_MISMATCH, "struct_bytes / abi_version do not match this library");
  if (p->num_tokens < 0 || p->num_kv_heads <= 0 || p->page_size <= 0 || p->num_pages < 0)
    return report_failure(ATREX_FA_INVALID_VALUE, "num_tokens, num_kv_heads, page_size or num_pages out of range");
  if (p->head_dim <= 0 || p->head_dim % 16 != 0)
    return report_failure(ATREX_FA_UNSUPPORTED, "head_dim must be a positive multiple of 16");
  if (p->num_tokens == 0) return ATREX_FA_OK;
  if (p->key == nullptr || p->value == nullptr || p->slot_mapping == nullptr)
    return report_failure(ATREX_FA_INVALID_VALUE, "key, value or slot_mapping is NULL");
  if (p->num_pages > 0 && (p->key_cache == nullptr || p->value_cache == nullptr || p->key_block_scale == nullptr ||
                           p->value_block_scale == nullptr))
    return report_failure(ATREX_FA_INVALID_VALUE, "a cache or a block-scale tensor is NULL");
  if (!aligned(p->key, 32) || !aligned(p->value, 32) || !aligned(p->key_out, 32) || !aligned(p->value_out, 32) ||
      !strides_ok({p->key_token_stride, p->key_head_stride, p->value_token_stride, p->value_head_stride}, 2, 32) ||
      (p->key_out && !strides_ok({p->key_out_token_stride, p->key_out_head_stride}, 2, 32)) ||
      (p->value_out && !strides_ok({p->value_out_token_stride, p->value_out_head_stride}, 2, 32)))
    return report_failure(ATREX_FA_UNSUPPORTED, "key / value / key_out / value_out rows must start on 32-byte boundaries");
  if (outs_alias(p))
    return report_failure(ATREX_FA_INVALID_VALUE, "key_out / value_out may be key / value themselves, but must not overlap "
                                                  "them, each other or themselves in any other way");
  if (!aligned(p->key_cache, 8) || !aligned(p->value_cache, 8) ||
      !strides_ok({p->key_cache_page_stride, p->key_cache_row_stride, p->key_cache_head_stride,
                   p->value_cache_page_stride, p->value_cache_row_stride, p->value_cache_head_stride}, 1, 8) ||
      !strides_ok({p->key_scale_page_stride, p->key_scale_row_stride, p->key_scale_head_stride,
                   p->value_scale_page_stride, p->value_scale_row_stride, p->value_scale_head_stride}, 1, 1))
    return report_failure(ATREX_FA_UNSUPPORTED, "cache rows must start on 8-byte boundaries; strides must not be negative");
  if (!strides_small({p->key_cache_page_stride, p->key_cache_row_stride, p->value_cache_page_stride, p->value_cache_row_stride,
                      p->key_scale_page_stride, p->key_scale_row_stride, p->value_scale_page_stride, p->value_scale_row_stride}))
    return report_failure(ATREX_FA_UNSUPPORTED, "a cache page or row stride of 4 GB or more");
  return ATREX_FA_OK;
}

enum Kernel { kDecode, kSingle, kDouble };   // mma.sync; tcgen05 with one 128-row subtile per item; with two
struct Resolved {
  Kernel kernel;
  bool parts;            // splits leave partial results in scratch for the combine kernel
  bool tiled;            // more than one row tile per request possible -> device plan
  int rows, row_tiles, splits;
  uint64_t off_order, off_prefix, off_lse, off_o, bytes;
};

int check_params(const atrex_kv4_sm100_params* pp) {
  if (pp == nullptr) return report_failure(ATREX_FA_INVALID_VALUE, "parameter block is NULL");
  const atrex_fa_sm100_params* p = &pp->fa;
  if (pp->struct_bytes != sizeof(*pp) || pp->abi_version != ATREX_KV4_SM100_ABI_VERSION ||
      p->struct_bytes != sizeof(*p) || p->abi_version != ATREX_FA_SM100_ABI_VERSION)
    return report_failure(ATREX_FA_ABI_MISMATCH, "struct_bytes / abi_version do not match this library");
  if (p->batch < 0 || p->total_q < 0 || p->num_pages < 0 || p->max_seqlen_q < 0 || p->max_seqlen_k < 0 ||
      p->max_pages_per_seq < 0 || p->num_splits < 0)
    return report_failure(ATREX_FA_INVALID_VALUE, "negative size");
  if (p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->num_q_heads % p->num_kv_heads != 0)
    return report_failure(ATREX_FA_INVALID_VALUE, "num_q_heads must be a positive multiple of num_kv_heads");
  if (p->cu_seqlens_q == nullptr || p->out == nullptr || (p->total_q > 0 && p->q == nullptr))
    return report_failure(ATREX_FA_INVALID_VALUE, "q, out or cu_seqlens_q is NULL");
  if (p->page_size <= 0 || p->block_table == nullptr || p->seqused_k == nullptr)
    return report_failure(ATREX_FA_INVALID_VALUE, "a 4-bit cache is paged: block_table, seqused_k and a page size");
  if (p->return_lse && p->lse == nullptr) return report_failure(ATREX_FA_INVALID_VALUE, "return_lse without an lse buffer");
  if (p->num_pages > 0 && (p->k == nullptr || p->v == nullptr || pp->k_block_scale == nullptr || pp->v_block_scale == nullptr))
    return report_failure(ATREX_FA_INVALID_VALUE, "a cache or a block-scale tensor is NULL");
  if (p->dtype != ATREX_FA_BF16) return report_failure(ATREX_FA_UNSUPPORTED, "q must be BF16");
  if (p->head_dim != 128 && p->head_dim != 256) return report_failure(ATREX_FA_UNSUPPORTED, "head_dim must be 128 or 256");
  if (p->page_size % 64 != 0 && p->page_size != 16 && p->page_size != 32)
    return report_failure(ATREX_FA_UNSUPPORTED, "page_size must be 16, 32 or a multiple of 64");
  if (p->num_splits > kMaxSplits) return report_failure(ATREX_FA_UNSUPPORTED, "num_splits above 256");
  if (p->softcap != 0.f || p->cp_world_size > 1 || p->q_descale != nullptr)
    return report_failure(ATREX_FA_UNSUPPORTED, "softcap, context parallelism and q_descale are not served over a 4-bit cache");
  if (!(p->softmax_scale > 0.f)) return report_failure(ATREX_FA_UNSUPPORTED, "softmax_scale must be positive");
  if (p->route != ATREX_FA_ROUTE_AUTO && p->route != ATREX_FA_ROUTE_MMA && p->route != ATREX_FA_ROUTE_UMMA)
    return report_failure(ATREX_FA_INVALID_VALUE, "unknown route");
  const unsigned scale_bytes = (unsigned)p->head_dim / 16;
  if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->k, 16) || !aligned(p->v, 16) ||
      !strides_ok({p->q_row_stride, p->q_head_stride, p->out_row_stride, p->out_head_stride}, 2, 16) ||
      !strides_ok({p->k_page_stride, p->k_row_stride, p->k_head_stride, p->v_page_stride, p->v_row_stride,
                   p->v_head_stride}, 1, 16))
    return report_failure(ATREX_FA_UNSUPPORTED, "q, k, v and out rows must start on 16-byte boundaries");
  if (!aligned(pp->k_block_scale, scale_bytes) || !aligned(pp->v_block_scale, scale_bytes) ||
      !strides_ok({pp->k_scale_page_stride, pp->k_scale_row_stride, pp->k_scale_head_stride, pp->v_scale_page_stride,
                   pp->v_scale_row_stride, pp->v_scale_head_stride}, 1, scale_bytes))
    return report_failure(ATREX_FA_UNSUPPORTED, "block-scale rows must start on boundaries of head_dim / 16 bytes");
  if (!strides_small({p->k_page_stride, p->k_row_stride, p->v_page_stride, p->v_row_stride, pp->k_scale_page_stride,
                      pp->k_scale_row_stride, pp->v_scale_page_stride, pp->v_scale_row_stride}))
    return report_failure(ATREX_FA_UNSUPPORTED, "a cache page or row stride of 4 GB or more");
  return ATREX_FA_OK;
}

uint64_t align_up(uint64_t x, uint64_t a) { return (x + a - 1) / a * a; }

// Which kernel and how many KV splits, from graph-static sizes only.
int resolve(const atrex_kv4_sm100_params* pp, int sm_count, Resolved* r) {
  const atrex_fa_sm100_params* p = &pp->fa;
  const int group = p->num_q_heads / p->num_kv_heads;
  const int64_t packed = (int64_t)p->max_seqlen_q * group;      // query rows per (request, KV head), at most
  const bool prefill = p->route == ATREX_FA_ROUTE_UMMA || (p->route == ATREX_FA_ROUTE_AUTO &&
                        packed > max_decode_rows((int64_t)p->batch * p->num_kv_heads, p->head_dim, sm_count));
  // Two-tile or single-tile, unsplit or by the split rule below (us, head_dim 128; requests, heads, query tokens, contexts):
  //   items that fill the SMs: 4, 64 / 8, 512 .. 2 048, 4 096 .. 16 384: 1 823 / 2 626;  1, 32 / 8, 2 048, 16 384: 542 / 863;
  //     64, 64 / 4, 9, 2 000 .. 8 000: 248 / 309;  16, 32 / 8, 200 .. 1 000, 1 000 .. 4 000: 625 / 573;  64 of 60 .. 200: 148 / 142
  //   items that leave SMs idle, where the two-tile kernel, which is never split, is the wrong choice: 1 over 16 384 keys,
  //     8 / 1 heads: 32 .. 128 tokens 263 / 41, 512: 263 / 78, 2 048: 263 / 232;  32 / 8 heads: 128: 265 / 97, 512: 264 / 235
  // A call with num_splits of 2 or more takes the single-tile kernel: with one that fills the SMs, about the second figure.
  r->kernel = !prefill ? kDecode
              : p->head_dim == 128 && packed > kv4_prefill_rows() && p->num_splits <= 1 ? kDouble : kSingle;
  r->rows = r->kernel == kDouble ? kv4_prefill2_rows()
            : prefill            ? kv4_prefill_rows()
                                 : kv4_decode_rows(p->head_dim, (int)(packed > 64 ? 64 : packed));
  r->tiled = r->kernel == kDouble || (prefill && packed > r->rows);
  // row tiles: of a request (mma.sync kernel, whose grid has them all), or of the call (tcgen05 kernel's work items)
  const int64_t tiles = !prefill ? (packed > r->rows ? (packed + r->rows - 1) / r->rows : 1)
                        : r->tiled  ? (int64_t)p->total_q * group / r->rows + p->batch
                                    : p->batch;
  const int64_t items = tiles * p->num_kv_heads * (prefill || p->batch == 0 ? 1 : p->batch);
  if (items * kMaxSplits > 0x7FFFFFFFll)
    return report_failure(ATREX_FA_UNSUPPORTED, "row tiles x KV heads x splits exceeds the 32-bit grid");
  r->row_tiles = (int)tiles;
  int64_t span = p->max_seqlen_k;               // keys a row tile can see, at most
  if (p->window_left >= 0 && (p->causal || p->window_right >= 0)) {
    const int64_t rows_q = r->tiled ? (r->rows + group - 1) / group + 1 : p->max_seqlen_q;
    const int64_t w = (int64_t)p->window_left + rows_q + (p->causal ? 0 : p->window_right) + 128;
    if (w < span) span = w;
  }
  const int64_t tile = prefill ? kv4_prefill_tile(p->head_dim) : 32, most = (span + tile - 1) / tile;
  int64_t splits = r->kernel == kDouble ? 1 : p->num_splits;
  if (splits == 0 && prefill) {
    // Items walk the SMs in rounds; an item costs about four tiles besides its own (Q rows, first scores, epilogue).
    // Splitting costs eight tiles (the combine kernel, the start of smaller items) and the partial results, of which
    // 1.5 MB written and read take a tile's 1.3 us.  An unsplit call counts an eighth more, because it waits for its
    // longest item and lengths vary; beyond three rounds nothing is split, nor into more than 256 MB.  The constants are
    // those with the least loss over 27 shapes measured with 1 .. 48 splits, 3 % on average, 18 % at most.  Microseconds by
    // splits, the rule's choice in brackets (requests, heads of D, query tokens, contexts):
    //   1, 64 / 4 of 128, 5, 16 384:  1: 226, 4: 68, 16: 29, [32: 25], 48: 37;    8, same, 8 192:  1: 120, [4: 43], 8: 48
    //   30, 64 / 4 of 128, 8, 500 .. 30 000:  1: 379, 4: 281, [6: 300];   all 20 000:  [1: 280], 2: 303, 6: 287
    //   40, 64 / 8 of 128, 10, 4 000 .. 16 000:  1: 424, [3: 373];   20, same, 9 .. 15, 1 000 .. 9 000:  1: 195, [3: 128], 5: 178
    //   16, 24 / 2 of 256, 1 .. 96, 97 .. 8 192:  1: 185, [3: 158], 6: 184;   90 .. 96, 8 192:  1: 361, [2: 419], 4: 476
    //   1, 64 / 8 of 256, 512, 16 384:  1: 680, [2: 731], 5: 748;   3, 32 / 8, ~1 000, 5 000 .. 12 974:  [1: 1 065], 3: 1 168
    const int64_t part = 4 * (int64_t)p->total_q * p->num_q_heads * (p->head_dim + 1);     // bytes of a split's results
    int64_t best = 0;                                                                      // in eighths of a tile
    splits = 1;
    for (int64_t s = 1; s <= most && s <= 64; ++s) {
      if (s > 1 && (items > 3 * (int64_t)sm_count || s * part > (256 << 20))) break;
      const int64_t tiles_long = ((items * s + sm_count - 1) / sm_count) * ((most + s - 1) / s + 4);
      const int64_t cost = s == 1 ? 9 * tiles_long : 8 * tiles_long + 64 + s * part / (192 << 10);
      if (s == 1 || cost < best) {
        best = cost;
        splits = s;
      }
    }
  } else if (splits == 0) {
    // Up to one wave of CTAs in splits of 16 tiles (four per warp) or more; three waves, which even out unlike lengths, if
    // that leaves 96 tiles or more, since a CTA costs ~3.5 us besides its tiles.  Microseconds by splits, D 128:
    //   512 items of 1 024 .. 16 384 keys: 1: 178, 2: 157, 3: 144, 6: 148, 12: 171;  600 of 2 000 keys: 1: 51, 2: 56, 4: 64
    //   160 items of 16 000: 1: 139, 2: 103, 5: 90, 8: 89, 16: 101;  128 of 8 000: 1: 56, 2: 45, 3: 41, 4: 50, 16: 56
    const int64_t wave = (int64_t)kv4_decode_resident(p->head_dim) * sm_count, n = items > 0 ? items : 1;
    const int64_t one = std::min(wave / n, most / 16), three = std::min((3 * wave + n - 1) / n, most / 96);
    splits = std::max(one, three);
  }
  if (splits > most) splits = most;
  if (splits > kMaxSplits) splits = kMaxSplits;
  if (splits < 1) splits = 1;
  r->splits = (int)splits;
  // Splits join inside the decode kernel while the whole call is one wave of CTAs; in larger calls clusters, which start
  // together, cost more than the combine kernel.  Microseconds, cluster / combine: 64 requests of 1 024 .. 16 384 keys,
  // 2 048 CTAs: 161 / 151; 512 CTAs at head_dim 128: 49.6 / 47.7, 55.8 / 49.5, 33.3 / 31.4; 320 and 400 at 256: 47.6 / 43.4,
  // 73.5 / 66.5.  Within a wave the cluster wins: one request of 4 097 keys 14.5 -> 12.5 (the kernel's first version).
  const int64_t wave = (int64_t)kv4_decode_resident(p->head_dim) * sm_count;
  r->parts = splits > 1 && !(r->kernel == kDecode && splits <= kv4_decode_max_cluster() && items * splits <= wave);
  uint64_t off = 0;
  r->off_order = off;
  if (r->tiled) off = align_up(off + 4ull * p->batch, 256);
  r->off_prefix = off;
  if (r->tiled) off = align_up(off + 4ull * (p->batch + 1), 256);
  r->off_lse = off;
  if (r->parts) off = align_up(off + 4ull * splits * p->total_q * p->num_q_heads, 256);
  r->off_o = off;
  if (r->parts) off = align_up(off + 4ull * splits * p->total_q * p->num_q_heads * p->head_dim, 256);
  r->bytes = off;
  return ATREX_FA_OK;
}

// The TMA descriptors of the code caches into the kernel's block.
int encode_code_maps(const atrex_fa_sm100_params* p, int box_rows, FwdParams* f) {
  const int row_bytes = p->head_dim / 2;
  int st;
  if (p->num_pages == 0) {        // no page exists and no copy is issued, but the descriptors must be valid: over q
    st = encode_byte_rows_map(&f->k_map, p->q, row_bytes, row_bytes, row_bytes, row_bytes, 1, 1, 1, 1, f->k_perm);
    if (st == ATREX_FA_OK)
      st = encode_byte_rows_map(&f->v_map, p->q, row_bytes, row_bytes, row_bytes, row_bytes, 1, 1, 1, 1, f->v_perm);
    return st;
  }
  st = encode_byte_rows_map(&f->k_map, p->k, row_bytes, p->k_head_stride, p->k_row_stride, p->k_page_stride,
                            p->num_kv_heads, p->page_size, p->num_pages, box_rows, f->k_perm);
  if (st == ATREX_FA_OK)
    st = encode_byte_rows_map(&f->v_map, p->v, row_bytes, p->v_head_stride, p->v_row_stride, p->v_page_stride,
                              p->num_kv_heads, p->page_size, p->num_pages, box_rows, f->v_perm);
  return st;
}

int prepare_current_device() {
  static std::atomic<int> prepared[64];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return report_failure(ATREX_FA_CUDA_ERROR, "cudaGetDevice", e);
  if (dev >= 0 && dev < 64 && prepared[dev].load(std::memory_order_acquire)) return ATREX_FA_OK;
  e = kv4_decode_prepare();
  if (e == cudaSuccess) e = kv4_prefill_prepare();
  if (e == cudaSuccess) e = kv4_prefill2_prepare();
  if (e != cudaSuccess) return report_failure(ATREX_FA_CUDA_ERROR, "cudaFuncSetAttribute (4-bit cache kernels)", e);
  if (dev >= 0 && dev < 64) prepared[dev].store(1, std::memory_order_release);
  return ATREX_FA_OK;
}

}  // namespace
}  // namespace atrex_sm100

using namespace atrex_sm100;

extern "C" {

int atrex_kv4_sm100_abi_version(void) { return ATREX_KV4_SM100_ABI_VERSION; }
size_t atrex_kv4_sm100_params_bytes(void) { return sizeof(atrex_kv4_sm100_params); }
size_t atrex_kv4_sm100_write_params_bytes(void) { return sizeof(atrex_kv4_sm100_write_params); }

int atrex_kv4_sm100_write(const atrex_kv4_sm100_write_params* p, void* stream) {
  clear_failure();
  int st = check_write(p);
  if (st != ATREX_FA_OK) return st;
  int sms = 0;
  st = current_sm_count(&sms);
  if (st != ATREX_FA_OK) return st;
  if (p->num_tokens == 0) return ATREX_FA_OK;
  Kv4WriteParams k;
  std::memset(&k, 0, sizeof(k));
  for (int i = 0; i < 2; ++i) {
    Kv4WriteSide& s = k.side[i];
    s.src = static_cast<const uint8_t*>(i ? p->value : p->key);
    s.codes = static_cast<uint8_t*>(i ? p->value_cache : p->key_cache);
    s.scales = static_cast<uint8_t*>(i ? p->value_block_scale : p->key_block_scale);
    s.out = static_cast<uint8_t*>(i ? p->value_out : p->key_out);
    s.factor = i ? p->v_factor : p->k_factor;
    s.src_token = 2 * (i ? p->value_token_stride : p->key_token_stride);
    s.src_head = 2 * (i ? p->value_head_stride : p->key_head_stride);
    s.out_token = 2 * (i ? p->value_out_token_stride : p->key_out_token_stride);
    s.out_head = 2 * (i ? p->value_out_head_stride : p->key_out_head_stride);
    s.factor_stride = i ? p->v_factor_stride : p->k_factor_stride;
    s.code = i ? cache_strides(p->value_cache_page_stride, p->value_cache_row_stride, p->value_cache_head_stride)
               : cache_strides(p->key_cache_page_stride, p->key_cache_row_stride, p->key_cache_head_stride);
    s.scale = i ? cache_strides(p->value_scale_page_stride, p->value_scale_row_stride, p->value_scale_head_stride)
                : cache_strides(p->key_scale_page_stride, p->key_scale_row_stride, p->key_scale_head_stride);
  }
  k.slot_mapping = reinterpret_cast<const long long*>(p->slot_mapping);
  k.slot_limit = (long long)p->num_pages * p->page_size;
  k.num_tokens = p->num_tokens;
  k.num_kv_heads = p->num_kv_heads;
  k.head_dim = p->head_dim;
  k.page_size = p->page_size;
  const cudaError_t e = kv4_write_launch(k, sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? ATREX_FA_OK : report_failure(ATREX_FA_CUDA_ERROR, "launch of the 4-bit cache write", e);
}

int atrex_kv4_sm100_plan(const atrex_kv4_sm100_params* p, atrex_fa_sm100_plan_info* plan) {
  clear_failure();
  if (plan == nullptr) return report_failure(ATREX_FA_INVALID_VALUE, "plan is NULL");
  int st = check_params(p);
  if (st != ATREX_FA_OK) return st;
  int sms = p->fa.sm_count;
  if (sms <= 0 && (st = current_sm_count(&sms)) != ATREX_FA_OK) return st;
  Resolved r;
  st = resolve(p, sms, &r);
  if (st != ATREX_FA_OK) return st;
  plan->route = r.kernel != kDecode ? ATREX_FA_ROUTE_UMMA : ATREX_FA_ROUTE_MMA;
  plan->num_splits = r.splits;
  plan->kernel_launches = 1 + (r.tiled ? 1 : 0) + (r.parts ? 1 : 0);
  plan->m_rows = r.rows;
  plan->workspace_bytes = r.bytes;
  return ATREX_FA_OK;
}

int atrex_kv4_sm100_forward(const atrex_kv4_sm100_params* pp, void* workspace, uint64_t workspace_bytes,
                            void* stream_ptr) {
  clear_failure();
  int st = check_params(pp);
  if (st != ATREX_FA_OK) return st;
  const atrex_fa_sm100_params* p = &pp->fa;
  int sms = 0;
  st = current_sm_count(&sms);
  if (st != ATREX_FA_OK) return st;
  Resolved r;
  st = resolve(pp, p->sm_count > 0 ? p->sm_count : sms, &r);
  if (st != ATREX_FA_OK) return st;
  if (r.bytes > 0 && (workspace == nullptr || workspace_bytes < r.bytes || !aligned(workspace, 256)))
    return report_failure(ATREX_FA_WORKSPACE_TOO_SMALL, "workspace missing, misaligned or too small");
  if (p->batch == 0 || p->total_q == 0) return ATREX_FA_OK;
  st = prepare_current_device();
  if (st != ATREX_FA_OK) return st;

  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  Kv4Params k;
  std::memset(static_cast<void*>(&k), 0, sizeof(k));
  FwdParams& f = k.f;
  if (r.kernel != kDecode) {
    int box = kv4_prefill_tile(p->head_dim);     // rows of one copy: the largest power of two that divides a tile and a page
    while (p->page_size % box != 0) box >>= 1;
    st = encode_code_maps(p, box, &f);
    if (st != ATREX_FA_OK) return st;
    f.box_rows = box;
  }
  f.q = p->q; f.out = p->out; f.lse = p->return_lse ? p->lse : nullptr;
  f.cu_seqlens_q = p->cu_seqlens_q;
  f.seqused_k = p->seqused_k;
  f.block_table = p->block_table;
  f.k_descale = p->k_descale; f.v_descale = p->v_descale;
  f.sink = static_cast<const __nv_bfloat16*>(p->sink);
  f.status = p->device_status;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (r.parts) {
    f.part_lse = reinterpret_cast<float*>(ws + r.off_lse);
    f.part_o = reinterpret_cast<float*>(ws + r.off_o);
  }
  f.q_row_stride = p->q_row_stride; f.q_head_stride = p->q_head_stride;
  f.out_row_stride = p->out_row_stride; f.out_head_stride = p->out_head_stride;
  f.block_table_row_stride = p->block_table_row_stride;
  f.k_descale_bs = p->k_descale_batch_stride; f.k_descale_hs = p->k_descale_head_stride;
  f.v_descale_bs = p->v_descale_batch_stride; f.v_descale_hs = p->v_descale_head_stride;
  f.batch = p->batch; f.total_q = p->total_q;
  f.num_pages = p->num_pages; f.page_size = p->page_size;
  f.num_q_heads = p->num_q_heads; f.num_kv_heads = p->num_kv_heads;
  f.group = p->num_q_heads / p->num_kv_heads;
  f.causal = p->causal ? 1 : 0;
  f.window_left = window_of(p->window_left);
  f.window_right = p->causal ? 0 : window_of(p->window_right);
  f.num_splits = r.splits;
  const int64_t cap = (int64_t)p->max_pages_per_seq * p->page_size;
  f.kv_cap = (int32_t)(cap > 0x7FFFFFFFll ? 0x7FFFFFFFll : cap);
  f.cp_world_size = 1;
  f.softmax_scale = p->softmax_scale;
  k.k = static_cast<const uint8_t*>(p->k); k.v = static_cast<const uint8_t*>(p->v);
  k.ks = static_cast<const uint8_t*>(pp->k_block_scale); k.vs = static_cast<const uint8_t*>(pp->v_block_scale);
  k.k_str = cache_strides(p->k_page_stride, p->k_row_stride, p->k_head_stride);
  k.v_str = cache_strides(p->v_page_stride, p->v_row_stride, p->v_head_stride);
  k.ks_str = cache_strides(pp->k_scale_page_stride, pp->k_scale_row_stride, pp->k_scale_head_stride);
  k.vs_str = cache_strides(pp->v_scale_page_stride, pp->v_scale_row_stride, pp->v_scale_head_stride);
  k.row_tiles = r.row_tiles;
  k.cluster = r.splits > 1 && !r.parts;
  f.num_row_tiles = r.row_tiles;
  cudaError_t e;
  if (r.tiled) {
    int32_t* order = reinterpret_cast<int32_t*>(ws + r.off_order);
    int32_t* prefix = reinterpret_cast<int32_t*>(ws + r.off_prefix);
    f.order = order;
    f.tile_prefix = prefix;
    if ((e = plan_launch(f, r.rows, order, prefix, stream)) != cudaSuccess)
      return report_failure(ATREX_FA_CUDA_ERROR, "launch of the plan kernel", e);
  }

  if (p->profile_event_begin != nullptr &&
      (e = cudaEventRecord(static_cast<cudaEvent_t>(p->profile_event_begin), stream)) != cudaSuccess)
    return report_failure(ATREX_FA_CUDA_ERROR, "cudaEventRecord(profile_event_begin)", e);
  if (p->sm_count > 0) sms = p->sm_count;
  e = r.kernel == kDouble   ? kv4_prefill2_launch(k, sms, stream)
      : r.kernel == kSingle ? kv4_prefill_launch(k, p->head_dim, sms, stream)
                            : kv4_decode_launch(k, p->head_dim, r.rows, stream);
  if (e != cudaSuccess) return report_failure(ATREX_FA_CUDA_ERROR, "launch of the 4-bit cache attention", e);
  if (p->profile_event_end != nullptr &&
      (e = cudaEventRecord(static_cast<cudaEvent_t>(p->profile_event_end), stream)) != cudaSuccess)
    return report_failure(ATREX_FA_CUDA_ERROR, "cudaEventRecord(profile_event_end)", e);
  if (r.parts && (e = combine_launch(f, p->head_dim, stream)) != cudaSuccess)
    return report_failure(ATREX_FA_CUDA_ERROR, "launch of the combine kernel", e);
  return ATREX_FA_OK;
}

}  // extern "C"
