// Attention over a 4-bit paged cache for few query rows: decode, speculative verify, and every call the tcgen05
// kernel does not take.
//
//   S^T = K Q^T,  P = 2^(S scale - m),  O^T = V^T P^T     per (request, KV head, 8 or 16 packed GQA rows, KV split)
//
// The cache is the M operand of mma.sync m16n8k16 (16 tokens of K, 16 head dimensions of V^T), the packed query rows
// are N: with 8 rows or fewer no tensor work is spent on padding, and a widened cache register is used for all rows.
// Both products are in FP16 with FP32 accumulators.  Widening E2M1 x E4M3 to FP16 is exact (fp4.cuh); a query row is
// scaled by a power of two so that its largest element is about 2^13 (exact too, down to 2^-27 of that), and P is
// stored as 2^7 p, so that probabilities down to 2^-31 of the row's reference keep their weight.
//
// One warp is one pipeline: 32 tokens at a time, private ring of kStages stages filled with cp.async by the warp
// itself, private online-softmax state; no CTA-wide barrier until the warps' states merge at the end.  The order of
// tokens inside a tile and of dimensions inside a row is free as long as both operands agree, and is chosen so that
// a lane's fragment is one 16-byte (K) or 8-byte (V) shared-memory load:
//   K: lane (g, t) of an m16 tile holds rows g and g + 8; its 32 dimensions are 32 t .. 32 t + 31 of each 128, four
//      at a time for the k16 steps (Q is loaded in the same order);
//   V: lane (g, t) holds dimensions 16 g .. 16 g + 15 of each 128 (one scale block) of the tokens t, 4 + t, 8 + t,
//      12 + t of every 16; MMA row g is an even dimension, row g + 8 the odd one behind it.  The nibbles of two
//      tokens are brought together before they are widened (one shift and one select per four pairs).
// The k index 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of P V belongs to those four tokens, so K's MMA row r holds token
// (r & 8) + 4 (r & 1) + ((r & 7) >> 1); P^T comes from S^T by one movmatrix per 8 x 8 block.
//
// Measured (32 / 8 heads of 128): one request of 4 097 keys 10.4 us; 64 requests of 1 024 .. 16 384 keys 144 us = 4.1 TB/s
// of codes and scales, 91 us at the measured copy rate; 300 of 1 000 keys 92 us (53).  What bounds it: instruction issue.
// A token and head costs ~19 warp instructions, of which 12 widen (convert, multiply by the block scale); three warps per
// scheduler, which is what 162 registers allow, issue in 0.6 of the cycles (math pipes busy and fixed latencies).  Four
// CTAs per SM in 128 registers: 158 us.  Codes by TMA: 154 against 144 (one lane's issue and polling cost more than eight
// cp.async a lane).  A CTA costs ~3.5 us besides its tiles, hence few splits (the rule is the launcher's).  Warps with
// equal shares of all tiles of the call: 138 us here, but 300 requests of 100 .. 4 000 keys 172 -> 188.
#include <type_traits>

#include <cooperative_groups.h>

#include "fp4.cuh"
#include "kv4_kernels.cuh"
#include "ptx.cuh"
#include "softmax_math.cuh"

namespace atrex_sm100 {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kMaxCluster = 8;            // portable cluster size
constexpr int kTile = 32;                 // tokens per warp and step
constexpr float kThreshold = 8.f;         // a row's reference is raised when its maximum grows by more than 2^8
constexpr float kShift = 7.f;             // P is stored as 2^7 p: at most 2^15

template <int D, int NB>
struct DecodeCfg {
  static constexpr int kRows = 8 * NB;                   // packed query rows per CTA
  static constexpr int kChunks = D / 128;                // 128-dimension parts of a row
  static constexpr int kRowBytes = D / 2, kScaleBytes = D / 16;
  static constexpr int kOffV = kTile * kRowBytes, kOffKs = 2 * kTile * kRowBytes;
  static constexpr int kOffVs = kOffKs + kTile * kScaleBytes;
  static constexpr int kStageBytes = 2 * kTile * (kRowBytes + kScaleBytes);
  static constexpr int kStages = D == 128 ? 3 : 2;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kMergePitch = D + 4;              // floats per packed row of a warp's partial O
  static constexpr int kMergeBytes = kWarps * kRows * kMergePitch * 4;
  static constexpr int kOffState = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;   // m and l of the warps, of the CTA
  static constexpr int kSmemBytes = kOffState + (2 * kWarps + 2) * kRows * 4;
};

// kBytes from global to shared memory, asynchronously; zeros where !ok (never so when kWhole).
template <int kBytes, bool kWhole>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool ok) {
  if (kBytes == 16 && kWhole) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  } else if (kBytes == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16u : 0u) : "memory");
  } else if (kWhole) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8u : 0u) : "memory");
  }
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Where 16-byte chunk `chunk` of a token's K / V row lies in its stage.  K rows are stored in MMA row order; the
// exclusive-ors spread the rows that one load instruction touches over the banks.
template <int D>
__device__ __forceinline__ int k_offset(int token, int chunk) {
  const int row = (token & 24) + 2 * (token & 3) + ((token >> 2) & 1);
  return row * (D / 2) + (D == 256 ? chunk ^ ((row & 1) << 2) : chunk) * 16;
}
template <int D>
__device__ __forceinline__ int v_offset(int token, int chunk) {
  return token * (D / 2) + (D == 256 ? chunk ^ ((token & 3) << 1) : chunk ^ (token & 2)) * 16;
}

template <int D, int NB>
__global__ void __launch_bounds__(kWarps * 32, NB == 2 ? 3 : 1) atrex_sm100_kv4_decode_kernel(const __grid_constant__ Kv4Params pp) {
  using C = DecodeCfg<D, NB>;
  const FwdParams& p = pp.f;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  // the splits of a row tile next to each other: up to eight form a cluster
  const int split = blockIdx.x % p.num_splits;
  int rest = blockIdx.x / p.num_splits;
  const int row_tile = rest % pp.row_tiles;
  rest /= pp.row_tiles;
  const int kvh = rest % p.num_kv_heads, b = rest / p.num_kv_heads;

  const int q_start = p.cu_seqlens_q[b];
  const int q_len = min(p.cu_seqlens_q[b + 1], p.total_q) - q_start;
  const int rows_total = q_len * p.group, row0 = row_tile * C::kRows;
  if (row0 >= rows_total || q_start < 0) return;
  int kv_len, k_start;
  request_kv(p, b, kv_len, k_start);
  const int off = request_off(p, b, kv_len, q_len);
  const int qi_lo = row0 / p.group, qi_hi = (min(rows_total, row0 + C::kRows) - 1) / p.group;
  int kv_end = kv_len, kv_begin = 0;
  if (p.window_right >= 0) kv_end = min(kv_len, right_bound(p, qi_hi + off));
  if (p.window_left >= 0) kv_begin = max(0, qi_lo + off - p.window_left);
  // keys lo .. hi - 1 that packed row r of this CTA sees
  auto row_keys = [&](int r, int& lo, int& hi) {
    const int qi = min((row0 + r) / p.group, q_len - 1);
    hi = p.window_right >= 0 ? min(kv_len, right_bound(p, qi + off)) : kv_len;
    lo = p.window_left >= 0 ? max(0, qi + off - p.window_left) : 0;
  };
  // keys every row of this CTA sees
  const int full_lo = p.window_left >= 0 ? max(0, qi_hi + off - p.window_left) : 0;
  const int full_hi = p.window_right >= 0 ? min(kv_len, right_bound(p, qi_lo + off)) : kv_len;
  int tile_lo = 0, n_tiles = 0;
  if (kv_end > kv_begin) {
    const int first = kv_begin / kTile, n = (kv_end + kTile - 1) / kTile - first;
    const int lo = (int)((long long)n * split / p.num_splits);
    const int hi = (int)((long long)n * (split + 1) / p.num_splits);
    tile_lo = first + lo;
    n_tiles = hi - lo;
  }
  const bool part_mode = p.num_splits > 1 && !pp.cluster;   // partial results go to scratch for the combine kernel
  if (n_tiles == 0 && part_mode) {
    if (threadIdx.x < C::kRows && row0 + threadIdx.x < rows_total) {
      const int row = row0 + threadIdx.x;
      p.part_lse[((int64_t)split * p.total_q + q_start + row / p.group) * p.num_q_heads + kvh * p.group + row % p.group] =
          -INFINITY;
    }
    return;
  }
  const int my_tiles = n_tiles > warp ? (n_tiles - warp + kWarps - 1) / kWarps : 0;

  // ---- the warp's copies ----
  uint8_t* ring = smem + warp * (C::kStages * C::kStageBytes);
  const int32_t* table = p.block_table + (int64_t)b * p.block_table_row_stride;
  const int shift = (p.page_size & (p.page_size - 1)) == 0 ? __ffs(p.page_size) - 1 : -1;
  // A tile lies in one page, or in two when pages have 16 rows.  Lane i holds the pages of the i-th of 32 tiles of this
  // warp: one load of the table per 32 tiles, a shuffle per tile.
  const bool two_pages = p.page_size == 16;
  const int tok_end = (tile_lo + n_tiles) * kTile;
  int page_batch[2] = {-1, -1};
  int fetched = 0;                                // tiles whose pages were handed out
  auto load_pages = [&]() {
    const int tok = (tile_lo + warp + (fetched + lane) * kWarps) * kTile;
    auto page_of = [&](int t) -> int {
      if (t >= kv_end) return -1;
      const int pg = table[shift >= 0 ? t >> shift : t / p.page_size];
      return pg < p.num_pages ? pg : -1;
    };
    page_batch[0] = tok < tok_end ? page_of(tok) : -1;
    page_batch[1] = two_pages && tok < tok_end ? page_of(tok + 16) : page_batch[0];
  };
  int next_page[2] = {-1, -1};
  auto fetch_pages = [&]() {
    if ((fetched & 31) == 0) load_pages();
    next_page[0] = __shfl_sync(0xffffffffu, page_batch[0], fetched & 31);
    next_page[1] = two_pages ? __shfl_sync(0xffffffffu, page_batch[1], fetched & 31) : next_page[0];
    ++fetched;
  };
  // Lane (row, chunk) of a copy moves 16-byte chunk `chunk` of the tokens row, row + kStep, ...  Page and row strides
  // are 32-bit numbers, so that an address is a chain of 32 x 32 + 64-bit multiply-adds: with 64-bit strides the copies
  // were 208 of the 677 instructions of a tile.
  constexpr int kPerRow = C::kRowBytes / 16, kStep = 32 / kPerRow;
  const int c_row = lane / kPerRow, c_chunk = lane % kPerRow;
  const int s_row = two_pages ? lane & 15 : lane;
  const uint8_t* k_lane = pp.k + kvh * pp.k_str.head + (uint64_t)c_row * pp.k_str.row + c_chunk * 16;
  const uint8_t* v_lane = pp.v + kvh * pp.v_str.head + (uint64_t)c_row * pp.v_str.row + c_chunk * 16;
  const uint8_t* ks_lane = pp.ks + kvh * pp.ks_str.head + (uint64_t)s_row * pp.ks_str.row;
  const uint8_t* vs_lane = pp.vs + kvh * pp.vs_str.head + (uint64_t)s_row * pp.vs_str.row;
  const uint32_t k_dst = smem_u32(ring) + k_offset<D>(c_row, c_chunk), v_dst = smem_u32(ring) + C::kOffV + v_offset<D>(c_row, c_chunk);
  const uint32_t ks_dst = smem_u32(ring) + C::kOffKs + ((lane & 24) + 2 * (lane & 3) + ((lane >> 2) & 1)) * C::kScaleBytes;
  const uint32_t vs_dst = smem_u32(ring) + C::kOffVs + lane * C::kScaleBytes;
  int copy_tok = (tile_lo + warp) * kTile;
  // The rows of one tile; kWhole: every token counts and has a page, otherwise the others become zeros.
  auto copy_rows = [&](uint32_t stage_off, auto whole_tag) {
    constexpr bool kWhole = decltype(whole_tag)::value;
    const uint32_t in_page = two_pages ? 0 : shift >= 0 ? copy_tok & (p.page_size - 1) : copy_tok % p.page_size;
    auto counts = [&](int token, int page) {
      return kWhole || (page >= 0 && copy_tok + token < kv_end && copy_tok + token >= kv_begin);
    };
    auto page_base = [](const uint8_t* lane_base, int page, uint32_t row, const CacheStrides& st) {
      return lane_base + (uint64_t)(uint32_t)max(page, 0) * st.page + (uint64_t)row * st.row;
    };
    const uint8_t *k0 = page_base(k_lane, next_page[0], in_page, pp.k_str), *k1 = k0;
    const uint8_t *v0 = page_base(v_lane, next_page[0], in_page, pp.v_str), *v1 = v0;
    uint32_t back = 0;                               // rows that the second page's base lies behind the first's
    if (two_pages) {
      k1 = page_base(k_lane, next_page[1], 0, pp.k_str);
      v1 = page_base(v_lane, next_page[1], 0, pp.v_str);
      back = 16;
    }
#pragma unroll
    for (int u = 0; u < kPerRow; ++u) {
      constexpr int kHalf = 16 / kStep;
      const bool second = u >= kHalf;
      const bool ok = counts(u * kStep + c_row, second ? next_page[1] : next_page[0]);
      const uint32_t row = u * kStep - (second ? back : 0);
      const uint8_t* k_src = (second ? k1 : k0) + (uint64_t)row * pp.k_str.row;
      const uint8_t* v_src = (second ? v1 : v0) + (uint64_t)row * pp.v_str.row;
      // offsets of token u * kStep + c_row, relative to c_row's, are known at compile time
      const uint32_t k_off = stage_off + k_offset<D>(u * kStep, 0), v_off = stage_off + v_offset<D>(u * kStep, 0);
      const uint32_t k_at = D == 256 && (u & 1) ? (k_dst ^ 64u) + k_off - 64u : k_dst + k_off;
      cp_async<16, kWhole>(k_at, k_src, ok);
      cp_async<16, kWhole>(v_dst + v_off, v_src, ok);
    }
    const int page = lane < 16 ? next_page[0] : next_page[1];
    const bool ok = counts(lane, page);
    cp_async<C::kScaleBytes, kWhole>(ks_dst + stage_off, page_base(ks_lane, page, in_page, pp.ks_str), ok);
    cp_async<C::kScaleBytes, kWhole>(vs_dst + stage_off, page_base(vs_lane, page, in_page, pp.vs_str), ok);
  };
  // Copies the next tile, whose pages were fetched, into `stage`; one commit group whatever happens.
  auto copy_tile = [&](int stage) {
    if (copy_tok < tok_end) {
      const uint32_t stage_off = stage * C::kStageBytes;
      if (copy_tok >= kv_begin && copy_tok + kTile <= kv_end && (next_page[0] | next_page[1]) >= 0)
        copy_rows(stage_off, std::true_type{});
      else
        copy_rows(stage_off, std::false_type{});
    }
    copy_tok += kWarps * kTile;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) {
    fetch_pages();
    copy_tile(s);
  }

  // ---- Q: FP16 fragments of packed rows 8 nb + g, the row's power of two folded into its score factor ----
  uint32_t qf[NB][C::kChunks][8][2];
  float factor[NB][2];                    // score factor (log2 units) of rows 8 nb + 2 t, 8 nb + 2 t + 1
  {
    const float dq = p.k_descale ? p.k_descale[b * p.k_descale_bs + kvh * p.k_descale_hs] : 1.f;
    const float scale_log2 = p.softmax_scale * dq * kLog2e;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = row0 + nb * 8 + g;
      uint4 raw[C::kChunks][4];
      uint32_t top = 0;                   // largest magnitude's BF16 bits
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          raw[c][u] = make_uint4(0, 0, 0, 0);
          if (row < rows_total) {
            const int qi = row / p.group, head = kvh * p.group + row % p.group;
            raw[c][u] = __ldg(reinterpret_cast<const uint4*>(
                reinterpret_cast<const __nv_bfloat16*>(p.q) + (int64_t)(q_start + qi) * p.q_row_stride +
                (int64_t)head * p.q_head_stride + c * 128 + t * 32 + u * 8));
          }
          const uint32_t w[4] = {raw[c][u].x, raw[c][u].y, raw[c][u].z, raw[c][u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float up, down;
      row_power(top, up, down);
      if (scale_log2 < 0.f) up = -up;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t w[4] = {raw[c][u].x, raw[c][u].y, raw[c][u].z, raw[c][u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            qf[nb][c][2 * u + (i >> 1)][i & 1] =
                pack_f16(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        factor[nb][i] = score_factor(__shfl_sync(0xffffffffu, down, 8 * t + 4 * i) * scale_log2, [&] {
          int lo, hi;
          row_keys(nb * 8 + 2 * t + i, lo, hi);
          return lo < hi;
        });
      }
    }
  }

  float o[C::kChunks * 8][NB][4];
  float m_run[NB][2], l_run[NB][2], neg[NB][2];       // reference, sum, kShift - reference
#pragma unroll
  for (int j = 0; j < C::kChunks * 8; ++j)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][nb][i] = 0.f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m_run[nb][i] = -INFINITY;
      l_run[nb][i] = 0.f;
      neg[nb][i] = kShift;
    }

  int stage = 0;
  for (int it = 0; it < my_tiles; ++it) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
    __syncwarp();                         // every lane's copies are in, and all have left the stage refilled next
    {
      int fill = stage + C::kStages - 1;
      if (fill >= C::kStages) fill -= C::kStages;
      fetch_pages();
      copy_tile(fill);
    }
    const uint8_t* st = ring + stage * C::kStageBytes;
    if (++stage == C::kStages) stage = 0;
    const int tok0 = (tile_lo + warp + it * kWarps) * kTile;

    // ---- S^T = K Q^T ----
    float s[2][NB][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[mt][nb][i] = 0.f;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        uint4 code[2];
        uint32_t scale[2];                // [row g / g + 8]: the scales of the first and second block of 16
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = mt * 16 + h * 8 + g;
          const int chunk = c * 4 + t;
          code[h] = *reinterpret_cast<const uint4*>(st + row * C::kRowBytes +
                                                    (D == 256 ? chunk ^ ((row & 1) << 2) : chunk) * 16);
          scale[h] = e4m3x2_to_f16x2(
              *reinterpret_cast<const uint16_t*>(st + C::kOffKs + row * C::kScaleBytes + c * 8 + 2 * t));
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t lo[4], hi[4];
          e2m1x8_to_f16x2(w == 0 ? code[0].x : w == 1 ? code[0].y : w == 2 ? code[0].z : code[0].w, lo);
          e2m1x8_to_f16x2(w == 0 ? code[1].x : w == 1 ? code[1].y : w == 2 ? code[1].z : code[1].w, hi);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[i] = w < 2 ? hmul2_low(lo[i], scale[0]) : hmul2_high(lo[i], scale[0]);
            hi[i] = w < 2 ? hmul2_low(hi[i], scale[1]) : hmul2_high(hi[i], scale[1]);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              mma_f16_16816(s[mt][nb], lo[2 * half], hi[2 * half], lo[2 * half + 1], hi[2 * half + 1],
                            qf[nb][c][2 * w + half][0], qf[nb][c][2 * w + half][1]);
        }
      }
    }

    // ---- masks, online softmax ----
    const bool need_mask = tok0 < full_lo || tok0 + kTile > full_hi;
    uint32_t pb[2][NB][2];                // P^T fragments
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (need_mask) {
        int lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) row_keys(nb * 8 + 2 * t + i, lo[i], hi[i]);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = g + (i & 2) * 4;
            const int key = tok0 + mt * 16 + (r & 8) + 4 * (r & 1) + ((r & 7) >> 1);
            if (key < lo[i & 1] || key >= hi[i & 1]) s[mt][nb][i] = -INFINITY;
          }
      }
      float mx[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mx[i] = fmaxf(fmaxf(s[0][nb][i], s[0][nb][i + 2]), fmaxf(s[1][nb][i], s[1][nb][i + 2])) * factor[nb][i];
      // The reference of a row moves only when its maximum has grown by more than 2^8 (P then stays below 2^15).
      if (__any_sync(0xffffffffu, mx[0] > m_run[nb][0] + kThreshold || mx[1] > m_run[nb][1] + kThreshold)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = mx[i];
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float m_new = fmaxf(m_run[nb][i], top);
          const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run[nb][i] - m_new);
          m_run[nb][i] = m_new;
          neg[nb][i] = m_new == -INFINITY ? kShift : kShift - m_new;
          l_run[nb][i] *= alpha;
#pragma unroll
          for (int j = 0; j < C::kChunks * 8; ++j) {
            o[j][nb][i] *= alpha;
            o[j][nb][i + 2] *= alpha;
          }
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          unpack2(fma2(pack2(s[mt][nb][i], s[mt][nb][i + 1]), pack2(factor[nb][0], factor[nb][1]),
                       pack2(neg[nb][0], neg[nb][1])), e[i], e[i + 1]);
          e[i] = fast_exp2(e[i]);
          e[i + 1] = fast_exp2(e[i + 1]);
          unpack2(add2(pack2(l_run[nb][0], l_run[nb][1]), pack2(e[i], e[i + 1])), l_run[nb][0], l_run[nb][1]);
        }
        pb[mt][nb][0] = movmatrix_trans(pack_f16(e[0], e[1]));
        pb[mt][nb][1] = movmatrix_trans(pack_f16(e[2], e[3]));
      }
    }

    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        uint2 code[4];
        uint32_t byte[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int token = mt * 16 + 4 * i + t;
          code[i] = *reinterpret_cast<const uint2*>(st + C::kOffV + v_offset<D>(token, c * 4 + (g >> 1)) + (g & 1) * 8);
          byte[i] = st[C::kOffVs + token * C::kScaleBytes + c * 8 + g];
        }
        const uint32_t s01 = e4m3x2_to_f16x2(byte[0] | (byte[1] << 8));
        const uint32_t s23 = e4m3x2_to_f16x2(byte[2] | (byte[3] << 8));
        constexpr uint32_t kLow = 0x0f0f0f0fu;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t x0 = w ? code[0].y : code[0].x, x1 = w ? code[1].y : code[1].x;
          const uint32_t x2 = w ? code[2].y : code[2].x, x3 = w ? code[3].y : code[3].x;
          uint32_t a0[4], a1[4], a2[4], a3[4];
          e2m1x8_to_f16x2((x0 & kLow) | ((x1 << 4) & ~kLow), a0);     // even dimensions of tokens 2 t, 2 t + 1
          e2m1x8_to_f16x2(((x0 >> 4) & kLow) | (x1 & ~kLow), a1);     // odd dimensions
          e2m1x8_to_f16x2((x2 & kLow) | ((x3 << 4) & ~kLow), a2);
          e2m1x8_to_f16x2(((x2 >> 4) & kLow) | (x3 & ~kLow), a3);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t f0 = hmul2_u32(a0[j], s01), f1 = hmul2_u32(a1[j], s01);
            const uint32_t f2 = hmul2_u32(a2[j], s23), f3 = hmul2_u32(a3[j], s23);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              mma_f16_16816(o[c * 8 + 4 * w + j][nb], f0, f1, f2, f3, pb[mt][nb][0], pb[mt][nb][1]);
          }
        }
      }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // ---- merge of the warps' states ----
  float* const merge = reinterpret_cast<float*>(smem);                 // [warp][row][kMergePitch], over the rings
  float* const s_m = reinterpret_cast<float*>(smem + C::kOffState);   // [warp][row]
  float* const s_l = s_m + kWarps * C::kRows;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float l = l_run[nb][i];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      if (g == 0) {
        s_m[warp * C::kRows + nb * 8 + 2 * t + i] = m_run[nb][i];
        s_l[warp * C::kRows + nb * 8 + 2 * t + i] = l;
      }
    }
  __syncthreads();                                                     // also: every warp is done with its ring
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = nb * 8 + 2 * t + i;
      float m = s_m[r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w * C::kRows + r]);
      const float resc = m == -INFINITY ? 0.f : fast_exp2(m_run[nb][i] - m);
      float* dst = merge + (warp * C::kRows + r) * C::kMergePitch;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float2*>(dst + c * 128 + 16 * g + 2 * j) =
              make_float2(o[c * 8 + j][nb][i] * resc, o[c * 8 + j][nb][i + 2] * resc);
    }
  __syncthreads();

  // ---- join the warps, and the splits of a cluster; normalise and store, four dimensions a thread ----
  const float dv = p.v_descale ? p.v_descale[b * p.v_descale_bs + kvh * p.v_descale_hs] : 1.f;
  constexpr int kCells = C::kRows * (D / 4);
  // The state of this CTA for row r, dimensions d .. d + 3: O relative to the maximum m, the sum l.
  auto join_warps = [&](int r, int d, float& m, float& l, float4& acc) {
    m = -INFINITY;
    l = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_m[w * C::kRows + r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = s_m[w * C::kRows + r];
      // without a maximum the sum is 0, or NaN where the query is
      l += s_l[w * C::kRows + r] * (mw == -INFINITY ? 1.f : fast_exp2(mw - m));
      const float4 part = *reinterpret_cast<const float4*>(merge + (w * C::kRows + r) * C::kMergePitch + d);
      acc.x += part.x;
      acc.y += part.y;
      acc.z += part.z;
      acc.w += part.w;
    }
  };
  auto finish = [&](int r, int d, float m, float l, float4 acc) {
    const int row = row0 + r;
    const int hd = kvh * p.group + row % p.group;
    const int64_t q_row = q_start + row / p.group;
    float sink = -INFINITY;
    if (p.sink != nullptr && !part_mode) sink = __bfloat162float(p.sink[hd]) * kLog2e;
    const float m_all = fmaxf(m, sink);
    const float m_use = m_all == -INFINITY ? 0.f : m_all;
    const float resc = fast_exp2(m - m_use);
    l *= resc;
    if (sink != -INFINITY) l += fast_exp2(sink - m_use + kShift);
    const float inv = l == 0.f ? 0.f : dv * resc / l;
    acc.x *= inv;
    acc.y *= inv;
    acc.z *= inv;
    acc.w *= inv;
    const float lse = l == 0.f ? -INFINITY : m_use + log2f(l) - kShift;
    if (part_mode) {
      const int64_t slot = ((int64_t)split * p.total_q + q_row) * p.num_q_heads + hd;
      *reinterpret_cast<float4*>(p.part_o + slot * D + d) = acc;
      if (d == 0) p.part_lse[slot] = lse;
    } else {
      uint2 v;
      v.x = pack_bf16(acc.x, acc.y);
      v.y = pack_bf16(acc.z, acc.w);
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + q_row * p.out_row_stride +
                                (int64_t)hd * p.out_head_stride + d) = v;
      if (d == 0 && p.lse != nullptr) p.lse[(int64_t)hd * p.total_q + q_row] = lse * kLn2;
    }
  };
  if (!pp.cluster) {
    for (int idx = threadIdx.x; idx < kCells; idx += kWarps * 32) {
      const int r = idx / (D / 4), d = (idx % (D / 4)) * 4;
      if (row0 + r >= rows_total) continue;
      float m, l;
      float4 acc;
      join_warps(r, d, m, l, acc);
      finish(r, d, m, l, acc);
    }
    return;
  }
  // The splits are the CTAs of one cluster: each leaves its joined state in its own shared memory (O over warp 0's
  // part), and after a cluster barrier every CTA takes a share of the outputs and reads all states.
  float* const cta_m = s_l + kWarps * C::kRows;
  float* const cta_l = cta_m + C::kRows;
  for (int idx = threadIdx.x; idx < kCells; idx += kWarps * 32) {
    const int r = idx / (D / 4), d = (idx % (D / 4)) * 4;
    float m, l;
    float4 acc;
    join_warps(r, d, m, l, acc);
    *reinterpret_cast<float4*>(merge + r * C::kMergePitch + d) = acc;
    if (d == 0) {
      cta_m[r] = m;
      cta_l[r] = l;
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int idx = split * kWarps * 32 + threadIdx.x; idx < kCells; idx += p.num_splits * kWarps * 32) {
    const int r = idx / (D / 4), d = (idx % (D / 4)) * 4;
    if (row0 + r >= rows_total) continue;
    float ms[kMaxCluster], m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) {
      ms[s] = s < p.num_splits ? *cluster.map_shared_rank(cta_m + r, s) : -INFINITY;
      m = fmaxf(m, ms[s]);
    }
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) {
      if (s >= p.num_splits) continue;
      const float w = ms[s] == -INFINITY ? 1.f : fast_exp2(ms[s] - m);      // 1: of zeros, or of a NaN query's NaN
      l += w * *cluster.map_shared_rank(cta_l + r, s);
      const float4 part = *reinterpret_cast<const float4*>(cluster.map_shared_rank(merge + r * C::kMergePitch + d, s));
      acc.x += w * part.x;
      acc.y += w * part.y;
      acc.z += w * part.z;
      acc.w += w * part.w;
    }
    finish(r, d, m, l, acc);
  }
  cluster.sync();                                                      // the others may still read this CTA's state
}

}  // namespace

int kv4_decode_resident(int head_dim) { return head_dim == 128 ? 3 : 2; }   // by registers

int kv4_decode_max_cluster() { return kMaxCluster; }
int kv4_decode_rows(int head_dim, int packed_rows) { return head_dim == 128 && packed_rows > 8 ? 16 : 8; }

#define ATREX_KV4_DECODE_VARIANTS(X) X(128, 1) X(128, 2) X(256, 1)

cudaError_t kv4_decode_prepare() {
  cudaError_t e;
#define X(D, NB)                                                                                                     \
  if ((e = cudaFuncSetAttribute(atrex_sm100_kv4_decode_kernel<D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                                DecodeCfg<D, NB>::kSmemBytes)) != cudaSuccess)                                     \
    return e;
  ATREX_KV4_DECODE_VARIANTS(X)
#undef X
  return cudaSuccess;
}

cudaError_t kv4_decode_launch(const Kv4Params& p, int head_dim, int rows, cudaStream_t stream) {
  // below 2^31: checked by the launcher
  const dim3 grid((unsigned)((long long)p.row_tiles * p.f.num_splits * p.f.num_kv_heads * p.f.batch));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  if (p.cluster) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.f.num_splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
  }
#define X(D, NB)                                                            \
  if (head_dim == D && rows == 8 * NB) {                                    \
    cfg.dynamicSmemBytes = DecodeCfg<D, NB>::kSmemBytes;                    \
    return cudaLaunchKernelEx(&cfg, atrex_sm100_kv4_decode_kernel<D, NB>, p); \
  }
  ATREX_KV4_DECODE_VARIANTS(X)
#undef X
  return cudaErrorInvalidValue;
}

}  // namespace atrex_sm100
