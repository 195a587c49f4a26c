// Attention over a 4-bit paged cache on tcgen05 tensor cores: prompts, chunks of prompts, wide verification steps.
//
// A work item is 128 packed GQA rows of one (request, KV head), optionally one KV split of them (fa_items.cuh).  The
// tensor-core side is that of the single-tile kernel (fa_umma1.cu): S0 | S1 | O in TMEM, Q K^T of the next tile issued
// while the softmax warps (two threads per row) work on this one, P read from TMEM.  What differs:
//
//   * both products are FP16: an E2M1 value times its E4M3 scale is exact in FP16 (fp4.cuh), P is stored as 2^7 p, and
//     a query row is brought into FP16's range by a power of two of its own, which rides in the row's score factor;
//   * warp 9 resolves work items one ahead into shared memory;
//   * warps 10 and 11 are the producers: codes by TMA, one box per page part of a tile; scales by cp.async, a row a lane,
//     those of keys that no row of the item sees become zeros (their codes may be anything, all codes are finite);
//   * warps 12-15 widen: a lane takes 128 values of one row of every K and V tile from the staging ring into the
//     128-byte-swizzled operand tile.  At the start of an item they bring its Q rows in, 32 each;
//   * Q lies in TMEM too (64 or 128 columns) and is the A operand from there, so that Q K^T reads only K from shared
//     memory, and the next item's Q rows may be prepared there meanwhile (verify, below: 111 -> 109 us).
//
// Measured: 64 requests x 4 query tokens, window 4 095, 64 / 4 heads of 128: 109 us (23 for the bytes); 16 requests of
// 1 .. 96 query tokens, 24 / 2 heads of 256, contexts of 97 .. 8 192: 158 us (33).  A tile of 128 rows by 128 keys takes
// ~2 550 cycles there (in long prompts 3 400, where the two-tile kernel takes 2 350), and three chains in it are about
// equally long: widening (two units of ~1 170 cycles on four warps), the softmax threads (half of a row each: load,
// exchange, exponentials, hand-over) and at head_dim 256 the tensor pipe (20 MMAs, ~88 cycles each).  Shortening one alone
// gained nothing: eight widening warps beside four softmax warps 109 -> 120 and 158 -> 164 us; pairs of warps per row piece
// 109 -> 124; the next unit's codes in registers early 109 -> 112; polynomial exponentials 109 -> 117; 128-key tiles at
// head_dim 256 155 -> 179.
//
// Every wait is bounded; on expiry the CTA records a code, drains its copies, frees TMEM and returns.
#define ATREX_MBAR_SPIN_INLINE   // setmaxnreg: no calls with their own register ABI
#include "fa_items.cuh"
#include "fp4.cuh"
#include "kv4_kernels.cuh"
#include "kv4_q.cuh"
#include "softmax_math.cuh"
#include "umma.cuh"

namespace atrex_sm100 {

namespace {

constexpr int kRing = 4;                              // operand ring slots of 32 KB
constexpr int kSoftmaxWarps = 8;                      // two threads per row
constexpr int kWidenWarps = 4;
constexpr int kThreads = 512;
// 512 threads launch with 128 registers each; 2 x 128 x (152 + 96) = 63 488 of the 65 536 leaves slack.
constexpr int kSoftmaxRegs = 152, kOtherRegs = 96;

template <int D>
struct Cfg {
  static constexpr int kSlotBytes = 32768;
  static constexpr int kRowBytes = D * 2;
  static constexpr int kBN = kSlotBytes / kRowBytes;          // keys per tile: 128 / 64
  static constexpr uint32_t kTmemCols = 512;
  static constexpr int kNKB = kRowBytes / 128;                // 128-byte column blocks per row
  static constexpr int kQBytes = kRows * kRowBytes;
  static constexpr int kQBlock = kRows * 128;
  static constexpr int kKVBlock = kBN * 128;
  static constexpr int kKStepsQK = kNKB * 4;
  static constexpr int kKStepsPV = kBN / 16;
  static constexpr int kPVStepBytes = 16 * 128;
  static constexpr float kThreshold = 8.f;                    // lazy-rescale threshold (log2 units)
  static constexpr float kShift = 7.f;                        // P is stored as 2^shift * p: at most 2^15
  // staging: a tile's codes (rows of D / 2 bytes, swizzled by TMA over that width), then its scales
  static constexpr int kCodeRow = D / 2, kScaleRow = D / 16;
  static constexpr int kCodeBytes = kBN * kCodeRow, kStageBytes = kCodeBytes + kBN * kScaleRow;
  static constexpr int kStages = D == 128 ? 6 : 3;
  static constexpr int kPieceRows = kBN / kWidenWarps;        // rows per widening warp and tile: 32 / 16
  static constexpr int kOffKV = kQBytes;                      // in front: where Q rows turn into TMEM lanes
  static constexpr int kOffStage = kOffKV + kRing * kSlotBytes;
  static constexpr int kOffXchg = kOffStage + kStages * kStageBytes;   // [parity][half][row] floats: row max / sum
  static constexpr int kOffFactor = kOffXchg + 2 * 2 * kRows * 4;      // [item parity][row] score factors
  static constexpr int kOffItem = kOffFactor + 2 * kRows * 4;
  static constexpr int kOffBar = kOffItem + 2 * 80;
  static constexpr uint32_t kQCol = 2 * kBN + D;              // TMEM columns: S0 | S1 | O | Q
  static_assert(kQCol + D / 2 <= 512, "S0 | S1 | O | Q must fit the 512 TMEM columns");
};
constexpr int kMaxStages = 6;
enum Bar { bQFull = 0, bQEmpty, bOFull, bOFinal, bItemFull, bItemEmpty = bItemFull + 2, bRowsFull = bItemEmpty + 2,
           bKVFull = bRowsFull + 2, bKVEmpty = bKVFull + kRing, bSFull = bKVEmpty + kRing, bPFull = bSFull + 2,
           bStageFull = bPFull + 2, bStageEmpty = bStageFull + kMaxStages, bCount = bStageEmpty + kMaxStages };
template <int D>
constexpr int smem_bytes() {
  return Cfg<D>::kOffBar + bCount * 8 + 16;
}
static_assert(smem_bytes<128>() <= 232448 && smem_bytes<256>() <= 232448, "shared memory of one CTA");

struct __align__(16) ItemSlot {
  Item256 it;
  int valid, kv_begin, kv_end;     // keys that some row of the item sees
  float scale_log2, dv;
  int pad[2];
};
static_assert(sizeof(ItemSlot) == 80, "five 16-byte vectors");

// One tile of keys for half a row, as in fa_umma1.cu: step 1 loads the thread's scores from TMEM, masks them and
// returns their (unscaled) maximum.
template <int D, bool kMask>
__device__ __forceinline__ float half_max(uint32_t s_tmem, uint32_t (&s)[Cfg<D>::kBN / 2], int col0, int vis_lo, int vis_hi) {
  constexpr int N = Cfg<D>::kBN / 2;
#pragma unroll
  for (int c = 0; c < N / 32; ++c) tmem_ld32(s_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
  tmem_ld_wait();
  if (kMask) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int col = col0 + i;
      if (col < vis_lo || col >= vis_hi) s[i] = 0xff800000u;  // -inf
    }
  }
  float mxv[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    mxv[0] = fmax3(mxv[0], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    mxv[1] = fmax3(mxv[1], __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
    mxv[2] = fmax3(mxv[2], __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
    mxv[3] = fmax3(mxv[3], __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
  }
  return fmaxf(fmaxf(mxv[0], mxv[1]), fmaxf(mxv[2], mxv[3]));
}

// Step 2: P = 2^(s * scale + neg_m) as FP16 pairs over the first columns of the thread's own score columns.
template <int D>
__device__ __forceinline__ float half_exp(uint32_t s_tmem, const uint32_t (&s)[Cfg<D>::kBN / 2], float scale_log2,
                                          float neg_m) {
  constexpr int N = Cfg<D>::kBN / 2;
  const f32x2 scale2 = pack2(scale_log2, scale_log2), negm2 = pack2(neg_m, neg_m);
  f32x2 sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
  for (int c = 0; c < N / 32; ++c) {
    uint32_t packed[16];
    exp32_f16(&s[c * 32], scale2, negm2, sum2, packed);
    tmem_st16(s_tmem + c * 16, packed);
  }
  return sum_of(sum2);
}

// A lane's piece: 128 values of one row of a staged tile into the operand tile, 16 bytes (8 values) at a time.
template <int D>
__device__ __forceinline__ void widen_piece(const uint8_t* stage, uint8_t* tile, int lane, int row_lo) {
  using C = Cfg<D>;
  const int row = row_lo + lane % C::kPieceRows, half = lane / C::kPieceRows;
  const uint8_t* codes = stage + row * C::kCodeRow;
  const int swizzle = D == 128 ? (row >> 1) & 3 : row & 7;
  const uint2 sc = *reinterpret_cast<const uint2*>(stage + C::kCodeBytes + row * C::kScaleRow + half * 8);
  uint8_t* dst = tile + (2 * half) * C::kKVBlock;
#pragma unroll
  for (int chunk = 0; chunk < 4; ++chunk) {                  // 32 values, two scales
    const uint4 raw = *reinterpret_cast<const uint4*>(codes + (((half * 4 + chunk) ^ swizzle) << 4));
    const uint32_t two = e4m3x2_to_f16x2(chunk < 2 ? sc.x >> (16 * chunk) : sc.y >> (16 * (chunk - 2)));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t f[4];
      e2m1x8_to_f16x2(w == 0 ? raw.x : w == 1 ? raw.y : w == 2 ? raw.z : raw.w, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = w < 2 ? hmul2_low(f[i], two) : hmul2_high(f[i], two);
      *reinterpret_cast<uint4*>(dst + (chunk >> 1) * C::kKVBlock + swz128(row, (chunk & 1) * 4 + w)) =
          make_uint4(f[0], f[1], f[2], f[3]);
    }
  }
}

// A bounded wait of a whole warp, which goes on or gives up as one: the TMEM accesses and warp barriers behind a wait need
// all of its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
// On expiry one lane reports and the warp leaves its loop.
#define KV4_WAIT_OR_BREAK(bar_ptr, parity, code)                  \
  if (!warp_wait((bar_ptr), (parity))) {                          \
    if (lane == 0) {                                              \
      if (p.status) atomicExch(p.status, (code));                 \
      atomicExch(abort_flag, 1);                                  \
    }                                                             \
    break;                                                        \
  }

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
atrex_sm100_kv4_prefill_kernel(const __grid_constant__ Kv4Params pp) {
  using C = Cfg<D>;
  constexpr int BN = C::kBN;
  const FwdParams& p = pp.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* q_smem = smem;
  uint8_t* kv_smem = smem + C::kOffKV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  ItemSlot* slots = reinterpret_cast<ItemSlot*>(smem + C::kOffItem);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + bCount);
  int* abort_flag = reinterpret_cast<int*>(bars + bCount + 1);
  float* row_factor = reinterpret_cast<float*>(smem + C::kOffFactor);

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  if ((smem_u32(smem) & 1023u) != 0u) {
    if (tid == 0 && p.status) atomicExch(p.status, kBadSmemAlignment);
    return;
  }
  if (tid == 0) {
    *abort_flag = 0;
    mbar_init(&bars[bQFull], kWidenWarps);
    mbar_init(&bars[bQEmpty], 1);
    mbar_init(&bars[bOFull], 1);
    mbar_init(&bars[bOFinal], 1);
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&bars[bKVFull + s], kWidenWarps);
      mbar_init(&bars[bKVEmpty + s], 1);
    }
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars[bStageFull + s], 64);          // 32 lanes with TMA bytes, 32 with scale copies
      mbar_init(&bars[bStageEmpty + s], kWidenWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars[bSFull + b], 1);
      mbar_init(&bars[bPFull + b], 2 * kRows);
      mbar_init(&bars[bItemFull + b], 1);
      mbar_init(&bars[bItemEmpty + b], kSoftmaxWarps + kWidenWarps + 3);   // and issuer, producers
      mbar_init(&bars[bRowsFull + b], kWidenWarps);
    }
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t o_col = 2 * BN;
  const int step = gridDim.x;

  if (warp >= 12) {
    // ------------------------------- widening -------------------------------
    setmaxnreg_dec<kOtherRegs>();
    const int row_lo = (warp - 12) * C::kPieceRows;
    for (uint32_t n_item = 0, done = 0;; ++n_item) {
      // the items only say how many tiles there are: K and V of each, in order
      KV4_WAIT_OR_BREAK(&bars[bItemFull + (n_item & 1u)], (n_item >> 1) & 1u, kWaitFullTimeout)
      const int valid = slots[n_item & 1u].valid, n_tiles = slots[n_item & 1u].it.n_tiles;
      __syncwarp();
      if (!valid) {
        if (lane == 0) mbar_arrive(&bars[bRowsFull + (n_item & 1u)]);    // the softmax warps read the slot behind it
        break;
      }
      {
        using Q = QRows<D, kRows / kWidenWarps, 8>;
        const ItemSlot& slot = slots[n_item & 1u];
        const int first = (warp - 12) * (kRows / kWidenWarps);
        const bool flip = slot.scale_log2 < 0.f;
        Q rows(p, first, slot.it.row0, slot.it.rows_total, slot.it.q_start, slot.it.kvh * p.group);
        rows.fetch();
        for (int k = 0; k < Q::kSteps; k += 8) {
          rows.store(q_smem, 0, C::kQBlock, row_factor + (n_item & 1u) * kRows, first + k * Q::kRpi, flip);
          if (k + 8 < Q::kSteps) rows.fetch();
        }
        __syncwarp();
        // Q's columns are free from the last Q K^T of the item before; a lane moves its own row
        if (n_item > 0) KV4_WAIT_OR_BREAK(&bars[bQEmpty], (n_item - 1u) & 1u, kWaitEmptyTimeout)
        __syncwarp();
        tcgen05_fence_after();
        const int r = first + lane;
#pragma unroll
        for (int kb = 0; kb < C::kNKB; ++kb) {
          uint32_t x[32];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(&x[4 * c]) = *reinterpret_cast<const uint4*>(q_smem + kb * C::kQBlock + swz128(r, c));
          tmem_st32(tmem_base + ((uint32_t)first << 16) + C::kQCol + kb * 32, x);
        }
        tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
      }
      if (lane == 0) {
        mbar_arrive(&bars[bQFull]);
        mbar_arrive(&bars[bRowsFull + (n_item & 1u)]);    // release: the row factors are written
        mbar_arrive(&bars[bItemEmpty + (n_item & 1u)]);
      }
      bool dead = false;
      for (int i = 0; i < 2 * n_tiles; ++i, ++done) {
        const uint32_t stage = done % C::kStages, slot = done % kRing;
        dead = true;
        KV4_WAIT_OR_BREAK(&bars[bStageFull + stage], (done / C::kStages) & 1u, kWaitFullTimeout)
        if (done >= (uint32_t)kRing) KV4_WAIT_OR_BREAK(&bars[bKVEmpty + slot], ((done / kRing) - 1u) & 1u, kWaitEmptyTimeout)
        dead = false;
        widen_piece<D>(smem + C::kOffStage + stage * C::kStageBytes, kv_smem + slot * C::kSlotBytes, lane, row_lo);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars[bKVFull + slot]);
          mbar_arrive(&bars[bStageEmpty + stage]);
        }
      }
      if (dead) break;
    }
    __syncwarp();
  } else if (warp >= 8) {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == 9) {
      // ------------------------------- items, one ahead -------------------------------
      if (lane == 0) {
        uint32_t n = 0;
        for (int item = blockIdx.x;; item += step, ++n) {
          ItemSlot* slot = slots + (n & 1u);
          if (n >= 2 && !mbar_wait(&bars[bItemEmpty + (n & 1u)], ((n >> 1) - 1u) & 1u)) {
            if (p.status) atomicExch(p.status, kWaitEmptyTimeout);
            atomicExch(abort_flag, 1);
            break;
          }
          const bool ok = decode_item256<BN>(p, item, slot->it) && *(volatile int*)abort_flag == 0;
          float dk = 1.f, dv = 1.f;
          if (ok) {
            const Item256& it = slot->it;
            const int qi_lo = it.row0 / p.group, qi_hi = min(it.q_len - 1, (it.row0 + kRows - 1) / p.group);
            slot->kv_end = p.window_right >= 0 ? min(it.kv_len, right_bound(p, qi_hi + it.off)) : it.kv_len;
            slot->kv_begin = p.window_left >= 0 ? max(0, qi_lo + it.off - p.window_left) : 0;
            if (p.k_descale) dk = p.k_descale[it.b * p.k_descale_bs + it.kvh * p.k_descale_hs];
            if (p.v_descale) dv = p.v_descale[it.b * p.v_descale_bs + it.kvh * p.v_descale_hs];
          }
          slot->valid = ok ? 1 : 0;
          slot->scale_log2 = p.softmax_scale * dk * kLog2e;
          slot->dv = dv;
          mbar_arrive(&bars[bItemFull + (n & 1u)]);      // release: the slot is written
          if (!ok) break;
        }
      }
      __syncwarp();
    } else if (warp >= 10) {
      // ------------------------------- producers -------------------------------
      constexpr int kPer = BN / 32;                    // rows of a tile per lane
      // Both walk every stage in order: a barrier's parity says which of two neighbouring phases is meant, so a warp
      // that skipped a stage's phases (K tiles or V tiles only, over an odd ring) would take an old one for its own.
      const bool codes = warp == 10;
      const int shift = (p.page_size & (p.page_size - 1)) == 0 ? __ffs(p.page_size) - 1 : -1;
      const int box_rows = p.box_rows;
      uint32_t n = 0;                                  // tiles of the run: K even, V odd
      for (uint32_t n_item = 0;; ++n_item) {
        KV4_WAIT_OR_BREAK(&bars[bItemFull + (n_item & 1u)], (n_item >> 1) & 1u, kWaitFullTimeout)
        const ItemSlot& slot = slots[n_item & 1u];
        if (!slot.valid) break;
        const int kv_begin = slot.kv_begin, kv_end = slot.kv_end, n_tiles = slot.it.n_tiles, kvh = slot.it.kvh;
        int tok0 = slot.it.tile_lo * BN;
        const int32_t* table = p.block_table + (int64_t)slot.it.b * p.block_table_row_stride;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[bItemEmpty + (n_item & 1u)]);
        const uint8_t* ks = pp.ks + kvh * pp.ks_str.head;
        const uint8_t* vs = pp.vs + kvh * pp.vs_str.head;
        // table entries of the rows lane, lane + 32, ... of a tile, as read: nothing looks at them before the next tile
        int page[kPer], next[kPer];
        auto fetch = [&](int t0, int (&out)[kPer]) {
#pragma unroll
          for (int u = 0; u < kPer; ++u) {
            const int t = t0 + u * 32 + lane;
            out[u] = t < kv_end ? table[shift >= 0 ? t >> shift : t / p.page_size] : -1;
          }
        };
        fetch(tok0, page);
        bool dead = false;
        for (int j = 0; j < n_tiles; ++j, tok0 += BN) {
          if (j + 1 < n_tiles) fetch(tok0 + BN, next);
#pragma unroll
          for (int u = 0; u < kPer; ++u)
            if (page[u] >= p.num_pages) page[u] = -1;
          for (int v = 0; v < 2; ++v, ++n) {
            const uint32_t stage = n % C::kStages;
            dead = true;
            if (n >= (uint32_t)C::kStages) KV4_WAIT_OR_BREAK(&bars[bStageEmpty + stage], ((n / C::kStages) - 1u) & 1u, kWaitEmptyTimeout)
            dead = false;
            uint8_t* dst = smem + C::kOffStage + stage * C::kStageBytes;
            uint64_t* full = &bars[bStageFull + stage];
            if (codes) {
              uint32_t bytes = 0;
#pragma unroll
              for (int u = 0; u < kPer; ++u)
                if (((u * 32 + lane) & (box_rows - 1)) == 0 && page[u] >= 0) bytes += box_rows * C::kCodeRow;
              mbar_arrive_expect_tx(full, bytes);
#pragma unroll
              for (int u = 0; u < kPer; ++u) {
                const int r = u * 32 + lane, t = tok0 + r;
                if ((r & (box_rows - 1)) == 0 && page[u] >= 0)
                  tma_load_kv(dst + r * C::kCodeRow, v ? &p.v_map : &p.k_map, full, 0, kvh,
                              shift >= 0 ? t & (p.page_size - 1) : t % p.page_size, page[u], v ? p.v_perm : p.k_perm);
              }
            } else {
              const CacheStrides& st = v ? pp.vs_str : pp.ks_str;
              const uint8_t* scales = v ? vs : ks;
#pragma unroll
              for (int u = 0; u < kPer; ++u) {
                const int r = u * 32 + lane, t = tok0 + r;
                const uint32_t in_page = shift >= 0 ? t & (p.page_size - 1) : t % p.page_size;
                const bool ok = page[u] >= 0 && t >= kv_begin;
                const uint8_t* src = scales + (uint64_t)(uint32_t)max(page[u], 0) * st.page + (uint64_t)in_page * st.row;
                const uint32_t to = smem_u32(dst + C::kCodeBytes + r * C::kScaleRow);
                if (C::kScaleRow == 8)
                  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(src), "r"(ok ? 8u : 0u) : "memory");
                else
                  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(ok ? 16u : 0u) : "memory");
              }
              asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
            }
            __syncwarp();
          }
          if (dead) break;
#pragma unroll
          for (int u = 0; u < kPer; ++u) page[u] = next[u];
        }
        if (dead) break;
      }
      // every copy must have landed before the CTA may exit
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (uint32_t back = 1; back <= (uint32_t)C::kStages && back <= n; ++back) {
        const uint32_t i = n - back;
        mbar_wait(&bars[bStageFull + i % C::kStages], (i / C::kStages) & 1u);
      }
      __syncwarp();
    } else if (warp == 8) {
    // ------------------------------- MMA issuer -------------------------------
    constexpr uint32_t kIdescQK = umma_idesc(kRows, BN, 0, 0, 0, 0);      // FP16 operands
    constexpr uint32_t kIdescPV = umma_idesc(kRows, D, 0, 0, 0, 1);
    const UmmaDesc k_desc0 = umma_desc_split(umma_desc_sw128(smem_u32(kv_smem), 16, 1024));
    const UmmaDesc v_desc0 = umma_desc_split(umma_desc_sw128(smem_u32(kv_smem), C::kKVBlock, 1024));
    uint32_t it_count = 0, base = 0, cp[2] = {0, 0};   // tile t of the CTA's run has K number 2t and V number 2t + 1
    bool dead = false;
    const uint32_t lead = lane == 0;
    auto issue_qk = [&](int buf, uint32_t slot) {
      const UmmaDesc kd = k_desc0 + (uint32_t)((slot * C::kSlotBytes) >> 4);
#pragma unroll
      for (int ks = 0; ks < C::kKStepsQK; ++ks) {
        const uint32_t koff = ((ks >> 2) * C::kKVBlock + (ks & 3) * 32) >> 4;
        umma_ts_f16_lead(lead, tmem_base + buf * BN, tmem_base + C::kQCol + ks * 8, kd + koff, kIdescQK, ks > 0);
      }
      umma_commit_lead(lead, &bars[bSFull + buf]);
      umma_commit_lead(lead, &bars[bKVEmpty + slot]);
    };
    while (!dead) {
      if (!warp_wait(&bars[bItemFull + (it_count & 1u)], (it_count >> 1) & 1u)) { dead = true; break; }
      const int valid = slots[it_count & 1u].valid, n_tiles = slots[it_count & 1u].it.n_tiles;
      __syncwarp();
      if (!valid) break;
      if (lane == 0) mbar_arrive(&bars[bItemEmpty + (it_count & 1u)]);
      if (!warp_wait(&bars[bQFull], it_count & 1u)) { dead = true; break; }
      tcgen05_fence_after();
      if (n_tiles == 0) {
        if (lane == 0) mbar_arrive(&bars[bQEmpty]);
        ++it_count;
        continue;
      }
      {
        const uint32_t slot_k = base % kRing;   // K(0)
        if (!warp_wait(&bars[bKVFull + slot_k], (base / kRing) & 1u)) { dead = true; break; }
        tcgen05_fence_after();
        issue_qk(0, slot_k);
        if (n_tiles == 1) umma_commit_lead(lead, &bars[bQEmpty]);   // Q is last read by the item's last Q K^T
      }
      for (int j = 0; j < n_tiles && !dead; ++j) {
        const uint32_t n_v = base + 2 * j + 1;   // V(j)
        if (j + 1 < n_tiles) {
          const uint32_t n_k = base + 2 * j + 2; // K(j+1)
          const uint32_t slot_k = n_k % kRing;
          if (!mbar_wait(&bars[bKVFull + slot_k], (n_k / kRing) & 1u)) { dead = true; break; }
          tcgen05_fence_after();
          issue_qk((j + 1) & 1, slot_k);         // its S buffer held P(j-1), consumed by the earlier P V
          if (j + 2 == n_tiles) umma_commit_lead(lead, &bars[bQEmpty]);
        }
        const uint32_t slot_v = n_v % kRing;
        if (!mbar_wait(&bars[bKVFull + slot_v], (n_v / kRing) & 1u)) { dead = true; break; }
        const int buf = j & 1;
        if (!mbar_wait(&bars[bPFull + buf], cp[buf] & 1u)) { dead = true; break; }
        ++cp[buf];
        tcgen05_fence_after();
        const UmmaDesc vd = v_desc0 + (uint32_t)((slot_v * C::kSlotBytes) >> 4);
#pragma unroll
        for (int ks = 0; ks < C::kKStepsPV; ++ks) {
          const uint32_t voff = (ks * C::kPVStepBytes) >> 4;
          // P of key half h sits over the first columns of that half's own score columns
          constexpr int kPerHalf = C::kKStepsPV / 2;
          const uint32_t pcol = buf * BN + (ks / kPerHalf) * (BN / 2) + (ks % kPerHalf) * 8;
          umma_ts_f16_lead(lead, tmem_base + o_col, tmem_base + pcol, vd + voff, kIdescPV, (j > 0) | (ks > 0));
        }
        umma_commit_lead(lead, &bars[bOFull]);
        if (j + 1 == n_tiles) umma_commit_lead(lead, &bars[bOFinal]);   // one phase per item with tiles: O is final
        umma_commit_lead(lead, &bars[bKVEmpty + slot_v]);
      }
      dead = __any_sync(0xffffffffu, dead);    // the lanes meet again: without a vote at each of the waits above
      if (dead) break;
      base += 2u * (uint32_t)n_tiles;
      ++it_count;
    }
    if (dead && lane == 0) {
      if (p.status) atomicExch(p.status, kWaitMmaTimeout);
      atomicExch(abort_flag, 1);
    }
    __syncwarp();
    }
  } else {
    // ------------- softmax warps: two threads per row, half of each tile's key columns each -------------
    setmaxnreg_inc<kSoftmaxRegs>();
    constexpr int N = BN / 2;                              // key columns per thread and tile
    const int h = warp >> 2;                               // which half of the key columns
    const int r = (warp & 3) * 32 + lane;                  // row = TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_tmem = tmem_base + lane_off + o_col + h * (D / 2);   // this thread's half of the O columns
    float* xchg = reinterpret_cast<float*>(smem + C::kOffXchg);            // [parity][half][row]
    constexpr int kGroupBar = 1, kGroup = kSoftmaxWarps * 32;
    uint32_t cs[2] = {0, 0}, co = 0, it_count = 0, cx = 0, n_final = 0;
    bool dead = false;
    for (; !dead; ++it_count) {
      const ItemSlot* item_slot = slots + (it_count & 1u);
      const bool got = mbar_wait(&bars[bRowsFull + (it_count & 1u)], (it_count >> 1) & 1u);
      // The slot stays this item's until the end of the epilogue, which reads the item again.
      Item256 it;
      bool valid = false;
      float scale_log2 = 0.f;
      if (got) {
        it = item_slot->it;
        valid = item_slot->valid != 0;
        scale_log2 = item_slot->scale_log2 * row_factor[(it_count & 1u) * kRows + r];
      }
      // leave together: no more items, an abort seen by the item warp, or a wait that expired in one thread
      if (group_barrier_or(kGroupBar, kGroup, !got || !valid || *(volatile int*)abort_flag != 0)) {
        if (!got) {
          if (p.status) atomicExch(p.status, kWaitFullTimeout);
          atomicExch(abort_flag, 1);
        }
        break;
      }
      const int qi = min((it.row0 + r) / p.group, max(it.q_len - 1, 0));
      const int vis_hi = p.window_right >= 0 ? min(it.kv_len, right_bound(p, qi + it.off)) : it.kv_len;
      const int vis_lo = p.window_left >= 0 ? max(0, qi + it.off - p.window_left) : 0;
      scale_log2 = score_factor(scale_log2, [&] { return vis_lo < vis_hi; });
      const int sqi_lo = it.row0 / p.group;
      const int sqi_hi = min(it.q_len - 1, (it.row0 + kRows - 1) / p.group);
      const int full_lo = p.window_left >= 0 ? max(0, sqi_hi + it.off - p.window_left) : 0;
      const int full_hi = p.window_right >= 0 ? min(it.kv_len, right_bound(p, sqi_lo + it.off)) : it.kv_len;
      float m_run = -INFINITY, l_run = 0.f;   // l_run: this thread's half of the row sum, in units of 2^kShift
      const int n_tiles = it.n_tiles, tile_lo = it.tile_lo;
      for (int j = 0; j < n_tiles; ++j) {
        const int buf = j & 1;
        const uint32_t s_tmem = tmem_base + lane_off + buf * BN + h * N;   // own scores; P goes over them
        const int tok0 = (tile_lo + j) * BN;
        const bool need_mask = tok0 < full_lo || tok0 + BN > full_hi;
        if (!warp_wait(&bars[bSFull + buf], cs[buf] & 1u)) dead = true;
        ++cs[buf];
        tcgen05_fence_after();
        uint32_t s[N];
        float mx = -INFINITY;
        if (!dead)
          mx = need_mask ? half_max<D, true>(s_tmem, s, tok0 + h * N, vis_lo, vis_hi)
                         : half_max<D, false>(s_tmem, s, tok0 + h * N, vis_lo, vis_hi);
        // row maximum = max of the two halves, exchanged through shared memory (double-buffered)
        float* slot = xchg + (cx & 1u) * (2 * kRows);
        ++cx;
        slot[h * kRows + r] = mx;
        if (group_barrier_or(kGroupBar, kGroup, dead)) { dead = true; break; }
        mx = fmaxf(mx, slot[(h ^ 1) * kRows + r]) * scale_log2;
        float alpha = 1.f;
        if (mx > m_run + C::kThreshold) {  // also the first finite maximum of the row
          alpha = fast_exp2(m_run - mx);
          m_run = mx;
        }
        const float neg_m = (m_run == -INFINITY ? 0.f : -m_run) + C::kShift;
        l_run = l_run * alpha + half_exp<D>(s_tmem, s, scale_log2, neg_m);
        if (j > 0) {
          // O(j-1) must be complete before it is rescaled; without a rescale this phase of the O barrier is only
          // counted (see fa_umma1.cu for why a later wait cannot take it for its own).
          const bool rescale = __any_sync(0xffffffffu, alpha != 1.f);
          if (rescale) {
            if (!warp_wait(&bars[bOFull], co & 1u)) dead = true;   // reported at the next group barrier
            tcgen05_fence_after();
          }
          ++co;
          if (!dead && rescale) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              uint32_t v[32];
              tmem_ld32(o_tmem + c * 32, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
              tmem_st32(o_tmem + c * 32, v);
            }
          }
        }
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(&bars[bPFull + buf]);
      }
      // Items without tiles have no phase here: two of them could pass before a slow warp looks, and a parity only tells
      // neighbouring phases apart.
      if (!dead && n_tiles > 0) {
        if (!warp_wait(&bars[bOFinal], n_final & 1u)) dead = true;
        ++n_final;
        ++co;
        tcgen05_fence_after();
      }
      // ---- epilogue: row sum = both halves; each thread normalises and stores its half of the O columns ----
      float* slot = xchg + (cx & 1u) * (2 * kRows);
      ++cx;
      slot[h * kRows + r] = l_run;
      if (group_barrier_or(kGroupBar, kGroup, dead)) {
        if (p.status) atomicExch(p.status, kWaitMmaTimeout);
        atomicExch(abort_flag, 1);
        dead = true;
        break;
      }
      const float l_row = l_run + slot[(h ^ 1) * kRows + r];
      const Item256 ie = item_slot->it;            // read again: see the top of the item loop
      const float dv = item_slot->dv;
      const int row = ie.row0 + r;
      const int hd = ie.kvh * p.group + row % p.group;
      const bool split_mode = ie.n_splits > 1;     // the combine kernel adds the sink and converts to BF16
      float sink_l2 = -INFINITY;
      if (p.sink != nullptr && !split_mode && row < ie.rows_total) sink_l2 = __bfloat162float(p.sink[hd]) * kLog2e;
      const float m_f = fmaxf(m_run, sink_l2);
      const float m_use = m_f == -INFINITY ? 0.f : m_f;
      const float resc = fast_exp2(m_run - m_use);
      float l = l_row * resc;                                        // in units of 2^kShift
      if (sink_l2 != -INFINITY) l += fast_exp2(sink_l2 - m_use + C::kShift);
      const float inv = (l == 0.f || ie.n_tiles == 0) ? 0.f : dv * resc / l;
      const int64_t q_row = ie.q_start + row / p.group;
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + q_row * p.out_row_stride +
                           (int64_t)hd * p.out_head_stride + h * (D / 2);
      const bool out_vec32 = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0 && (p.out_row_stride & 15) == 0 &&
                             (p.out_head_stride & 15) == 0;
      const int64_t part_slot = ((int64_t)ie.split * p.total_q + q_row) * p.num_q_heads + hd;
      float* part = split_mode ? p.part_o + part_slot * D + h * (D / 2) : nullptr;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t v[32];
        if (ie.n_tiles > 0) {
          tmem_ld32(o_tmem + c * 32, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        if (row < ie.rows_total && split_mode) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(part + c * 32 + i) =
                make_float4(__uint_as_float(v[i]) * inv, __uint_as_float(v[i + 1]) * inv,
                            __uint_as_float(v[i + 2]) * inv, __uint_as_float(v[i + 3]) * inv);
        } else if (row < ie.rows_total) {
          store_bf16_row32(dst + c * 32, v, inv, out_vec32);
        }
      }
      if (h == 0 && row < ie.rows_total) {
        const float lse_l2 = l == 0.f ? -INFINITY : m_use + log2f(l) - C::kShift;
        if (split_mode) p.part_lse[part_slot] = lse_l2;
        else if (p.lse != nullptr) p.lse[(int64_t)hd * p.total_q + q_row] = lse_l2 * kLn2;
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[bItemEmpty + (it_count & 1u)]);   // warp 9 may resolve item n + 2 into the slot
    }
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 8) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

}  // namespace

int kv4_prefill_rows() { return kRows; }
int kv4_prefill_tile(int head_dim) { return head_dim == 128 ? Cfg<128>::kBN : Cfg<256>::kBN; }

cudaError_t kv4_prefill_prepare() {
  const cudaError_t e = cudaFuncSetAttribute(atrex_sm100_kv4_prefill_kernel<128>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<128>());
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(atrex_sm100_kv4_prefill_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              smem_bytes<256>());
}

cudaError_t kv4_prefill_launch(const Kv4Params& p, int head_dim, int sm_count, cudaStream_t stream) {
  const long long items = (long long)p.f.num_row_tiles * p.f.num_kv_heads * p.f.num_splits;
  const unsigned grid = (unsigned)(items < sm_count ? (items < 1 ? 1 : items) : sm_count);
  if (head_dim == 128)
    return launch_kernel(atrex_sm100_kv4_prefill_kernel<128>, dim3(grid), dim3(kThreads), smem_bytes<128>(), stream, p);
  return launch_kernel(atrex_sm100_kv4_prefill_kernel<256>, dim3(grid), dim3(kThreads), smem_bytes<256>(), stream, p);
}

}  // namespace atrex_sm100
