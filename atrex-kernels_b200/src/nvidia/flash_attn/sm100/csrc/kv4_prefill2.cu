// Attention over a 4-bit paged cache on tcgen05 tensor cores, head_dim 128, 256 packed GQA rows (two 128-row subtiles)
// per work item: prompts and chunks of prompts.
//
// The tensor-core side is that of the BF16 kernel (fa_umma.cu): S0 | S1 | O0 | O1 fill TMEM, one softmax thread per row,
// P handed over in two halves of 64 keys, the issuer alternating between the subtiles.  Every K / V tile serves 256
// rows, so its widening from 4 bits costs half of what it costs the single-tile kernel (kv4_prefill.cu) per product.
//
//   warps 0-7    softmax (184 registers)
//   warp 8       tcgen05.mma issuer
//   warp 9       resolves work items one ahead into shared memory
//   warp 10      producer of codes: TMA, one box per page part of a 128-key tile
//   warp 11      producer of scales: cp.async, four rows a lane; those of keys that no row of the item sees become zeros
//                (their codes may be anything, all codes are finite).  With one warp for both, the widening warps waited
//                1 000 - 1 500 cycles per K tile for its staging
//   warps 12-15  widening: 32 rows each of every tile, from the staging ring into the FP16 operand ring; at the start of
//                an item its Q rows, 64 each (a row is scaled by a power of two that joins its score factor)
//
// Measured: 4 chunks of 512 .. 2 048 tokens over contexts of 4 096 .. 16 384, 64 / 8 heads of 128: 1.83 ms = 950 TFLOP/s
// (the single-tile kernel: 2.63 ms; where it wins, the launcher says).  What bounds it: a subtile's chain of softmax
// (~1 900 cycles per 128 keys, waiting for its own instructions, their fetch included: polynomial exponentials, which free
// the special-function units, made it 1 930 -> 2 270 us) and the two products behind it (512 each), of which the other
// subtile covers what it can.
//
// Both products are FP16: E2M1 x E4M3 is exact there (fp4.cuh), P is stored as 2^7 p.  Every wait is bounded; on expiry
// the CTA records a code, drains its copies, frees TMEM and returns.
#define ATREX_MBAR_SPIN_INLINE
#include "fp4.cuh"
#include "kv4_kernels.cuh"
#include "kv4_q.cuh"
#include "softmax_math.cuh"
#include "umma.cuh"

namespace atrex_sm100 {

namespace {

constexpr int kBM = 128;                      // rows per Q subtile (UMMA M)
constexpr int kBN = 128;                      // keys per tile
constexpr int kHD = 128;                      // head dimension
constexpr int kTileBytes = kBN * kHD * 2;     // one K, V or Q operand tile: 32 KB
constexpr int kBlockBytes = kBN * 128;        // one 64-element column block of a tile
constexpr int kSlots = 4;                     // operand ring: K(j), V(j), K(j+1), V(j+1)
constexpr int kStages = 3;                    // staging ring of 4-bit tiles
constexpr int kCodeBytes = kBN * 64, kStageBytes = kBN * 72;
constexpr int kThreads = 512;
constexpr int kRowsPerItem = 2 * kBM;
constexpr uint32_t kTmemCols = 512;
constexpr int kWidenWarps = 4;
constexpr float kShift = 7.f;                 // P is stored as 2^7 p: at most 2^15 with the rescale threshold of 2^8
constexpr float kThreshold = 8.f;
// 512 threads launch with 128 registers each.  2 x 128 x (184 + 64) = 63 488 of the 65 536: the split leaves slack.
constexpr int kSoftmaxRegs = 184, kOtherRegs = 64;

constexpr int kOffKV = 2 * kTileBytes;
constexpr int kOffStage = kOffKV + kSlots * kTileBytes;
constexpr int kOffFactor = kOffStage + kStages * kStageBytes;       // [item parity][row] score factors
constexpr int kOffItem = kOffFactor + 2 * kRowsPerItem * 4;
enum Bar { kQFull = 0, kQEmpty, kItemFull, kItemEmpty = kItemFull + 2, kRowsFull = kItemEmpty + 2, kKVFull = kRowsFull + 2,
           kKVEmpty = kKVFull + kSlots, kStageFull = kKVEmpty + kSlots, kStageEmpty = kStageFull + kStages,
           kSFull = kStageEmpty + kStages, kPFull = kSFull + 2, kPLast = kPFull + 2, kOFull = kPLast + 2,
           kNumBars = kOFull + 2 };

// One work item, resolved by warp 9 into one of two slots.
struct __align__(16) Item {
  int valid, b, kvh, row0, q_start, q_len, rows_total, kv_len, off, tile_lo, n_tiles, kv_begin, kv_end;
  float scale_log2, dv;
  int pad;
};
static_assert(sizeof(Item) == 64, "four 16-byte vectors");
constexpr int kOffBar = kOffItem + 2 * 64;
constexpr int kOffMisc = kOffBar + kNumBars * 8;
constexpr int kSmemBytes = kOffMisc + 16;
static_assert(kSmemBytes <= 232448, "shared memory of one CTA");

// Items are KV-head-major, heaviest request first, last (heaviest causal) row tile first: the CTAs in flight read one
// head of the cache, which stays in L2 (see fa_umma.cu).
__device__ __forceinline__ void resolve_item(const FwdParams& p, int item, Item& it) {
  it.valid = 0;
  const int total_tiles = p.tile_prefix[p.batch];
  if (total_tiles <= 0) return;
  it.kvh = item / total_tiles;
  if (it.kvh >= p.num_kv_heads) return;
  const int tile_rank = item - it.kvh * total_tiles;
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.tile_prefix[mid] <= tile_rank) lo = mid; else hi = mid;
  }
  const int b = p.order[lo];
  const int tiles_b = p.tile_prefix[lo + 1] - p.tile_prefix[lo];
  const int row0 = (tiles_b - 1 - (tile_rank - p.tile_prefix[lo])) * kRowsPerItem;
  const int q_start = p.cu_seqlens_q[b], q_len = p.cu_seqlens_q[b + 1] - q_start;
  int kv_len, k_start;
  request_kv(p, b, kv_len, k_start);
  const int off = request_off(p, b, kv_len, q_len);
  const int qi_lo = row0 / p.group, qi_hi = min(q_len - 1, (row0 + kRowsPerItem - 1) / p.group);
  it.kv_end = p.window_right >= 0 ? min(kv_len, right_bound(p, qi_hi + off)) : kv_len;
  it.kv_begin = p.window_left >= 0 ? max(0, qi_lo + off - p.window_left) : 0;
  it.tile_lo = it.n_tiles = 0;
  if (it.kv_end > it.kv_begin) {
    it.tile_lo = it.kv_begin / kBN;
    it.n_tiles = (it.kv_end + kBN - 1) / kBN - it.tile_lo;
  }
  it.b = b;
  it.row0 = row0;
  it.q_start = q_start;
  it.q_len = q_len;
  it.rows_total = q_len * p.group;
  it.kv_len = kv_len;
  it.off = off;
  const float dk = p.k_descale ? p.k_descale[b * p.k_descale_bs + it.kvh * p.k_descale_hs] : 1.f;
  it.dv = p.v_descale ? p.v_descale[b * p.v_descale_bs + it.kvh * p.v_descale_hs] : 1.f;
  it.scale_log2 = p.softmax_scale * dk * kLog2e;
  it.valid = 1;
}

// First step of a tile for one row (= one thread), as in fa_umma.cu: scores into registers, masked columns -inf, the
// running maximum by the lazy-rescale rule.  Returns the factor for the O and the row sum accumulated so far.
template <bool kMask>
__device__ __forceinline__ float tile_max(uint32_t s_tmem, uint32_t (&s)[kBN], float scale_log2, int tok0, int vis_lo,
                                          int vis_hi, float& m_run) {
  float mxv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) mxv[i] = -INFINITY;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half == 0) {
#pragma unroll
      for (int c = 0; c < kBN / 64; ++c) tmem_ld32(s_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
    }
    tmem_ld_wait();
    if (half == 0) {
#pragma unroll
      for (int c = kBN / 64; c < kBN / 32; ++c)
        tmem_ld32(s_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
    }
    if (kMask) {
#pragma unroll
      for (int i = half * (kBN / 2); i < (half + 1) * (kBN / 2); ++i) {
        const int col = tok0 + i;
        if (col < vis_lo || col >= vis_hi) s[i] = 0xff800000u;  // -inf
      }
    }
#pragma unroll
    for (int i = half * (kBN / 2); i < (half + 1) * (kBN / 2); i += 16) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        mxv[u] = fmax3(mxv[u], __uint_as_float(s[i + 2 * u]), __uint_as_float(s[i + 2 * u + 1]));
    }
  }
  mxv[0] = fmaxf(mxv[0], mxv[4]); mxv[1] = fmaxf(mxv[1], mxv[5]);
  mxv[2] = fmaxf(mxv[2], mxv[6]); mxv[3] = fmaxf(mxv[3], mxv[7]);
  const float mx = fmaxf(fmaxf(mxv[0], mxv[1]), fmaxf(mxv[2], mxv[3])) * scale_log2;
  float alpha = 1.f;
  if (mx > m_run + kThreshold) {  // also the first finite maximum of the row
    alpha = fast_exp2(m_run - mx);
    m_run = mx;
  }
  return alpha;
}

// Second step, for 64-key half `half`: P = 2^(s * scale + neg_m) as FP16 pairs over the S columns.
__device__ __forceinline__ void tile_exp(uint32_t s_tmem, const uint32_t (&s)[kBN], int half, f32x2 scale2, f32x2 negm2,
                                         f32x2 (&sum2)[2]) {
  uint32_t packed[32];
  exp32_f16(&s[half * 64], scale2, negm2, sum2, *reinterpret_cast<uint32_t(*)[16]>(&packed[0]));
  exp32_f16(&s[half * 64 + 32], scale2, negm2, sum2, *reinterpret_cast<uint32_t(*)[16]>(&packed[16]));
  tmem_st32(s_tmem + half * 32, packed);
}

// 128 values of one row of a staged tile into the 128-byte-swizzled operand tile, 8 at a time.
__device__ __forceinline__ void widen_row(const uint8_t* stage, uint8_t* tile, int row) {
  const uint2 sc = *reinterpret_cast<const uint2*>(stage + kCodeBytes + row * 8);
  // Rolled: the loops of a scheduler's warps fill its instruction cache (chunk case 1 920 -> 1 805 us; two chunks: 1 905)
#pragma unroll 1
  for (int chunk = 0; chunk < 4; ++chunk) {                  // 32 values, two scales
    const uint4 raw = *reinterpret_cast<const uint4*>(stage + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
    const uint32_t two = e4m3x2_to_f16x2(chunk < 2 ? sc.x >> (16 * chunk) : sc.y >> (16 * (chunk - 2)));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t f[4];
      e2m1x8_to_f16x2(w == 0 ? raw.x : w == 1 ? raw.y : w == 2 ? raw.z : raw.w, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = w < 2 ? hmul2_low(f[i], two) : hmul2_high(f[i], two);
      *reinterpret_cast<uint4*>(tile + (chunk >> 1) * kBlockBytes + swz128(row, (chunk & 1) * 4 + w)) =
          make_uint4(f[0], f[1], f[2], f[3]);
    }
  }
}

// A bounded wait that expired: one lane reports.
#define KV4_REPORT(code)                              \
  if (lane == 0) {                                    \
    if (p.status) atomicExch(p.status, (code));       \
    atomicExch(abort_flag, 1);                        \
  }
// A warp goes on or leaves its loop as one: TMEM accesses and warp barriers behind a wait need all of its lanes.  The tile
// loops of issuer and producers hold neither, because a vote there costs (chunk case, us: 1 835; at every wait 1 900, in
// place of the producers' barrier behind a stage 1 885): their lanes give up one by one and the warp votes once an item.
#define KV4_WAIT(bar_index, parity, code)                                          \
  if (!__all_sync(0xffffffffu, mbar_wait(&bars[bar_index], (parity)))) {           \
    KV4_REPORT(code)                                                               \
    break;                                                                         \
  }
#define KV4_LANE_WAIT(bar_index, parity) \
  if (!mbar_wait(&bars[bar_index], (parity))) break;

__global__ void __launch_bounds__(kThreads, 1)
atrex_sm100_kv4_prefill2_kernel(const __grid_constant__ Kv4Params pp) {
  const FwdParams& p = pp.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* q_smem = smem;
  uint8_t* kv_smem = smem + kOffKV;
  uint8_t* stage_smem = smem + kOffStage;
  float* row_factor = reinterpret_cast<float*>(smem + kOffFactor);
  Item* slots = reinterpret_cast<Item*>(smem + kOffItem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOffMisc);
  int* abort_flag = reinterpret_cast<int*>(smem + kOffMisc + 4);

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  if ((smem_u32(smem) & 1023u) != 0u) {
    if (tid == 0 && p.status) atomicExch(p.status, kBadSmemAlignment);
    return;
  }
  if (tid == 0) {
    *abort_flag = 0;
    mbar_init(&bars[kQFull], kWidenWarps);
    mbar_init(&bars[kQEmpty], 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[kItemFull + s], 1);
      mbar_init(&bars[kItemEmpty + s], 15);          // issuer, producers, widening and softmax warps
      mbar_init(&bars[kRowsFull + s], kWidenWarps);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bars[kKVFull + s], kWidenWarps);
      mbar_init(&bars[kKVEmpty + s], 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars[kStageFull + s], 64);          // 32 lanes with TMA bytes, 32 with scale copies
      mbar_init(&bars[kStageEmpty + s], kWidenWarps);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bars[kSFull + w], 1);
      mbar_init(&bars[kPFull + w], kBM);
      mbar_init(&bars[kPLast + w], kBM);
      mbar_init(&bars[kOFull + w], 1);
    }
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= 12) {
    // ------------------------------- widening -------------------------------
    setmaxnreg_dec<kOtherRegs>();
    const int row = (warp - 12) * 32 + lane;
    for (uint32_t n_item = 0, done = 0;; ++n_item) {
      // the items only say how many tiles there are: K and V of each, in order
      KV4_WAIT(kItemFull + (n_item & 1u), (n_item >> 1) & 1u, kWaitFullTimeout)
      const int valid = slots[n_item & 1u].valid, n_tiles = slots[n_item & 1u].n_tiles;
      __syncwarp();
      if (!valid) {
        if (lane == 0) mbar_arrive(&bars[kRowsFull + (n_item & 1u)]);    // the softmax warps read the slot behind it
        break;
      }
      {
        using Q = QRows<kHD, kRowsPerItem / kWidenWarps, 4>;
        const Item& it = slots[n_item & 1u];
        const int first = (warp - 12) * (kRowsPerItem / kWidenWarps);
        const bool flip = it.scale_log2 < 0.f;
        Q rows(p, first, it.row0, it.rows_total, it.q_start, it.kvh * p.group);
        rows.fetch();
        // Q is free from the last Q K^T of the item before
        if (n_item > 0) KV4_WAIT(kQEmpty, (n_item - 1u) & 1u, kWaitEmptyTimeout)
        for (int k = 0; k < Q::kSteps; k += 4) {
          rows.store(q_smem, kTileBytes, kBlockBytes, row_factor + (n_item & 1u) * kRowsPerItem, first + k * Q::kRpi, flip);
          if (k + 4 < Q::kSteps) rows.fetch();
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[kQFull]);
        mbar_arrive(&bars[kRowsFull + (n_item & 1u)]);    // release: the row factors are written
        mbar_arrive(&bars[kItemEmpty + (n_item & 1u)]);
      }
      bool dead = false;
      for (int i = 0; i < 2 * n_tiles; ++i, ++done) {
        const uint32_t stage = done % kStages, slot = done % kSlots;
        dead = true;
        KV4_WAIT(kStageFull + stage, (done / kStages) & 1u, kWaitFullTimeout)
        if (done >= (uint32_t)kSlots) KV4_WAIT(kKVEmpty + slot, ((done / kSlots) - 1u) & 1u, kWaitEmptyTimeout)
        dead = false;
        widen_row(stage_smem + stage * kStageBytes, kv_smem + slot * kTileBytes, row);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars[kKVFull + slot]);
          mbar_arrive(&bars[kStageEmpty + stage]);
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
        for (int item = blockIdx.x;; item += gridDim.x, ++n) {
          Item* slot = slots + (n & 1u);
          if (n >= 2 && !mbar_wait(&bars[kItemEmpty + (n & 1u)], ((n >> 1) - 1u) & 1u)) {
            KV4_REPORT(kWaitEmptyTimeout)
            break;
          }
          resolve_item(p, item, *slot);
          if (*(volatile int*)abort_flag) slot->valid = 0;
          const bool valid = slot->valid != 0;
          mbar_arrive(&bars[kItemFull + (n & 1u)]);              // release: the slot is written
          if (!valid) break;
        }
      }
      __syncwarp();
    } else if (warp >= 10) {
      // ------------------------------- producers -------------------------------
      // Both walk every stage in order: a barrier's parity says which of two neighbouring phases is meant, so a warp
      // that skipped a stage's phases (K tiles or V tiles only, over an odd ring) would take an old one for its own.
      const bool codes = warp == 10;
      const int shift = (p.page_size & (p.page_size - 1)) == 0 ? __ffs(p.page_size) - 1 : -1;
      const int box_rows = p.box_rows;
      uint32_t n = 0;                                  // tiles of the run: K even, V odd
      for (uint32_t n_item = 0;; ++n_item) {
        KV4_WAIT(kItemFull + (n_item & 1u), (n_item >> 1) & 1u, kWaitFullTimeout)
        const Item& it = slots[n_item & 1u];
        if (!it.valid) break;
        const int kv_begin = it.kv_begin, kv_end = it.kv_end, n_tiles = it.n_tiles, kvh = it.kvh;
        int tok0 = it.tile_lo * kBN;
        const int32_t* table = p.block_table + (int64_t)it.b * p.block_table_row_stride;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kItemEmpty + (n_item & 1u)]);
        const uint8_t* ks = pp.ks + kvh * pp.ks_str.head;
        const uint8_t* vs = pp.vs + kvh * pp.vs_str.head;
        // table entries of the rows lane, lane + 32, ... of a tile, as read: nothing looks at them before the next tile
        int page[4], next[4];
        auto fetch = [&](int t0, int (&out)[4]) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int t = t0 + u * 32 + lane;
            out[u] = t < kv_end ? table[shift >= 0 ? t >> shift : t / p.page_size] : -1;
          }
        };
        fetch(tok0, page);
        bool dead = false;
        for (int j = 0; j < n_tiles; ++j, tok0 += kBN) {
          if (j + 1 < n_tiles) fetch(tok0 + kBN, next);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (page[u] >= p.num_pages) page[u] = -1;
          for (int v = 0; v < 2; ++v, ++n) {
            const uint32_t stage = n % kStages;
            dead = true;
            if (n >= (uint32_t)kStages) KV4_LANE_WAIT(kStageEmpty + stage, ((n / kStages) - 1u) & 1u)
            dead = false;
            uint8_t* dst = stage_smem + stage * kStageBytes;
            uint64_t* full = &bars[kStageFull + stage];
            if (codes) {
              uint32_t bytes = 0;
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (((u * 32 + lane) & (box_rows - 1)) == 0 && page[u] >= 0) bytes += box_rows * 64;
              mbar_arrive_expect_tx(full, bytes);
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int r = u * 32 + lane, t = tok0 + r;
                if ((r & (box_rows - 1)) == 0 && page[u] >= 0)
                  tma_load_kv(dst + r * 64, v ? &p.v_map : &p.k_map, full, 0, kvh,
                              shift >= 0 ? t & (p.page_size - 1) : t % p.page_size, page[u], v ? p.v_perm : p.k_perm);
              }
            } else {
              const CacheStrides& st = v ? pp.vs_str : pp.ks_str;
              const uint8_t* scales = v ? vs : ks;
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int r = u * 32 + lane, t = tok0 + r;
                const uint32_t in_page = shift >= 0 ? t & (p.page_size - 1) : t % p.page_size;
                const bool ok = page[u] >= 0 && t >= kv_begin;
                const uint8_t* src = scales + (uint64_t)(uint32_t)max(page[u], 0) * st.page + (uint64_t)in_page * st.row;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst + kCodeBytes + r * 8)),
                             "l"(src), "r"(ok ? 8u : 0u)
                             : "memory");
              }
              asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
            }
          }
          if (dead) break;
#pragma unroll
          for (int u = 0; u < 4; ++u) page[u] = next[u];
        }
        if (__any_sync(0xffffffffu, dead)) {
          KV4_REPORT(kWaitEmptyTimeout)
          break;
        }
      }
      // every copy must have landed before the CTA may exit
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (uint32_t back = 1; back <= (uint32_t)kStages && back <= n; ++back) {
        const uint32_t i = n - back;
        mbar_wait(&bars[kStageFull + i % kStages], (i / kStages) & 1u);
      }
      __syncwarp();
    } else if (warp == 8) {
      // ------------------------------- MMA issuer -------------------------------
      constexpr uint32_t kIdescQK = umma_idesc(kBM, kBN, 0, 0, 0, 0);      // FP16 operands
      constexpr uint32_t kIdescPV = umma_idesc(kBM, kHD, 0, 0, 0, 1);
      uint32_t seq = 0, cp[2] = {0, 0};
      const UmmaDesc q_desc0 = umma_desc_split(umma_desc_sw128(smem_u32(q_smem), 16, 1024));
      const UmmaDesc k_desc0 = umma_desc_split(umma_desc_sw128(smem_u32(kv_smem), 16, 1024));
      const UmmaDesc v_desc0 = umma_desc_split(umma_desc_sw128(smem_u32(kv_smem), kBlockBytes, 1024));
      const uint32_t lead = lane == 0;
      auto issue_qk = [&](int w, uint32_t slot) {
        const UmmaDesc qd = q_desc0 + (uint32_t)((w * kTileBytes) >> 4);
        const UmmaDesc kd = k_desc0 + (uint32_t)((slot * kTileBytes) >> 4);
#pragma unroll
        for (int ks = 0; ks < kHD / 16; ++ks) {
          const uint32_t koff = ((ks >> 2) * kBlockBytes + (ks & 3) * 32) >> 4;
          umma_ss_f16_lead(lead, tmem_base + w * kBN, qd + koff, kd + koff, kIdescQK, ks > 0);
        }
        umma_commit_lead(lead, &bars[kSFull + w]);
      };
      for (uint32_t n_item = 0;; ++n_item) {
        KV4_WAIT(kItemFull + (n_item & 1u), (n_item >> 1) & 1u, kWaitFullTimeout)
        const int valid = slots[n_item & 1u].valid, n_tiles = slots[n_item & 1u].n_tiles;
        __syncwarp();
        if (!valid) break;
        if (lane == 0) mbar_arrive(&bars[kItemEmpty + (n_item & 1u)]);
        KV4_WAIT(kQFull, n_item & 1u, kWaitFullTimeout)
        if (n_tiles == 0) {              // nothing to multiply, but the Q tile must be released
          if (lane == 0) mbar_arrive(&bars[kQEmpty]);
          continue;
        }
        bool dead = false;
        uint32_t slot_k = seq % kSlots;
        KV4_WAIT(kKVFull + slot_k, (seq / kSlots) & 1u, kWaitFullTimeout)
        ++seq;
        tcgen05_fence_after();
        issue_qk(0, slot_k);
        issue_qk(1, slot_k);
        umma_commit_lead(lead, &bars[kKVEmpty + slot_k]);
        if (n_tiles == 1) umma_commit_lead(lead, &bars[kQEmpty]);   // Q is last read by the item's last Q K^T
        for (int j = 0; j < n_tiles; ++j) {
          const bool more = j + 1 < n_tiles;
          const uint32_t slot_v = seq % kSlots;
          dead = true;
          KV4_LANE_WAIT(kKVFull + slot_v, (seq / kSlots) & 1u)
          ++seq;
          uint32_t slot_k2 = 0;
          if (more) {
            slot_k2 = seq % kSlots;
            KV4_LANE_WAIT(kKVFull + slot_k2, (seq / kSlots) & 1u)
            ++seq;
          }
          int w = 0;
          for (; w < 2; ++w) {
            KV4_LANE_WAIT(kPFull + w, cp[w] & 1u)
            ++cp[w];
            tcgen05_fence_after();
            const UmmaDesc vd = v_desc0 + (uint32_t)((slot_v * kTileBytes) >> 4);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma_ts_f16_lead(lead, tmem_base + 2 * kBN + w * kHD, tmem_base + w * kBN + ks * 8,
                               vd + (uint32_t)((ks * 2048) >> 4), kIdescPV, (j > 0) | (ks > 0));
            KV4_LANE_WAIT(kPLast + w, (cp[w] - 1) & 1u)
            tcgen05_fence_after();
#pragma unroll
            for (int ks = 4; ks < 8; ++ks)
              umma_ts_f16_lead(lead, tmem_base + 2 * kBN + w * kHD, tmem_base + w * kBN + ks * 8,
                               vd + (uint32_t)((ks * 2048) >> 4), kIdescPV, 1u);
            umma_commit_lead(lead, &bars[kOFull + w]);
            if (more) issue_qk(w, slot_k2);
          }
          if (w < 2) break;
          dead = false;
          umma_commit_lead(lead, &bars[kKVEmpty + slot_v]);
          if (more) umma_commit_lead(lead, &bars[kKVEmpty + slot_k2]);
          if (j + 2 == n_tiles) umma_commit_lead(lead, &bars[kQEmpty]);
        }
        if (__any_sync(0xffffffffu, dead)) {
          KV4_REPORT(kWaitMmaTimeout)
          break;
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------- softmax, O kept in TMEM -------------------------------
    setmaxnreg_inc<kSoftmaxRegs>();
    const int w = warp >> 2;                                   // subtile
    const int r = (warp & 3) * 32 + lane;                      // row inside the subtile = TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem_base + lane_off + w * kBN;
    const uint32_t o_tmem = tmem_base + lane_off + 2 * kBN + w * kHD;
    uint32_t cs = 0, co = 0;
    for (uint32_t n_item = 0;; ++n_item) {
      // row factors are written behind the item itself
      KV4_WAIT(kRowsFull + (n_item & 1u), (n_item >> 1) & 1u, kWaitFullTimeout)
      const Item& it = slots[n_item & 1u];
      if (!it.valid) break;
      const int sub_row0 = it.row0 + w * kBM;
      const int n_tiles = it.n_tiles, tile_lo = it.tile_lo;
      float scale_log2 = it.scale_log2 * row_factor[(n_item & 1u) * kRowsPerItem + w * kBM + r];
      int vis_lo, vis_hi, full_lo, full_hi;
      {
        const int q_last = max(it.q_len - 1, 0), off = it.off, kv_len = it.kv_len;
        const int qi = min((sub_row0 + r) / p.group, q_last);
        vis_hi = p.window_right >= 0 ? min(kv_len, right_bound(p, qi + off)) : kv_len;
        vis_lo = p.window_left >= 0 ? max(0, qi + off - p.window_left) : 0;
        const int sqi_lo = sub_row0 / p.group, sqi_hi = min(it.q_len - 1, (sub_row0 + kBM - 1) / p.group);
        full_lo = p.window_left >= 0 ? max(0, sqi_hi + off - p.window_left) : 0;
        full_hi = p.window_right >= 0 ? min(kv_len, right_bound(p, sqi_lo + off)) : kv_len;
      }
      scale_log2 = score_factor(scale_log2, [&] { return vis_lo < vis_hi; });
      bool dead = false;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < n_tiles; ++j) {
        const int tok0 = (tile_lo + j) * kBN;
        const bool need_mask = tok0 < full_lo || tok0 + kBN > full_hi;
        dead = true;
        KV4_WAIT(kSFull + w, cs & 1u, kWaitMmaTimeout)
        dead = false;
        ++cs;
        tcgen05_fence_after();
        uint32_t s[kBN];
        const float alpha = need_mask ? tile_max<true>(s_tmem, s, scale_log2, tok0, vis_lo, vis_hi, m_run)
                                      : tile_max<false>(s_tmem, s, scale_log2, tok0, vis_lo, vis_hi, m_run);
        if (j > 0) {
          // O(j-1) is complete: S(j), waited for above, was committed behind P V(j-1) (see fa_umma.cu)
          ++co;
          if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
            for (int c = 0; c < kHD / 16; ++c) {
              uint32_t v[16];
              tmem_ld16(o_tmem + c * 16, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
              tmem_st16(o_tmem + c * 16, v);
            }
          }
        }
        const float neg_m = kShift - (m_run == -INFINITY ? 0.f : m_run);
        const f32x2 scale2 = pack2(scale_log2, scale_log2), negm2 = pack2(neg_m, neg_m);
        f32x2 sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
        tile_exp(s_tmem, s, 0, scale2, negm2, sum2);
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(&bars[kPFull + w]);
        tile_exp(s_tmem, s, 1, scale2, negm2, sum2);
        l_run = l_run * alpha + sum_of(sum2);
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(&bars[kPLast + w]);
      }
      if (dead) break;
      if (n_tiles > 0) {
        KV4_WAIT(kOFull + w, co & 1u, kWaitMmaTimeout)
        ++co;
        tcgen05_fence_after();
      }
      // ---- epilogue: O from TMEM, normalise, store the BF16 row and the natural-log LSE ----
      const int row = sub_row0 + r;
      const int hd = it.kvh * p.group + row % p.group;
      const bool in = row < it.rows_total;
      const int64_t q_row = it.q_start + row / p.group;
      float sink_l2 = -INFINITY;
      if (p.sink != nullptr && in) sink_l2 = __bfloat162float(p.sink[hd]) * kLog2e;
      const float m_f = fmaxf(m_run, sink_l2);
      const float m_use = m_f == -INFINITY ? 0.f : m_f;
      const float resc = fast_exp2(m_run - m_use);
      float l = l_run * resc;                                        // in units of 2^kShift
      if (sink_l2 != -INFINITY) l += fast_exp2(sink_l2 - m_use + kShift);
      const float inv = (l == 0.f || n_tiles == 0) ? 0.f : it.dv * resc / l;
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + q_row * p.out_row_stride +
                           (int64_t)hd * p.out_head_stride;
      const bool out_vec32 = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0 && (p.out_row_stride & 15) == 0 &&
                             (p.out_head_stride & 15) == 0;
#pragma unroll
      for (int c = 0; c < kHD / 32; ++c) {
        uint32_t v[32];
        if (n_tiles > 0) {           // warp-uniform
          tmem_ld32(o_tmem + c * 32, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        if (in) store_bf16_row32(dst + c * 32, v, inv, out_vec32);
      }
      if (in && p.lse != nullptr)
        p.lse[(int64_t)hd * p.total_q + q_row] = l == 0.f ? -INFINITY : (m_use + log2f(l) - kShift) * kLn2;
      // the next item's first P V overwrites O only after this warp's next P arrival, i.e. after these loads
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kItemEmpty + (n_item & 1u)]);
    }
  }

  // All roles meet here (every wait above is bounded), then the allocating warp frees TMEM.
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 8) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace

int kv4_prefill2_rows() { return kRowsPerItem; }

cudaError_t kv4_prefill2_prepare() {
  return cudaFuncSetAttribute(atrex_sm100_kv4_prefill2_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
}

cudaError_t kv4_prefill2_launch(const Kv4Params& p, int sm_count, cudaStream_t stream) {
  const long long items = (long long)p.f.num_row_tiles * p.f.num_kv_heads;
  const unsigned grid = (unsigned)(items < sm_count ? (items < 1 ? 1 : items) : sm_count);
  return launch_kernel(atrex_sm100_kv4_prefill2_kernel, dim3(grid), dim3(kThreads), kSmemBytes, stream, p);
}

}  // namespace atrex_sm100
