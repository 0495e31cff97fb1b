// Matrix products of the cross entropy over many symbols: one kernel on CTA pairs (tcgen05 cta_group::2), four uses.
//
//   STATS   z = x W^T, of which only each row's running maximum and sum of exponentials over a span of symbols is kept,
//           and the logit of the row's own symbol
//   PROB    d = (exp(z - lse) - [symbol]) g over a piece of the symbols, rounded to 16 bits for the products that follow
//   OUT_X   dx = d W       (W's symbols are the contraction)
//   OUT_W   dW = d^T x     (the positions are the contraction)
//
// Both CTAs of a pair hold 128 rows of the 256 x BN tile and half of its columns' operand: a stage of 64 contraction values is 16 KB + 16 KB to
// a CTA, which TMA brings (no multicast) and signals at the leader's barrier, whose one thread issues the MMAs for both tensor
// cores.  The accumulator is double-buffered in tensor memory, so that what is done with a tile (8 warps, a row and half
// of the columns to a thread) runs beside the products of the next one.  Operands are taken as they lie: x and W by rows, d and W and x for the
// gradients across them (MN-major).
//
// Tiles and spans end where they should for the pairs to have equal shares: a tile may have any multiple of 32 columns for its MMAs.  Where the tiles of a
// gradient do not fill the pairs evenly, the last ones are cut along the contraction into parts, which a further launch adds.
//
// 32-bit operands (WIDE) come as three planes of bfloat16 whose sum they are, exactly: 8 + 8 + 8 of the 24 digits.  Six products of planes, the
// smallest first, leave out what is below 2^-24 of a product of two numbers.  Each plane of 64 contraction values is a stage of its own, and is used for
// 8 or 12 MMAs.  (TMA takes some 2.5 cycles for each row of a box, of 64 bytes or 128: rows of 64 took longer than their MMAs.)  The tensor core cuts
// off what does not fit its accumulator, half a unit of the last place for each of many additions; so each 64 contraction values have an
// accumulator of their own, which is added to sums in registers, and tiles are 192 columns, whose sums are 96 registers of a thread.  The logits of 16-bit operands
// are added up like that too, every `drain` k-blocks (8192 values in one accumulator: off by 1e-3 where float32 is by 1e-5).
#pragma once

#include "divisor.cuh"
#include "packs.cuh"
#include "ptx.cuh"

namespace tb200 {

enum EntropyMode { ENTROPY_STATS, ENTROPY_PROB, ENTROPY_OUT_X, ENTROPY_OUT_W };

// What OUT_X and OUT_W do with a product.
enum EntropyDest {
  DEST_FINAL,      // rounded to the result's type
  DEST_SUM,        // written to a 32-bit sum
  DEST_SUM_ADD,    // added to it
  DEST_FINAL_ADD,  // added to it, rounded and written to the result
};

template <int MODE_, bool WIDE_>
struct EntropyCfg {
  static constexpr int MODE = MODE_;
  static constexpr bool WIDE = WIDE_;
  static constexpr bool A_MN = MODE == ENTROPY_OUT_W;
  static constexpr bool B_MN = MODE == ENTROPY_OUT_X || MODE == ENTROPY_OUT_W;
  static constexpr int BM = 128;  // rows of a CTA
  static constexpr int BN = WIDE ? 192 : 256;
  static constexpr int BNH = BN / 2;
  static constexpr int BK = 64;
  static constexpr int NS = 6;
  static constexpr int PLANES = WIDE ? 3 : 1;
  static constexpr int MN_BOX = 64 * BK * 2;  // 64 rows or columns of an MN-major operand
  static constexpr int A_TILE = BM * BK * 2;
  static constexpr int B_BOXES = (BNH + 63) / 64;
  static constexpr int B_TILE = B_MN ? B_BOXES * MN_BOX : BNH * BK * 2;
  static constexpr int STAGE = A_TILE + B_TILE;  // (WIDE: of one plane)
  static constexpr int EPI_WARPS = 8;
  static constexpr int NTHREADS = (4 + EPI_WARPS) * 32;
  static constexpr int BOX = 32 * 128;
  static constexpr int COLS = BNH;  // columns of a thread: the two halves of the tile go to four warps each
  static constexpr int BUF_COLS = 256;
  static constexpr int TMEM_COLS = 2 * BUF_COLS;
  static constexpr int NBAR = 2 * NS + 4;
  static constexpr int SMEM_BYTES = 1024 + NS * STAGE + EPI_WARPS * BOX + NBAR * 8 + 16;
  static_assert(SMEM_BYTES <= 232448, "shared memory capacity");
};

struct EntropyParams {
  int rows, cols;         // of the product
  int kblocks;              // of the contraction
  int tiles_m;              // row tiles
  int units_n, unit_cols;   // a unit is a row tile and so many columns,
  int tile_cols;            // gone over in tiles of these: one tile but for STATS
  int group;                // row tiles that are gone over together
  int whole;                // units that are one pair's
  int shared;               // and those behind them whose contraction is cut
  int splits, kb_split;     // into parts of so many k-blocks
  Divisor by_group, by_rows, by_last, by_shared;  // a group's units, its row tiles, those of the last group; `shared`
  int b_row, b_k;         // where the piece begins in W: as rows of the product's columns, as contraction values
  uint32_t idesc;
  int drain;              // k-blocks of an accumulator, where not WIDE
  int half;               // 16-bit operands are float16 and not bfloat16
  // STATS: [units_n * 2][rows] of maximum and sum, and the logits of the rows' own symbols
  float2* stats;
  float* picked;
  int* arrived;           // set to zero for the launch that joins them
  // STATS, PROB and OUT_X
  const void* target;
  int target_wide;        // 64 bits
  int64_t ignore;
  int64_t symbols;        // (not OUT_X)
  // PROB
  const float* lse;
  const float* dloss;     // [rows], or one number
  int per_row;
  float* factors;         // what dloss is multiplied by; what the gradients are
  uint16_t* d;            // [planes][rows][d_pitch]
  int64_t d_pitch, d_plane;
  // OUT
  int dest;               // of whole tiles
  void* out;              // rows of `out_pitch` elements
  int64_t out_pitch;
  int out_vec;            // its rows are on boundaries of 16 bytes
  int direct;             // of 32 bytes
  int boxed;              // 32-bit results of OUT_W leave through TMA
  float* sum;             // [rows][sum_pitch], what earlier pieces gave
  int64_t sum_pitch;
  float* part;            // [shared][splits][256][tile_cols]
  int* status;
};

// f16 or bf16 operands, fp32 accumulator: descriptor of MMAs of m rows, but for their columns n, as n / 8 from bit 17 on; `half`: float16.
__host__ __device__ constexpr uint32_t umma_idesc_16(int m, bool half, bool a_mn, bool b_mn) {
  return (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// Shared-memory descriptor of an MN-major operand of 16-bit elements: boxes of 64 consecutive rows or columns (128 bytes) by BK contraction
// values with the 128-byte swizzle, one after the other (leading byte offset); groups of eight contraction values are 1024 bytes apart
// (stride byte offset).  One MMA (16 contraction values) spans two groups: the next adds 2048 bytes, 128 to the encoded address.
__device__ __forceinline__ uint64_t umma_desc_mn16_sw128(uint32_t smem_addr, uint32_t box_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((box_bytes >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

__device__ __forceinline__ void umma_16_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// TMA load into this CTA's shared memory whose bytes are counted at a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* tmap, uint32_t leader_bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// The 16 high bits of two numbers, each a bfloat16 (cut off, not rounded), and what they leave of a number, exactly.  Three of these take one apart.  (An infinity
// leaves a NaN.)
__device__ __forceinline__ uint32_t plane_bits(float x0, float x1) { return __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632); }
__device__ __forceinline__ float plane_rest(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// What the largest |dloss| stands for in d; 0: dloss as it is, times the share of a position.  What is common to all positions is rounded with each d, the same way
// each time (1/6 of "mean" in bfloat16 by 0.1 %, and with it the gradients of a few positions), so 16-bit d leave it to their products.  In float16 the
// largest is 2^15, so that a probability of 2^-29 still has all of its digits; of bfloat16 one for each position keeps its own, and its range.
__host__ __device__ constexpr float entropy_scale(bool wide, int half, int per_row) { return wide ? 0.f : half ? 32768.f : per_row ? 0.f : 1.f; }
// What dloss is multiplied by in d, and what dx and dW are multiplied by, for the largest finite |dloss| and the number of targets that are not ignored.
__device__ __forceinline__ float2 entropy_factors(float top, int count, int mean, float scale) {
  const float share = mean ? 1.f / static_cast<float>(max(count, 1)) : 1.f;
  if (scale == 0.f) return make_float2(share, 1.f);
  top = top == 0.f ? 1.f : fmaxf(top, 0x1p-100f);
  return make_float2(scale / top, top * share * (1.f / scale));
}

__device__ __forceinline__ int64_t entropy_target(const EntropyParams& p, int64_t row) {
  return p.target_wide ? static_cast<const int64_t*>(p.target)[row] : static_cast<int64_t>(static_cast<const int32_t*>(p.target)[row]);
}

// 32 bytes, a whole sector, as one access of a thread.
__device__ __forceinline__ void store_sector(void* to, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
               "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ void load_sector(uint32_t (&w)[8], const void* from) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(from)
               : "memory");
}

// Two numbers as 16-bit ones.
__device__ __forceinline__ uint32_t pack16(float x0, float x1, int half) {
  if (half) {
    const __half2 x = __floats2half2_rn(x0, x1);
    return *reinterpret_cast<const uint32_t*>(&x);
  }
  const __nv_bfloat162 x = __floats2bfloat162_rn(x0, x1);
  return *reinterpret_cast<const uint32_t*>(&x);
}

// Four elements of a result, in row `row` from column `col` on (those before column `end`).
template <class T>
__device__ __forceinline__ void entropy_put(const EntropyParams& p, int row, int col, float4 x, int end) {
  T* out = static_cast<T*>(p.out) + static_cast<int64_t>(row) * p.out_pitch + col;
  Pack<T, 4 * static_cast<int>(sizeof(T))> y;
  y.v[0] = from_float<T>(x.x);
  y.v[1] = from_float<T>(x.y);
  y.v[2] = from_float<T>(x.z);
  y.v[3] = from_float<T>(x.w);
  if (p.out_vec && col + 4 <= end) {
    *reinterpret_cast<Pack<T, 4 * static_cast<int>(sizeof(T))>*>(out) = y;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < end) out[e] = y.v[e];
  }
}

template <class Cfg>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Cfg::NTHREADS, 1)
entropy_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_out,
               const EntropyParams p) {
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BNH = Cfg::BNH, BK = Cfg::BK, NS = Cfg::NS, MODE = Cfg::MODE;
  constexpr bool WIDE = Cfg::WIDE;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* boxes = smem + NS * Cfg::STAGE;  // one to an epilogue warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(boxes + Cfg::EPI_WARPS * Cfg::BOX);
  uint64_t* full = bars;              // [NS] (leader's copy is used) the bytes of both CTAs landed
  uint64_t* stage_empty = bars + NS;  // [NS] the MMAs that read the stage are done (committed by the leader)
  uint64_t* acc_full = bars + 2 * NS;  // [2] accumulator complete (committed by the leader)
  uint64_t* acc_empty = acc_full + 2;  // [2] (leader's copy is used) read by the epilogues of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const uint32_t rank = warp_uniform(cluster_ctarank());
  const bool leader = rank == 0;
  const AbortCtl ctl{abort_flag, p.status};

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&stage_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 2 * Cfg::EPI_WARPS);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  cluster_sync_all();  // (both CTAs exist and have their barriers before anything crosses between them, the allocation too)
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);

  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  pdl_launch_dependents();
  pdl_wait();
  if constexpr (MODE == ENTROPY_STATS) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.arrived = 0;
  }

  // tile(t) for each tile of this pair in turn; leaves when one returns false.  A group of row tiles is gone over column by column: the pairs
  // that run at the same time share rows and columns through the L2 cache.
  struct Tile {
    int tm, un;       // row tile, column unit
    int n0, n1;       // columns
    int mma;          // columns of its MMAs: the multiple of 32 that holds them
    int k0, k1;       // k-blocks
    int part;         // where it goes if it is a part of a shared tile, else -1
    bool first, last;  // of its unit
  };
  const auto walk = [&](auto&& tile) {
    const auto unit = [&](int u, int k0, int k1, int part) {
      const int of_group = p.group * p.units_n;
      const int g = p.by_group(u), r = u - g * of_group;
      const int rows_here = min(p.group, p.tiles_m - g * p.group);
      Tile t;
      t.un = rows_here == p.group ? p.by_rows(r) : p.by_last(r);
      t.tm = g * p.group + r - t.un * rows_here;
      t.k0 = k0;
      t.k1 = k1;
      t.part = part;
      const int begin = t.un * p.unit_cols, end = min(begin + p.unit_cols, p.cols);
      for (t.n0 = begin; t.n0 < end; t.n0 = t.n1) {
        t.n1 = min(t.n0 + p.tile_cols, end);
        t.mma = (t.n1 - t.n0 + 31) & ~31;
        t.first = t.n0 == begin;
        t.last = t.n1 == end;
        if (!tile(t)) return false;
      }
      return true;
    };
    if constexpr (MODE == ENTROPY_OUT_X || MODE == ENTROPY_OUT_W) {
      // Part by part, so that pairs which run at the same time have the same contraction values: with parts of equal length for all
      // pairs, each from another place on, the operands came from memory again and again (2048 x 1024 of 50021 float16: 237 us, with two even parts 147).
      for (int u = pair; u < p.whole + p.shared * p.splits; u += npairs) {
        const int v = u - p.whole;
        if (v < 0) {
          if (!unit(u, 0, p.kblocks, -1)) return;
        } else {
          const int ks = p.by_shared(v), s = v - ks * p.shared, k0 = ks * p.kb_split;
          if (!unit(p.whole + s, k0, min(p.kblocks, k0 + p.kb_split), s * p.splits + ks)) return;
        }
      }
    } else {
      for (int u = pair; u < p.whole; u += npairs)
        if (!unit(u, 0, p.kblocks, -1)) return;
    }
  };
  const int drain = WIDE ? 1 : p.drain;  // k-blocks of an accumulator
  // The sums of a 256-column tile take 128 registers of a thread: the warps that copy and multiply hand theirs over.  (All that the block was launched
  // with, which launch_products makes sure of: 128 x 72 + 256 x 216 = 384 x 168.)
  if (warp < 4) {
    if constexpr (!WIDE) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer (this CTA's halves)
      // (Here and in the issuer the whole warp runs the loop and one elected lane issues: control flow and addresses are uniform and stay in
      // uniform registers.  One lane in a branch of its own took some 600 cycles for a stage whose MMAs take 512, or 256 where WIDE.)
      uint32_t it = 0;
      bool ok = true;
      walk([&](const Tile& t) {
        const int a0 = t.tm * (2 * BM) + static_cast<int>(rank) * BM;
        const int b0 = p.b_row + t.n0 + static_cast<int>(rank) * (t.mma >> 1);
        for (int kb = t.k0; kb < t.k1; ++kb) {
          const int ka = kb * BK, kw = p.b_k + kb * BK;
#pragma unroll
          for (int i = 0; i < Cfg::PLANES; ++i, ++it) {
            const int plane = WIDE ? (i + 2) % 3 : 0;  // 2, 0, 1
            const uint32_t s = it % NS;
            if (!(ok = mbar_wait_warp(&stage_empty[s], ((it / NS) & 1) ^ 1, ctl, STATUS_TIMEOUT_PRODUCER))) return false;
            if (elect_one_sync()) {
              if (leader) mbar_arrive_expect_tx(&full[s], 2 * Cfg::STAGE);
              const uint32_t bar = map_to_cta(smem_u32(&full[s]), 0);
              uint8_t* a = smem + s * Cfg::STAGE;
              uint8_t* b = a + Cfg::A_TILE;
              if constexpr (Cfg::A_MN) {
#pragma unroll
                for (int g = 0; g < BM / 64; ++g) tma_load_3d_pair(a + g * Cfg::MN_BOX, &tmap_a, bar, a0 + g * 64, ka, plane);
              } else {
                tma_load_3d_pair(a, &tmap_a, bar, ka, a0, plane);
              }
              if constexpr (Cfg::B_MN) {
#pragma unroll
                for (int g = 0; g < Cfg::B_BOXES; ++g) tma_load_3d_pair(b + g * Cfg::MN_BOX, &tmap_b, bar, b0 + g * 64, kw, plane);
              } else {
                tma_load_3d_pair(b, &tmap_b, bar, kw, b0, plane);
              }
            }
            __syncwarp();
          }
        }
        return true;
      });
      // The leader's commits arrive on both CTAs' stage_empty barriers: this CTA stays until the last ones are in.
      for (uint32_t d = ok ? min(it, static_cast<uint32_t>(NS)) : 0u; ok && d > 0; --d)
        ok = mbar_wait_warp(&stage_empty[(it - d) % NS], ((it - d) / NS) & 1, ctl, STATUS_TIMEOUT_PRODUCER);
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer (leader only)
      if (leader) {
        constexpr uint32_t STAGE_ENC = Cfg::STAGE >> 4;
        constexpr uint32_t a_step = Cfg::A_MN ? 128 : 2, b_step = Cfg::B_MN ? 128 : 2;  // 16 contraction values
        const uint32_t a_at = smem_u32(smem), b_at = a_at + Cfg::A_TILE;
        const uint64_t da0 = Cfg::A_MN ? umma_desc_mn16_sw128(a_at, Cfg::MN_BOX) : umma_desc_k_sw128(a_at);
        const uint64_t db0 = Cfg::B_MN ? umma_desc_mn16_sw128(b_at, Cfg::MN_BOX) : umma_desc_k_sw128(b_at);
        uint32_t s = 0, ph = 0, accs = 0;
        const auto advance = [&] {
          if (++s == NS) {
            s = 0;
            ph ^= 1;
          }
        };
        // rows of stage sa by columns of stage sb
        const auto multiply = [&](uint32_t d, uint32_t idesc, uint32_t sa, uint32_t sb, bool add) {
          const uint64_t da = da0 + sa * STAGE_ENC, db = db0 + sb * STAGE_ENC;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) umma_16_ss_pair(d, da + a_step * k, db + b_step * k, idesc, add || k > 0 ? 1u : 0u);
        };
        const auto free_stage = [&](uint32_t stage) { umma_commit_pair_mcast(smem_u32(&stage_empty[stage]), 3); };
        walk([&](const Tile& t) {
          const uint32_t idesc = p.idesc | static_cast<uint32_t>(t.mma >> 3) << 17;
          int sum_end = t.k0;  // of the k-blocks of this accumulator
          for (int kb = t.k0; kb < t.k1; ++kb) {
            const uint32_t buf = accs & 1, d = tmem_base + buf * Cfg::BUF_COLS;
            const bool begin = kb == sum_end;
            if (begin) {
              sum_end = min(kb + drain, t.k1);
              if (!mbar_wait_warp(&acc_empty[buf], ((accs >> 1) & 1) ^ 1, ctl, STATUS_TIMEOUT_MMA)) return false;
            }
            if (!mbar_wait_warp(&full[s], ph, ctl, STATUS_TIMEOUT_MMA)) return false;
            const bool done = kb + 1 == sum_end;
            if constexpr (WIDE) {
              // planes 2, 0 and 1 in three stages (of six: the three have the same parity of the wait); the first is free again after a third of the MMAs
              const uint32_t s2 = s, s0 = s + 1, s1 = s + 2;
              if (!mbar_wait_warp(&full[s0], ph, ctl, STATUS_TIMEOUT_MMA)) return false;
              tc_fence_after_sync();
              if (elect_one_sync()) {
                multiply(d, idesc, s2, s0, false);
                multiply(d, idesc, s0, s2, true);
                free_stage(s2);
              }
              __syncwarp();
              if (!mbar_wait_warp(&full[s1], ph, ctl, STATUS_TIMEOUT_MMA)) return false;
              tc_fence_after_sync();
              if (elect_one_sync()) {
                multiply(d, idesc, s1, s1, true);
                multiply(d, idesc, s1, s0, true);
                multiply(d, idesc, s0, s1, true);
                free_stage(s1);
                multiply(d, idesc, s0, s0, true);
                free_stage(s0);
                umma_commit_pair_mcast(smem_u32(&acc_full[buf]), 3);
              }
              advance();
              advance();
            } else {
              tc_fence_after_sync();
              if (elect_one_sync()) {
                multiply(d, idesc, s, s, !begin);
                free_stage(s);
                if (done) umma_commit_pair_mcast(smem_u32(&acc_full[buf]), 3);
              }
            }
            __syncwarp();
            advance();
            if (done) ++accs;
          }
          return true;
        });
      }
    }
  } else {
    if constexpr (!WIDE) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------------ epilogue: a row and half of the tile's columns to a thread
    const int q = warp & 3, h = (warp - 4) >> 2;
    uint8_t* box = boxes + (warp - 4) * Cfg::BOX;
    constexpr int CHUNKS = Cfg::COLS / 32;
    uint32_t accs = 0;
    static_assert(CHUNKS == 3 || CHUNKS == 4);
    float sum[CHUNKS][32];  // what the accumulators of a tile add up to

    // of the unit's row (STATS), of the tile's row (PROB)
    float top = -INFINITY, total = 0.f, lse = 0.f, g = 0.f;
    int64_t target = -1;
    bool ignored = false;
    const float alpha = MODE == ENTROPY_OUT_X || MODE == ENTROPY_OUT_W ? p.factors[1] : 1.f;
    const float factor = MODE == ENTROPY_PROB ? p.factors[0] : 1.f;

    walk([&](const Tile& t) {
      const int row0 = t.tm * (2 * BM) + static_cast<int>(rank) * BM + q * 32;  // of the warp
      const int row = row0 + lane;
      const int col0 = t.n0 + h * Cfg::COLS;                                    // of the thread
      const bool valid = row < p.rows;
      // (what comes from memory is looked at when the products are there)
      int64_t own = p.ignore;
      float own_lse = 0.f, own_dloss = 0.f;
      if constexpr (MODE == ENTROPY_STATS || MODE == ENTROPY_PROB) {
        if (t.first && valid) {
          own = entropy_target(p, row);
          if constexpr (MODE == ENTROPY_PROB) {
            own_lse = p.lse[row];
            own_dloss = p.dloss[p.per_row ? row : 0];
          }
        }
      }
      if constexpr (MODE == ENTROPY_OUT_X) {
        if (valid) own = entropy_target(p, row);
      }
      // chunks of 32 columns that this thread has in the tile
      const bool rows_exist = t.tm * (2 * BM) + static_cast<int>(rank) * BM < p.rows;
      const int chunks = rows_exist ? max(0, min(CHUNKS, (t.n1 - col0 + 31) >> 5)) : 0;

      // Results leave straight from registers, a sector of 32 bytes of its row to a thread: beside TMA and the MMAs there is no bandwidth of shared memory
      // left (through it the planes of a WIDE tile took 11 600 cycles, of which the exponentials 2 800).  Where the rows do not begin on sectors they go
      // through a box in shared memory, in rows of 128 bytes, and 32-bit ones of a short contraction too, from there by TMA (`boxed`).
      // 16-bit results, two to a word: chunk c of this thread's row into its half of the box; with the second half (or the last chunk) the box to memory.
      const auto box16 = [&](const uint32_t (&w)[16], int c, int c0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(box + lane * 128 + ((((c & 1) * 4 + j) ^ (lane & 7)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        if ((c & 1) == 0 && c + 1 < chunks) return;
        __syncwarp();
        const int begin = c0 - (c & 1) * 32, end = min(c0 + 32, t.n1);
        uint16_t* out = static_cast<uint16_t*>(p.out);
        if (p.out_vec) {
          const int cb = begin + (lane & 7) * 8;
#pragma unroll 2
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (row0 + r < p.rows && cb < end)
              *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row0 + r) * p.out_pitch + cb) = *reinterpret_cast<const uint4*>(box + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          }
        } else {
#pragma unroll 4
          for (int i = 0; i < 64; ++i) {
            const int r = i >> 1, at = (i & 1) * 32 + lane;
            if (row0 + r < p.rows && begin + at < end)
              out[static_cast<int64_t>(row0 + r) * p.out_pitch + begin + at] =
                  *reinterpret_cast<const uint16_t*>(box + r * 128 + (((at >> 3) ^ (r & 7)) << 4) + (at & 7) * 2);
          }
        }
        __syncwarp();
      };
      // 32 columns of the product from column c0 on.  (One copy of this code, in a loop over the chunks: unrolled over them it is fetched as slowly
      // as it is long, 8 000 cycles for a chunk.)
      const auto process = [&](float (&v)[32], int c) {
        const int c0 = col0 + c * 32;
        if constexpr (MODE == ENTROPY_STATS) {
          if (c0 + 32 > t.n1) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c0 + e >= t.n1) v[e] = -INFINITY;
          }
          const int at = target < t.n1 && target >= c0 && target < c0 + 32 ? static_cast<int>(target) - c0 : -1;
          if (__any_sync(0xffffffffu, at >= 0)) {
            float z = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) z = at == e ? v[e] : z;
            if (valid && at >= 0) p.picked[row] = z;
          }
          float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int e = 4; e < 32; ++e) m[e & 3] = fmaxf(m[e & 3], v[e]);
          const float now = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top);
          const float base = now == -INFINITY ? 0.f : now;
          float s[4] = {total * ex2_approx((top - base) * LOG2E_F), 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float e0, e1;
            exp_shifted_x2(v[e], v[e + 1], base, e0, e1);  // (multiplied first, a maximum from 1.5e9 on has an exponential of 0 or infinity)
            s[e & 3] += e0;
            s[(e + 1) & 3] += e1;
          }
          total = (s[0] + s[1]) + (s[2] + s[3]);
          top = now;
        } else if constexpr (MODE == ENTROPY_PROB) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float e0, e1;
            exp_shifted_x2(v[e], v[e + 1], lse, e0, e1);
            v[e] = e0 * g;
            v[e + 1] = e1 * g;
          }
          const int at = target >= c0 && target < c0 + 32 ? static_cast<int>(target) - c0 : -1;
          if (__any_sync(0xffffffffu, ignored || at >= 0)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if (at == e) v[e] -= g;
              if (ignored) v[e] = 0.f;  // (whatever its logits are)
            }
          }
          // Tiles have multiples of 32 columns here, and so has d.
          uint16_t* to = p.d + static_cast<int64_t>(row) * p.d_pitch + c0;
#pragma unroll 1
          for (int plane = 0; plane < Cfg::PLANES; ++plane, to += p.d_plane) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if constexpr (WIDE) {
                w[e] = plane_bits(v[2 * e], v[2 * e + 1]);
                v[2 * e] = plane_rest(v[2 * e]);
                v[2 * e + 1] = plane_rest(v[2 * e + 1]);
              } else {
                w[e] = pack16(v[2 * e], v[2 * e + 1], p.half);
              }
            }
            if (valid) {
              store_sector(to, w);
              store_sector(to + 16, w + 8);
            }
          }
        } else {
          if (!WIDE) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= alpha;
          }
          if constexpr (MODE == ENTROPY_OUT_X) {
            if (__any_sync(0xffffffffu, ignored)) {
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = ignored ? 0.f : v[e];  // (d is zero there, and 0 times an infinite weight is not)
            }
          }
          const auto as_bits = [&](int e) { return __float_as_uint(v[e]); };
          const auto store_floats = [&](float* to) {  // scratch memory, whose rows are on sectors
            if (!valid) return;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (c0 + 8 * j < t.n1) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = as_bits(8 * j + e);
                store_sector(to + 8 * j, w);
              }
            }
          };
          if (t.part >= 0) {
            store_floats(p.part + (static_cast<int64_t>(t.part) * (2 * BM) + static_cast<int>(rank) * BM + q * 32 + lane) * p.tile_cols + (c0 - t.n0));
            return;
          }
          if (p.dest != DEST_FINAL) {
            float* sums = p.sum + static_cast<int64_t>(row) * p.sum_pitch + c0;
            if (p.dest != DEST_SUM && valid) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (c0 + 8 * j < t.n1) {
                  uint32_t y[8];
                  load_sector(y, sums + 8 * j);
#pragma unroll
                  for (int e = 0; e < 8; ++e) v[8 * j + e] += __uint_as_float(y[e]);
                }
              }
            }
            if (p.dest != DEST_FINAL_ADD) {
              store_floats(sums);
              return;
            }
          }
          if constexpr (WIDE) {
            float* out = static_cast<float*>(p.out);
            if (p.boxed) {
              if (lane == 0) tma_store_wait_read<0>();
              __syncwarp();
            } else if (p.direct) {
              store_floats(out + static_cast<int64_t>(row) * p.out_pitch + c0);
              return;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            if (p.boxed) fence_proxy_async_smem();
            __syncwarp();
            if (p.boxed) {
              if (lane == 0 && row0 < p.rows) {
                tma_store_3d(&tmap_out, box, c0, row0, 0);
                tma_store_commit();
              }
              return;
            }
            if (p.out_vec) {
              const int cb = c0 + (lane & 7) * 4;
#pragma unroll 2
              for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + (lane >> 3);
                if (row0 + r < p.rows && cb < t.n1)
                  *reinterpret_cast<float4*>(out + static_cast<int64_t>(row0 + r) * p.out_pitch + cb) =
                      *reinterpret_cast<const float4*>(box + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
              }
            } else {
#pragma unroll 4
              for (int r = 0; r < 32; ++r) {
                if (row0 + r < p.rows && c0 + lane < t.n1)
                  out[static_cast<int64_t>(row0 + r) * p.out_pitch + c0 + lane] =
                      *reinterpret_cast<const float*>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
              }
            }
            __syncwarp();
          } else {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack16(v[2 * e], v[2 * e + 1], p.half);
            if (p.direct) {
              uint16_t* to = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(row) * p.out_pitch + c0;
              if (valid && c0 < t.n1) store_sector(to, w);
              if (valid && c0 + 16 < t.n1) store_sector(to + 16, w + 8);
            } else {
              box16(w, c, c0);
            }
          }
        }
      };

      for (int kb = t.k0; kb < t.k1; kb += drain, ++accs) {
        const uint32_t buf = accs & 1;
        if (!mbar_wait_warp(&acc_full[buf], (accs >> 1) & 1, ctl, STATUS_TIMEOUT_EPILOGUE)) return false;
        tc_fence_after_sync();
        const uint32_t empty = map_to_cta(smem_u32(&acc_empty[buf]), 0);
        const uint32_t at = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * Cfg::BUF_COLS + h * Cfg::COLS;
        if (kb == t.k0) {
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c)
            if (c < chunks) tmem_ld_32x32(at + c * 32, reinterpret_cast<uint32_t(&)[32]>(sum[c]));
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            if (c < chunks) {
              uint32_t ld[32];
              tmem_ld_32x32(at + c * 32, ld);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) sum[c][e] += __uint_as_float(ld[e]);
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(empty);
      }
      if constexpr (MODE == ENTROPY_STATS || MODE == ENTROPY_PROB) {
        if (t.first) {
          top = -INFINITY;
          total = 0.f;
          ignored = own == p.ignore;
          target = ignored ? -1 : own - p.b_row;
          lse = own_lse;
          g = ignored ? 0.f : own < 0 || own >= p.symbols ? __int_as_float(0x7fc00000) : own_dloss * factor;
        }
      }
      if constexpr (MODE == ENTROPY_OUT_X) ignored = own == p.ignore;
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float low = c == 0 ? sum[0][e] : sum[1][e], high = c == 2 || CHUNKS == 3 ? sum[2][e] : sum[CHUNKS - 1][e];
          v[e] = c < 2 ? low : high;
        }
        process(v, c);
      }
      if constexpr (MODE == ENTROPY_STATS) {
        if (t.last && valid) p.stats[(static_cast<int64_t>(t.un) * 2 + h) * p.rows + row] = make_float2(top, total);
      }
      return true;
    });
    if (WIDE && MODE == ENTROPY_OUT_W && lane == 0) tma_store_wait_all();
  }

  // ------------------------------------------------------------------ teardown
  // Neither CTA may leave while the other can still signal into its shared memory or use its half of the tensor memory.
  tc_fence_before_sync();
  cluster_sync_all();
  if (*abort_flag) {  // copies in flight still write into this block's shared memory
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
  }
  cluster_sync_all();
}

}  // namespace tb200
