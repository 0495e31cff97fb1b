// The products of the cross entropy for few rows of x (up to 64 at a time), which are bound by reading W: STATS, PROB and OUT_X with the operands'
// roles exchanged.  W's symbols (STATS, PROB) or columns (OUT_X) are the 128 rows of an MMA and the rows of x or d its columns, a multiple of 16
// of them, so that no copies and no MMAs are spent on rows that do not exist; one CTA to an SM, each with an even share of W.
//
// 16-bit W goes from TMA to the MMAs as it lies.  32-bit W (WIDE) is read as it lies, too, and not as planes that were written before: four warps take each stage
// apart and store its three planes to tensor memory, as the MMAs' row operand.  (W's planes written and read again: 64 rows of x,
// 50000 x 2048 symbols in float32, 376 us.)  x and d come as planes; they are small.
#pragma once

#include "entropy_kernel.cuh"

namespace tb200 {

template <int MODE_, bool WIDE_>
struct FewCfg {
  static constexpr int MODE = MODE_;
  static constexpr bool WIDE = WIDE_;
  static constexpr bool A_MN = MODE == ENTROPY_OUT_X;
  static constexpr int BM = 128;
  static constexpr int BN = 64;
  static constexpr int BK = 64;
  static constexpr int PLANES = WIDE ? 3 : 1;
  static constexpr int A_TILE = BM * BK * (WIDE ? 4 : 2);
  static constexpr int B_TILE = PLANES * BN * BK * 2;
  static constexpr int NSA = WIDE ? 3 : 8;  // stages of W
  static constexpr int NSB = WIDE ? 4 : 8;  // of the other operand
  static constexpr int MN_BOX = 64 * BK * 2;
  static constexpr int RAW_BOX = A_TILE / (A_MN ? 4 : 2);  // WIDE: boxes of 32 elements
  static constexpr int EPI_WARPS = 8;
  static constexpr int CUT_WARPS = WIDE ? 4 : 0;  // that take W apart
  static constexpr int NTHREADS = (4 + EPI_WARPS + CUT_WARPS) * 32;
  static constexpr int A_COL = 2 * BN;       // tensor memory: two accumulators, then two stages of W's planes
  static constexpr int A_COLS = 3 * BK / 2;  // of a stage
  static constexpr int TMEM_COLS = WIDE ? 512 : 128;
  static constexpr int NBAR = 2 * NSA + 2 * NSB + 8;
  static constexpr int SMEM_BYTES = 1024 + NSA * A_TILE + NSB * B_TILE + NBAR * 8 + 16 + EPI_WARPS * 32 * 16;
  static_assert(SMEM_BYTES <= 232448, "shared memory capacity");
};

struct FewParams {
  int rows;              // of x
  int length;            // of W's side: symbols of the piece (STATS, PROB), columns (OUT_X)
  int kblocks;
  int spans, span, tile;  // W's side: so many spans of so many symbols or columns, gone over in tiles of these (up to 128)
  int splits, kb_split;   // OUT_X: parts of the contraction
  int units;              // spans x splits x parts of 64 rows
  int mma_n;              // columns of the MMAs
  int a_bytes, b_bytes;   // of a stage's copies
  uint32_t idesc;
  int mean;              // PROB: dloss is that of the mean
  const void *x, *weight;  // STATS: as they were given, for the logits of the rows' own symbols
  int64_t x_stride, weight_stride;
  int width;
  EntropyParams e;        // what the forms have in common with those of entropy_kernel
};

__device__ __forceinline__ void umma_16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A from tensor memory: a row to a lane, two 16-bit contraction values to a column.
__device__ __forceinline__ void umma_16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// For each of 32 columns (v[e]: column e of this lane's row), in lane e: f over the rows of the warp.
template <class F>
__device__ __forceinline__ float columns_to_lanes(float (&v)[32], int lane, F f) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int e = 0; e < d; ++e) {
      const float keep = upper ? v[e + d] : v[e], send = upper ? v[e] : v[e + d];
      v[e] = f(keep, __shfl_xor_sync(0xffffffffu, send, d));
    }
  }
  return v[0];
}

// x[row] W[symbol], by a warp.
template <class T>
__device__ __forceinline__ float logit(const FewParams& p, int64_t row, int64_t symbol, int lane) {
  const T *x = static_cast<const T*>(p.x) + row * p.x_stride, *w = static_cast<const T*>(p.weight) + symbol * p.weight_stride;
  float s = 0.f;
#pragma unroll 8
  for (int c = lane; c < p.width; c += 32) s = fmaf(to_float(x[c]), to_float(w[c]), s);
  return warp_sum(s);
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::NTHREADS, 1)
entropy_few_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ FewParams p) {
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BK = Cfg::BK, NSA = Cfg::NSA, NSB = Cfg::NSB, MODE = Cfg::MODE;
  constexpr bool WIDE = Cfg::WIDE;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* b_base = smem + NSA * Cfg::A_TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(b_base + NSB * Cfg::B_TILE);
  uint64_t* a_full = bars;                 // [NSA] W's bytes landed
  uint64_t* a_empty = a_full + NSA;        // [NSA] read by the MMAs, or (WIDE) by the warps that take it apart
  uint64_t* b_full = a_empty + NSA;        // [NSB]
  uint64_t* b_empty = b_full + NSB;        // [NSB]
  uint64_t* acc_full = b_empty + NSB;      // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2]
  uint64_t* cut_full = acc_empty + 2;      // [2] WIDE: planes in tensor memory
  uint64_t* cut_empty = cut_full + 2;      // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(cut_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* of_done = reinterpret_cast<int*>(tmem_slot + 2);          // [2] STATS: warps of a half of the rows that have left their part
  uint8_t* of_rows = reinterpret_cast<uint8_t*>(tmem_slot + 4);  // [8][32 * 16] PROB: what each epilogue warp needs of its rows of x
  float2* of_stats = reinterpret_cast<float2*>(of_rows);         // [8][32] STATS: those parts

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const AbortCtl ctl{abort_flag, p.e.status};

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    of_done[0] = of_done[1] = 0;
    for (int s = 0; s < NSA; ++s) {
      mbar_init(&a_full[s], 1);
      mbar_init(&a_empty[s], WIDE ? Cfg::CUT_WARPS : 1);
    }
    for (int s = 0; s < NSB; ++s) {
      mbar_init(&b_full[s], 1);
      mbar_init(&b_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], Cfg::EPI_WARPS);
      mbar_init(&cut_full[s], WIDE ? Cfg::CUT_WARPS : 1);
      mbar_init(&cut_empty[s], 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  pdl_launch_dependents();
  pdl_wait();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);

  const int drain = WIDE ? 1 : p.e.drain;  // k-blocks of an accumulator
  struct Tile {
    int span, ks;      // which span and which part of the contraction
    int n0;            // first row of x
    int m0, m1;        // symbols, or columns of W
    int k0, k1;
    bool first, last;  // of its unit
  };
  const auto walk = [&](auto&& tile) {
    for (int u = blockIdx.x; u < p.units; u += gridDim.x) {  // (STATS, PROB: one)
      const int of_tile = p.spans * p.splits;
      Tile t;
      t.n0 = u / of_tile * BN;
      const int r = u % of_tile;
      t.ks = r / p.spans;
      t.span = r - t.ks * p.spans;
      t.k0 = t.ks * p.kb_split;
      t.k1 = min(p.kblocks, t.k0 + p.kb_split);
      const int begin = t.span * p.span, end = min(begin + p.span, p.length);
      for (t.m0 = begin; t.m0 < end; t.m0 = t.m1) {
        t.m1 = min(t.m0 + p.tile, end);
        t.first = t.m0 == begin;
        t.last = t.m1 == end;
        if (!tile(t)) return;
      }
    }
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    uint32_t it = 0;
    bool ok = true;
    walk([&](const Tile& t) {
      for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
        const uint32_t sa = it % NSA, sb = it % NSB;
        if (!(ok = mbar_wait_warp(&a_empty[sa], ((it / NSA) & 1) ^ 1, ctl, STATUS_TIMEOUT_PRODUCER))) return false;
        if (elect_one_sync()) {
          mbar_arrive_expect_tx(&a_full[sa], p.a_bytes);
          uint8_t* a = smem + sa * Cfg::A_TILE;
          const int k = p.e.b_k + kb * BK, m = p.e.b_row + t.m0;
          if constexpr (Cfg::A_MN) {
#pragma unroll
            for (int g = 0; g < (WIDE ? 4 : 2); ++g)
              tma_load_3d(a + g * (WIDE ? Cfg::RAW_BOX : Cfg::MN_BOX), &tmap_a, &a_full[sa], m + g * (WIDE ? 32 : 64), k, 0);
          } else {
#pragma unroll
            for (int g = 0; g < (WIDE ? 2 : 1); ++g) tma_load_3d(a + g * Cfg::RAW_BOX, &tmap_a, &a_full[sa], k + g * 32, m, 0);
          }
        }
        __syncwarp();
        if (!(ok = mbar_wait_warp(&b_empty[sb], ((it / NSB) & 1) ^ 1, ctl, STATUS_TIMEOUT_PRODUCER))) return false;
        if (elect_one_sync()) {
          mbar_arrive_expect_tx(&b_full[sb], p.b_bytes);
#pragma unroll
          for (int plane = 0; plane < Cfg::PLANES; ++plane)
            tma_load_3d(b_base + sb * Cfg::B_TILE + plane * (BN * BK * 2), &tmap_b, &b_full[sb], kb * BK, t.n0, plane);
        }
        __syncwarp();
      }
      return true;
    });
    // The MMAs' commits arrive on this CTA's barriers: it stays until the last ones are in.
    for (uint32_t d = ok ? min(it, static_cast<uint32_t>(NSB)) : 0u; ok && d > 0; --d)
      ok = mbar_wait_warp(&b_empty[(it - d) % NSB], ((it - d) / NSB) & 1, ctl, STATUS_TIMEOUT_PRODUCER);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const uint64_t da0 = Cfg::A_MN ? umma_desc_mn16_sw128(smem_u32(smem), Cfg::MN_BOX) : umma_desc_k_sw128(smem_u32(smem));
    const uint64_t db0 = umma_desc_k_sw128(smem_u32(b_base));
    uint32_t it = 0, accs = 0;
    walk([&](const Tile& t) {
      int sum_end = t.k0;  // of the k-blocks of this accumulator
      for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
        const uint32_t sa = it % NSA, sb = it % NSB, buf = accs & 1, d = tmem_base + buf * BN;
        const bool begin = kb == sum_end;
        if (begin) {
          sum_end = min(kb + drain, t.k1);
          if (!mbar_wait_warp(&acc_empty[buf], ((accs >> 1) & 1) ^ 1, ctl, STATUS_TIMEOUT_MMA)) return false;
        }
        if (!mbar_wait_warp(&b_full[sb], (it / NSB) & 1, ctl, STATUS_TIMEOUT_MMA)) return false;
        if (WIDE) {
          if (!mbar_wait_warp(&cut_full[it & 1], (it >> 1) & 1, ctl, STATUS_TIMEOUT_MMA)) return false;
        } else {
          if (!mbar_wait_warp(&a_full[sa], (it / NSA) & 1, ctl, STATUS_TIMEOUT_MMA)) return false;
        }
        tc_fence_after_sync();
        const bool done = kb + 1 == sum_end;
        if (elect_one_sync()) {
          const uint64_t db = db0 + sb * (Cfg::B_TILE >> 4);
          if constexpr (WIDE) {
            constexpr int plane_a[6] = {2, 0, 1, 1, 0, 0}, plane_b[6] = {0, 2, 1, 0, 1, 0};  // the smallest products first
            const uint32_t at = tmem_base + Cfg::A_COL + (it & 1) * Cfg::A_COLS;
#pragma unroll
            for (int x = 0; x < 6; ++x)
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                umma_16_ts(d, at + plane_a[x] * (BK / 2) + k * 8, db + plane_b[x] * (BN * BK * 2 >> 4) + 2 * k, p.idesc, x > 0 || k > 0 ? 1u : 0u);
            umma_commit(&cut_empty[it & 1]);
          } else {
            const uint64_t da = da0 + sa * (Cfg::A_TILE >> 4);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) umma_16_ss(d, da + (Cfg::A_MN ? 128 : 2) * k, db + 2 * k, p.idesc, !begin || k > 0 ? 1u : 0u);
            umma_commit(&a_empty[sa]);
          }
          umma_commit(&b_empty[sb]);
          if (done) umma_commit(&acc_full[buf]);
        }
        __syncwarp();
        if (done) ++accs;
      }
      return true;
    });
  } else if (warp == 2) {
    // ------------------------------------------------------------------ STATS: the logits of the rows' own symbols, a row to a CTA
    if constexpr (MODE == ENTROPY_STATS) {
      if (blockIdx.x == 0 && lane == 0) *p.e.arrived = 0;
      for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t t = entropy_target(p.e, row);
        if (t < 0 || t >= p.e.symbols) continue;
        float z;
        if constexpr (WIDE) {
          z = logit<float>(p, row, t, lane);
        } else {
          z = p.e.half ? logit<__half>(p, row, t, lane) : logit<__nv_bfloat16>(p, row, t, lane);
        }
        if (lane == 0) p.e.picked[row] = z;
      }
    }
  } else if (warp >= 4 && warp < 12) {
    // ------------------------------------------------------------------ epilogue: a row of the MMAs and 32 of their columns to a thread
    const int q = warp & 3, h = (warp - 4) >> 2;
    uint32_t accs = 0;
    float sum[32];
    float top = -INFINITY, total = 0.f;  // STATS: of row h * 32 + lane of x, over the warp's symbols of the unit
    const float alpha = MODE == ENTROPY_OUT_X ? p.e.factors[1] : 1.f;
    int64_t* of_target = reinterpret_cast<int64_t*>(of_rows + (warp - 4) * (32 * 16));
    float* of_lse = reinterpret_cast<float*>(of_target + 32);
    float* of_g = of_lse + 32;

    float factor = 1.f;
    if constexpr (MODE == ENTROPY_PROB) {  // (few rows: each warp finds this for itself)
      float largest = 0.f;
      int count = 0;
      for (int i = lane; i < p.rows; i += 32) {
        if (entropy_target(p.e, i) == p.e.ignore) continue;
        ++count;
        const float g = fabsf(p.e.dloss[p.e.per_row ? i : 0]);
        if (g < INFINITY) largest = fmaxf(largest, g);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        count += __shfl_xor_sync(0xffffffffu, count, o);
      }
      const float2 f = entropy_factors(largest, count, p.mean, entropy_scale(Cfg::WIDE, p.e.half, p.e.per_row));
      factor = f.x;
      if (blockIdx.x == 0 && threadIdx.x == 128) p.e.factors[1] = f.y;  // for the products that follow
    }

    walk([&](const Tile& t) {
      const int m = t.m0 + q * 32 + lane;  // symbol of the piece, or column
      const bool valid = m < t.m1;
      const int n = t.n0 + h * 32;         // first row of x
      const int count = max(0, min(32, p.rows - n));
      if constexpr (MODE == ENTROPY_STATS) {
        if (t.first) {
          top = -INFINITY;
          total = 0.f;
        }
      }
      if constexpr (MODE == ENTROPY_PROB) {
        if (t.first) {
          const int64_t to = lane < count ? entropy_target(p.e, n + lane) : p.e.ignore;
          const bool ignored = to == p.e.ignore;
          const float lse = lane < count ? p.e.lse[n + lane] : 0.f;
          __syncwarp();
          of_target[lane] = ignored ? -1 : to - p.e.b_row;
          of_lse[lane] = ignored ? INFINITY : lse;  // (no lse is that: infinite logits make it NaN)
          of_g[lane] = ignored ? 0.f : to < 0 || to >= p.e.symbols ? __int_as_float(0x7fc00000) : p.e.dloss[p.e.per_row ? n + lane : 0] * factor;
          __syncwarp();
        }
      }
      unsigned ignored = 0;  // OUT_X: rows whose d is zero, which 0 times an infinite weight is not
      if constexpr (MODE == ENTROPY_OUT_X) ignored = __ballot_sync(0xffffffffu, lane < count && entropy_target(p.e, n + lane) == p.e.ignore);
      for (int kb = t.k0; kb < t.k1; kb += drain, ++accs) {
        const uint32_t buf = accs & 1;
        if (!mbar_wait_warp(&acc_full[buf], (accs >> 1) & 1, ctl, STATUS_TIMEOUT_EPILOGUE)) return false;
        tc_fence_after_sync();
        if (count > 0) {
          uint32_t ld[32];
          tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BN + h * 32, ld);
          tmem_ld_wait();
          if (kb == t.k0) {
#pragma unroll
            for (int e = 0; e < 32; ++e) sum[e] = __uint_as_float(ld[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) sum[e] += __uint_as_float(ld[e]);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
      }
      if (count == 0) return true;
      if constexpr (MODE == ENTROPY_STATS) {
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = sum[e] = valid ? sum[e] : -INFINITY;
        const float high = columns_to_lanes(v, lane, [](float a, float b) { return fmaxf(a, b); });
        const float now = fmaxf(top, high), base = now == -INFINITY ? 0.f : now;
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = ex2_approx((sum[e] - __shfl_sync(0xffffffffu, base, e)) * LOG2E_F);
        total = total * ex2_approx((top - base) * LOG2E_F) + columns_to_lanes(v, lane, [](float a, float b) { return a + b; });
        top = now;
        if (t.last) {
          // the four warps of these rows of x leave theirs to the last one of them (a CTA has one unit: this happens once)
          of_stats[(h * 4 + q) * 32 + lane] = make_float2(top, total);
          __threadfence_block();
          __syncwarp();
          const int order = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(&of_done[h], 1) : 0, 0);
          if (order == 3) {
            __threadfence_block();
            float m4 = -INFINITY, s4 = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) m4 = fmaxf(m4, of_stats[(h * 4 + k) * 32 + lane].x);
            const float b4 = m4 == -INFINITY ? 0.f : m4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 a = of_stats[(h * 4 + k) * 32 + lane];
              s4 = fmaf(a.y, ex2_approx((a.x - b4) * LOG2E_F), s4);
            }
            if (lane < count) p.e.stats[static_cast<int64_t>(t.span) * p.rows + n + lane] = make_float2(m4, s4);
          }
        }
      } else if constexpr (MODE == ENTROPY_PROB) {
        if (valid) {
          uint16_t* to = p.e.d + static_cast<int64_t>(n) * p.e.d_pitch + m;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (e < count) {
              const float lse = of_lse[e], g = of_g[e];
              float x = lse == INFINITY ? 0.f : exp_shifted(sum[e], lse) * g;
              if (of_target[e] == m) x -= g;
              if constexpr (WIDE) {
#pragma unroll
                for (int plane = 0; plane < 3; ++plane) {
                  to[e * p.e.d_pitch + plane * p.e.d_plane] = static_cast<uint16_t>(__float_as_uint(x) >> 16);
                  x = plane_rest(x);
                }
              } else {
                to[e * p.e.d_pitch] = static_cast<uint16_t>(pack16(x, 0.f, p.e.half));
              }
            }
          }
        }
      } else {
        if (valid) {
          // a column of W and the rows of x to a thread: neighbouring lanes write neighbouring elements of dx
          float* part = p.e.part + (static_cast<int64_t>(t.ks) * p.rows + n) * p.e.sum_pitch + m;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (e < count) part[e * p.e.sum_pitch] = ignored >> e & 1 ? 0.f : sum[e] * alpha;
          }
        }
      }
      return true;
    });
  } else if (WIDE && warp >= 12) {
    // ------------------------------------------------------------------ W's stages taken apart: a row of the MMAs to a thread
    const int r = (warp - 12) * 32 + lane;
    uint32_t it = 0;
    walk([&](const Tile& t) {
      for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
        const uint32_t sa = it % NSA, buf = it & 1;
        if (!mbar_wait_warp(&a_full[sa], (it / NSA) & 1, ctl, STATUS_TIMEOUT_TRANSFORM)) return false;
        if (!mbar_wait_warp(&cut_empty[buf], ((it >> 1) & 1) ^ 1, ctl, STATUS_TIMEOUT_TRANSFORM)) return false;
        tc_fence_after_sync();
        const uint8_t* a = smem + sa * Cfg::A_TILE;
        const uint32_t at = tmem_base + (static_cast<uint32_t>((warp - 12) * 32) << 16) + Cfg::A_COL + buf * Cfg::A_COLS;
#pragma unroll
        for (int g = 0; g < 2; ++g) {  // 32 contraction values: 16 columns of each plane
          float v[32];
          if constexpr (Cfg::A_MN) {
            const uint8_t* box = a + (r >> 5) * Cfg::RAW_BOX;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const int kk = g * 32 + k;
              v[k] = *reinterpret_cast<const float*>(box + kk * 128 + ((((r & 31) >> 2) ^ (kk & 7)) << 4) + (r & 3) * 4);
            }
          } else {
            const uint8_t* box = a + g * Cfg::RAW_BOX + r * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float4 x = *reinterpret_cast<const float4*>(box + ((c ^ (r & 7)) << 4));
              v[4 * c] = x.x;
              v[4 * c + 1] = x.y;
              v[4 * c + 2] = x.z;
              v[4 * c + 3] = x.w;
            }
          }
#pragma unroll
          for (int plane = 0; plane < 3; ++plane) {
            float w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              w[k] = __uint_as_float(plane_bits(v[2 * k], v[2 * k + 1]));
              v[2 * k] = plane_rest(v[2 * k]);
              v[2 * k + 1] = plane_rest(v[2 * k + 1]);
            }
            tmem_st_32x16(at + plane * (BK / 2) + g * 16, w);
          }
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&a_empty[sa]);
          mbar_arrive(&cut_full[buf]);
        }
      }
      return true;
    });
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {  // copies in flight still write into this block's shared memory
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace tb200
