// Sampling of one symbol per row of logits from given exponential noise.
//
//   p_i = exp((x_i - max x) / T).  In the order of falling x (equal ones by index): the first top_k; of these the fewest whose sum of p
//   reaches top_p times theirs; of these the ones with p >= min_p.  Of what is kept, the symbol with the largest p_i / noise_i, and
//   log(p_i / sum of p kept).
//
// For exponential noise the largest p / noise falls on i with probability p_i / sum p.  No place on a cumulative sum decides, and so no order
// of additions: what is kept is a prefix of the sorted row, and only its end depends on sums.
//
// A row belongs to a cluster of blocks, each of which holds its slice in shared memory.  No row is sorted.  Filters find the end of the
// kept prefix from a histogram of (max - x) / T in steps of 1/16 (a factor of 1.06 of p): the bins down to one that surely reach far
// enough hold some tens to hundreds of symbols as a rule, which the first block of the cluster gathers, sorts and finishes alone.  Where there
// are more than it has room for (flat rows, many equal values), the end is found by radix selection over the bits of x and then over
// the index.  Counts and, as multiples of a power of two, masses are added as integers, so that a result does not depend on the order of
// the atomic additions.
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "../../include/triturus_b200.h"
#include "packs.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = 2048;  // symbols that are sorted

struct SampleArgs {
  const void* logits;
  const float* noise;
  int64_t* token;
  float* logprob;  // may be nullptr
  int64_t logits_stride, noise_stride;
  int symbols;
  int slice;       // of a block, a multiple of 8
  const float* temperature;  // [rows], or nullptr: the number beside it
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature0, top_p0, min_p0;
  int top_k0;
};

struct Shared {
  unsigned long long list[kList];
  uint32_t count[kBins];     // the block's
  uint32_t mass[kBins];      // the block's, as multiples of 2^-clz(count)
  uint32_t all_count[kBins]; // the cluster's
  double all_mass[kBins];
  float red[2][kWarps];
  int red_i[2][kWarps];
  float out_f[4];            // read by the other blocks
  int out_i[4];
  double pick_d[2];
  uint32_t pick[4];
  uint32_t listed;
};

// A word of another block's shared memory.
__device__ __forceinline__ uint32_t peer_u32(const void* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long peer_u64(const void* p, int rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ float peer_f32(const void* p, int rank) { return __uint_as_float(peer_u32(p, rank)); }

// All threads of the row's blocks.
template <int C>
__device__ __forceinline__ void row_sync() {
  if (C > 1)
    cluster_sync_all();
  else
    __syncthreads();
}

// Bits in the order of the values.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// What the blocks of a row share of it.
struct Row {
  float top;      // its largest value
  float k2;       // log2(e) / T
  uint32_t ckey;  // kept so far: keys above ckey, and of those equal to it the indexes up to cidx
  int cidx;
};
__device__ __forceinline__ float prob(const Row& r, float x) { return ex2_approx((x - r.top) * r.k2); }
__device__ __forceinline__ bool keeps(const Row& r, uint32_t key, int idx) { return key > r.ckey || (key == r.ckey && idx <= r.cidx); }

// The block's slice: element j (0 ... slice) is symbol first + j of the row, those below 0 and from `symbols` on are -inf.
template <class T, bool HELD>
struct Slice {
  const T* row;
  float* held;
  int first, size, symbols;
  __device__ __forceinline__ float at(int j) const {
    if (HELD) return held[j];
    const int i = first + j;
    if (i < 0 || i >= symbols) return -INFINITY;
    return fminf(to_float(row[i]), FLT_MAX) + 0.f;
  }
};

// Loads the slice; the thread's largest value, and whether it saw a NaN.  Infinity counts as the largest number, -0 as 0.
template <class T, bool HELD>
__device__ __forceinline__ void load_slice(const Slice<T, HELD>& s, float& top, int& nan) {
  constexpr int N = Pack<T, 16>::N;
  top = -INFINITY;
  nan = 0;
  for (int j = static_cast<int>(threadIdx.x) * N; j < s.size; j += kThreads * N) {
    const int i = s.first + j;
    float v[N];
    if (i >= 0 && i + N <= s.symbols) {
      const Pack<T, 16> p = *reinterpret_cast<const Pack<T, 16>*>(s.row + i);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = to_float(p.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = i + e >= 0 && i + e < s.symbols ? to_float(s.row[i + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      nan |= v[e] != v[e];
      v[e] = fminf(v[e], FLT_MAX) + 0.f;
      top = fmaxf(top, v[e]);
      if (HELD) s.held[j + e] = v[e];
    }
  }
}

// Sum over the row of a value of each thread: warps, the block, then the blocks by rank.  Every thread has it.
template <int C>
__device__ __forceinline__ float row_sum(float v, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = block_sum(v, sh.red[0], warp, lane, kWarps);
  if (C == 1) {
    __syncthreads();
    return v;
  }
  if (threadIdx.x == 0) sh.out_f[1] = v;
  cluster_sync_all();
  float s = 0.f;
#pragma unroll
  for (int r = 0; r < C; ++r) s += peer_f32(&sh.out_f[1], r);
  cluster_sync_all();
  return s;
}

// The cluster's counts (and masses, each block's in units of its own) from the blocks' ones.  `mass_of_bin(b)`: p at the upper end of a bin.
template <int C, class F>
__device__ __forceinline__ void merge_bins(Shared& sh, bool masses, F mass_of_bin) {
  row_sync<C>();
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    uint32_t n = 0;
    double m = 0.0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const uint32_t c = C > 1 ? peer_u32(&sh.count[b], r) : sh.count[b];
      n += c;
      if (masses && c != 0) m += ldexp(static_cast<double>(C > 1 ? peer_u32(&sh.mass[b], r) : sh.mass[b]), -__clz(static_cast<int>(c)));
    }
    sh.all_count[b] = n;
    if (masses) sh.all_mass[b] = n != 0 ? m * static_cast<double>(mass_of_bin(b)) : 0.0;
  }
  row_sync<C>();
}

// The end of the prefix of the kept symbols whose number, or mass, first reaches `target` (more than nothing, at most what there is), by
// radix selection over all of the row.  Sets r.ckey and r.cidx.
template <int C, class T, bool HELD>
__device__ void select_end(const Slice<T, HELD>& s, Shared& sh, Row& r, bool by_mass, double target) {
  const int tid = threadIdx.x;
  uint32_t hi = key_of(r.top), lo = max(r.ckey, key_of(-FLT_MAX));
  double above = 0.0;
  uint32_t ties = 0;
  for (;;) {
    const uint32_t range = hi - lo;
    const int shift = max(0, 24 - __clz(static_cast<int>(range)));  // at most 256 bins
    for (int b = tid; b < kBins; b += kThreads) sh.count[b] = sh.mass[b] = 0;
    __syncthreads();
    for (int j = tid; j < s.size; j += kThreads) {
      const float x = s.at(j);
      const uint32_t key = key_of(x);
      if (x > -INFINITY && key >= lo && key <= hi && keeps(r, key, s.first + j)) atomicAdd(&sh.count[(hi - key) >> shift], 1u);
    }
    auto upper = [&](int b) { return fminf(value_of(hi - (static_cast<uint32_t>(b) << shift)), r.top); };
    if (by_mass) {
      __syncthreads();
      for (int j = tid; j < s.size; j += kThreads) {
        const float x = s.at(j);
        const uint32_t key = key_of(x);
        if (x > -INFINITY && key >= lo && key <= hi && keeps(r, key, s.first + j)) {
          const int b = static_cast<int>((hi - key) >> shift);
          // (the count's bits and the mass's make 32: no overflow)
          const float e = fminf(ex2_approx((x - upper(b)) * r.k2), 1.f);
          atomicAdd(&sh.mass[b], static_cast<uint32_t>(ldexpf(e, __clz(static_cast<int>(sh.count[b])))));
        }
      }
    }
    merge_bins<C>(sh, by_mass, [&](int b) { return prob(r, upper(b)); });
    if (tid == 0) {
      double sum = above;
      int b = 0, last = 0;
      double before = above;
      for (; b < kBins; ++b) {
        if (sh.all_count[b] == 0) continue;
        last = b;
        before = sum;
        sum += by_mass ? sh.all_mass[b] : static_cast<double>(sh.all_count[b]);
        if (sum >= target) break;
      }
      sh.pick[0] = static_cast<uint32_t>(last);
      sh.pick[1] = sh.all_count[last];
      sh.pick_d[0] = before;
    }
    __syncthreads();
    const uint32_t b = sh.pick[0];
    ties = sh.pick[1];
    above = sh.pick_d[0];
    hi -= b << shift;
    lo = max(lo, hi - ((1u << shift) - 1u));
    __syncthreads();
    if (shift == 0) break;
  }
  // all that is left has one value: the first few by index
  const double each = by_mass ? static_cast<double>(prob(r, value_of(hi))) : 1.0;
  const double wanted = each > 0.0 ? ceil((target - above) / each) : 1.0;
  uint32_t want = wanted < 1.0 ? 1u : wanted < static_cast<double>(ties) ? static_cast<uint32_t>(wanted) : ties;
  int from = 0, to = s.symbols;  // the index is in [from, to)
  if (want < ties) {
    while (to - from > 1) {
      const int width = (to - from + kBins - 1) / kBins;
      for (int b = tid; b < kBins; b += kThreads) sh.count[b] = 0;
      __syncthreads();
      for (int j = tid; j < s.size; j += kThreads) {
        const int i = s.first + j;
        if (i >= from && i < to && key_of(s.at(j)) == hi && keeps(r, hi, i)) atomicAdd(&sh.count[(i - from) / width], 1u);
      }
      merge_bins<C>(sh, false, [](int) { return 0.f; });
      if (tid == 0) {
        uint32_t sum = 0;
        int b = 0;
        while (b < kBins - 1 && sum + sh.all_count[b] < want) sum += sh.all_count[b++];
        sh.pick[0] = static_cast<uint32_t>(b);
        sh.pick[1] = sum;
      }
      __syncthreads();
      from += static_cast<int>(sh.pick[0]) * width;
      to = min(to, from + width);
      want -= sh.pick[1];
      __syncthreads();
    }
    r.cidx = from;
  } else if (hi != r.ckey) {
    r.cidx = INT32_MAX;
  }
  r.ckey = hi;
}

// The better of two candidates: the larger score, of equal ones the lower index.
__device__ __forceinline__ void better(float& score, int& idx, float s2, int i2) {
  if (s2 > score || (s2 == score && i2 < idx)) {
    score = s2;
    idx = i2;
  }
}

// The block's best candidate and sum, in all threads of warp 0.
__device__ __forceinline__ void block_best(float& score, int& idx, float& sum, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(score, idx, __shfl_xor_sync(0xffffffffu, score, o), __shfl_xor_sync(0xffffffffu, idx, o));
  sum = warp_sum(sum);
  if (lane == 0) {
    sh.red[0][warp] = score;
    sh.red[1][warp] = sum;
    sh.red_i[0][warp] = idx;
  }
  __syncthreads();
  if (warp == 0) {
    score = lane < kWarps ? sh.red[0][lane] : -1.f;
    idx = lane < kWarps ? sh.red_i[0][lane] : INT32_MAX;
    sum = warp_sum(lane < kWarps ? sh.red[1][lane] : 0.f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) better(score, idx, __shfl_xor_sync(0xffffffffu, score, o), __shfl_xor_sync(0xffffffffu, idx, o));
  }
}

__device__ __forceinline__ void write_answer(const SampleArgs& p, int64_t row, const Row& r, int idx, float x, float sum) {
  p.token[row] = idx;
  if (p.logprob != nullptr) p.logprob[row] = (x - r.top) * r.k2 * 0.6931471805599453f - logf(sum);
}

template <class T, bool HELD, int C>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t row = blockIdx.x / C;

  Slice<T, HELD> s;
  s.row = static_cast<const T*>(p.logits) + row * p.logits_stride;
  s.held = reinterpret_cast<float*>(smem_raw + sizeof(Shared));
  // the row's slices begin on 16-byte boundaries of memory
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(s.row) & 15) / sizeof(T));
  s.first = rank * p.slice - skip;
  s.size = p.slice;
  s.symbols = p.symbols;
  const float* noise = p.noise + row * p.noise_stride;

  float temperature = p.temperature != nullptr ? p.temperature[row] : p.temperature0;
  int top_k = p.top_k != nullptr ? p.top_k[row] : p.top_k0;
  float top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p0;
  const float min_p = fminf(p.min_p != nullptr ? p.min_p[row] : p.min_p0, 1.f);
  if (!(temperature > 0.f)) {  // the most probable symbol
    temperature = 1.f;
    top_k = 1;
  }

  float top;
  int nan;
  load_slice(s, top, nan);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) {
    sh.red[0][warp] = top;
    sh.red_i[0][warp] = nan;
  }
  if (tid == 0) sh.listed = 0;
  for (int b = tid; b < kBins; b += kThreads) sh.count[b] = 0;
  __syncthreads();
  top = -INFINITY;
  nan = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    top = fmaxf(top, sh.red[0][w]);
    nan |= sh.red_i[0][w];
  }
  if (C > 1) {
    if (tid == 0) {
      sh.out_f[0] = top;
      sh.out_i[0] = nan;
    }
    cluster_sync_all();
#pragma unroll
    for (int q = 0; q < C; ++q) {
      top = fmaxf(top, peer_f32(&sh.out_f[0], q));
      nan |= static_cast<int>(peer_u32(&sh.out_i[0], q));
    }
  } else {
    __syncthreads();
  }
  Row r;
  r.top = top;
  r.k2 = fminf(fmaxf(LOG2E_F / temperature, 1e-38f), FLT_MAX);
  r.ckey = 0;
  r.cidx = INT32_MAX;

  if (nan || top == -INFINITY) {  // (the same for all blocks of the row)
    if (rank == 0 && tid == 0) {
      p.token[row] = -1;
      if (p.logprob != nullptr) p.logprob[row] = nan ? NAN : -INFINITY;
    }
    if (C > 1) cluster_sync_all();
    return;
  }

  bool by_count = top_k > 0 && top_k < p.symbols;
  const bool by_mass = top_p < 1.f;
  if (by_count || by_mass) {
    // ---- the histogram
    const float to_bin = r.k2 * (16.f / LOG2E_F);
    auto bin_of = [&](float x) { return static_cast<int>(fminf((r.top - x) * to_bin, 255.f)); };
    float z = 0.f;
    for (int j = tid; j < s.size; j += kThreads) {
      const float x = s.at(j);
      if (x > -INFINITY) {
        atomicAdd(&sh.count[bin_of(x)], 1u);
        z += prob(r, x);
      }
    }
    if (!by_count) z = row_sum<C>(z, sh);
    merge_bins<C>(sh, false, [](int) { return 0.f; });
    if (tid < 32) {
      // lane l has bins 8 l ... 8 l + 7
      uint32_t n[8], total = 0;
      float least[8], mass = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[i] = sh.all_count[lane * 8 + i];
        total += n[i];
        least[i] = lane * 8 + i < kBins - 1 ? static_cast<float>(n[i]) * ex2_approx(-LOG2E_F / 16.f * static_cast<float>(lane * 8 + i + 1)) : 0.f;
        mass += least[i];
      }
      uint32_t upto = total;
      float mass_upto = mass;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
        const float f = __shfl_up_sync(0xffffffffu, mass_upto, o);
        if (lane >= o) {
          upto += u;
          mass_upto += f;
        }
      }
      const uint32_t everything = __shfl_sync(0xffffffffu, upto, 31);
      uint32_t cum = upto - total;
      float cum_mass = mass_upto - mass;
      int bin = kBins;  // the first that surely reaches the end
      uint32_t listed = 0;
      const bool count_first = by_count && static_cast<uint32_t>(top_k) < everything;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cum += n[i];
        cum_mass += least[i];
        const bool there = count_first ? cum >= static_cast<uint32_t>(top_k) : by_mass && !by_count && cum_mass >= top_p * z * 1.0001f;
        if (there && bin == kBins) {
          bin = lane * 8 + i;
          listed = cum;
        }
      }
      const unsigned who = __ballot_sync(0xffffffffu, bin < kBins);
      const int src = who != 0 ? __ffs(static_cast<int>(who)) - 1 : 31;
      bin = __shfl_sync(0xffffffffu, bin, src);
      listed = who != 0 ? __shfl_sync(0xffffffffu, listed, src) : everything;
      if (lane == 0) {
        sh.pick[0] = static_cast<uint32_t>(min(bin, kBins - 1));
        sh.pick[1] = listed;
      }
    }
    __syncthreads();
    const int end_bin = static_cast<int>(sh.pick[0]);
    const uint32_t listed = sh.pick[1];

    if (listed <= kList) {
      // ---- few enough: the first block sorts them
      for (int j = tid; j < s.size; j += kThreads) {
        const float x = s.at(j);
        if (x > -INFINITY && bin_of(x) <= end_bin) {
          const uint32_t at = atomicAdd(&sh.listed, 1u);
          sh.list[at] = static_cast<unsigned long long>(~key_of(x)) << 32 | static_cast<uint32_t>(s.first + j);
        }
      }
      row_sync<C>();
      if (rank == 0) {
        int have = static_cast<int>(sh.listed);
        for (int q = 1; q < C; ++q) {
          const int more = static_cast<int>(peer_u32(&sh.listed, q));
          for (int i = tid; i < more; i += kThreads) sh.list[have + i] = peer_u64(&sh.list[i], q);
          have += more;
        }
        int size = 2;
        while (size < have) size *= 2;
        for (int i = have + tid; i < size; i += kThreads) sh.list[i] = ~0ull;
        __syncthreads();
        for (int span = 2; span <= size; span *= 2) {
          for (int step = span / 2; step > 0; step /= 2) {
            for (int i = tid; i < size / 2; i += kThreads) {
              const int a = 2 * i - (i & (step - 1)), b = a + step;
              const unsigned long long u = sh.list[a], v = sh.list[b];
              if ((u > v) == ((a & span) == 0)) {
                sh.list[a] = v;
                sh.list[b] = u;
              }
            }
            __syncthreads();
          }
        }
        // the thread's part of the sorted list, and the sum of p before it
        constexpr int kPart = kList / kThreads;
        if (by_count) have = min(have, top_k);
        float pr[kPart], sum = 0.f;
#pragma unroll
        for (int i = 0; i < kPart; ++i) {
          const int at = tid * kPart + i;
          pr[i] = at < have ? prob(r, value_of(~static_cast<uint32_t>(sh.list[at] >> 32))) : 0.f;
          sum += pr[i];
        }
        float upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float f = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += f;
        }
        if (lane == 31) sh.red[0][warp] = upto;
        __syncthreads();
        float before = upto - sum, all = 0.f;
        if (lane == 0) before = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) before += sh.red[0][w];
          all += sh.red[0][w];
        }
        __syncthreads();
        const float goal = by_mass ? top_p * (by_count ? all : z) : INFINITY;
        float score = -1.f, kept = 0.f;
        int idx = INT32_MAX;
#pragma unroll
        for (int i = 0; i < kPart; ++i) {
          const int at = tid * kPart + i;
          if (at < have && (before < goal || at == 0) && pr[i] >= min_p) {
            const int sym = static_cast<int>(static_cast<uint32_t>(sh.list[at]));
            better(score, idx, pr[i] / noise[sym], sym);
            kept += pr[i];
          }
          before += pr[i];
        }
        block_best(score, idx, kept, sh);
        if (tid == 0) write_answer(p, row, r, idx == INT32_MAX ? -1 : idx, idx == INT32_MAX ? r.top : fminf(to_float(s.row[idx]), FLT_MAX), kept);
      }
      if (C > 1) cluster_sync_all();  // (the other blocks' lists are read until here)
      return;
    }
    // ---- too many
    if (by_count) {
      uint32_t possible = 0;
      for (int b = 0; b < kBins; ++b) possible += sh.all_count[b];
      __syncthreads();
      if (static_cast<uint32_t>(top_k) < possible) select_end<C>(s, sh, r, false, static_cast<double>(top_k));
      if (by_mass) {
        z = 0.f;
        for (int j = tid; j < s.size; j += kThreads) {
          const float x = s.at(j);
          if (x > -INFINITY && keeps(r, key_of(x), s.first + j)) z += prob(r, x);
        }
        z = row_sum<C>(z, sh);
      }
    }
    __syncthreads();
    if (by_mass) select_end<C>(s, sh, r, true, fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(z));
    __syncthreads();
  }

  // ---- all that is kept
  float score = -1.f, kept = 0.f;
  int idx = INT32_MAX;
#pragma unroll 4
  for (int j = tid; j < s.size; j += kThreads) {
    const float x = s.at(j);
    const int i = s.first + j;
    const float pr = prob(r, x);
    if (x > -INFINITY && pr >= min_p && keeps(r, key_of(x), i)) {
      better(score, idx, pr / __ldg(noise + i), i);
      kept += pr;
    }
  }
  block_best(score, idx, kept, sh);
  if (C > 1) {
    if (tid == 0) {
      sh.out_f[2] = score;
      sh.out_f[3] = kept;
      sh.out_i[2] = idx;
    }
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
#pragma unroll
      for (int q = 1; q < C; ++q) {
        better(score, idx, peer_f32(&sh.out_f[2], q), static_cast<int>(peer_u32(&sh.out_i[2], q)));
        kept += peer_f32(&sh.out_f[3], q);
      }
    }
    cluster_sync_all();
  }
  if (rank == 0 && tid == 0)
    write_answer(p, row, r, idx == INT32_MAX ? -1 : idx, idx == INT32_MAX ? r.top : fminf(to_float(s.row[idx]), FLT_MAX), kept);
}

// ----------------------------------------------------------------------------- launches

constexpr int kMostHeld = 48 * 1024;  // symbols of a slice that shared memory holds

template <class T, bool HELD, int C>
int run_sample(const SampleArgs& p, int64_t rows, cudaStream_t stream) {
  const size_t smem = sizeof(Shared) + (HELD ? static_cast<size_t>(p.slice) * sizeof(float) : 0);
  static std::atomic<bool> set[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TRITURUS_B200_ELAUNCH;
  if (HELD && !set[dev]) {
    if (cudaFuncSetAttribute(sample_kernel<T, HELD, C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(Shared) + kMostHeld * sizeof(float))) != cudaSuccess)
      return TRITURUS_B200_ELAUNCH;
    set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * C), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, HELD, C>, p) == cudaSuccess ? TRITURUS_B200_OK : TRITURUS_B200_ELAUNCH;
}

template <class T>
int sample_rows(SampleArgs p, int64_t rows, cudaStream_t stream) {
  const int64_t most = static_cast<int64_t>(p.symbols) + 16 / static_cast<int64_t>(sizeof(T));  // (with what lies before a 16-byte boundary)
  int c = 1;
  while (c < 8 && (most > c * 16384 || (rows * c * 2 <= device_sms() && most > c * 4096))) c *= 2;
  p.slice = static_cast<int>((((most + c - 1) / c) + 7) / 8 * 8);
  if (p.slice > kMostHeld) return run_sample<T, false, 8>(p, rows, stream);
  switch (c) {
    case 1: return run_sample<T, true, 1>(p, rows, stream);
    case 2: return run_sample<T, true, 2>(p, rows, stream);
    case 4: return run_sample<T, true, 4>(p, rows, stream);
    default: return run_sample<T, true, 8>(p, rows, stream);
  }
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" int triturus_b200_sample(const void* logits, const float* noise, int64_t* token, float* logprob, int64_t rows, int64_t symbols,
                                    int64_t logits_stride, int64_t noise_stride, int type, const float* temperature, float temperature0,
                                    const int32_t* top_k, int32_t top_k0, const float* top_p, float top_p0, const float* min_p, float min_p0,
                                    void* stream) {
  if (rows < 0 || symbols <= 0 || symbols > (1 << 30) || type < TRITURUS_B200_TYPE_F32 || type > TRITURUS_B200_TYPE_F16) return TRITURUS_B200_EINVAL;
  if (rows > INT32_MAX / 8) return TRITURUS_B200_EINVAL;
  if (rows == 0) return TRITURUS_B200_OK;
  if (logits == nullptr || noise == nullptr || token == nullptr) return TRITURUS_B200_EINVAL;
  if (!aligned_to(logits, type == TRITURUS_B200_TYPE_F32 ? 4 : 2) || !aligned_to(noise, 4) || !aligned_to(token, 8) || !aligned_to(logprob, 4) ||
      !aligned_to(temperature, 4) || !aligned_to(top_k, 4) || !aligned_to(top_p, 4) || !aligned_to(min_p, 4))
    return TRITURUS_B200_EALIGN;
  SampleArgs p = {};
  p.logits = logits;
  p.noise = noise;
  p.token = token;
  p.logprob = logprob;
  p.logits_stride = logits_stride;
  p.noise_stride = noise_stride;
  p.symbols = static_cast<int>(symbols);
  p.temperature = temperature;
  p.temperature0 = temperature0;
  p.top_k = top_k;
  p.top_k0 = top_k0;
  p.top_p = top_p;
  p.top_p0 = top_p0;
  p.min_p = min_p;
  p.min_p0 = min_p0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return type == TRITURUS_B200_TYPE_F32    ? sample_rows<float>(p, rows, st)
         : type == TRITURUS_B200_TYPE_BF16 ? sample_rows<__nv_bfloat16>(p, rows, st)
                                           : sample_rows<__half>(p, rows, st);
}
