// Sampling of one symbol per row of logits from given exponential noise.
//
//   p_i = exp((x_i - max x) / T).  In the order of falling x (equal ones by index): the first top_k; of these the fewest whose sum of p
//   reaches top_p times theirs; of these the ones with p >= min_p.  Of what is kept, the symbol with the largest p_i / noise_i, and
//   log(p_i / sum of p kept).
//
// For exponential noise the largest p / noise falls on i with probability p_i / sum p.  No place on a cumulative sum decides, and so no order
// of additions: what is kept is a prefix of the sorted row, and only its end depends on sums.
//
// A row belongs to a cluster of up to eight blocks with a slice each, held in shared memory or, where that is too little, read again from the L2 cache.
// No row is sorted.
//
// Nothing filtered: one pass over logits and noise (200 x 10007 in float32 8.2 us a call; 256 x 131072 84 us = 3.2 TB/s).  min_p alone: the same pass behind
// one for the maximum, with all of the noise (256 x 131072 100 us).
//
// A small top_k: a block's own symbols below the k-th largest of its threads' maxima cannot be among the row's first k; what remains, some
// tens of symbols of each block, the first block gathers, sorts and finishes alone (1 x 32768, top_k 50 and top_p 0.9: 11.5 us a call, 9.3 of the
// GPU, half a dozen steps that wait for each other).
//
// Else the end of the kept prefix is found from a histogram of (max - x) / T in steps of 1/16, a factor of 1.06 of p.  The numbers in its bins give the
// bin where a number of symbols is reached, and an estimate of the one where a mass is; the masses are then added in fine steps around
// that, and have to confirm the estimate.  The threads set apart the few percent that can still be kept, so that only these are gone over from
// there on.  The symbols of the one fine bin that is left are gathered and narrowed down; where they are too many for that (flat rows), the end is found
// by radix selection over the bits of x and then over the index.  Numbers and, as multiples of a power of two, masses are added as integers, so
// that a result does not depend on the order of the atomic additions.
//
// 256 x 131072 in float32 with top_p 0.95, at a temperature that leaves 2 % of the symbols, takes 146 us, seven times what reading the logits
// does: three passes over each row (maximum, histogram, setting apart) of 11, 21 and 11 us to a wave of 148 rows, where 11 is what the L2 cache takes to hand out so much, and some 15 us of
// steps that wait for the cluster; the instructions of the histogram bound its pass (ncu: issue 47 %, DRAM 16 %).  Where more symbols remain
// than the threads can set apart, each of the later steps goes over the row again: 361 us with 9 % of them (temperature 1; 0.8 leaves the 2).
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "../../include/triturus_b200.h"
#include "key_range.cuh"
#include "packs.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = 2048;  // symbols that the first block of a row can gather
constexpr int kKept = 16;    // symbols of a slice in shared memory that a thread can set apart
constexpr size_t kKeptBytes = kThreads * kKept * sizeof(uint16_t);
constexpr int kCopied = 16;  // ... and of one that is not, with their values
constexpr int kFew = kThreads / 2;  // a small top_k

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

struct alignas(16) Shared {
  unsigned long long list[kList];
  double all_mass[kBins];
  double pick_d;
  uint32_t count[kBins];      // the block's
  uint32_t mass[kBins];       // the block's, as multiples of 2^-clz(count)
  uint32_t all_count[kBins];  // the cluster's
  uint32_t fine_count[kBins];
  uint32_t all_fine[kBins];
  float red[2][kWarps];
  int red_i[2][kWarps];
  // read by the other blocks, each written once or with a row_sync between
  float out_ref, out_top, out_z, out_sure, out_cut, out_score, out_sum;
  int out_cidx, out_idx;
  uint32_t out_lo, out_hi;
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

// Bits in the order of the values; -0 is 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// A place in the sorted row, lower ones first.
__device__ __forceinline__ unsigned long long place_of(float x, int idx) {
  return static_cast<unsigned long long>(~key_of(x)) << 32 | static_cast<uint32_t>(idx);
}
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float kStep = LOG2E_F / 16.f;  // of a bin, in powers of two of p
constexpr float kMean = 0.96929f;        // of p over a bin, in units of its upper end: 16 (1 - e^(-1/16))
constexpr int kHeavy = 96;               // bins of p > 0.0025, where a few symbols can be most of the row

// What the blocks of a row share of it.
struct Row {
  float top;      // its largest value
  float k2;       // log2(e) / T
  float to_bin;   // 16 / T
  float cut;      // kept so far: values above cut, and of those equal to it the indexes up to cidx
  int cidx;
};
// (the whole part of a number below 2^23 stands in the last bits of its sum with 2^23: no conversion)
__device__ __forceinline__ int whole_part(float t) { return __float_as_int(__fadd_rz(t, 8388608.f)) & 0x3ff; }
__device__ __forceinline__ float bin_place(const Row& r, float x) { return (r.top - x) * r.to_bin; }
__device__ __forceinline__ float prob_at(float place) { return ex2_approx(place * -kStep); }
__device__ __forceinline__ float prob(const Row& r, float x) { return prob_at(bin_place(r, x)); }
// (a symbol so far below the top that 32 bits do not hold how far has p = 0: it is in no bin, as one of -inf)
constexpr int kNoBin = 0x7fff;
__device__ __forceinline__ int bin_of(const Row& r, float x) {
  const float t = bin_place(r, x);
  return t < FLT_MAX ? whole_part(fminf(t, 255.f)) : kNoBin;
}
__device__ __forceinline__ bool keeps(const Row& r, float x, int idx) { return x > r.cut || (x == r.cut && idx <= r.cidx); }

// The block's slice: element j (0 ... size) is symbol first + j of the row, those below 0 and from `symbols` on are -inf.
template <class T, bool HELD>
struct Slice {
  const T* row;
  float* held;
  int first, size, symbols;
  bool apart;            // the thread has set apart which of its elements can still be kept:
  int kept_count;        // so many, kThreads places apart
  uint16_t* kept;        // HELD: their numbers
  float* kept_x;         // else their values
  int* kept_j;           // and numbers
  __device__ __forceinline__ float at(int j) const {
    if (HELD) return held[j];
    const int i = first + j;
    return i < 0 || i >= symbols ? -INFINITY : min_nan(to_float(row[i]), FLT_MAX);
  }
};

// Loads the slice; the thread's largest value, NaN if it saw one.
template <class T, bool HELD>
__device__ __forceinline__ float load_slice(const Slice<T, HELD>& s) {
  constexpr int N = Pack<T, 16>::N;
  float top = -INFINITY;
#pragma unroll 4
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
    for (int e = 0; e < N; ++e) top = max_nan(top, v[e]);
    if (HELD) {
#pragma unroll
      for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(s.held + j + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
  }
  return top;
}

// The N elements from j on, of memory where the slice is not held; -inf from the slice's end on.
template <class T, int N>
__device__ __forceinline__ void load_elements(const Slice<T, false>& s, int j, float (&v)[N]) {
  const int i = s.first + j;
  if (i >= 0 && i + N <= s.symbols && j < s.size) {
    const Pack<T, 16> p = *reinterpret_cast<const Pack<T, 16>*>(s.row + i);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = min_nan(to_float(p.v[e]), FLT_MAX);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = j < s.size ? s.at(j + e) : -INFINITY;
  }
}
template <class T, int N>
__device__ __forceinline__ void load_elements(const Slice<T, true>& s, int j, float (&v)[N]) {
  float4 p = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  if (j < s.size) p = *reinterpret_cast<const float4*>(s.held + j);
  v[0] = p.x;
  v[1] = p.y;
  v[2] = p.z;
  v[3] = p.w;
}
template <class T, bool HELD>
constexpr int kRun = HELD ? 4 : Pack<T, 16>::N;  // elements of one load
template <class T, bool HELD>
constexpr int kRuns = HELD ? 2 : 16 / Pack<T, 16>::N;  // loads under way: what f does may keep the compiler from starting them early

// The noise of the N elements from j on; `noise` is the slice's, `four`: it begins on a 16-byte boundary.
template <class T, bool HELD, int N>
__device__ __forceinline__ void load_noise(const Slice<T, HELD>& s, const float* noise, bool four, int j, float (&q)[N]) {
  const int i = s.first + j;
  if (four && i >= 0 && i + N <= s.symbols && j < s.size) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(noise + j + e));
      q[e] = f.x;
      q[e + 1] = f.y;
      q[e + 2] = f.z;
      q[e + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = j < s.size && i + e >= 0 && i + e < s.symbols ? __ldg(noise + j + e) : 1.f;
  }
}

// f(x, j) for the thread's elements of the slice.
template <class T, bool HELD, class F>
__device__ __forceinline__ void for_slice(const Slice<T, HELD>& s, F f) {
  constexpr int N = kRun<T, HELD>, U = kRuns<T, HELD>;
#pragma unroll 1
  for (int j = static_cast<int>(threadIdx.x) * N; j < s.size; j += kThreads * N * U) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) load_elements(s, j + u * kThreads * N, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) f(v[u][e], j + u * kThreads * N + e);
  }
}
// ... or for all of the thread's that can still be kept, where those were set apart.
template <class T, bool HELD, class F>
__device__ __forceinline__ void for_kept(const Slice<T, HELD>& s, F f) {
  if (s.apart) {
    for (int i = 0; i < s.kept_count; ++i) {
      const int j = HELD ? s.kept[i * kThreads] : s.kept_j[i * kThreads];
      f(HELD ? s.held[j] : s.kept_x[i * kThreads], j);
    }
  } else {
    for_slice(s, f);
  }
}

// Sets apart the symbols of the bins up to `last`, each thread its own.  What follows goes over some percent of the slice.
template <class T, bool HELD>
__device__ __forceinline__ void set_apart(Slice<T, HELD>& s, const Row& r, int last) {
  constexpr int kMost = HELD ? kKept : kCopied;
  const float limit = last < kBins - 1 ? static_cast<float>(last + 1) : FLT_MAX;
  int n = 0;
  for_slice(s, [&](float x, int j) {
    if (bin_place(r, x) < limit) {
      const int at = min(n, kMost - 1) * kThreads;
      if (HELD) {
        s.kept[at] = static_cast<uint16_t>(j);
      } else {
        s.kept_x[at] = x;
        s.kept_j[at] = j;
      }
      ++n;
    }
  });
  if (n <= kMost) {  // (else the thread goes over all of its part, as before)
    s.apart = true;
    s.kept_count = n;
  }
}

__device__ __forceinline__ void clear_bins(uint32_t* bins) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) bins[b] = 0;
}

// A mass is counted in units of 2^-clz(count) of the p at the upper end of its bin: the count's bits and the mass's make 32, no overflow.
__device__ __forceinline__ uint32_t mass_units(float share, uint32_t count) {
  return __float2uint_rn(fminf(share, 1.f) * __int_as_float((127 + min(__clz(static_cast<int>(count)), 31)) << 23));
}
__device__ __forceinline__ double unit_of(uint32_t count) {
  return __hiloint2double((1023 - min(__clz(static_cast<int>(count)), 31)) << 20, 0);
}

// The cluster's counts (and masses, each block's in units of its own) from the blocks' ones.  `upper(b)`: the p that bin b's masses are
// multiples of.  The blocks' bins are read until the next row_sync.
template <int C, class F>
__device__ __forceinline__ void merge_bins(Shared& sh, bool counts, bool masses, F upper) {
  row_sync<C>();
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    uint32_t n = 0;
    double m = 0.0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const uint32_t c = C > 1 ? peer_u32(&sh.count[b], r) : sh.count[b];
      n += c;
      if (masses) m += static_cast<double>(C > 1 ? peer_u32(&sh.mass[b], r) : sh.mass[b]) * unit_of(c);
    }
    if (counts) sh.all_count[b] = n;
    if (masses) sh.all_mass[b] = m > 0.0 ? m * static_cast<double>(upper(b)) : 0.0;
  }
  __syncthreads();
}

// Warp 0: the first bin with something where the running sum of `value(b)` from `start` on reaches `target`, or -1; *before: the sum before
// it, *filled: the last bin with something, or -1, and *before_filled.  Lane l has bins 8 l ... 8 l + 7.
template <class V>
struct Found {
  int bin, filled;
  V before, before_filled;
};
template <class V, class F>
__device__ __forceinline__ Found<V> first_bin(V start, V target, F value) {
  const int lane = threadIdx.x & 31;
  V v[8], total = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = value(lane * 8 + i);
    total += v[i];
  }
  V upto = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  V sum = __shfl_up_sync(0xffffffffu, upto, 1);
  sum = start + (lane == 0 ? V(0) : sum);
  Found<V> f = {-1, -1, sum, sum};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const V next = sum + v[i];
    if (v[i] > 0) {
      f.filled = lane * 8 + i;
      f.before_filled = sum;
      if (next >= target && f.bin < 0) {
        f.bin = lane * 8 + i;
        f.before = sum;
      }
    }
    sum = next;
  }
  const unsigned who = __ballot_sync(0xffffffffu, f.bin >= 0), any = __ballot_sync(0xffffffffu, f.filled >= 0);
  const int first = who != 0 ? __ffs(static_cast<int>(who)) - 1 : 0, last = any != 0 ? 31 - __clz(static_cast<int>(any)) : 0;
  f.bin = __shfl_sync(0xffffffffu, f.bin, first);
  f.before = __shfl_sync(0xffffffffu, f.before, first);
  f.filled = __shfl_sync(0xffffffffu, f.filled, last);
  f.before_filled = __shfl_sync(0xffffffffu, f.before_filled, last);
  return f;
}
// The mass of a bin with `count` symbols.  What lies far enough below the top has p = 0 in 32 bits, but is something all the same: a bin that is empty
// must not be taken for the end.
__device__ __forceinline__ double mass_of(double mass, uint32_t count) { return count == 0 ? 0.0 : fmax(mass, 1e-300); }
// ... and the last one with something where none reaches it: the sums were rounded on two ways.
template <class V>
__device__ __forceinline__ int bin_or_last(const Found<V>& f, V* before) {
  *before = f.bin >= 0 ? f.before : f.before_filled;
  return max(f.bin >= 0 ? f.bin : f.filled, 0);
}

// Sorts list[0 ... n) and fills it up to the next power of two.  A list of up to 128 by counting for each what is before it.
__device__ __forceinline__ void sort_list(unsigned long long* list, int n) {
  if (n <= 128) {
    constexpr int kShare = kThreads / 128;  // threads to an element
    const int i = static_cast<int>(threadIdx.x) / kShare, part = static_cast<int>(threadIdx.x) % kShare;
    const unsigned long long mine = i < n ? list[i] : ~0ull;
    int before = 0;
    for (int j = part; j < n; j += kShare) before += list[j] < mine;
#pragma unroll
    for (int o = 1; o < kShare; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    __syncthreads();
    if (part == 0 && i < n) list[before] = mine;
    __syncthreads();
    return;
  }
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + static_cast<int>(threadIdx.x); i < size; i += kThreads) list[i] = ~0ull;
  __syncthreads();
  for (int span = 2; span <= size; span *= 2) {
    for (int step = span / 2; step > 0; step /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const unsigned long long u = list[a], v = list[b];
        if ((u > v) == ((a & span) == 0)) {
          list[a] = v;
          list[b] = u;
        }
      }
      __syncthreads();
    }
  }
}

// The first block's list and behind it the others', each fetched by warps of its own; their number.
template <int C>
__device__ __forceinline__ int gather_lists(Shared& sh) {
  if (C == 1) return static_cast<int>(sh.listed);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mine = lane < C ? static_cast<int>(peer_u32(&sh.listed, lane)) : 0;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < C; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  constexpr int kEach = kWarps / C;
  const int q = warp / kEach, more = __shfl_sync(0xffffffffu, mine, q), from = __shfl_sync(0xffffffffu, upto, q) - more;
  if (q > 0)
    for (int i = (warp % kEach) * 32 + lane; i < more; i += kEach * 32) sh.list[from + i] = peer_u64(&sh.list[i], q);
  __syncthreads();
  return __shfl_sync(0xffffffffu, upto, C - 1);
}

// The sums of p before each of the thread's kPart symbols of the sorted list's first `have`, and of all of them.
constexpr int kPart = kList / kThreads;
__device__ __forceinline__ void sorted_sums(Shared& sh, const Row& r, int have, float (&pr)[kPart], float& before, float& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPart; ++i) {
    const int at = static_cast<int>(threadIdx.x) * kPart + i;
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
  before = __shfl_up_sync(0xffffffffu, upto, 1);
  if (lane == 0) before = 0.f;
  __syncthreads();
  all = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh.red[0][w];
    all += sh.red[0][w];
  }
  __syncthreads();
}

// The end of the prefix of the kept symbols whose number, or mass, with the `above` of keys above `hi`, first reaches `target`, by radix selection over
// the keys of lo ... hi.  Sets r.cut and r.cidx.
template <int C, class T, bool HELD>
__device__ __forceinline__ void select_end(const Slice<T, HELD>& s, Shared& sh, Row& r, bool by_mass, double target, uint32_t lo, uint32_t hi, double above) {
  uint32_t ties = 0;
#pragma unroll 1
  for (int round = 0; round < kKeyRounds; ++round) {
    const KeyRange range = {lo, hi};
    const int shift = range.shift();
    clear_bins(sh.count);
    clear_bins(sh.mass);
    __syncthreads();
    for_kept(s, [&](float x, int j) {
      const uint32_t key = key_of(x);
      if (key >= lo && key <= hi && keeps(r, x, s.first + j)) atomicAdd(&sh.count[(hi - key) >> shift], 1u);
    });
    auto upper = [&](int b) { return fminf(value_of(hi - (static_cast<uint32_t>(b) << shift)), r.top); };
    if (by_mass) {
      __syncthreads();
      for_kept(s, [&](float x, int j) {
        const uint32_t key = key_of(x);
        if (key >= lo && key <= hi && keeps(r, x, s.first + j)) {
          const int b = static_cast<int>((hi - key) >> shift);
          atomicAdd(&sh.mass[b], mass_units(ex2_approx((x - upper(b)) * r.k2), sh.count[b]));
        }
      });
    }
    merge_bins<C>(sh, true, by_mass, [&](int b) { return prob(r, upper(b)); });
    if (threadIdx.x < 32) {
      double before;
      const int b = bin_or_last(
          first_bin<double>(above, target, [&](int i) { return by_mass ? mass_of(sh.all_mass[i], sh.all_count[i]) : static_cast<double>(sh.all_count[i]); }),
          &before);
      if (threadIdx.x == 0) {
        sh.pick[0] = static_cast<uint32_t>(b);
        sh.pick[1] = sh.all_count[b];
        sh.pick_d = before;
      }
    }
    __syncthreads();
    const uint32_t b = sh.pick[0];
    ties = sh.pick[1];
    above = sh.pick_d;
    const KeyRange left = range.bin_downwards(b, shift);
    lo = left.lo;
    hi = left.hi;
    row_sync<C>();  // (all have read the bins)
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
      clear_bins(sh.count);
      __syncthreads();
      for_kept(s, [&](float x, int j) {
        const int i = s.first + j;
        if (i >= from && i < to && key_of(x) == hi && keeps(r, x, i)) atomicAdd(&sh.count[(i - from) / width], 1u);
      });
      merge_bins<C>(sh, true, false, [](int) { return 0.f; });
      if (threadIdx.x < 32) {
        uint32_t before;
        const int b = bin_or_last(first_bin<uint32_t>(0u, want, [&](int i) { return sh.all_count[i]; }), &before);
        if (threadIdx.x == 0) {
          sh.pick[0] = static_cast<uint32_t>(b);
          sh.pick[1] = before;
        }
      }
      __syncthreads();
      from += static_cast<int>(sh.pick[0]) * width;
      to = min(to, from + width);
      want -= sh.pick[1];
      row_sync<C>();
    }
    r.cidx = from;
  } else if (value_of(hi) != r.cut) {
    r.cidx = INT32_MAX;
  }
  r.cut = value_of(hi);
}

// One round of radix selection over list[0 ... n), by the upper halves of the places (the values) or, BY_INDEX, the lower ones: those in lo ... hi are in
// question and `above` (a number or mass) lies before them; narrows the range to the bin where `target` is reached.  Returns how many are in it.
template <bool BY_INDEX>
__device__ __forceinline__ uint32_t half_of(unsigned long long place) {
  return static_cast<uint32_t>(BY_INDEX ? place : place >> 32);
}
template <bool BY_INDEX>
__device__ __forceinline__ uint32_t narrow_list(Shared& sh, const Row& r, int n, bool by_mass, double target, uint32_t& lo, uint32_t& hi, double& above) {
  const KeyRange range = {lo, hi};
  const int shift = range.shift();
  clear_bins(sh.count);
  clear_bins(sh.mass);
  __syncthreads();
  auto upper = [&](int b) { return fminf(value_of(~(lo + (static_cast<uint32_t>(b) << shift))), r.top); };
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t k = half_of<BY_INDEX>(sh.list[i]);
    if (k >= lo && k <= hi) atomicAdd(&sh.count[(k - lo) >> shift], 1u);
  }
  __syncthreads();
  if (by_mass) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t k = half_of<BY_INDEX>(sh.list[i]);
      if (k >= lo && k <= hi) {
        const int b = static_cast<int>((k - lo) >> shift);
        atomicAdd(&sh.mass[b], mass_units(ex2_approx((value_of(~k) - upper(b)) * r.k2), sh.count[b]));
      }
    }
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    double before;
    const int b = bin_or_last(first_bin<double>(above, target, [&](int i) {
                                const uint32_t c = sh.count[i];
                                if (!by_mass || c == 0) return static_cast<double>(c);
                                return mass_of(static_cast<double>(sh.mass[i]) * unit_of(c) * static_cast<double>(prob(r, upper(i))), c);
                              }),
                              &before);
    if (threadIdx.x == 0) {
      sh.pick[0] = static_cast<uint32_t>(b);
      sh.pick[1] = sh.count[b];
      sh.pick_d = before;
    }
  }
  __syncthreads();
  above = sh.pick_d;
  const KeyRange left = range.bin_upwards(sh.pick[0], shift);
  lo = left.lo;
  hi = left.hi;
  const uint32_t in = sh.pick[1];
  __syncthreads();
  return in;
}

// The range of those halves.
template <bool BY_INDEX>
__device__ __forceinline__ void range_of_list(Shared& sh, int n, uint32_t& lo, uint32_t& hi) {
  lo = 0xffffffffu;
  hi = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t k = half_of<BY_INDEX>(sh.list[i]);
    lo = min(lo, k);
    hi = max(hi, k);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    sh.red_i[0][warp] = static_cast<int>(lo);
    sh.red_i[1][warp] = static_cast<int>(hi);
  }
  __syncthreads();
  lo = __reduce_min_sync(0xffffffffu, lane < kWarps ? static_cast<uint32_t>(sh.red_i[0][lane]) : 0xffffffffu);
  hi = __reduce_max_sync(0xffffffffu, lane < kWarps ? static_cast<uint32_t>(sh.red_i[1][lane]) : 0u);
  __syncthreads();
}

// Keeps those of list[0 ... n) whose halves are in lo ... hi; their number.  (Each thread has its own in registers meanwhile.)
template <bool BY_INDEX>
__device__ __forceinline__ int filter_list(Shared& sh, int n, uint32_t lo, uint32_t hi) {
  unsigned long long mine[kPart];
#pragma unroll
  for (int i = 0; i < kPart; ++i) {
    const int at = static_cast<int>(threadIdx.x) + i * kThreads;
    mine[i] = at < n ? sh.list[at] : 0ull;
  }
  if (threadIdx.x == 0) sh.pick[2] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPart; ++i) {
    const uint32_t k = half_of<BY_INDEX>(mine[i]);
    if (static_cast<int>(threadIdx.x) + i * kThreads < n && k >= lo && k <= hi) sh.list[atomicAdd(&sh.pick[2], 1u)] = mine[i];
  }
  __syncthreads();
  n = static_cast<int>(sh.pick[2]);
  __syncthreads();
  return n;
}

// The place in list[0 ... n) where, with the `above` before the list, `target` is reached.  The list is lost.  (n > 0, as the list is that of a bin
// with something; behind an empty one all is kept.)
__device__ __forceinline__ unsigned long long end_in_list(Shared& sh, const Row& r, int n, bool by_mass, double target, double above) {
  if (n == 0) return place_of(-INFINITY, INT32_MAX);
  uint32_t lo, hi, in = static_cast<uint32_t>(n);
  range_of_list<false>(sh, n, lo, hi);
  while (in > 128 && lo != hi) in = narrow_list<false>(sh, r, n, by_mass, target, lo, hi, above);
  n = filter_list<false>(sh, n, lo, hi);
  if (n > 128) {  // that many of one value: a number of them, by index
    const double each = by_mass ? static_cast<double>(prob(r, value_of(~lo))) : 1.0;
    const double wanted = each > 0.0 ? ceil((target - above) / each) : 1.0;
    target = fmin(fmax(wanted, 1.0), static_cast<double>(n));
    above = 0.0;
    by_mass = false;
    range_of_list<true>(sh, n, lo, hi);
    while (in > 128) in = narrow_list<true>(sh, r, n, false, target, lo, hi, above);
    n = filter_list<true>(sh, n, lo, hi);
  }
  sort_list(sh.list, n);
  if (by_mass) {
    float pr[kPart], before, all;
    sorted_sums(sh, r, n, pr, before, all);
    if (threadIdx.x == 0) sh.pick[0] = static_cast<uint32_t>(n - 1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPart; ++i) {
      before += pr[i];
      const int at = static_cast<int>(threadIdx.x) * kPart + i;
      if (at < n && above + static_cast<double>(before) >= target) atomicMin(&sh.pick[0], static_cast<uint32_t>(at));
    }
    __syncthreads();
    return sh.list[sh.pick[0]];
  }
  return sh.list[min(max(static_cast<int>(target - above) - 1, 0), n - 1)];
}

// The row's largest of a value of each thread, NaN where one is; `slot` is read by the other blocks.
template <int C>
__device__ __forceinline__ float row_max(float v, Shared& sh, float* slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) sh.red[0][threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.red[0][0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = max_nan(v, sh.red[0][w]);
  if (C > 1) {
    if (threadIdx.x == 0) *slot = v;
    cluster_sync_all();
#pragma unroll
    for (int q = 0; q < C; ++q) v = max_nan(v, peer_f32(slot, q));
  } else {
    __syncthreads();
  }
  return v;
}

// The row's histogram of what is kept so far, in bins up to `last`: the blocks' in sh.count, all of it in sh.all_count.  Where `want_sum`, returns the row's
// sum of p, and leaves in sh.all_mass an estimate of the bins' masses: of the first kHeavy from their p, of the others from their numbers.
template <int C, class T, bool HELD>
__device__ __forceinline__ float histogram(const Slice<T, HELD>& s, Shared& sh, const Row& r, int last, bool want_sum) {
  clear_bins(sh.count);
  clear_bins(sh.mass);
  __syncthreads();
  float z = 0.f;
  const float limit = last < kBins - 1 ? static_cast<float>(last + 1) : FLT_MAX;
  const int unit_bits = min(__clz(s.size), 31);  // (no overflow, should all of the slice be in one bin)
  const float unit = __int_as_float((127 + unit_bits) << 23);
  if (r.cut == -INFINITY) {
    for_slice(s, [&](float x, int) {
      const float t = bin_place(r, x);  // (infinite for -inf)
      const float pr = prob_at(t);
      if (t < limit) {
        const int b = whole_part(fminf(t, 255.f));
        atomicAdd(&sh.count[b], 1u);
        if (want_sum && t < static_cast<float>(kHeavy)) atomicAdd(&sh.mass[b], __float2uint_rn(fminf(pr, 1.f) * unit));
      }
      z += pr;
    });
  } else {
    for_kept(s, [&](float x, int j) {
      if (keeps(r, x, s.first + j)) {
        const int b = bin_of(r, x);
        if (b < kBins) {
          atomicAdd(&sh.count[b], 1u);
          if (want_sum && b < kHeavy) atomicAdd(&sh.mass[b], __float2uint_rn(fminf(prob(r, x), 1.f) * unit));
        }
        z += prob(r, x);
      }
    });
  }
  if (want_sum) {
    z = block_sum(z, sh.red[0], threadIdx.x >> 5, threadIdx.x & 31, kWarps);
    if (threadIdx.x == 0) sh.out_z = z;
  }
  row_sync<C>();
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    uint32_t n = 0;
    float m = 0.f;
#pragma unroll
    for (int q = 0; q < C; ++q) {
      n += C > 1 ? peer_u32(&sh.count[b], q) : sh.count[b];
      if (want_sum && b < kHeavy) m += static_cast<float>(C > 1 ? peer_u32(&sh.mass[b], q) : sh.mass[b]);
    }
    sh.all_count[b] = n;
    if (want_sum) sh.all_mass[b] = b < kHeavy ? m / unit : b < kBins - 1 ? static_cast<float>(n) * (kMean * ex2_approx(-kStep * static_cast<float>(b))) : 0.f;
  }
  __syncthreads();
  if (!want_sum) return 0.f;
  z = 0.f;
#pragma unroll
  for (int q = 0; q < C; ++q) z += C > 1 ? peer_f32(&sh.out_z, q) : sh.out_z;
  return z;
}

// False, and nothing done, where `all_bins` has to be set.
template <int C, class T, bool HELD>
__device__ __forceinline__ bool find_end(Slice<T, HELD>& s, Shared& sh, Row& r, bool by_mass, double target, int last_bin, bool all_bins, int rank) {
  const int tid = threadIdx.x;
  const bool kept_before = s.apart;
  // The bin of the end: by number it is known, by mass estimated, and two bins to either side are taken for certain, which the masses
  // themselves confirm; else all bins are in question.
  if (tid < 32) {
    if (by_mass) {
      const Found<float> f = first_bin<float>(0.f, static_cast<float>(target), [&](int b) { return static_cast<float>(sh.all_mass[b]); });
      const bool guess = !all_bins && f.bin >= 0;
      if (tid == 0) {
        sh.pick[0] = static_cast<uint32_t>(guess ? max(f.bin - 2, 0) : 0);
        sh.pick[1] = static_cast<uint32_t>(guess ? min(f.bin + 2, last_bin) : last_bin);
      }
    } else {
      uint32_t before;
      const int b = bin_or_last(first_bin<uint32_t>(0u, static_cast<uint32_t>(target), [&](int i) { return sh.all_count[i]; }), &before);
      if (tid == 0) {
        sh.pick[0] = sh.pick[1] = static_cast<uint32_t>(b);
        sh.pick_d = static_cast<double>(before);
      }
    }
  }
  if (tid == 0) sh.listed = 0;
  clear_bins(sh.fine_count);
  row_sync<C>();  // (all have read the masses that the estimate is of)
  clear_bins(sh.mass);
  __syncthreads();
  const int from = static_cast<int>(sh.pick[0]), to = static_cast<int>(sh.pick[1]);
  double above = sh.pick_d;
  // (in the bins from ... to that are left, a step as fine as 256 bins allow)
  const float scale = by_mass ? static_cast<float>(kBins) / static_cast<float>(to + 1 - from) : 1.f;
  auto fine_of = [&](float x) {
    const float t = bin_place(r, x);
    if (!(t < FLT_MAX)) return kNoBin;
    if (!by_mass) return whole_part(fminf(t, 255.f)) - from;
    if (t < static_cast<float>(from)) return -1;
    return t < static_cast<float>(to + 1) || to == kBins - 1 ? whole_part(fminf((t - static_cast<float>(from)) * scale, 255.f)) : kNoBin;
  };
  int bin = 0;
  uint32_t in_bin;
  {
    uint32_t mine = 0;  // how many of the block's symbols are in the bins up to `to`
    for (int b = tid & 31; b <= to; b += 32) mine += sh.count[b];
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (!s.apart && mine <= kThreads * (HELD ? kKept : kCopied) / 2) set_apart(s, r, to);
  }
  if (by_mass) {
    const float fine_step = kStep / scale;
    for_kept(s, [&](float x, int j) {
      if (keeps(r, x, s.first + j)) {
        const int b = fine_of(x);
        if (b >= 0 && b < kBins) atomicAdd(&sh.fine_count[b], 1u);
      }
    });
    __syncthreads();
    float sure = 0.f;
    for_kept(s, [&](float x, int j) {
      if (keeps(r, x, s.first + j)) {
        const int b = fine_of(x);
        const float e = (x - r.top) * r.k2;
        if (b < 0)
          sure += ex2_approx(e);
        else if (b < kBins)
          atomicAdd(&sh.mass[b], mass_units(ex2_approx(e + (kStep * static_cast<float>(from) + fine_step * static_cast<float>(b))), sh.fine_count[b]));
      }
    });
    sure = block_sum(sure, sh.red[0], tid >> 5, tid & 31, kWarps);
    if (tid == 0) sh.out_sure = sure;
    row_sync<C>();
    for (int b = tid; b < kBins; b += kThreads) {
      uint32_t n = 0;
      double m = 0.0;
#pragma unroll
      for (int q = 0; q < C; ++q) {
        const uint32_t c = C > 1 ? peer_u32(&sh.fine_count[b], q) : sh.fine_count[b];
        n += c;
        m += static_cast<double>(C > 1 ? peer_u32(&sh.mass[b], q) : sh.mass[b]) * unit_of(c);
      }
      sh.all_fine[b] = n;
      sh.all_mass[b] = m * static_cast<double>(ex2_approx(-(kStep * static_cast<float>(from) + fine_step * static_cast<float>(b))));
    }
    __syncthreads();
    if (tid < 32) {
      double before;
      above = 0.0;
#pragma unroll
      for (int q = 0; q < C; ++q) above += static_cast<double>(C > 1 ? peer_f32(&sh.out_sure, q) : sh.out_sure);
      const Found<double> f = first_bin<double>(above, target, [&](int i) { return mass_of(sh.all_mass[i], sh.all_fine[i]); });
      const int b = bin_or_last(f, &before);
      if (tid == 0) {
        sh.pick[2] = static_cast<uint32_t>(b);
        sh.pick[3] = (f.bin >= 0 || to == last_bin) && (above < target || from == 0);
        sh.pick_d = before;
      }
    }
    __syncthreads();
    if (!sh.pick[3]) {
      s.apart = kept_before;
      row_sync<C>();  // (all have read the bins)
      return false;
    }
    bin = static_cast<int>(sh.pick[2]);
    above = sh.pick_d;
    in_bin = sh.all_fine[bin];
  } else {
    in_bin = sh.all_count[from];
  }
  if (in_bin <= kList) {
    for_kept(s, [&](float x, int j) {
      if (keeps(r, x, s.first + j) && fine_of(x) == bin) sh.list[atomicAdd(&sh.listed, 1u)] = place_of(x, s.first + j);
    });
    row_sync<C>();
    if (rank == 0) {
      const unsigned long long place = end_in_list(sh, r, gather_lists<C>(sh), by_mass, target, above);
      if (tid == 0) {
        sh.out_cut = value_of(~static_cast<uint32_t>(place >> 32));
        sh.out_cidx = static_cast<int>(static_cast<uint32_t>(place));
      }
    }
    row_sync<C>();
    r.cut = C > 1 ? peer_f32(&sh.out_cut, 0) : sh.out_cut;
    r.cidx = static_cast<int>(C > 1 ? peer_u32(&sh.out_cidx, 0) : sh.out_cidx);
    return true;
  }
  // the range of the bin's keys
  uint32_t lo = 0xffffffffu, hi = 0;
  for_kept(s, [&](float x, int j) {
    if (keeps(r, x, s.first + j) && fine_of(x) == bin) {
      lo = min(lo, key_of(x));
      hi = max(hi, key_of(x));
    }
  });
  if (tid == 0) {
    sh.out_lo = 0xffffffffu;
    sh.out_hi = 0;
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  __syncthreads();
  if ((tid & 31) == 0) {
    atomicMin(&sh.out_lo, lo);
    atomicMax(&sh.out_hi, hi);
  }
  row_sync<C>();
  lo = 0xffffffffu;
  hi = 0;
#pragma unroll
  for (int q = 0; q < C; ++q) {
    lo = min(lo, C > 1 ? peer_u32(&sh.out_lo, q) : sh.out_lo);
    hi = max(hi, C > 1 ? peer_u32(&sh.out_hi, q) : sh.out_hi);
  }
  row_sync<C>();
  select_end<C>(s, sh, r, by_mass, target, lo, hi, above);
  return true;
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

template <class T, bool HELD>
__device__ __forceinline__ void write_answer(const SampleArgs& p, int64_t row, const Slice<T, HELD>& s, const Row& r, int idx, float sum) {
  const bool none = idx == INT32_MAX;  // (noise that is no number)
  p.token[row] = none ? -1 : idx;
  if (p.logprob != nullptr)
    p.logprob[row] = none ? NAN : (fminf(to_float(s.row[idx]), FLT_MAX) - r.top) * r.k2 * 0.6931471805599453f - logf(sum);
}

template <class T, bool HELD, int C>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  const int tid = threadIdx.x;
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t row = blockIdx.x / C;

  Slice<T, HELD> s;
  s.row = static_cast<const T*>(p.logits) + row * p.logits_stride;
  s.held = reinterpret_cast<float*>(smem_raw + sizeof(Shared) + kKeptBytes);
  // the row's slices begin on 16-byte boundaries of memory
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(s.row) & 15) / sizeof(T));
  s.first = rank * p.slice - skip;
  s.size = p.slice;
  s.symbols = p.symbols;
  s.apart = false;
  s.kept_count = 0;
  s.kept = reinterpret_cast<uint16_t*>(smem_raw + sizeof(Shared)) + tid;
  s.kept_x = reinterpret_cast<float*>(smem_raw + sizeof(Shared)) + tid;
  s.kept_j = reinterpret_cast<int*>(smem_raw + sizeof(Shared)) + kCopied * kThreads + tid;
  const float* noise = p.noise + row * p.noise_stride;

  float temperature = p.temperature != nullptr ? p.temperature[row] : p.temperature0;
  int top_k = p.top_k != nullptr ? p.top_k[row] : p.top_k0;
  float top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p0;
  const float min_p = fminf(p.min_p != nullptr ? p.min_p[row] : p.min_p0, 1.f);
  if (!(temperature > 0.f)) {  // the most probable symbol
    temperature = 1.f;
    top_k = 1;
  }

  Row r;
  r.k2 = fminf(fmaxf(LOG2E_F / temperature, 1e-38f), FLT_MAX);
  r.to_bin = fminf(r.k2 / kStep, FLT_MAX);
  r.cut = -INFINITY;
  r.cidx = INT32_MIN;
  const bool by_count = top_k > 0 && top_k < p.symbols, by_mass = top_p < 1.f;
  // a symbol with p below (1 - top_p) / symbols is behind the end of what top_p keeps: all such ones together have less than 1 - top_p, the first
  // alone has 1
  const int mass_bins = by_mass && !by_count ? static_cast<int>(fminf(16.f * logf(static_cast<float>(p.symbols) / (1.f - fmaxf(top_p, 0.f))) + 1.f, 255.f)) : kBins - 1;
  if (tid == 0) sh.listed = 0;
  clear_bins(sh.count);
  clear_bins(sh.mass);
  float score = 0.f, kept = 0.f;  // of what is kept: the best p / noise and the sum of p
  int idx = INT32_MAX;
  float mine = -INFINITY, top;
  bool scanned = false;
  if constexpr (!HELD) {
    // ---- Where nothing is filtered, memory is read once: p is taken in units of that of the largest of the row's first few thousand
    // symbols, which cancels in the end.
    if (!by_count && !by_mass && !(min_p > 0.f)) {
      constexpr int N = kRun<T, HELD>, U = kRuns<T, HELD>;
      float ref = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[N];
        load_elements(s, tid * N + u * kThreads * N, v);
#pragma unroll
        for (int e = 0; e < N; ++e) ref = max_nan(ref, v[e]);
      }
      ref = row_max<C>(ref, sh, &sh.out_ref);
      if (ref > -INFINITY && ref < FLT_MAX) {
        r.top = ref;
        const float* mine_noise = noise + s.first;
        const bool four = (reinterpret_cast<uintptr_t>(mine_noise) & 15) == 0;
#pragma unroll 1
        for (int j0 = tid * N; j0 < s.size; j0 += kThreads * N * U) {
          float x[U][N], q[U][N];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            load_elements(s, j0 + u * kThreads * N, x[u]);
            load_noise(s, mine_noise, four, j0 + u * kThreads * N, q[u]);
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float pr = prob(r, x[u][e]), sc = __fdividef(pr, q[u][e]);
              mine = max_nan(mine, x[u][e]);
              kept += pr;
              if (sc > score) {  // (-inf has p = 0, which no score is below)
                score = sc;
                idx = s.first + j0 + u * kThreads * N + e;
              }
            }
        }
        top = row_max<C>(mine, sh, &sh.out_top);
        scanned = !((top - ref) * r.to_bin > 512.f);  // (else p is too large for its units)
        if (!scanned) {
          score = kept = 0.f;
          idx = INT32_MAX;
          row_sync<C>();
        }
      }
    }
  }
  if (!scanned) {
    mine = load_slice(s);
    top = row_max<C>(mine, sh, &sh.out_top);
  }
  // (the same for all blocks of the row)
  if (!(top > -INFINITY)) {
    if (rank == 0 && tid == 0) {
      p.token[row] = -1;
      if (p.logprob != nullptr) p.logprob[row] = top;
    }
    if (C > 1) cluster_sync_all();
    return;
  }
  if (top == INFINITY) {  // counts as the largest number
    top = FLT_MAX;
    if (HELD)
      for (int j = tid; j < s.size; j += kThreads) s.held[j] = fminf(s.held[j], FLT_MAX);
    __syncthreads();
  }
  if (!scanned) r.top = top;
  if (by_count && top_k <= kFew) {
    // ---- what is below the k-th largest of the threads' maxima is not among the first k
    const int mine_bin = bin_of(r, mine);
    if (mine_bin < kBins) atomicAdd(&sh.count[mine_bin], 1u);
    __syncthreads();
    if (tid < 32) {
      const Found<uint32_t> f = first_bin<uint32_t>(0u, static_cast<uint32_t>(top_k), [&](int b) { return sh.count[b]; });
      if (tid == 0) sh.pick[0] = static_cast<uint32_t>(f.bin >= 0 ? f.bin : kBins - 1);
    }
    __syncthreads();
    const int bound = static_cast<int>(sh.pick[0]);
    for_slice(s, [&](float x, int j) {
      if (bin_of(r, x) <= bound) {
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kList) sh.list[at] = place_of(x, s.first + j);
      }
    });
    row_sync<C>();
    uint32_t listed = 0;
#pragma unroll
    for (int q = 0; q < C; ++q) listed += C > 1 ? peer_u32(&sh.listed, q) : sh.listed;
    if (listed <= kList) {
      if (rank == 0) {
        int n = gather_lists<C>(sh);
        if (n > 128) {  // the first few of them, or all of the last value's
          uint32_t lo, hi, first;
          double above = 0.0;
          range_of_list<false>(sh, n, lo, hi);
          first = lo;
          narrow_list<false>(sh, r, n, false, static_cast<double>(top_k), lo, hi, above);
          n = filter_list<false>(sh, n, first, hi);
        }
        sort_list(sh.list, n);
        const int have = min(n, top_k);
        float pr[kPart], before, all;
        sorted_sums(sh, r, have, pr, before, all);
        const float goal = by_mass ? top_p * all : INFINITY;
        float score = -1.f, kept = 0.f;
        int idx = INT32_MAX;
#pragma unroll
        for (int i = 0; i < kPart; ++i) {
          const int at = tid * kPart + i;
          if (at < have && (before < goal || at == 0) && pr[i] >= min_p) {
            const int symbol = static_cast<int>(static_cast<uint32_t>(sh.list[at]));
            better(score, idx, __fdividef(pr[i], __ldg(noise + symbol)), symbol);
            kept += pr[i];
          }
          before += pr[i];
        }
        block_best(score, idx, kept, sh);
        if (tid == 0) write_answer(p, row, s, r, idx, kept);
      }
      if (C > 1) cluster_sync_all();  // (the other blocks' lists are read until here)
      return;
    }
    row_sync<C>();
  }
  // ---- the ends of what top_k keeps, then of what top_p does
  bool count_next = by_count, mass_next = by_mass, all_bins = false;
  double target = 0.0;
#pragma unroll 1
  while (count_next || mass_next) {
    const bool mass = !count_next;
    const int last_bin = mass ? mass_bins : kBins - 1;
    if (!all_bins) {
      const float z = histogram<C>(s, sh, r, last_bin, mass);
      target = mass ? static_cast<double>(fmaxf(top_p, 0.f)) * static_cast<double>(z) : static_cast<double>(top_k);
    }
    if (find_end<C>(s, sh, r, mass, target, last_bin, all_bins, rank)) {
      if (mass) mass_next = false;
      count_next = false;
    } else {
      all_bins = true;
    }
  }

  // ---- all that is kept
  // (the noise is fetched for several at once: its latency is what this takes)
  auto weigh = [&](float x, int j) {
    const float pr = prob(r, x);
    return keeps(r, x, s.first + j) && pr >= min_p ? pr : -1.f;
  };
  auto add = [&](float pr, float q, int j) {  // (by rising index: of equal scores the first stays)
    if (pr >= 0.f) {
      const float sc = __fdividef(pr, q);
      if (sc > score) {
        score = sc;
        idx = s.first + j;
      }
      kept += pr;
    }
  };
  if (scanned) {
    // (done above)
  } else if (s.apart) {
    for (int i = 0; i < s.kept_count; i += 4) {
      float pr[4], q[4];
      int j[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pr[e] = -1.f;
        q[e] = 1.f;
        j[e] = 0;
        if (i + e < s.kept_count) {
          j[e] = HELD ? s.kept[(i + e) * kThreads] : s.kept_j[(i + e) * kThreads];
          pr[e] = weigh(HELD ? s.held[j[e]] : s.kept_x[(i + e) * kThreads], j[e]);
        }
        if (pr[e] >= 0.f) q[e] = __ldg(noise + s.first + j[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) add(pr[e], q[e], j[e]);
    }
  } else {
    constexpr int N = kRun<T, HELD>, U = kRuns<T, HELD>;
    const float* mine_noise = noise + s.first;
    const bool four = (reinterpret_cast<uintptr_t>(mine_noise) & 15) == 0;
    const bool all = r.cut == -INFINITY && !(min_p > 0.f);
#pragma unroll 1
    for (int j0 = tid * N; j0 < s.size; j0 += kThreads * N * U) {
      float x[U][N], q[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * kThreads * N;
        load_elements(s, j, x[u]);
        load_noise(s, mine_noise, four, j, q[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * kThreads * N;
        if (all) {  // (-inf has p = 0, which no score is below)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float pr = prob(r, x[u][e]), sc = __fdividef(pr, q[u][e]);
            if (sc > score) {
              score = sc;
              idx = s.first + j + e;
            }
            kept += pr;
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) add(weigh(x[u][e], j + e), q[u][e], j + e);
        }
      }
    }
  }
  block_best(score, idx, kept, sh);
  if (C > 1) {
    if (tid == 0) {
      sh.out_score = score;
      sh.out_sum = kept;
      sh.out_idx = idx;
    }
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
#pragma unroll
      for (int q = 1; q < C; ++q) {
        better(score, idx, peer_f32(&sh.out_score, q), static_cast<int>(peer_u32(&sh.out_idx, q)));
        kept += peer_f32(&sh.out_sum, q);
      }
    }
    cluster_sync_all();
  }
  if (rank == 0 && tid == 0) write_answer(p, row, s, r, idx, kept);
}

// ----------------------------------------------------------------------------- launches

constexpr size_t kMostShared = 227 * 1024;
constexpr int kMostHeld = (kMostShared - sizeof(Shared) - kKeptBytes) / sizeof(float) / 8 * 8;  // symbols of a slice that shared memory holds
static_assert(kMostHeld <= 1 << 16, "their numbers have 16 bits");
constexpr size_t shared_bytes(bool held, int slice) {
  return sizeof(Shared) + (held ? kKeptBytes + static_cast<size_t>(slice) * sizeof(float) : kThreads * kCopied * 8);
}
static_assert(shared_bytes(true, kMostHeld) <= kMostShared && shared_bytes(false, 0) <= kMostShared, "");

template <class T, bool HELD, int C>
int run_sample(const SampleArgs& p, int64_t rows, cudaStream_t stream) {
  static_assert(sizeof(Shared) % 16 == 0, "the slice is read four at a time");
  const size_t smem = shared_bytes(HELD, p.slice);
  static std::atomic<bool> set[64];
  int dev = 0;
  if (code_of(cudaGetDevice(&dev)) != TRITURUS_B200_OK || dev < 0 || dev >= 64) return TRITURUS_B200_ELAUNCH;
  if (!set[dev]) {
    const int rc = code_of(cudaFuncSetAttribute(sample_kernel<T, HELD, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostShared)));
    if (rc != TRITURUS_B200_OK) return rc;
    set[dev] = true;
  }
  const cudaLaunchAttribute cluster = cluster_of(C);
  return launch_of(sample_kernel<T, HELD, C>, dim3(static_cast<unsigned>(rows * C)), kThreads, smem, stream, C > 1 ? &cluster : nullptr, p);
}

template <class T, bool HELD>
int run_sample(const SampleArgs& p, int64_t rows, int c, cudaStream_t stream) {
  switch (c) {
    case 1: return run_sample<T, HELD, 1>(p, rows, stream);
    case 2: return run_sample<T, HELD, 2>(p, rows, stream);
    case 4: return run_sample<T, HELD, 4>(p, rows, stream);
    default: return run_sample<T, HELD, 8>(p, rows, stream);
  }
}

// Blocks to a row: as many as the GPU holds at once (two to an SM, by their registers), if they have 4096 symbols each; in any case enough that a
// block has no more than 64 K symbols (and what lies before a 16-byte boundary).  With fewer its threads set a larger share apart, with more there are
// fewer steps of a cluster and less to do for it: 256 x 131072 in float32, us, in blocks of 32 K / 64 K / 128 K symbols: top_p 0.95 at temperature
// 0.6 156 / 120 / 127, 0.8 182 / 146 / 317, 1.0 292 / 361 / 392, 1.2 426 / 381 / 405; unfiltered 98 / 84 / 76.  A slice is held in shared memory where two
// such blocks fit an SM or one to an SM is all there is; else it is read again from the L2 cache.
template <class T>
int sample_rows(SampleArgs p, int64_t rows, cudaStream_t stream) {
  const int64_t most = static_cast<int64_t>(p.symbols) + 16 / static_cast<int64_t>(sizeof(T));  // (with what lies before a 16-byte boundary)
  const int64_t sms = device_sms();
  int c = 1;
  while (c < 8 && (most > c * INT64_C(65552) || (rows * c <= sms && most > c * 4096))) c *= 2;
  p.slice = static_cast<int>((((most + c - 1) / c) + 7) / 8 * 8);
  const bool held = p.slice <= 16400 || (rows * c <= sms && p.slice <= kMostHeld);
  return held ? run_sample<T, true>(p, rows, c, stream) : run_sample<T, false>(p, rows, c, stream);
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
