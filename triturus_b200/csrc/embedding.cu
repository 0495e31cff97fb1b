// Rows of a table by symbol, and the table's gradient.
//
//   y[i] = s W[t_i];    dW[v] = s sum over {i: t_i = v} of dy[i]
//
// The lookup moves each row once, 16 bytes to a thread and four of them under way; bound by memory.
//
// The gradient adds rows of dy that belong to the same symbol.  Atomics would add them in any order, so the positions are sorted by
// symbol first, with a stable radix sort of up to 9 bits a pass: every block counts its digits, adds up the blocks' counts before it and places its
// items, ranked by warp and by warps.  Up to kClusterSort positions that is one launch, whose first cluster of eight blocks sorts, with the counts in
// each other's shared memory; beyond, two launches a pass.  Blocks beside those fill the table with zeros.  Then groups of threads walk tiles of sorted
// positions: a thread keeps its 16 bytes of columns as 32-bit sums and writes them where a symbol's run ends.  A run over a border of
// two tiles is left in the workspace in parts, which a last launch adds in their order: frequent symbols are spread over many
// blocks, and the same call gives the same result each time.  Few positions are not sorted but compared with
// each other.  Bound by memory: dy read once, the table written once.
#include <algorithm>

#include "packs.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int kLeastTile = 8;        // sorted positions of a group of threads
constexpr int kMostTile = 128;
constexpr int kMostTiles = 4096;     // (more positions than these take longer tiles)
constexpr int kSortThreads = 1024;
constexpr int kMostDigits = 512;
constexpr int kMostSortBlocks = 128;
constexpr int kSortCluster = 8;
constexpr int kRounds = 4;             // items of a thread at a time
constexpr int kClusterSort = 1 << 14;  // positions (16384: 17 us in one launch of 8 blocks, 65536: 47, and 35 in four launches of 64)
// Bytes of the table that are filled beside a launch of the sort; what is left over by a launch of its own, which is faster (1 GB: 148 and 190 us).
constexpr int64_t kFillBeside = 64 << 20, kFillCount = 16 << 20, kFillPlace = 48 << 20;
constexpr int kGroup = 128;          // threads of a block that adds rows
// Positions that are not sorted, and blocks of kDirectLanes vectors for them, at most (each looks through all positions).  Microseconds of the whole call in bfloat16
// without and with the sort: 512 rows of width 512 and 5000 symbols 8.0 and 16.7, 1024 of width 1024 (2048 blocks) 10.7 and 19, 1000 of 2048 (4000) 16.1 and 20.2,
// 1000 of 4096 (8000) 26.9 and 22.6.  All of one symbol: 1000 of 512 23.5 and 26.8, with a table of 100 MB 54 and 42.
constexpr int kDirect = 1024;
constexpr int64_t kDirectBlocks = 4096;
constexpr int kDirectThreads = 256;
constexpr int kDirectLanes = 64;
constexpr int kMostSlabs = 65535;    // of a row, in the second dimension of a grid
constexpr int kJoins = 2;            // groups of them that add the parts of a run

// A symbol of a list of 64- or 32-bit ones.
__device__ __forceinline__ int64_t token_at(const void* tokens, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(tokens)[i] : static_cast<int64_t>(static_cast<const int32_t*>(tokens)[i]);
}

// 16 bytes from any multiple of an element's size: where they are not on a 16-byte boundary, two vectors around them.  [lo, hi) is the
// tensor's memory, beyond which nothing is read.  In two steps, for a thread that has several under way: what the first one loads is not looked at before the
// second (with one after the other the sums of 5003 x 1537 float32 rows took 22 us for 11).
template <class T, bool ALIGNED>
struct Window {
  uint4 a, b;
  const T* p;
  int s;  // bytes behind the boundary; -1: too near to an end of the memory
  __device__ __forceinline__ void begin(const T* from, const char* lo, const char* hi) {
    p = from;
    if constexpr (ALIGNED) {
      a = *reinterpret_cast<const uint4*>(from);
    } else {
      s = static_cast<int>(reinterpret_cast<uintptr_t>(from) & 15);
      const char* g = reinterpret_cast<const char*>(from) - s;
      if (s != 0 && (g < lo || g + 32 > hi)) s = -1;
      if (s >= 0) a = *reinterpret_cast<const uint4*>(g);
      if (s > 0) b = *reinterpret_cast<const uint4*>(g + 16);
    }
  }
  __device__ __forceinline__ uint4 end() const {
    if constexpr (ALIGNED) return a;
    if (s < 0) {
      Pack<T, 16> r;
#pragma unroll
      for (int e = 0; e < Pack<T, 16>::N; ++e) r.v[e] = p[e];
      return *reinterpret_cast<const uint4*>(&r);
    }
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (s & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (s & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const int bits = (s & 3) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// ----------------------------------------------------------------------------- lookup

struct LookupArgs {
  const void* tokens;
  const void* weight;
  void* y;
  const char *lo, *hi;  // the table's memory
  int64_t count, symbols, stride;
  int width, wide, lanes;  // lanes: threads of a row, a power of two
  float scale;
};

template <class T, bool SCALED>
__device__ __forceinline__ uint4 scaled(uint4 bits, float scale) {
  if (!SCALED) return bits;
  Pack<T, 16> p = *reinterpret_cast<Pack<T, 16>*>(&bits);
#pragma unroll
  for (int e = 0; e < Pack<T, 16>::N; ++e) p.v[e] = from_float<T>(to_float(p.v[e]) * scale);
  return *reinterpret_cast<uint4*>(&p);
}

template <class T, bool SCALED, bool ALIGNED>
__global__ void __launch_bounds__(256) embedding_kernel(const LookupArgs p) {
  constexpr int N = Pack<T, 16>::N;
  const int lane = static_cast<int>(threadIdx.x) & (p.lanes - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / p.lanes) + threadIdx.x / p.lanes;
  if (row >= p.count) return;
  const int64_t t = token_at(p.tokens, p.wide, row);
  T* dst = static_cast<T*>(p.y) + row * p.width;
  if (t < 0 || t >= p.symbols) {  // no such symbol: no number either
    for (int c = lane; c < p.width; c += p.lanes) dst[c] = from_float<T>(__int_as_float(0x7fc00000));
    return;
  }
  const T* src = static_cast<const T*>(p.weight) + t * p.stride;
  const int head = min(p.width, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / sizeof(T)));
  const int body = (p.width - head) / N;
  for (int v = lane; v < body; v += 4 * p.lanes) {
    Window<T, ALIGNED> r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v + u * p.lanes < body) r[u].begin(src + head + (v + u * p.lanes) * N, p.lo, p.hi);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v + u * p.lanes < body) *reinterpret_cast<uint4*>(dst + head + (v + u * p.lanes) * N) = scaled<T, SCALED>(r[u].end(), p.scale);
  }
  const int rest = p.width - body * N;  // what lies before the first and behind the last vector
  for (int e = lane; e < rest; e += p.lanes) {
    const int c = e < head ? e : body * N + e;
    dst[c] = SCALED ? from_float<T>(to_float(src[c]) * p.scale) : src[c];
  }
}

// ----------------------------------------------------------------------------- sort

struct SortArgs {
  const void* tokens;  // of the first pass
  int64_t symbols, padding;
  const int32_t *keys, *at;  // of later passes: symbols and positions
  int32_t *keys_out, *at_out;
  int* counts;  // [blocks][digits]
  int count, per_block, blocks, wide, shift, digits;
};

// What a position is sorted by: its symbol; `symbols` where it has no gradient to give.
__device__ __forceinline__ int key_at(const SortArgs& p, int i) {
  if (p.keys != nullptr) return p.keys[i];
  const int64_t t = token_at(p.tokens, p.wide, i);
  return static_cast<int>(t < 0 || t >= p.symbols || t == p.padding ? p.symbols : t);
}

// `bytes` of the table filled with zeros by blocks of kSortThreads, of which this is number `block` of `blocks`.
__device__ __forceinline__ void fill_table(char* table, int64_t bytes, int block, int blocks) {
  const int64_t head = min(bytes, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(table) & 15)) & 15)), body = (bytes - head) / 16;
  uint4* to = reinterpret_cast<uint4*>(table + head);
  const int64_t first = static_cast<int64_t>(block) * kSortThreads + threadIdx.x, step = static_cast<int64_t>(blocks) * kSortThreads;
  for (int64_t i = first; i < body; i += step) to[i] = make_uint4(0, 0, 0, 0);
  if (first < 32) {  // before and behind the vectors, two bytes at a time
    uint16_t *a = reinterpret_cast<uint16_t*>(table), *b = reinterpret_cast<uint16_t*>(table + head + body * 16);
    if (2 * first < head) a[first] = 0;
    if (head + body * 16 + 2 * first < bytes) b[first] = 0;
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs p, char* table, int64_t bytes) {
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= p.blocks) {
    fill_table(table, bytes, static_cast<int>(blockIdx.x) - p.blocks, static_cast<int>(gridDim.x) - p.blocks);
    return;
  }
  pdl_wait();
  __shared__ int n[kMostDigits];
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) n[d] = 0;
  __syncthreads();
  const int begin = static_cast<int>(blockIdx.x) * p.per_block, end = min(p.count, begin + p.per_block);
  for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += kSortThreads) atomicAdd(&n[(key_at(p, i) >> p.shift) & (p.digits - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) p.counts[static_cast<int>(blockIdx.x) * p.digits + d] = n[d];
}

struct SortSpace {
  int next[kMostDigits];                                  // where the block's next item of a digit goes
  uint16_t of_warp[kSortThreads / 32][kMostDigits];       // items of a digit in a warp, then in the warps before
  int sums[kSortThreads / 32];
};

// next[digit] for the items of lower digits in all blocks (`all`: of this thread's digit) and those of this digit in the blocks before.
__device__ __forceinline__ void sort_begin(const SortArgs& p, SortSpace& sp, int all, int before) {
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  int upto = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sp.sums[warp] = upto;
  __syncthreads();
  int lower = 0;
  for (int w = 0; w < warp; ++w) lower += sp.sums[w];
  if (tid < p.digits) sp.next[tid] = lower + upto - all + before;
}
// The block's items in their order, up to kRounds to a thread at a time: a warp has consecutive ones, 32 in each round.
__device__ __forceinline__ void sort_place(const SortArgs& p, SortSpace& sp, int begin, int end) {
  constexpr int W = kSortThreads / 32;
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  for (int base = begin; base < end; base += kRounds * kSortThreads) {
    const int rounds = min(kRounds, (end - base + kSortThreads - 1) / kSortThreads), first = base + warp * rounds * 32 + lane;
    int key[kRounds], at[kRounds], digit[kRounds], rank[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int i = first + r * 32;
      const bool valid = r < rounds && i < end;
      key[r] = valid ? key_at(p, i) : 0;
      at[r] = valid && p.at != nullptr ? p.at[i] : i;
      digit[r] = valid ? (key[r] >> p.shift) & (p.digits - 1) : -1;
    }
    for (int i = lane; i < p.digits; i += 32) sp.of_warp[warp][i] = 0;
    __syncwarp();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (r < rounds) {
        const unsigned same = __match_any_sync(0xffffffffu, digit[r]);
        const int before = __popc(same & ((1u << lane) - 1)), so_far = digit[r] >= 0 ? sp.of_warp[warp][digit[r]] : 0;
        rank[r] = so_far + before;
        __syncwarp();
        if (digit[r] >= 0 && before == 0) sp.of_warp[warp][digit[r]] = static_cast<uint16_t>(so_far + __popc(same));
        __syncwarp();
      }
    }
    __syncthreads();
    int total = 0;
    if (tid < p.digits) {
#pragma unroll 8
      for (int w = 0; w < W; ++w) {
        const int n = sp.of_warp[w][tid];
        sp.of_warp[w][tid] = static_cast<uint16_t>(total);
        total += n;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (digit[r] >= 0) {
        const int to = sp.next[digit[r]] + sp.of_warp[warp][digit[r]] + rank[r];
        p.keys_out[to] = key[r];
        p.at_out[to] = at[r];
      }
    }
    __syncthreads();
    if (tid < p.digits) sp.next[tid] += total;
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortArgs p, char* table, int64_t bytes) {
  __shared__ SortSpace sp;
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= p.blocks) {
    fill_table(table, bytes, static_cast<int>(blockIdx.x) - p.blocks, static_cast<int>(gridDim.x) - p.blocks);
    return;
  }
  pdl_wait();
  const int tid = static_cast<int>(threadIdx.x);
  int before = 0, all = 0;
  if (tid < p.digits) {
    for (int b = 0; b < p.blocks; ++b) {
      const int n = p.counts[b * p.digits + tid];
      all += n;
      before += b < static_cast<int>(blockIdx.x) ? n : 0;
    }
  }
  sort_begin(p, sp, all, before);
  __syncthreads();
  const int begin = static_cast<int>(blockIdx.x) * p.per_block;
  sort_place(p, sp, begin, min(p.count, begin + p.per_block));
}

// All passes in one launch: the first cluster sorts, the others fill `bytes` of the table with zeros.  `keys` and `at`: two lists each.
__global__ void __cluster_dims__(kSortCluster, 1, 1) __launch_bounds__(kSortThreads)
sort_cluster_kernel(SortArgs p, int32_t* keys0, int32_t* keys1, int32_t* at0, int32_t* at1, int passes, int each, char* table, int64_t bytes) {
  __shared__ SortSpace sp;
  __shared__ int counts[kMostDigits];
  const int tid = static_cast<int>(threadIdx.x);
  pdl_launch_dependents();
  if (blockIdx.x >= kSortCluster) {
    fill_table(table, bytes, static_cast<int>(blockIdx.x) - kSortCluster, static_cast<int>(gridDim.x) - kSortCluster);
    return;
  }
  const int begin = min(p.count, static_cast<int>(blockIdx.x) * p.per_block), end = min(p.count, begin + p.per_block);
  for (int pass = 0; pass < passes; ++pass) {
    p.shift = pass * each;
    p.keys_out = pass & 1 ? keys1 : keys0;
    p.at_out = pass & 1 ? at1 : at0;
    for (int d = tid; d < p.digits; d += kSortThreads) counts[d] = 0;
    __syncthreads();
    for (int i = begin + tid; i < end; i += kSortThreads) atomicAdd(&counts[(key_at(p, i) >> p.shift) & (p.digits - 1)], 1);
    cluster_sync_all();
    int before = 0, all = 0;
    if (tid < p.digits) {
#pragma unroll
      for (uint32_t b = 0; b < kSortCluster; ++b) {
        int n;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(n) : "r"(map_to_cta(smem_u32(&counts[tid]), b)) : "memory");
        all += n;
        before += b < blockIdx.x ? n : 0;
      }
    }
    sort_begin(p, sp, all, before);
    __syncthreads();
    sort_place(p, sp, begin, end);
    cluster_sync_all();  // (all have read each other's counts, and what they wrote is seen)
    p.keys = p.keys_out;
    p.at = p.at_out;
  }
}

// ----------------------------------------------------------------------------- sums

struct SumArgs {
  const void* dy;
  const char *lo, *hi;  // its memory
  const int32_t *keys, *at;
  void* dweight;
  float* part;  // [tiles][2][pitch], by slots: of the run that began before the tile, and of the one that goes on behind it
  int64_t stride, pitch;  // pitch: a multiple of 16 bytes of elements, so of four (32 bits) or eight
  int count, symbols, width, tile, lanes;
  int slots;  // vectors of a row, and one more where rows are off 16-byte boundaries
  int slab;   // of the launch's first blocks: of `lanes` (or, the same where it is not 0, kGroup) vectors of a row
  int base;   // elements that the table's first is behind such a boundary
  float scale;
};

// A thread's columns of symbol key's row begin `slot` vectors behind the 16-byte boundary at or before the row (so that the row is written in whole vectors wherever it
// lies): with the first of them before the row for the first thread of a row that is off one.
template <class T>
__device__ __forceinline__ int column_of(const SumArgs& p, int key, int slot) {
  constexpr int N = Pack<T, 16>::N;
  return slot * N - static_cast<int>((static_cast<uint32_t>(p.base) + static_cast<uint32_t>(key) * static_cast<uint32_t>(p.width)) & (N - 1));
}
template <class T>
__device__ __forceinline__ void store_row(const SumArgs& p, int key, int slot, const float* acc) {
  constexpr int N = Pack<T, 16>::N;
  const int c = column_of<T>(p, key, slot);
  T* dst = static_cast<T*>(p.dweight) + static_cast<int64_t>(key) * p.width + c;
  Pack<T, 16> r;
#pragma unroll
  for (int e = 0; e < N; ++e) r.v[e] = from_float<T>(acc[e] * p.scale);
  if (c >= 0 && c + N <= p.width) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(&r);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e >= 0 && c + e < p.width) dst[e] = r.v[e];
  }
}

// A thread's columns of a row of dy, in two steps as above.
template <class T, bool ALIGNED>
struct Columns {
  Window<T, ALIGNED> w;
  int c;
  __device__ __forceinline__ void begin(const SumArgs& p, int at, int column) {
    c = column;
    if (inside(p)) w.begin(static_cast<const T*>(p.dy) + at * p.stride + c, p.lo, p.hi);
    w.p = static_cast<const T*>(p.dy) + at * p.stride + c;
  }
  __device__ __forceinline__ bool inside(const SumArgs& p) const { return ALIGNED || (c >= 0 && c + Pack<T, 16>::N <= p.width); }
  __device__ __forceinline__ uint4 end(const SumArgs& p) const {
    if (inside(p)) return w.end();
    Pack<T, 16> r;
#pragma unroll
    for (int e = 0; e < Pack<T, 16>::N; ++e) r.v[e] = c + e >= 0 && c + e < p.width ? w.p[e] : from_float<T>(0.f);
    return *reinterpret_cast<const uint4*>(&r);
  }
};

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kGroup) embedding_sum_kernel(const SumArgs p) {
  constexpr int N = Pack<T, 16>::N, kAhead = 4;  // rows of a thread under way (65536 x 4096 bfloat16, the whole step: 424 us, 8: 446, 16: 500)
  const int groups = kGroup / p.lanes;
  const int64_t tile = static_cast<int64_t>(blockIdx.x) * groups + threadIdx.x / p.lanes;
  const int slot = (p.slab + static_cast<int>(blockIdx.y)) * p.lanes + (static_cast<int>(threadIdx.x) & (p.lanes - 1));
  const int64_t first = tile * p.tile;
  pdl_launch_dependents();
  pdl_wait();
  if (first >= p.count || slot >= p.slots) return;
  const int begin = static_cast<int>(first), end = static_cast<int>(min(first + p.tile, static_cast<int64_t>(p.count)));
  float* part = p.part + tile * 2 * p.pitch + slot * N;
  const int before = begin > 0 ? p.keys[begin - 1] : -1, behind = end < p.count ? p.keys[end] : -1;
  float acc[N];
  int run = -1;  // the symbol whose rows are in acc
  bool head = false;
  const auto leave = [&](bool last) {
    if (run < 0) return;
    if (head || (last && run == behind)) {
      float4* to = reinterpret_cast<float4*>(part + (head ? 0 : p.pitch));
#pragma unroll
      for (int e = 0; e < N / 4; ++e) to[e] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
    } else {
      store_row<T>(p, run, slot, acc);
    }
  };
  // (the symbols and positions of the next rows are fetched with the rows before them)
  int key[kAhead], at[kAhead];
  const auto fetch = [&](int i) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      key[u] = i + u < end ? p.keys[i + u] : p.symbols;
      at[u] = i + u < end ? p.at[i + u] : 0;
    }
  };
  fetch(begin);
  for (int i = begin; i < end; i += kAhead) {
    Columns<T, ALIGNED> row[kAhead];
    int now[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      now[u] = key[u];
      if (key[u] < p.symbols) row[u].begin(p, at[u], ALIGNED ? slot * N : column_of<T>(p, key[u], slot));
    }
    if (now[0] >= p.symbols) break;  // (they are the last ones)
    fetch(i + kAhead);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (now[u] >= p.symbols) break;
      const uint4 bits = row[u].end(p);
      const Pack<T, 16> r = *reinterpret_cast<const Pack<T, 16>*>(&bits);
      if (now[u] != run) {
        leave(false);
        run = now[u];
        head = i + u == begin && run == before;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = to_float(r.v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += to_float(r.v[e]);
      }
    }
  }
  leave(true);
}

// Runs over the borders of tiles: the block of the tile in which one begins adds its parts.
template <class T>
__global__ void __launch_bounds__(kGroup * kJoins) embedding_join_kernel(const SumArgs p) {
  constexpr int N = Pack<T, 16>::N, THREADS = kGroup * kJoins;
  __shared__ int ends;
  __shared__ float sums[kJoins][N][kGroup];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tile;
  const int begin = static_cast<int>(first);
  const int64_t end = first + p.tile;
  if (end >= p.count) return;
  const int run = p.keys[end - 1];
  if (run >= p.symbols || p.keys[end] != run) return;                         // none goes on
  if (begin > 0 && p.keys[begin] == run && p.keys[begin - 1] == run) return;  // it began before
  // how many tiles behind this one it reaches: a thread to a tile looks whether it goes on behind that
  int tiles = 1;
  for (int64_t base = end;; base += static_cast<int64_t>(THREADS) * p.tile) {
    if (threadIdx.x == 0) ends = THREADS;
    __syncthreads();
    const int64_t next = base + (static_cast<int64_t>(threadIdx.x) + 1) * p.tile;  // where the tile behind that begins
    if (next >= p.count || p.keys[next - 1] != run || p.keys[next] != run) atomicMin(&ends, static_cast<int>(threadIdx.x));
    __syncthreads();
    const int here = ends;
    tiles += here;
    if (here < THREADS) break;
    __syncthreads();
  }
  // each of the kJoins groups of threads has a share of the parts (the first one first of all the part of this tile); of few parts the first one all
  const int group = static_cast<int>(threadIdx.x) / kGroup, lane = static_cast<int>(threadIdx.x) % kGroup;
  const bool alone = tiles < 4 * kJoins;
  if (alone && group != 0) return;
  const int slot = (p.slab + static_cast<int>(blockIdx.y)) * kGroup + lane;
  const bool mine = slot < p.slots;
  alignas(16) float acc[N] = {};
  const float4* part = reinterpret_cast<const float4*>(p.part + (static_cast<int64_t>(blockIdx.x) * 2 + 1) * p.pitch + slot * N);
  if (mine) {
    const int each = alone ? tiles : (tiles + kJoins - 1) / kJoins, last = min(tiles, (group + 1) * each);
    if (group == 0) {
#pragma unroll
      for (int e = 0; e < N / 4; ++e) *reinterpret_cast<float4*>(acc + 4 * e) = part[e];
    }
    part += p.pitch / 4;  // the first part of the next tile
#pragma unroll 8
    for (int k = group * each; k < last; ++k) {
#pragma unroll
      for (int e = 0; e < N / 4; ++e) {
        const float4 x = part[static_cast<int64_t>(k) * (p.pitch / 2) + e];
        acc[4 * e] += x.x;
        acc[4 * e + 1] += x.y;
        acc[4 * e + 2] += x.z;
        acc[4 * e + 3] += x.w;
      }
    }
  }
  if (!alone) {
#pragma unroll
    for (int e = 0; e < N; ++e) sums[group][e][lane] = acc[e];
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int g = 1; g < kJoins; ++g)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += sums[g][e][lane];
    }
  }
  if (group == 0 && mine) store_row<T>(p, run, slot, acc);
}

// ----------------------------------------------------------------------------- few positions

__global__ void __launch_bounds__(kSortThreads) embedding_fill_kernel(char* table, int64_t bytes) {
  pdl_launch_dependents();
  fill_table(table, bytes, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
}

// Without a sort: the block of a position looks through all of them for its symbol and, where none of them comes earlier, adds up the rows of
// those that have it, a consecutive share of them to each group of threads.  All but the last store runs beside the launch that fills the table.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kDirectThreads) embedding_direct_kernel(const SumArgs p, const void* tokens, int wide, int64_t padding) {
  constexpr int N = Pack<T, 16>::N, kAhead = 8, kRounds = kDirect / kDirectThreads, kWarps = kDirectThreads / 32;
  static_assert(kRounds * kWarps == 32, "a lane to each warp's round");
  __shared__ uint16_t list[kDirect];
  __shared__ int before[kRounds][kWarps], found;
  __shared__ float sums[kDirectThreads / kDirectLanes - 1][N][kDirectLanes];
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, warp_lane = tid & 31, here = static_cast<int>(blockIdx.x);
  const int64_t own = token_at(tokens, wide, here);
  unsigned same[kRounds];
  bool earlier = own < 0 || own >= p.symbols || own == padding;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int i = r * kDirectThreads + tid;
    const bool match = i < p.count && token_at(tokens, wide, i) == own;
    earlier = earlier || (match && i < here);
    same[r] = __ballot_sync(0xffffffffu, match);
    if (warp_lane == 0) before[r][warp] = __popc(same[r]);
  }
  if (__syncthreads_or(earlier)) {
    pdl_wait();
    return;
  }
  if (warp == 0) {
    int* n = &before[0][0] + warp_lane;
    const int mine = *n;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (warp_lane >= o) upto += v;
    }
    *n = upto - mine;
    if (warp_lane == 31) found = upto;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (same[r] >> warp_lane & 1) list[before[r][warp] + __popc(same[r] & ((1u << warp_lane) - 1))] = static_cast<uint16_t>(r * kDirectThreads + tid);
  __syncthreads();

  const int groups = kDirectThreads / kDirectLanes, group = tid / kDirectLanes, lane = tid % kDirectLanes;
  const int slot = static_cast<int>(blockIdx.y) * kDirectLanes + lane, key = static_cast<int>(own);
  const int each = (found + groups - 1) / groups, end = min(found, (group + 1) * each);
  const bool mine = slot < p.slots;
  float acc[N] = {};
  if (mine) {
    const int column = ALIGNED ? slot * N : column_of<T>(p, key, slot);
    for (int i = group * each; i < end; i += kAhead) {
      Columns<T, ALIGNED> row[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u < end) row[u].begin(p, list[i + u], column);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i + u >= end) break;
        const uint4 bits = row[u].end(p);
        const Pack<T, 16> r = *reinterpret_cast<const Pack<T, 16>*>(&bits);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += to_float(r.v[e]);
      }
    }
  }
  if (found > 1) {
    if (group > 0) {
#pragma unroll
      for (int e = 0; e < N; ++e) sums[group - 1][e][lane] = acc[e];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int g = 0; g < groups - 1; ++g)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += sums[g][e][lane];
    }
  }
  pdl_wait();
  if (group == 0 && mine) store_row<T>(p, key, slot, acc);
}

// ----------------------------------------------------------------------------- host

bool type_ok(int type) { return type >= TRITURUS_B200_TYPE_F32 && type <= TRITURUS_B200_TYPE_F16; }
int size_of(int type) { return type == TRITURUS_B200_TYPE_F32 ? 4 : 2; }
bool sizes_ok(int64_t count, int64_t symbols, int64_t width, int type, int token_bytes) {
  return count >= 0 && count <= (1ll << 30) && symbols > 0 && symbols < (1ll << 30) && width > 0 && width <= (1ll << 30) && type_ok(type) &&
         (token_bytes == 4 || token_bytes == 8);
}
template <class F>
int by_type(int type, F fn) {
  return type == TRITURUS_B200_TYPE_F32 ? fn(0.f) : type == TRITURUS_B200_TYPE_BF16 ? fn(__nv_bfloat16()) : fn(__half());
}

// The least power of two that is not below n, of at most `most`.
int lanes_for(int64_t n, int most) {
  int l = 1;
  while (l < most && l < n) l <<= 1;
  return l;
}
// Vectors of a row, and one more.
int64_t slots_of(int64_t width, int size) { return (width * size + 15) / 16 + 1; }
int64_t part_pitch(int64_t width, int size) { return slots_of(width, size) * (16 / size); }
// Sorted positions of a tile: some 12 blocks of threads to an SM, between latency (few long tiles) and the parts of runs over borders (many short ones).
int tile_of(int64_t count, int64_t width, int size) {
  const int64_t vectors = (width * size + 15) / 16;
  const int64_t tile = count * vectors / (static_cast<int64_t>(kGroup) * 12 * device_sms());
  return static_cast<int>(std::max<int64_t>(std::clamp<int64_t>(tile, kLeastTile, kMostTile), (count + kMostTiles - 1) / kMostTiles));
}

struct SumSpace {  // the workspace: keys and positions twice, the counts, the parts
  size_t list, counts, part, bytes;
};
SumSpace space_of(int64_t count, int64_t width, int size) {
  const auto up = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
  SumSpace s;
  s.list = up(static_cast<size_t>(count) * 4);
  s.counts = up(static_cast<size_t>(kMostSortBlocks) * kMostDigits * 4);
  const int64_t tile = tile_of(count, width, size), tiles = (count + tile - 1) / tile;
  s.part = up(static_cast<size_t>(tiles) * 2 * static_cast<size_t>(part_pitch(width, size)) * 4);
  s.bytes = 4 * s.list + s.counts + s.part;
  return s;
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" {

int triturus_b200_embedding(const void* tokens, int token_bytes, const void* weight, void* y, int64_t count, int64_t symbols, int64_t width,
                            int64_t weight_stride, int type, float scale, void* stream) {
  if (!sizes_ok(count, symbols, width, type, token_bytes)) return TRITURUS_B200_EINVAL;
  if (count == 0) return TRITURUS_B200_OK;
  if (tokens == nullptr || weight == nullptr || y == nullptr) return TRITURUS_B200_EINVAL;
  const int size = size_of(type);
  if (!aligned_to(tokens, token_bytes) || !aligned_to(weight, size) || !aligned_to(y, size)) return TRITURUS_B200_EALIGN;
  LookupArgs p = {};
  p.tokens = tokens;
  p.weight = weight;
  p.y = y;
  const int64_t far = (symbols - 1) * weight_stride * size;
  p.lo = static_cast<const char*>(weight) + std::min<int64_t>(far, 0);
  p.hi = static_cast<const char*>(weight) + std::max<int64_t>(far, 0) + width * size;
  p.count = count;
  p.symbols = symbols;
  p.stride = weight_stride;
  p.width = static_cast<int>(width);
  p.wide = token_bytes == 8;
  p.lanes = lanes_for((width * size / 16 + 3) / 4, 256);
  p.scale = scale;
  const int64_t rows = 256 / p.lanes;
  const dim3 grid(static_cast<unsigned>((count + rows - 1) / rows));
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    const bool aligned = aligned_to(weight, 16) && aligned_to(y, 16) && width * size % 16 == 0 && weight_stride * size % 16 == 0;
    const auto run = [&](auto kern) { return launch_of(kern, grid, 256, 0, static_cast<cudaStream_t>(stream), nullptr, p); };
    if (scale == 1.f) return aligned ? run(embedding_kernel<T, false, true>) : run(embedding_kernel<T, false, false>);
    return aligned ? run(embedding_kernel<T, true, true>) : run(embedding_kernel<T, true, false>);
  });
}

size_t triturus_b200_embedding_backward_workspace_bytes(int64_t count, int64_t symbols, int64_t width, int type) {
  return sizes_ok(count, symbols, width, type, 8) ? space_of(count, width, size_of(type)).bytes : 0;
}

int triturus_b200_embedding_backward(const void* dy, const void* tokens, int token_bytes, void* dweight, int64_t count, int64_t symbols,
                                     int64_t width, int64_t dy_stride, int type, float scale, int64_t padding, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (!sizes_ok(count, symbols, width, type, token_bytes) || dweight == nullptr) return TRITURUS_B200_EINVAL;
  const int size = size_of(type);
  if (!aligned_to(dweight, size)) return TRITURUS_B200_EALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (count > 0) {
    if (dy == nullptr || tokens == nullptr || workspace == nullptr) return TRITURUS_B200_EINVAL;
    if (!aligned_to(dy, size) || !aligned_to(tokens, token_bytes) || !aligned_to(workspace, 16)) return TRITURUS_B200_EALIGN;
    if (workspace_bytes < space_of(count, width, size).bytes) return TRITURUS_B200_EWORKSPACE;
  }
  const int64_t table = symbols * width * size;
  int rc = TRITURUS_B200_OK;
  if (count == 0) return code_of(cudaMemsetAsync(dweight, 0, static_cast<size_t>(table), st));

  SumArgs p = {};
  p.dy = dy;
  const int64_t far = (count - 1) * dy_stride * size;
  p.lo = static_cast<const char*>(dy) + std::min<int64_t>(far, 0);
  p.hi = static_cast<const char*>(dy) + std::max<int64_t>(far, 0) + width * size;
  p.dweight = dweight;
  p.stride = dy_stride;
  p.pitch = part_pitch(width, size);
  p.count = static_cast<int>(count);
  p.symbols = static_cast<int>(symbols);
  p.width = static_cast<int>(width);
  p.tile = tile_of(count, width, size);
  p.scale = scale;
  const bool off = width * size % 16 != 0 || !aligned_to(dweight, 16);
  const int64_t vectors = slots_of(width, size);  // (room for one more than rows on boundaries have)
  p.slots = static_cast<int>(off ? vectors : vectors - 1);
  p.base = static_cast<int>(reinterpret_cast<uintptr_t>(dweight) % 16) / size;
  const bool aligned = !off && aligned_to(dy, 16) && dy_stride * size % 16 == 0;
  const int64_t direct_slabs = (p.slots + kDirectLanes - 1) / kDirectLanes;
  if (count <= kDirect && count * direct_slabs <= kDirectBlocks) {
    const int64_t beside = std::min(table, kFillBeside), rest = table - beside;
    const int64_t fills = std::clamp<int64_t>(beside / (16 * kSortThreads * 4), 1, device_sms());
    if (rest > 0) rc = code_of(cudaMemsetAsync(static_cast<char*>(dweight) + beside, 0, static_cast<size_t>(rest), st));
    if (rc == TRITURUS_B200_OK)
      rc = launch_of(embedding_fill_kernel, dim3(static_cast<unsigned>(fills)), kSortThreads, 0, st, nullptr, static_cast<char*>(dweight), beside);
    if (rc != TRITURUS_B200_OK) return rc;
    return by_type(type, [&](auto t) {
      using T = decltype(t);
      const cudaLaunchAttribute dependent = dependent_launch();
      return launch_of(aligned ? embedding_direct_kernel<T, true> : embedding_direct_kernel<T, false>,
                       dim3(static_cast<unsigned>(count), static_cast<unsigned>(direct_slabs)), kDirectThreads, 0, st, &dependent, p, tokens,
                       token_bytes == 8 ? 1 : 0, padding);
    });
  }

  const SumSpace space = space_of(count, width, size);
  char* ws = static_cast<char*>(workspace);
  const auto list = [&](int i) { return reinterpret_cast<int32_t*>(ws + i * space.list); };
  SortArgs s = {};
  s.tokens = tokens;
  s.symbols = symbols;
  s.padding = padding;
  s.counts = reinterpret_cast<int*>(ws + 4 * space.list);
  s.count = static_cast<int>(count);
  s.wide = token_bytes == 8;
  int bits = 1;
  while ((symbols >> bits) != 0) ++bits;  // (of 0 ... symbols)
  const int passes = (bits + 8) / 9, each = (bits + passes - 1) / passes;
  s.digits = 1 << each;
  const auto per_block = [&](int64_t blocks) { return static_cast<int>((count + blocks * kSortThreads - 1) / (blocks * kSortThreads)) * kSortThreads; };
  if (count <= kClusterSort) {
    const int64_t beside = std::min(table, kFillBeside), rest = table - beside;
    const int64_t fills = std::clamp<int64_t>(beside / (16 * kSortThreads * 4), 1, 2 * device_sms());
    if (rest > 0) rc = code_of(cudaMemsetAsync(static_cast<char*>(dweight) + beside, 0, static_cast<size_t>(rest), st));
    if (rc == TRITURUS_B200_OK) {
      s.per_block = per_block(kSortCluster);
      const int64_t grid = (kSortCluster + fills + kSortCluster - 1) / kSortCluster * kSortCluster;
      rc = launch_of(sort_cluster_kernel, dim3(static_cast<unsigned>(grid)), kSortThreads, 0, st, nullptr, s, list(0), list(1), list(2), list(3), passes, each,
                     static_cast<char*>(dweight), beside);
    }
    s.keys = list((passes - 1) & 1);
    s.at = list(2 + ((passes - 1) & 1));
  } else {
    s.per_block = per_block(kMostSortBlocks);
    s.blocks = static_cast<int>((count + s.per_block - 1) / s.per_block);
    const int64_t beside = std::min(table, passes * (kFillCount + kFillPlace));
    if (table > beside) rc = code_of(cudaMemsetAsync(static_cast<char*>(dweight) + beside, 0, static_cast<size_t>(table - beside), st));
    int64_t filled = 0;
    bool first = true;
    const cudaLaunchAttribute dependent = dependent_launch();
    const auto run = [&](void (*kern)(SortArgs, char*, int64_t), int64_t most) {
      const int64_t bytes = std::min(most, beside - filled);
      const int64_t blocks = bytes == 0 ? 0 : std::clamp<int64_t>(bytes / (16 * kSortThreads * 4), 1, device_sms());
      const int code = launch_of(kern, dim3(static_cast<unsigned>(s.blocks + blocks)), kSortThreads, 0, st, first ? nullptr : &dependent, s,
                                 static_cast<char*>(dweight) + filled, bytes);
      filled += bytes;
      first = false;
      return code;
    };
    for (int pass = 0; pass < passes && rc == TRITURUS_B200_OK; ++pass) {
      s.shift = pass * each;
      s.keys_out = list(pass & 1);
      s.at_out = list(2 + (pass & 1));
      rc = run(sort_count_kernel, kFillCount);
      if (rc == TRITURUS_B200_OK) rc = run(sort_place_kernel, kFillPlace);
      s.keys = s.keys_out;
      s.at = s.at_out;
    }
  }
  if (rc != TRITURUS_B200_OK) return rc;

  p.keys = s.keys;
  p.at = s.at;
  p.part = reinterpret_cast<float*>(ws + 4 * space.list + space.counts);
  p.lanes = lanes_for(p.slots, kGroup);
  const int64_t tiles = (count + p.tile - 1) / p.tile, groups = kGroup / p.lanes;
  const int slabs = (p.slots + p.lanes - 1) / p.lanes;
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    const cudaLaunchAttribute dependent = dependent_launch();
    int code = TRITURUS_B200_OK;
    for (p.slab = 0; p.slab < slabs && code == TRITURUS_B200_OK; p.slab += kMostSlabs) {
      const unsigned here = static_cast<unsigned>(std::min(slabs - p.slab, kMostSlabs));
      code = launch_of(aligned ? embedding_sum_kernel<T, true> : embedding_sum_kernel<T, false>, dim3(static_cast<unsigned>((tiles + groups - 1) / groups), here), kGroup, 0, st, &dependent, p);
      if (code == TRITURUS_B200_OK && tiles > 1)
        code = launch_of(embedding_join_kernel<T>, dim3(static_cast<unsigned>(tiles), here), kGroup * kJoins, 0, st, &dependent, p);
    }
    return code;
  });
}

}  // extern "C"
