// The norm of many tensors taken as one vector, and their scaling to a limit.
//
//   n = sqrt(sum x^2) or max |x| over all elements of all tensors;  c = min(1, limit / (n + 1e-6));  x <- c x
//
// The tensors are cut into chunks of kChunk bytes that begin on 16-byte boundaries of memory (the first of a tensor may begin with a partial
// vector), and each block has a run of them.  Bound by memory: all is read once for the norm and, where the norm is above the limit, read again
// and written.  First launch: each block's sum of squares, in 64 bits.  Second launch: every block adds those sums in the same order, so
// that all have the same n, and scales its chunks, the last one first: what the first launch read last is still in the L2 cache.  Where c is
// 1 nothing is written.
//
// Measured on one B200: the norm alone of 1 GB and more at the copy bandwidth (146 us a GB), 120 MB 24.7 us; with the product 120 MB 59.8 us, 1.46 GB 717 us =
// 0.94 of three passes.  The second read of what the L2 cache still holds saves little, since the last call's written lines leave the cache
// at the same time.  (Of the blocks' four 16-byte loads under way and the next four, ncu: DRAM 63 and 61 %.)
//
// A few small tensors are one launch: a cluster of blocks that keep their chunks in registers from the sum to the product (15 chunks in 12 tensors: 4.7 us of the
// GPU, 8.2 a call with its Python).
#include <algorithm>
#include <cstring>

#include "../../include/triturus_b200.h"
#include "packs.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int kChunk = 32768;
constexpr int kThreads = 512;
constexpr int kVectors = kChunk / 16 / kThreads;  // of a chunk, to a thread
constexpr int kMostTensors = 1024;                // of one launch: what fits its parameters
constexpr int kMostBlocks = 1024;

template <int MOST>
struct TensorList {
  void* data[MOST];
  int64_t bytes[MOST];
  uint32_t first[MOST];  // number of the tensor's first chunk
  uint8_t type[MOST];
  int count;
  uint32_t chunks;
};

struct ClipArgs {
  double* sums;     // a block's sum of squares, or its largest magnitude
  int sums_here;    // number of the launch's first one
  int sums_in_all;
  double limit;
  float* norm;
  int largest;      // the norm is the largest magnitude
};

struct Chunk {
  uint8_t* base;   // on a 16-byte boundary: the chunk's first byte, if the tensor began there
  int begin, end;  // the tensor's bytes of the chunk
  int type;
};

// A place in the list: a chunk and its tensor.
struct Cursor {
  uint32_t chunk;
  int tensor;
};
template <int MOST>
__device__ __forceinline__ Cursor cursor_at(const TensorList<MOST>& l, uint32_t c) {
  int lo = 0, hi = l.count;  // the last tensor whose first chunk is not behind c
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= c)
      lo = mid;
    else
      hi = mid;
  }
  return {c, lo};
}
template <int MOST>
__device__ __forceinline__ Chunk chunk_at(const TensorList<MOST>& l, const Cursor& at) {
  const uintptr_t data = reinterpret_cast<uintptr_t>(l.data[at.tensor]);
  const int skip = static_cast<int>(data & 15);
  const int64_t off = static_cast<int64_t>(at.chunk - l.first[at.tensor]) * kChunk;
  const int64_t left = skip + l.bytes[at.tensor] - off;
  Chunk k;
  k.base = reinterpret_cast<uint8_t*>(data - skip) + off;
  k.begin = off == 0 ? skip : 0;
  k.end = static_cast<int>(left < kChunk ? left : kChunk);
  k.type = l.type[at.tensor];
  return k;
}

// The vectors of a chunk that are the thread's, as bits; what lies outside of the tensor is zero.
struct Bits {
  uint4 v[kVectors];
};
__device__ __forceinline__ int offset_of(int i) { return (i * kThreads + static_cast<int>(threadIdx.x)) * 16; }
__device__ __forceinline__ void load_chunk(const Chunk& k, Bits& b) {
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int o = offset_of(i);
    if (o >= k.begin && o + 16 <= k.end) {
      b.v[i] = *reinterpret_cast<const uint4*>(k.base + o);
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 8; ++h)
        if (o + 2 * h >= k.begin && o + 2 * h < k.end) w[h / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(k.base + o + 2 * h)) << (h % 2 * 16);
      b.v[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
__device__ __forceinline__ void store_chunk(const Chunk& k, const Bits& b) {
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int o = offset_of(i);
    if (o >= k.begin && o + 16 <= k.end) {
      __stcs(reinterpret_cast<uint4*>(k.base + o), b.v[i]);
    } else {
      const uint32_t w[4] = {b.v[i].x, b.v[i].y, b.v[i].z, b.v[i].w};
#pragma unroll
      for (int h = 0; h < 8; ++h)
        if (o + 2 * h >= k.begin && o + 2 * h < k.end) *reinterpret_cast<uint16_t*>(k.base + o + 2 * h) = static_cast<uint16_t>(w[h / 2] >> (h % 2 * 16));
    }
  }
}

// f(numbers) for each vector, with T's N numbers of it.
template <class T, class F>
__device__ __forceinline__ void for_vectors(const Bits& b, F f) {
  constexpr int N = Pack<T, 16>::N;
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const Pack<T, 16> p = *reinterpret_cast<const Pack<T, 16>*>(&b.v[i]);
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_float(p.v[e]);
    f(x);
  }
}
// What the elements are multiplied by: c, then unit.  A factor below the least normal number has no 24 digits of its own; it is held in units of
// 2^-126, else unit is 1.
struct Factor {
  float c, unit;
  __device__ __forceinline__ bool one() const { return c == 1.f; }
};
template <class T>
__device__ __forceinline__ void scale_bits(Bits& b, Factor f) {
  constexpr int N = Pack<T, 16>::N;
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    Pack<T, 16>& p = *reinterpret_cast<Pack<T, 16>*>(&b.v[i]);
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = from_float<T>(to_float(p.v[e]) * f.c * f.unit);
  }
}
__device__ __forceinline__ void scale_bits(Bits& b, int type, Factor f) {
  if (type == TRITURUS_B200_TYPE_F32)
    scale_bits<float>(b, f);
  else if (type == TRITURUS_B200_TYPE_BF16)
    scale_bits<__nv_bfloat16>(b, f);
  else
    scale_bits<__half>(b, f);
}

// Adds the squares of a chunk's elements.  A vector's squares are added in 32 bits where they neither overflow nor lose digits
// below the least normal number, else in 64 bits: a norm that 32 bits can hold is not lost to its square.  The largest magnitude is held as
// bits: those of a NaN are above those of infinity.
struct Sum {
  double squares;
  uint32_t most;
};
template <class T>
__device__ __forceinline__ void add_bits(const Bits& b, bool largest, Sum& sum) {
  constexpr int N = Pack<T, 16>::N;
  if (largest) {
    for_vectors<T>(b, [&](const float(&x)[N]) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum.most = max(sum.most, __float_as_uint(x[e]) & 0x7fffffffu);
    });
  } else {
    for_vectors<T>(b, [&](const float(&x)[N]) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) s = fmaf(x[e], x[e], s);
      if (s > 1e-25f && s < 1e38f) {
        sum.squares += static_cast<double>(s);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) sum.squares = fma(static_cast<double>(x[e]), static_cast<double>(x[e]), sum.squares);
      }
    });
  }
}
__device__ __forceinline__ void add_bits(const Bits& b, int type, bool largest, Sum& sum) {
  if (type == TRITURUS_B200_TYPE_F32)
    add_bits<float>(b, largest, sum);
  else if (type == TRITURUS_B200_TYPE_BF16)
    add_bits<__nv_bfloat16>(b, largest, sum);
  else
    add_bits<__half>(b, largest, sum);
}
__device__ __forceinline__ double sum_of(const Sum& sum, bool largest) {
  return largest ? static_cast<double>(__uint_as_float(sum.most)) : sum.squares;
}

__device__ __forceinline__ double combine(double a, double b, bool largest) {
  if (!largest) return a + b;
  return b > a || b != b ? b : a;  // (a NaN stays: b > NaN is false)
}

// The sum (or largest) of a block's values, in thread 0.
__device__ __forceinline__ double block_combine(double v, double* part, bool largest) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = combine(v, __shfl_down_sync(0xffffffffu, v, o), largest);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = threadIdx.x < kThreads / 32 ? part[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = combine(v, __shfl_down_sync(0xffffffffu, v, o), largest);
  }
  return v;
}

// The norm and the factor from the sum of all, for thread 0.
__device__ __forceinline__ Factor factor_of(const ClipArgs& p, double sum, float* norm) {
  const double n = p.largest ? sum : sqrt(sum);
  *norm = static_cast<float>(n);
  // (a norm beyond 32 bits still has its factor; a NaN among the elements makes all of them NaN)
  if (n + 1e-6 <= p.limit) return {1.f, 1.f};
  const double c = p.limit / (n + 1e-6);
  return c < 0x1p-126 ? Factor{static_cast<float>(c * 0x1p126), 0x1p-126f} : Factor{static_cast<float>(c), 1.f};
}

// The block's run of chunks.
__device__ __forceinline__ uint32_t run_start(uint32_t chunks, uint32_t block, uint32_t blocks) {
  return static_cast<uint32_t>(static_cast<uint64_t>(chunks) * block / blocks);
}

template <int MOST>
__global__ void __launch_bounds__(kThreads) norm_parts_kernel(const __grid_constant__ TensorList<MOST> l, const ClipArgs p) {
  __shared__ double part[kThreads / 32];
  pdl_launch_dependents();  // (all blocks are resident: the next launch's take their places as they leave)
  Sum sum = {0.0, 0};
  Cursor at = cursor_at(l, run_start(l.chunks, blockIdx.x, gridDim.x));
  const uint32_t end = run_start(l.chunks, blockIdx.x + 1, gridDim.x);
  if (at.chunk < end) {
    Chunk k = chunk_at(l, at);
    Bits now;
    load_chunk(k, now);
    for (;;) {  // (the next chunk is under way while one is added)
      const int type = k.type;
      Bits next;
      const bool more = ++at.chunk < end;
      if (more) {
        if (at.tensor + 1 < l.count && at.chunk >= l.first[at.tensor + 1]) ++at.tensor;
        k = chunk_at(l, at);
        load_chunk(k, next);
      }
      add_bits(now, type, p.largest, sum);
      if (!more) break;
      now = next;
    }
  }
  const double v = block_combine(sum_of(sum, p.largest), part, p.largest);
  if (threadIdx.x == 0) p.sums[p.sums_here + blockIdx.x] = v;
}

// `scale` == 0: the norm alone (one block).
template <int MOST>
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ TensorList<MOST> l, const ClipArgs p, int scale) {
  __shared__ double part[kThreads / 32];
  __shared__ Factor factor;
  const uint32_t begin = run_start(l.chunks, blockIdx.x, gridDim.x);
  Cursor at = {0, 0};
  Chunk k = {};
  Bits now;
  if (scale) {  // (no launch before this one writes the elements, but for an earlier list's: they are read while it ends)
    at = cursor_at(l, run_start(l.chunks, blockIdx.x + 1, gridDim.x) - 1);  // (no more blocks than chunks)
    k = chunk_at(l, at);
    load_chunk(k, now);
  }
  pdl_wait();
  double v = 0.0;
  for (int i = threadIdx.x; i < p.sums_in_all; i += kThreads) v = combine(v, p.sums[i], p.largest);
  v = block_combine(v, part, p.largest);
  if (threadIdx.x == 0) {
    float n;
    factor = factor_of(p, v, &n);
    if (blockIdx.x == 0 && p.sums_here == 0) *p.norm = n;
  }
  __syncthreads();
  const Factor c = factor;
  if (!scale || c.one()) return;
  for (;;) {
    const Chunk here = k;
    Bits next;
    const bool more = at.chunk > begin;
    if (more) {
      --at.chunk;
      if (at.chunk < l.first[at.tensor]) --at.tensor;
      k = chunk_at(l, at);
      load_chunk(k, next);
    }
    scale_bits(now, here.type, c);
    store_chunk(here, now);
    if (!more) break;
    now = next;
  }
}

// All in one launch, for up to C * kHeld chunks: the blocks of a cluster hold them.
constexpr int kHeld = 2;
template <int C>
__global__ void __launch_bounds__(kThreads) clip_small_kernel(const __grid_constant__ TensorList<64> l, const ClipArgs p, int scale) {
  __shared__ double part[kThreads / 32];
  __shared__ double block_sum;
  __shared__ Factor factor;
  Chunk k[kHeld];
  Bits held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const uint32_t c = blockIdx.x + i * C;
    if (c < l.chunks) {
      k[i] = chunk_at(l, cursor_at(l, c));
      load_chunk(k[i], held[i]);
    }
  }
  Sum sum = {0.0, 0};
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (blockIdx.x + i * C < l.chunks) add_bits(held[i], k[i].type, p.largest, sum);
  double v = block_combine(sum_of(sum, p.largest), part, p.largest);
  if (threadIdx.x == 0) block_sum = v;
  if (C > 1) cluster_sync_all();
  if (threadIdx.x == 0) {
    if (C > 1) {
      v = 0.0;
      for (int q = 0; q < C; ++q) {
        double other;
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(other) : "r"(map_to_cta(smem_u32(&block_sum), q)) : "memory");
        v = combine(v, other, p.largest);
      }
    }
    float n;
    factor = factor_of(p, v, &n);
    if (blockIdx.x == 0) *p.norm = n;
  }
  __syncthreads();
  const Factor c = factor;
  if (scale && !c.one()) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (blockIdx.x + i * C < l.chunks) {
        scale_bits(held[i], k[i].type, c);
        store_chunk(k[i], held[i]);
      }
  }
  if (C > 1) cluster_sync_all();  // (the others' sums are read until here)
}

// ----------------------------------------------------------------------------- launches

int blocks_for(uint32_t chunks) { return static_cast<int>(std::min<int64_t>(chunks, std::min(kMostBlocks, device_sms() * 2))); }

// Tensors [from, to) that have elements, as a list; false: more chunks than 32 bits count.
template <int MOST>
bool fill_list(TensorList<MOST>* l, void* const* data, const int64_t* numels, const int* types, int64_t from, int64_t to) {
  l->count = 0;
  int64_t chunks = 0;
  for (int64_t i = from; i < to; ++i) {
    if (numels[i] == 0) continue;
    const int64_t bytes = numels[i] * (types[i] == TRITURUS_B200_TYPE_F32 ? 4 : 2);
    l->data[l->count] = data[i];
    l->bytes[l->count] = bytes;
    l->first[l->count] = static_cast<uint32_t>(chunks);
    l->type[l->count] = static_cast<uint8_t>(types[i]);
    ++l->count;
    chunks += ((static_cast<int64_t>(reinterpret_cast<uintptr_t>(data[i]) & 15)) + bytes + kChunk - 1) / kChunk;
  }
  l->chunks = static_cast<uint32_t>(chunks);
  return chunks <= INT64_C(0x7fffffff);
}

template <int C>
int run_small(const TensorList<64>& l, const ClipArgs& p, int scale, cudaStream_t stream) {
  const cudaLaunchAttribute cluster = cluster_of(C);
  return launch_of(clip_small_kernel<C>, dim3(C), kThreads, 0, stream, C > 1 ? &cluster : nullptr, l, p, scale);
}

template <int MOST>
int run_clip(void* const* data, const int64_t* numels, const int* types, int64_t count, ClipArgs p, int scale, cudaStream_t stream) {
  const int64_t lists = std::max<int64_t>(1, (count + MOST - 1) / MOST);
  const cudaLaunchAttribute dependent = dependent_launch();
  TensorList<MOST> l;
  p.sums_in_all = 0;
  for (int64_t i = 0; i < lists; ++i) {
    if (!fill_list(&l, data, numels, types, i * MOST, std::min(count, (i + 1) * MOST))) return TRITURUS_B200_EINVAL;
    if constexpr (MOST == 64) {
      if (l.chunks <= kHeld) return run_small<1>(l, p, scale, stream);
      if (l.chunks <= 8 * kHeld) return run_small<8>(l, p, scale, stream);
    }
    p.sums_here = p.sums_in_all;
    const int blocks = blocks_for(l.chunks);
    p.sums_in_all += blocks;
    if (blocks == 0) continue;
    const int rc = launch_of(norm_parts_kernel<MOST>, dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream, nullptr, l, p);
    if (rc != TRITURUS_B200_OK) return rc;
  }
  for (int64_t i = 0; i < (scale ? lists : 1); ++i) {
    if (lists > 1 && !fill_list(&l, data, numels, types, i * MOST, std::min(count, (i + 1) * MOST))) return TRITURUS_B200_EINVAL;
    p.sums_here = i == 0 ? 0 : 1;
    const int blocks = scale ? std::max(1, blocks_for(l.chunks)) : 1;
    const int work = scale && l.chunks > 0;
    if (i > 0 && !work) continue;
    const int rc = launch_of(clip_kernel<MOST>, dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream, &dependent, l, p, work);
    if (rc != TRITURUS_B200_OK) return rc;
  }
  return TRITURUS_B200_OK;
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" {

size_t triturus_b200_clip_grad_norm_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  return static_cast<size_t>(std::max<int64_t>(1, (count + kMostTensors - 1) / kMostTensors)) * kMostBlocks * sizeof(double);
}

int triturus_b200_clip_grad_norm(void* const* tensors, const int64_t* numels, const int* types, int64_t count, double max_norm, int largest,
                                 int scale, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (count < 0 || norm == nullptr || workspace == nullptr || (count > 0 && (tensors == nullptr || numels == nullptr || types == nullptr)))
    return TRITURUS_B200_EINVAL;
  if (!(max_norm >= 0.0)) return TRITURUS_B200_EINVAL;
  for (int64_t i = 0; i < count; ++i) {
    if (numels[i] < 0 || types[i] < TRITURUS_B200_TYPE_F32 || types[i] > TRITURUS_B200_TYPE_F16) return TRITURUS_B200_EINVAL;
    if (numels[i] > 0 && tensors[i] == nullptr) return TRITURUS_B200_EINVAL;
    if (numels[i] > 0 && !aligned_to(tensors[i], types[i] == TRITURUS_B200_TYPE_F32 ? 4 : 2)) return TRITURUS_B200_EALIGN;
  }
  if (!aligned_to(norm, 4) || !aligned_to(workspace, 8)) return TRITURUS_B200_EALIGN;
  if (workspace_bytes < triturus_b200_clip_grad_norm_workspace_bytes(count)) return TRITURUS_B200_EWORKSPACE;
  ClipArgs p = {};
  p.sums = static_cast<double*>(workspace);
  p.limit = max_norm;
  p.norm = norm;
  p.largest = largest;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return count <= 64 ? run_clip<64>(tensors, numels, types, count, p, scale, st)
                     : run_clip<kMostTensors>(tensors, numels, types, count, p, scale, st);
}

}  // extern "C"
