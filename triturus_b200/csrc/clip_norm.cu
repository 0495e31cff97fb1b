// The norm of many tensors taken as one vector, and their scaling to a limit.
//
//   n = sqrt(sum x^2) or max |x| over all elements of all tensors;  c = min(1, limit / (n + 1e-6));  x <- c x
//
// The tensors are cut into chunks of kChunk bytes that begin on 16-byte boundaries of memory (the first of a tensor may begin with
// a partial vector), and the blocks take the chunks in turn.  First launch: each block's sum of squares, in 64 bits.  Second launch: every
// block adds those sums in the same order, so that all have the same n, and scales its chunks; it goes through them backwards, because
// what the first launch read last is still in the L2 cache.  Where c is 1 nothing is written.
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
  uint8_t* base;     // on a 16-byte boundary: the chunk's first byte, if the tensor began there
  int begin, end;    // the tensor's bytes of the chunk
  int type;
};

template <int MOST>
__device__ __forceinline__ Chunk find_chunk(const TensorList<MOST>& l, uint32_t c) {
  int lo = 0, hi = l.count;  // the last tensor whose first chunk is not behind c
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= c)
      lo = mid;
    else
      hi = mid;
  }
  const uintptr_t at = reinterpret_cast<uintptr_t>(l.data[lo]);
  const int skip = static_cast<int>(at & 15);
  const int64_t off = static_cast<int64_t>(c - l.first[lo]) * kChunk;
  const int64_t left = skip + l.bytes[lo] - off;
  Chunk k;
  k.base = reinterpret_cast<uint8_t*>(at - skip) + off;
  k.begin = off == 0 ? skip : 0;
  k.end = static_cast<int>(left < kChunk ? left : kChunk);
  k.type = l.type[lo];
  return k;
}

// The vectors of a chunk that are the thread's; elements outside of the tensor are zeros.
template <class T>
__device__ __forceinline__ void load_chunk(const Chunk& k, Pack<T, 16> (&v)[kVectors]) {
  constexpr int N = Pack<T, 16>::N;
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int o = (i * kThreads + static_cast<int>(threadIdx.x)) * 16;
    if (o >= k.begin && o + 16 <= k.end) {
      v[i] = *reinterpret_cast<const Pack<T, 16>*>(k.base + o);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int at = o + e * static_cast<int>(sizeof(T));
        v[i].v[e] = from_float<T>(0.f);
        if (at >= k.begin && at < k.end) v[i].v[e] = *reinterpret_cast<const T*>(k.base + at);
      }
    }
  }
}

template <class T>
__device__ __forceinline__ void scale_chunk(const Chunk& k, float c) {
  constexpr int N = Pack<T, 16>::N;
  Pack<T, 16> v[kVectors];
  load_chunk<T>(k, v);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int o = (i * kThreads + static_cast<int>(threadIdx.x)) * 16;
#pragma unroll
    for (int e = 0; e < N; ++e) v[i].v[e] = from_float<T>(to_float(v[i].v[e]) * c);
    if (o >= k.begin && o + 16 <= k.end) {
      *reinterpret_cast<Pack<T, 16>*>(k.base + o) = v[i];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int at = o + e * static_cast<int>(sizeof(T));
        if (at >= k.begin && at < k.end) *reinterpret_cast<T*>(k.base + at) = v[i].v[e];
      }
    }
  }
}

// Adds the squares of a chunk's elements.  A vector's squares are added in 32 bits where they neither overflow nor lose digits
// below the least normal number, else in 64 bits: a norm that 32 bits can hold is not lost to its square.
template <class T>
__device__ __forceinline__ void add_squares(const Chunk& k, double& sum) {
  constexpr int N = Pack<T, 16>::N;
  Pack<T, 16> v[kVectors];
  load_chunk<T>(k, v);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = to_float(v[i].v[e]);
      s = fmaf(x, x, s);
    }
    if (s > 1e-25f && s < 1e38f) {
      sum += static_cast<double>(s);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double x = static_cast<double>(to_float(v[i].v[e]));
        sum = fma(x, x, sum);
      }
    }
  }
}

// The largest magnitude, as bits: those of a NaN are above those of infinity.
template <class T>
__device__ __forceinline__ void raise_largest(const Chunk& k, uint32_t& most) {
  constexpr int N = Pack<T, 16>::N;
  Pack<T, 16> v[kVectors];
  load_chunk<T>(k, v);
#pragma unroll
  for (int i = 0; i < kVectors; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) most = max(most, __float_as_uint(to_float(v[i].v[e])) & 0x7fffffffu);
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

template <int MOST>
__global__ void __launch_bounds__(kThreads) norm_parts_kernel(const __grid_constant__ TensorList<MOST> l, const ClipArgs p) {
  __shared__ double part[kThreads / 32];
  double sum = 0.0;
  uint32_t most = 0;
  for (uint32_t c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const Chunk k = find_chunk(l, c);
    if (!p.largest) {
      if (k.type == TRITURUS_B200_TYPE_F32)
        add_squares<float>(k, sum);
      else if (k.type == TRITURUS_B200_TYPE_BF16)
        add_squares<__nv_bfloat16>(k, sum);
      else
        add_squares<__half>(k, sum);
    } else {
      if (k.type == TRITURUS_B200_TYPE_F32)
        raise_largest<float>(k, most);
      else if (k.type == TRITURUS_B200_TYPE_BF16)
        raise_largest<__nv_bfloat16>(k, most);
      else
        raise_largest<__half>(k, most);
    }
  }
  pdl_launch_dependents();
  if (p.largest) sum = static_cast<double>(__uint_as_float(most));
  sum = block_combine(sum, part, p.largest);
  if (threadIdx.x == 0) p.sums[p.sums_here + blockIdx.x] = sum;
}

// `scale` == 0: the norm alone (one block).
template <int MOST>
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ TensorList<MOST> l, const ClipArgs p, int scale) {
  __shared__ double part[kThreads / 32];
  __shared__ float factor;
  pdl_wait();
  double v = 0.0;
  for (int i = threadIdx.x; i < p.sums_in_all; i += kThreads) v = combine(v, p.sums[i], p.largest);
  v = block_combine(v, part, p.largest);
  if (threadIdx.x == 0) {
    const double n = p.largest ? v : sqrt(v);
    // (a norm beyond 32 bits still has its factor; a NaN among the elements makes all of them NaN)
    factor = n + 1e-6 <= p.limit ? 1.f : static_cast<float>(p.limit / (n + 1e-6));
    if (blockIdx.x == 0 && p.sums_here == 0) *p.norm = static_cast<float>(n);
  }
  __syncthreads();
  const float c = factor;
  if (!scale || c == 1.f) return;
  const uint32_t last = (l.chunks - 1 - blockIdx.x) / gridDim.x;  // (no more blocks than chunks)
  for (uint32_t i = 0; i <= last; ++i) {
    const Chunk k = find_chunk(l, blockIdx.x + (last - i) * gridDim.x);
    if (k.type == TRITURUS_B200_TYPE_F32)
      scale_chunk<float>(k, c);
    else if (k.type == TRITURUS_B200_TYPE_BF16)
      scale_chunk<__nv_bfloat16>(k, c);
    else
      scale_chunk<__half>(k, c);
  }
}

// ----------------------------------------------------------------------------- launches

int blocks_for(uint32_t chunks) { return static_cast<int>(std::min<int64_t>(chunks, std::min(kMostBlocks, device_sms() * 4))); }

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

template <int MOST, class Kern, class... More>
bool launch(Kern kern, int blocks, bool dependent, cudaStream_t stream, const TensorList<MOST>& l, const ClipArgs& p, More... more) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, l, p, more...) == cudaSuccess;
}

template <int MOST>
int run_clip(void* const* data, const int64_t* numels, const int* types, int64_t count, ClipArgs p, int scale, cudaStream_t stream) {
  const int64_t lists = std::max<int64_t>(1, (count + MOST - 1) / MOST);
  TensorList<MOST> l;
  p.sums_in_all = 0;
  for (int64_t i = 0; i < lists; ++i) {
    if (!fill_list(&l, data, numels, types, i * MOST, std::min(count, (i + 1) * MOST))) return TRITURUS_B200_EINVAL;
    p.sums_here = p.sums_in_all;
    const int blocks = blocks_for(l.chunks);
    p.sums_in_all += blocks;
    if (blocks > 0 && !launch<MOST>(norm_parts_kernel<MOST>, blocks, false, stream, l, p)) return TRITURUS_B200_ELAUNCH;
  }
  for (int64_t i = 0; i < (scale ? lists : 1); ++i) {
    if (lists > 1 && !fill_list(&l, data, numels, types, i * MOST, std::min(count, (i + 1) * MOST))) return TRITURUS_B200_EINVAL;
    p.sums_here = i == 0 ? 0 : 1;
    const int blocks = scale ? std::max(1, blocks_for(l.chunks)) : 1;
    const int work = scale && l.chunks > 0;
    if (i > 0 && !work) continue;
    if (!launch<MOST>(clip_kernel<MOST>, blocks, true, stream, l, p, work)) return TRITURUS_B200_ELAUNCH;
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
