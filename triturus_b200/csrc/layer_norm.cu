// Layer norm over the last dimension and its gradients.
//
//   mean = sum(x) / D,  rstd = 1 / sqrt(sum((x - mean)^2) / D + eps),  h = (x - mean) rstd,  y = h w + b
//   with g = dy w:  dx = rstd (g - sum(g) / D - h sum(g h) / D),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// Bound by memory: 2 row lengths are moved forwards and 3 backwards.  A block of threads goes from row to row; each thread has the same columns in
// every row, fetches them some rows ahead into shared memory that only it uses (cp.async: no registers and no barrier for what is
// under way), and backwards keeps its columns' shares of dw and db in registers until the end.  Rows of up to 512 elements belong to a
// warp.
//
// Everything between the loads and the stores is in 32 bits.  The variance is the sum of squares about the mean and not the
// difference of two sums: a feature at a high level would cancel its digits.  Nothing here adds atomically: the results
// of a call are the same each time.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/triturus_b200.h"
#include "packs.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

struct NormArgs {
  const void* x;
  const void* dy;
  const void* weight;  // nullptr: all ones
  const void* bias;    // nullptr: zeros
  void* y;             // forward: y, backward: dx; contiguous
  float* mean;
  float* rstd;
  float* part;         // backward: [blocks, 2, width], the sums of a block's rows: dw, then db
  int64_t rows;
  int64_t x_stride, dy_stride;
  int width;
  int stages;          // rows under way: 1, 2 or 4
  int weight32;        // weight, bias and their gradients are 32-bit (else of x's type)
  float eps;
};

// BYTES from global to shared memory without a register.  (16-bit rows on odd addresses: a plain load.)
template <int BYTES>
__device__ __forceinline__ void fetch(void* dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  else if constexpr (BYTES == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  else
    *static_cast<uint16_t*>(dst) = *static_cast<const uint16_t*>(src);
}
__device__ __forceinline__ void wait_for_row(int stages) {
  if (stages == 4)
    cp_async_wait<3>();
  else if (stages == 2)
    cp_async_wait<1>();
  else
    cp_async_wait<0>();
}

// How the elements of a row are dealt out: vectors of N elements, vector v to thread v % TH of the row's group of TH threads, NV to a thread.  What
// lies behind the row's end is never fetched and stays zero.
template <class T, int BYTES, int NV, int TH>
struct Deal {
  using P = Pack<T, BYTES>;
  static constexpr int N = P::N;
  int left;  // vectors of the row from the thread's first one on
  int first_column;
  __device__ __forceinline__ Deal(int t, int width) : left(width / N - t), first_column(t * N) {}
  __device__ __forceinline__ bool has(int i) const { return left > i * TH; }
  __device__ __forceinline__ int column(int i) const { return first_column + i * TH * N; }
};

// The thread's weights, zeros behind the row's end.
template <class T, class D, int NV>
__device__ __forceinline__ void load_weights(const D& d, const void* w, int weight32, float fill, float (&out)[NV][D::N]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < D::N; ++e) {
      out[i][e] = d.has(i) ? fill : 0.f;
      if (w != nullptr && d.has(i))
        out[i][e] = weight32 ? __ldg(static_cast<const float*>(w) + d.column(i) + e) : to_float(static_cast<const T*>(w)[d.column(i) + e]);
    }
}

// The sums over a group of TH threads of K values, in each of them.  A group of warps meets at a barrier of its own; two calls in a row use different
// `part`.
template <int TH, int K, int WARPS>
__device__ __forceinline__ void group_sums(float (&v)[K], float (*part)[WARPS], int group) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if constexpr (TH > 32) {
    constexpr int kWarps = TH / 32;
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) part[k][threadIdx.x >> 5] = v[k];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TH) : "memory");
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* mine = part[k] + group * kWarps;
      if constexpr (kWarps <= 4) {
        v[k] = mine[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) v[k] += mine[w];
      } else {
        v[k] = warp_sum(lane < kWarps ? mine[lane] : 0.f);
      }
    }
  }
}
template <int TH, int WARPS>
__device__ __forceinline__ float group_sum(float v, float (*part)[WARPS], int group) {
  float one[1] = {v};
  group_sums<TH>(one, part, group);
  return one[0];
}

template <class T, int BYTES, int NV, int TH, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK >= 512 ? 1 : 768 / BLOCK) norm_forward_kernel(const NormArgs p) {
  using D = Deal<T, BYTES, NV, TH>;
  using P = typename D::P;
  constexpr int kGroups = BLOCK / TH;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part[2][BLOCK / 32];
  const int group = threadIdx.x / TH, t = threadIdx.x % TH;
  const D d(t, p.width);
  P* const ring = reinterpret_cast<P*>(smem) + threadIdx.x;
  const float inv = 1.f / static_cast<float>(p.width);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group, step = static_cast<int64_t>(gridDim.x) * kGroups;
  auto ask = [&](int64_t row, int stage) {
    if (row < p.rows) {
      const T* x = static_cast<const T*>(p.x) + row * p.x_stride + d.first_column;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (d.has(i)) fetch<BYTES>(&ring[(stage * NV + i) * BLOCK], x + i * TH * D::N);
    }
    cp_async_commit();
  };
  for (int s = 0; s < p.stages; ++s) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (!d.has(i)) ring[(s * NV + i) * BLOCK] = P{};
    ask(first + s * step, s);
  }
  float weight[NV][D::N], bias[NV][D::N];
  load_weights<T>(d, p.weight, p.weight32, 1.f, weight);
  load_weights<T>(d, p.bias, p.weight32, 0.f, bias);
  int stage = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    wait_for_row(p.stages);
    float v[NV][D::N], s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const P x = ring[(stage * NV + i) * BLOCK];
#pragma unroll
      for (int e = 0; e < D::N; ++e) s += v[i][e] = to_float(x.v[e]);
    }
    const float mean = group_sum<TH>(s, part, group) * inv;
    ask(row + p.stages * step, stage);  // (the values are in registers: they are part of the sum)
    stage = stage + 1 == p.stages ? 0 : stage + 1;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < D::N; ++e) {
        v[i][e] = d.has(i) ? v[i][e] - mean : 0.f;
        q = fmaf(v[i][e], v[i][e], q);
      }
    const float rstd = 1.f / sqrtf(fmaf(group_sum<TH>(q, part + 1, group), inv, p.eps));
    if (t == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(p.y) + row * p.width + d.first_column;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (d.has(i)) {
        P o;
#pragma unroll
        for (int e = 0; e < D::N; ++e) o.v[e] = from_float<T>(fmaf(v[i][e] * rstd, weight[i][e], bias[i][e]));
        *reinterpret_cast<P*>(y + i * TH * D::N) = o;
      }
  }
}

template <class T>
__device__ __forceinline__ float weight_at(const void* w, int weight32, int c, float fill) {
  return w == nullptr ? fill : weight32 ? static_cast<const float*>(w)[c] : to_float(static_cast<const T*>(w)[c]);
}

// Rows that do not fit a block's registers: read three times, from the L2 cache after the first.
template <class T>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(const NormArgs p) {
  __shared__ float part[2][32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const float inv = 1.f / static_cast<float>(p.width);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    float s = 0.f;
    for (int c = t; c < p.width; c += 1024) s += to_float(x[c]);
    const float mean = block_sum(s, part[0], warp, lane, 32) * inv;
    float q = 0.f;
    for (int c = t; c < p.width; c += 1024) {
      const float d = to_float(x[c]) - mean;
      q += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(q, part[1], warp, lane, 32) * inv + p.eps);
    if (t == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(p.y) + row * p.width;
    for (int c = t; c < p.width; c += 1024) {
      const float w = weight_at<T>(p.weight, p.weight32, c, 1.f), b = weight_at<T>(p.bias, p.weight32, c, 0.f);
      y[c] = from_float<T>((to_float(x[c]) - mean) * rstd * w + b);
    }
  }
}

// dx of a block's rows, and the block's share of dw and db.  The block is kBack threads, as many groups as rows fit it.
constexpr int kBack = 512;
template <class T, int BYTES, int NV, int TH>
__global__ void __launch_bounds__(kBack) norm_backward_kernel(const NormArgs p) {
  using D = Deal<T, BYTES, NV, TH>;
  using P = typename D::P;
  constexpr int kGroups = kBack / TH;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part[2][2][kBack / 32];
  const int group = threadIdx.x / TH, t = threadIdx.x % TH;
  const D d(t, p.width);
  P* const ring = reinterpret_cast<P*>(smem) + threadIdx.x;
  const float inv = 1.f / static_cast<float>(p.width);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group, step = static_cast<int64_t>(gridDim.x) * kGroups;
  auto ask = [&](int64_t row, int stage) {
    if (row < p.rows) {
      const T* x = static_cast<const T*>(p.x) + row * p.x_stride + d.first_column;
      const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride + d.first_column;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (d.has(i)) {
          fetch<BYTES>(&ring[(stage * 2 * NV + i) * kBack], x + i * TH * D::N);
          fetch<BYTES>(&ring[(stage * 2 * NV + NV + i) * kBack], dy + i * TH * D::N);
        }
    }
    cp_async_commit();
  };
  for (int s = 0; s < p.stages; ++s) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (!d.has(i)) ring[(s * 2 * NV + i) * kBack] = ring[(s * 2 * NV + NV + i) * kBack] = P{};
    ask(first + s * step, s);
  }
  float weight[NV][D::N];
  load_weights<T>(d, p.weight, p.weight32, 1.f, weight);
  float mean = 0.f, rstd = 0.f;
  if (first < p.rows) {
    mean = p.mean[first];
    rstd = p.rstd[first];
  }
  float dw[NV][D::N], db[NV][D::N];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < D::N; ++e) dw[i][e] = db[i][e] = 0.f;
  int stage = 0, odd = 0;
  for (int64_t row = first; row < p.rows; row += step, odd ^= 1) {
    float next_mean = 0.f, next_rstd = 0.f;
    if (row + step < p.rows) {
      next_mean = p.mean[row + step];
      next_rstd = p.rstd[row + step];
    }
    wait_for_row(p.stages);
    float sums_of[2] = {0.f, 0.f};  // of g and g h
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const P x = ring[(stage * 2 * NV + i) * kBack], dy = ring[(stage * 2 * NV + NV + i) * kBack];
#pragma unroll
      for (int e = 0; e < D::N; ++e) {
        const float dd = to_float(dy.v[e]), h = (to_float(x.v[e]) - mean) * rstd, g = dd * weight[i][e];
        sums_of[0] += g;
        sums_of[1] = fmaf(g, h, sums_of[1]);
        dw[i][e] = fmaf(dd, h, dw[i][e]);
        db[i][e] += dd;
      }
    }
    group_sums<TH>(sums_of, part[odd], group);
    const float mg = sums_of[0] * inv, mgh = sums_of[1] * inv;
    T* dx = static_cast<T*>(p.y) + row * p.width + d.first_column;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const P x = ring[(stage * 2 * NV + i) * kBack], dy = ring[(stage * 2 * NV + NV + i) * kBack];
      P o;
#pragma unroll
      for (int e = 0; e < D::N; ++e) {
        const float h = (to_float(x.v[e]) - mean) * rstd;
        o.v[e] = from_float<T>(rstd * fmaf(-h, mgh, fmaf(to_float(dy.v[e]), weight[i][e], -mg)));
      }
      if (d.has(i)) *reinterpret_cast<P*>(dx + i * TH * D::N) = o;
    }
    ask(row + p.stages * step, stage);  // (what the stage held went into the stores)
    stage = stage + 1 == p.stages ? 0 : stage + 1;
    mean = next_mean;
    rstd = next_rstd;
  }
  float* mine = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.width;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (d.has(i)) {
#pragma unroll
        for (int e = 0; e < D::N; ++e) {
          mine[d.column(i) + e] = dw[i][e];
          mine[p.width + d.column(i) + e] = db[i][e];
        }
      }
  } else {  // the groups' shares, added in their order
    cp_async_wait<0>();
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (d.has(i)) {
#pragma unroll
          for (int e = 0; e < D::N; ++e) sums[group * p.width + d.column(i) + e] = which == 0 ? dw[i][e] : db[i][e];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < p.width; c += kBack) {
        float v = sums[c];
#pragma unroll
        for (int g = 1; g < kGroups; ++g) v += sums[g * p.width + c];
        mine[which * p.width + c] = v;
      }
    }
  }
}

// Rows that do not fit a block's registers, first half: dx, one block to a row.
template <class T>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(const NormArgs p) {
  __shared__ float part[2][32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const float inv = 1.f / static_cast<float>(p.width);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float sg = 0.f, sgh = 0.f;
    for (int c = t; c < p.width; c += 1024) {
      const float w = weight_at<T>(p.weight, p.weight32, c, 1.f);
      const float g = to_float(dy[c]) * w;
      sg += g;
      sgh += g * ((to_float(x[c]) - mean) * rstd);
    }
    const float mg = block_sum(sg, part[0], warp, lane, 32) * inv;
    const float mgh = block_sum(sgh, part[1], warp, lane, 32) * inv;
    T* dx = static_cast<T*>(p.y) + row * p.width;
    for (int c = t; c < p.width; c += 1024) {
      const float w = weight_at<T>(p.weight, p.weight32, c, 1.f);
      const float h = (to_float(x[c]) - mean) * rstd;
      dx[c] = from_float<T>(rstd * (to_float(dy[c]) * w - mg - h * mgh));
    }
  }
}

// ... and second half: dw and db, a block of 256 columns over the rows of one of gridDim.y groups.
template <class T>
__global__ void __launch_bounds__(256) norm_backward_columns_kernel(const NormArgs p) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= p.width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float d = to_float((static_cast<const T*>(p.dy) + row * p.dy_stride)[c]);
    dw += d * ((to_float((static_cast<const T*>(p.x) + row * p.x_stride)[c]) - p.mean[row]) * p.rstd[row]);
    db += d;
  }
  float* mine = p.part + static_cast<int64_t>(blockIdx.y) * 2 * p.width;
  mine[c] = dw;
  mine[p.width + c] = db;
}

// dw and db from the blocks' shares [blocks, 2, width]: 32 columns to a block, its warps add every 16th share.
template <class W>
__global__ void __launch_bounds__(512) norm_reduce_kernel(const float* __restrict__ part, W* __restrict__ dweight, W* __restrict__ dbias,
                                                          int blocks, int width) {
  __shared__ float sums[16][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  W* out = blockIdx.y == 0 ? dweight : dbias;
  if (out == nullptr) return;
  pdl_wait();
  float s = 0.f;
  if (c < width) {
#pragma unroll 4
    for (int b = warp; b < blocks; b += 16) s += part[(static_cast<int64_t>(b) * 2 + blockIdx.y) * width + c];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sums[i][lane];
    out[c] = from_float<W>(s);
  }
}

// ----------------------------------------------------------------------------- launches

int size_of(int type) { return type == TRITURUS_B200_TYPE_F32 ? 4 : 2; }
bool type_ok(int type) { return type >= TRITURUS_B200_TYPE_F32 && type <= TRITURUS_B200_TYPE_F16; }

// The widest access that a tensor's rows allow: 16 bytes, else 4, else 2 (16-bit types).
int vector_bytes(const void* base, int64_t stride, int64_t rows, int64_t width, int size) {
  for (int bytes : {16, 4}) {
    if (aligned_to(base, bytes) && width * size % bytes == 0 && (rows == 1 || stride * size % bytes == 0)) return bytes;
  }
  return size;
}

constexpr int kMostShared = 220 * 1024;
constexpr int kEach = 16;  // elements of a thread, twice that in the longest rows

// The blocks of a kernel that an SM holds, 0 where something failed.
template <class Kern>
int blocks_of_sm(Kern kern, std::atomic<int> (&known)[64], int threads, size_t smem) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) return 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem) != cudaSuccess || n <= 0) return 0;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Rows under way, of what shared memory holds.
constexpr int stages_for(size_t row_bytes, int bytes) {
  return bytes < 4 ? 1 : 4 * row_bytes <= kMostShared ? 4 : 2 * row_bytes <= kMostShared ? 2 : 1;
}

template <class T, int BYTES, int NV, int TH>
int run_forward(NormArgs p, cudaStream_t stream) {
  constexpr int BLOCK = TH < 128 ? 128 : TH, kGroups = BLOCK / TH;
  constexpr size_t row_bytes = static_cast<size_t>(BLOCK) * NV * BYTES;
  constexpr int stages = stages_for(row_bytes, BYTES);
  static std::atomic<int> known[64];
  const auto kern = norm_forward_kernel<T, BYTES, NV, TH, BLOCK>;
  const int fit = blocks_of_sm(kern, known, BLOCK, stages * row_bytes);
  if (fit == 0) return TRITURUS_B200_ELAUNCH;
  p.stages = stages;
  const int64_t blocks = std::min<int64_t>((p.rows + kGroups - 1) / kGroups, static_cast<int64_t>(device_sms()) * fit);
  kern<<<static_cast<unsigned>(blocks), BLOCK, stages * row_bytes, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRITURUS_B200_OK : TRITURUS_B200_ELAUNCH;
}

// Blocks of the backward pass: each has a share of dw and db to write and to be added.
int most_shares(int64_t rows) { return static_cast<int>(std::min<int64_t>(rows, device_sms())); }

template <class T, int BYTES, int NV, int TH>
int run_backward(NormArgs p, int* blocks, cudaStream_t stream) {
  constexpr int kGroups = kBack / TH;
  constexpr size_t row_bytes = static_cast<size_t>(kBack) * NV * BYTES * 2;
  constexpr int stages = stages_for(row_bytes, BYTES);
  constexpr size_t smem = std::max<size_t>(stages * row_bytes, kGroups > 1 ? static_cast<size_t>(kBack) * NV * BYTES / sizeof(T) * sizeof(float) : 0);
  static std::atomic<int> known[64];
  const auto kern = norm_backward_kernel<T, BYTES, NV, TH>;
  if (blocks_of_sm(kern, known, kBack, smem) == 0) return TRITURUS_B200_ELAUNCH;
  p.stages = stages;
  *blocks = static_cast<int>(std::min<int64_t>((p.rows + kGroups - 1) / kGroups, device_sms()));
  kern<<<static_cast<unsigned>(*blocks), kBack, smem, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRITURUS_B200_OK : TRITURUS_B200_ELAUNCH;
}

// run(NV, TH) as constants: the fewest threads that hold a row with kEach elements each.
template <class T, int BYTES, class F>
int by_width(int64_t width, F run) {
  constexpr int NV = kEach / Pack<T, BYTES>::N;
  using C = std::integral_constant<int, NV>;
  if (width <= 32 * kEach) return run(C(), std::integral_constant<int, 32>());
  if (width <= 64 * kEach) return run(C(), std::integral_constant<int, 64>());
  if (width <= 128 * kEach) return run(C(), std::integral_constant<int, 128>());
  if (width <= 256 * kEach) return run(C(), std::integral_constant<int, 256>());
  if (width <= 512 * kEach) return run(C(), std::integral_constant<int, 512>());
  return run(std::integral_constant<int, 2 * NV>(), std::integral_constant<int, 512>());
}
constexpr int64_t kLongest = 1024 * kEach;  // rows that by_width takes

// fn(bytes) as a constant.
template <class T, class F>
int by_bytes(int bytes, F fn) {
  if (bytes == 16) return fn(std::integral_constant<int, 16>());
  if (bytes == 4) return fn(std::integral_constant<int, 4>());
  return fn(std::integral_constant<int, static_cast<int>(sizeof(T))>());
}

template <class T>
int forward(const NormArgs& p, cudaStream_t stream) {
  constexpr int SIZE = static_cast<int>(sizeof(T));
  if (p.width > kLongest) {
    norm_forward_long_kernel<T><<<static_cast<unsigned>(std::min<int64_t>(p.rows, device_sms() * 2)), 1024, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? TRITURUS_B200_OK : TRITURUS_B200_ELAUNCH;
  }
  const int bytes = std::min(vector_bytes(p.x, p.x_stride, p.rows, p.width, SIZE), vector_bytes(p.y, p.width, p.rows, p.width, SIZE));
  return by_bytes<T>(bytes, [&](auto b) {
    return by_width<T, b()>(p.width, [&](auto nv, auto th) { return run_forward<T, b(), nv(), th()>(p, stream); });
  });
}

template <class W>
int run_reduce(const NormArgs& p, void* dweight, void* dbias, int blocks, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.width + 31) / 32), 2, 1);
  cfg.blockDim = dim3(512, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_reduce_kernel<W>, p.part, static_cast<W*>(dweight), static_cast<W*>(dbias), blocks, p.width) == cudaSuccess
             ? TRITURUS_B200_OK
             : TRITURUS_B200_ELAUNCH;
}

template <class T>
int backward(const NormArgs& p, void* dweight, void* dbias, cudaStream_t stream) {
  constexpr int SIZE = static_cast<int>(sizeof(T));
  int blocks = 0, rc;
  if (p.width > kLongest) {
    blocks = most_shares(std::min<int64_t>(p.rows, 64));
    norm_backward_long_kernel<T><<<static_cast<unsigned>(std::min<int64_t>(p.rows, device_sms() * 2)), 1024, 0, stream>>>(p);
    norm_backward_columns_kernel<T><<<dim3(static_cast<unsigned>((p.width + 255) / 256), static_cast<unsigned>(blocks)), 256, 0, stream>>>(p);
    rc = cudaGetLastError() == cudaSuccess ? TRITURUS_B200_OK : TRITURUS_B200_ELAUNCH;
  } else {
    const int bytes = std::min({vector_bytes(p.x, p.x_stride, p.rows, p.width, SIZE), vector_bytes(p.dy, p.dy_stride, p.rows, p.width, SIZE),
                                vector_bytes(p.y, p.width, p.rows, p.width, SIZE)});
    rc = by_bytes<T>(bytes, [&](auto b) {
      return by_width<T, b()>(p.width, [&](auto nv, auto th) { return run_backward<T, b(), nv(), th()>(p, &blocks, stream); });
    });
  }
  if (rc != TRITURUS_B200_OK || (dweight == nullptr && dbias == nullptr)) return rc;
  return p.weight32 ? run_reduce<float>(p, dweight, dbias, blocks, stream) : run_reduce<T>(p, dweight, dbias, blocks, stream);
}

// fn(T()) for the type of the elements.
template <class F>
int by_type(int type, F fn) {
  return type == TRITURUS_B200_TYPE_F32 ? fn(0.f) : type == TRITURUS_B200_TYPE_BF16 ? fn(__nv_bfloat16()) : fn(__half());
}

bool norm_sizes_ok(int64_t rows, int64_t width, int type, int weight_type) {
  return rows >= 0 && width > 0 && width <= (1 << 30) && type_ok(type) && (weight_type == type || weight_type == TRITURUS_B200_TYPE_F32);
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" {

int triturus_b200_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, int64_t rows,
                             int64_t width, int64_t x_stride, int type, int weight_type, float eps, void* stream) {
  if (!norm_sizes_ok(rows, width, type, weight_type)) return TRITURUS_B200_EINVAL;
  if (rows == 0) return TRITURUS_B200_OK;
  if (x == nullptr || y == nullptr) return TRITURUS_B200_EINVAL;
  const int size = size_of(type);
  if (!aligned_to(x, size) || !aligned_to(y, size) || !aligned_to(weight, size_of(weight_type)) || !aligned_to(bias, size_of(weight_type)) ||
      !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return TRITURUS_B200_EALIGN;
  NormArgs p = {};
  p.x = x;
  p.weight = weight;
  p.bias = bias;
  p.y = y;
  p.mean = mean;
  p.rstd = rstd;
  p.rows = rows;
  p.x_stride = x_stride;
  p.width = static_cast<int>(width);
  p.weight32 = weight_type == TRITURUS_B200_TYPE_F32;
  p.eps = eps;
  return by_type(type, [&](auto t) { return forward<decltype(t)>(p, static_cast<cudaStream_t>(stream)); });
}

size_t triturus_b200_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width, int type) {
  if (!norm_sizes_ok(rows, width, type, type)) return 0;
  return static_cast<size_t>(most_shares(rows)) * 2 * static_cast<size_t>(width) * sizeof(float);
}

int triturus_b200_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd, void* dx,
                                      void* dweight, void* dbias, int64_t rows, int64_t width, int64_t dy_stride, int64_t x_stride,
                                      int type, int weight_type, void* workspace, size_t workspace_bytes, void* stream) {
  if (!norm_sizes_ok(rows, width, type, weight_type)) return TRITURUS_B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int size = size_of(type);
  if (rows == 0) {  // sums over no rows
    for (void* d : {dweight, dbias})
      if (d != nullptr && cudaMemsetAsync(d, 0, static_cast<size_t>(width) * size_of(weight_type), st) != cudaSuccess) return TRITURUS_B200_ELAUNCH;
    return TRITURUS_B200_OK;
  }
  if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || dx == nullptr || workspace == nullptr) return TRITURUS_B200_EINVAL;
  if (!aligned_to(dy, size) || !aligned_to(x, size) || !aligned_to(dx, size) || !aligned_to(weight, size_of(weight_type)) ||
      !aligned_to(dweight, size_of(weight_type)) || !aligned_to(dbias, size_of(weight_type)) || !aligned_to(mean, 4) || !aligned_to(rstd, 4) ||
      !aligned_to(workspace, 16))
    return TRITURUS_B200_EALIGN;
  if (workspace_bytes < triturus_b200_layer_norm_backward_workspace_bytes(rows, width, type)) return TRITURUS_B200_EWORKSPACE;
  NormArgs p = {};
  p.x = x;
  p.dy = dy;
  p.weight = weight;
  p.y = dx;
  p.mean = const_cast<float*>(mean);
  p.rstd = const_cast<float*>(rstd);
  p.part = static_cast<float*>(workspace);
  p.rows = rows;
  p.x_stride = x_stride;
  p.dy_stride = dy_stride;
  p.width = static_cast<int>(width);
  p.weight32 = weight_type == TRITURUS_B200_TYPE_F32;
  return by_type(type, [&](auto t) { return backward<decltype(t)>(p, dweight, dbias, st); });
}

}  // extern "C"
