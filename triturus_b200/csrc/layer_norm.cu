// Layer norm over the last dimension and its gradients.
//
//   mean = sum(x) / D,  rstd = 1 / sqrt(sum((x - mean)^2) / D + eps),  h = (x - mean) rstd,  y = h w + b
//   with g = dy w:  dx = rstd (g - sum(g) / D - h sum(g h) / D),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// Everything between the loads and the stores is in 32 bits.  The variance is the sum of squares about the mean and not the
// difference of two sums: a feature at a high level would cancel its digits.  Nothing here adds atomically: the results
// of a call are the same each time.
#include <algorithm>

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
  int weight32;        // weight, bias and their gradients are 32-bit (else of x's type)
  float eps;
};

// Weights or biases of the thread's elements [c0, c0 + N), as floats.
template <class T, int BYTES>
__device__ __forceinline__ void load_weights(const void* w, int weight32, int c0, float fill, float (&out)[Pack<T, BYTES>::N]) {
  constexpr int N = Pack<T, BYTES>::N;
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = fill;
  if (w == nullptr) return;
  if (weight32) {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = __ldg(static_cast<const float*>(w) + c0 + e);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = to_float(static_cast<const T*>(w)[c0 + e]);
  }
}

// A row is `nv` vectors of N elements (BYTES divides the rows' bytes, pitch and base), vector v belongs to thread v % threads.
// `threads` are those of a row: a warp (WARP, blockDim.y rows to a block) or the block.
template <class T, int BYTES, int NV, bool WARP>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const NormArgs p) {
  using P = Pack<T, BYTES>;
  constexpr int N = P::N;
  __shared__ float part[2][32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, threads = blockDim.x, warps = threads >> 5;
  const int nv = p.width / N;
  const float inv = 1.f / static_cast<float>(p.width);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? blockDim.y : 1);
  for (int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y : blockIdx.x; row < p.rows; row += step) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    P v[NV];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * threads;
      if (c < nv) v[i] = *reinterpret_cast<const P*>(x + c * N);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * threads < nv) {
#pragma unroll
        for (int e = 0; e < N; ++e) s += to_float(v[i].v[e]);
      }
    const float mean = (WARP ? warp_sum(s) : block_sum(s, part[0], warp, lane, warps)) * inv;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * threads < nv) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float d = to_float(v[i].v[e]) - mean;
          q += d * d;
        }
      }
    const float var = (WARP ? warp_sum(q) : block_sum(q, part[1], warp, lane, warps)) * inv;
    const float rstd = 1.f / sqrtf(var + p.eps);
    if (t == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(p.y) + row * p.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * threads;
      if (c < nv) {
        float w[N], b[N];
        load_weights<T, BYTES>(p.weight, p.weight32, c * N, 1.f, w);
        load_weights<T, BYTES>(p.bias, p.weight32, c * N, 0.f, b);
        P o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = from_float<T>((to_float(v[i].v[e]) - mean) * rstd * w[e] + b[e]);
        *reinterpret_cast<P*>(y + c * N) = o;
      }
    }
  }
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
      float w[1], b[1];
      load_weights<T, sizeof(T)>(p.weight, p.weight32, c, 1.f, w);
      load_weights<T, sizeof(T)>(p.bias, p.weight32, c, 0.f, b);
      y[c] = from_float<T>((to_float(x[c]) - mean) * rstd * w[0] + b[0]);
    }
  }
}

// dx of a block's rows, and the block's share of dw and db: a thread has the same columns in every row and keeps their sums.
template <class T, int BYTES, int NV>
__global__ void __launch_bounds__(1024) norm_backward_kernel(const NormArgs p) {
  using P = Pack<T, BYTES>;
  constexpr int N = P::N;
  __shared__ float part[2][2][32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, threads = blockDim.x, warps = threads >> 5;
  const int nv = p.width / N;
  const float inv = 1.f / static_cast<float>(p.width);
  float w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + i * threads;
    if (c < nv) load_weights<T, BYTES>(p.weight, p.weight32, c * N, 1.f, w[i]);
#pragma unroll
    for (int e = 0; e < N; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  int odd = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, odd ^= 1) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
    const float mean = p.mean[row], rstd = p.rstd[row];
    P v[NV], d[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * threads;
      if (c < nv) {
        v[i] = *reinterpret_cast<const P*>(x + c * N);
        d[i] = *reinterpret_cast<const P*>(dy + c * N);
      }
    }
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * threads < nv) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float dd = to_float(d[i].v[e]), h = (to_float(v[i].v[e]) - mean) * rstd, g = dd * w[i][e];
          sg += g;
          sgh += g * h;
          dw[i][e] += dd * h;
          db[i][e] += dd;
        }
      }
    sg = warp_sum(sg);
    sgh = warp_sum(sgh);
    if (lane == 0) {
      part[odd][0][warp] = sg;
      part[odd][1][warp] = sgh;
    }
    __syncthreads();
    const float mg = warp_sum(lane < warps ? part[odd][0][lane] : 0.f) * inv;
    const float mgh = warp_sum(lane < warps ? part[odd][1][lane] : 0.f) * inv;
    T* dx = static_cast<T*>(p.y) + row * p.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * threads;
      if (c < nv) {
        P o;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float h = (to_float(v[i].v[e]) - mean) * rstd;
          o.v[e] = from_float<T>(rstd * (to_float(d[i].v[e]) * w[i][e] - mg - h * mgh));
        }
        *reinterpret_cast<P*>(dx + c * N) = o;
      }
    }
  }
  float* mine = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.width;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t + i * threads;
    if (c < nv) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        mine[c * N + e] = dw[i][e];
        mine[p.width + c * N + e] = db[i][e];
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
      float w[1];
      load_weights<T, sizeof(T)>(p.weight, p.weight32, c, 1.f, w);
      const float g = to_float(dy[c]) * w[0];
      sg += g;
      sgh += g * ((to_float(x[c]) - mean) * rstd);
    }
    const float mg = block_sum(sg, part[0], warp, lane, 32) * inv;
    const float mgh = block_sum(sgh, part[1], warp, lane, 32) * inv;
    T* dx = static_cast<T*>(p.y) + row * p.width;
    for (int c = t; c < p.width; c += 1024) {
      float w[1];
      load_weights<T, sizeof(T)>(p.weight, p.weight32, c, 1.f, w);
      const float h = (to_float(x[c]) - mean) * rstd;
      dx[c] = from_float<T>(rstd * (to_float(dy[c]) * w[0] - mg - h * mgh));
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

// dw and db from the blocks' shares [blocks, 2, width]: 32 columns to a block, its warps add every 8th share.
template <class W>
__global__ void __launch_bounds__(256) norm_reduce_kernel(const float* __restrict__ part, W* __restrict__ dweight, W* __restrict__ dbias,
                                                          int blocks, int width) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  W* out = blockIdx.y == 0 ? dweight : dbias;
  if (out == nullptr) return;
  pdl_wait();
  float s = 0.f;
  if (c < width)
    for (int b = warp; b < blocks; b += 8) s += part[(static_cast<int64_t>(b) * 2 + blockIdx.y) * width + c];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][lane];
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

struct RowShape {
  int threads;  // of a row
  int nv;       // vectors to a thread; 0: the row does not fit
};
// The fewest threads that hold a row with at most `most` vectors each.
RowShape row_shape(int64_t vectors, int most, int least_threads) {
  for (int threads = least_threads; threads <= 1024; threads *= 2) {
    if (vectors <= static_cast<int64_t>(threads) * most) return {threads, static_cast<int>((vectors + threads - 1) / threads)};
  }
  return {0, 0};
}

template <class T, int BYTES, int NV>
void run_forward(const NormArgs& p, int threads, cudaStream_t stream) {
  const int sms = device_sms();
  if (threads == 32) {
    const int64_t blocks = std::min<int64_t>((p.rows + 7) / 8, static_cast<int64_t>(sms) * 8);
    norm_forward_kernel<T, BYTES, NV, true><<<static_cast<unsigned>(blocks), dim3(32, 8), 0, stream>>>(p);
  } else {
    const int64_t blocks = std::min<int64_t>(p.rows, static_cast<int64_t>(sms) * (2048 / threads));
    norm_forward_kernel<T, BYTES, NV, false><<<static_cast<unsigned>(blocks), threads, 0, stream>>>(p);
  }
}

template <class T, int BYTES>
bool forward_by_size(const NormArgs& p, cudaStream_t stream) {
  constexpr int N = Pack<T, BYTES>::N;
  constexpr int MOST = BYTES == 16 ? 4 : 16;
  const RowShape s = row_shape(p.width / N, MOST, 32);
  if (s.nv == 0) return false;
  if (s.nv <= MOST / 4)
    run_forward<T, BYTES, MOST / 4>(p, s.threads, stream);
  else if (s.nv <= MOST / 2)
    run_forward<T, BYTES, MOST / 2>(p, s.threads, stream);
  else
    run_forward<T, BYTES, MOST>(p, s.threads, stream);
  return true;
}

template <class T>
int forward(const NormArgs& p, cudaStream_t stream) {
  constexpr int SIZE = static_cast<int>(sizeof(T));
  const int bytes = std::min(vector_bytes(p.x, p.x_stride, p.rows, p.width, SIZE), vector_bytes(p.y, p.width, p.rows, p.width, SIZE));
  const bool done = bytes == 16  ? forward_by_size<T, 16>(p, stream)
                    : bytes == 4 ? forward_by_size<T, 4>(p, stream)
                                 : forward_by_size<T, SIZE>(p, stream);
  if (!done) norm_forward_long_kernel<T><<<static_cast<unsigned>(std::min<int64_t>(p.rows, device_sms() * 2)), 1024, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRITURUS_B200_OK : TRITURUS_B200_ELAUNCH;
}

struct BackwardPlan {
  int bytes, threads, nv;  // nv == 0: the kernels for long rows
  int blocks;              // shares of dw and db
};

BackwardPlan plan_backward(int64_t rows, int64_t width, int size, int bytes) {
  BackwardPlan b = {bytes, 0, 0, 0};
  const int n = bytes / size;
  const RowShape s = row_shape(width / n, 16 / n, 128);
  b.threads = s.threads;
  b.nv = s.nv;
  if (s.nv == 0)
    b.blocks = static_cast<int>(std::min<int64_t>(rows, 64));
  else
    b.blocks = static_cast<int>(std::min<int64_t>(rows, device_sms() * std::max(1, std::min(4, 1024 / s.threads))));
  return b;
}

template <class T, int BYTES>
void run_backward(const NormArgs& p, const BackwardPlan& b, cudaStream_t stream) {
  constexpr int N = Pack<T, BYTES>::N;
  constexpr int MOST = 16 / N;  // 16 elements to a thread at most
  if (b.nv <= MOST / 2)
    norm_backward_kernel<T, BYTES, MOST / 2><<<b.blocks, b.threads, 0, stream>>>(p);
  else
    norm_backward_kernel<T, BYTES, MOST><<<b.blocks, b.threads, 0, stream>>>(p);
}

template <class W>
int run_reduce(const float* part, void* dweight, void* dbias, int blocks, int width, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((width + 31) / 32), 2, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_reduce_kernel<W>, part, static_cast<W*>(dweight), static_cast<W*>(dbias), blocks, width) == cudaSuccess
             ? TRITURUS_B200_OK
             : TRITURUS_B200_ELAUNCH;
}

template <class T>
int backward(const NormArgs& p, const BackwardPlan& b, void* dweight, void* dbias, cudaStream_t stream) {
  if (b.nv == 0) {
    norm_backward_long_kernel<T><<<static_cast<unsigned>(std::min<int64_t>(p.rows, device_sms() * 2)), 1024, 0, stream>>>(p);
    norm_backward_columns_kernel<T><<<dim3(static_cast<unsigned>((p.width + 255) / 256), static_cast<unsigned>(b.blocks)), 256, 0, stream>>>(p);
  } else if (b.bytes == 16) {
    run_backward<T, 16>(p, b, stream);
  } else if (b.bytes == 4) {
    run_backward<T, 4>(p, b, stream);
  } else {
    run_backward<T, sizeof(T)>(p, b, stream);
  }
  if (cudaGetLastError() != cudaSuccess) return TRITURUS_B200_ELAUNCH;
  if (dweight == nullptr && dbias == nullptr) return TRITURUS_B200_OK;
  return p.weight32 ? run_reduce<float>(p.part, dweight, dbias, b.blocks, p.width, stream)
                    : run_reduce<T>(p.part, dweight, dbias, b.blocks, p.width, stream);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return type == TRITURUS_B200_TYPE_F32    ? forward<float>(p, st)
         : type == TRITURUS_B200_TYPE_BF16 ? forward<__nv_bfloat16>(p, st)
                                           : forward<__half>(p, st);
}

size_t triturus_b200_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width, int type) {
  if (!norm_sizes_ok(rows, width, type, type)) return 0;
  int blocks = 0;  // (the shares are fewer or more by the alignment of the operands: room for either)
  for (int bytes : {16, 4, size_of(type)})
    if (width * size_of(type) % bytes == 0) blocks = std::max(blocks, plan_backward(rows, width, size_of(type), bytes).blocks);
  return static_cast<size_t>(blocks) * 2 * static_cast<size_t>(width) * sizeof(float);
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
  const int bytes = std::min({vector_bytes(x, x_stride, rows, width, size), vector_bytes(dy, dy_stride, rows, width, size),
                              vector_bytes(dx, width, rows, width, size)});
  const BackwardPlan b = plan_backward(rows, width, size, bytes);
  return type == TRITURUS_B200_TYPE_F32    ? backward<float>(p, b, dweight, dbias, st)
         : type == TRITURUS_B200_TYPE_BF16 ? backward<__nv_bfloat16>(p, b, dweight, dbias, st)
                                           : backward<__half>(p, b, dweight, dbias, st);
}

}  // extern "C"
