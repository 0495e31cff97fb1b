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
// Measured on one B200 (copy bandwidth 6.54 TB/s): forward 16384 x 2048 bfloat16 26.7 us = 5.0 TB/s, 16384 x 8192 111-117 us = 4.6-4.8; backward 16384 x 8192
// 159 us = 5.1 TB/s with the shares of dw and db; 4000 x 16384 float32 99 and 138 us = 5.3 and 5.7.  What is missing is the time of a row's steps in turn (issue
// 0.5-0.6 of a scheduler's cycles): more rows under way than four change nothing.  Rows off 16-byte boundaries come element by element and are
// bound by instructions: 5003 x 1537 float32 16.5 and 29 us = 3.7 and 3.2 TB/s, 20000 x 1001 bfloat16 45 and 72 us = 1.8 and 1.7 (20000 x 1000: 21 and 34).
// Rows beyond 16384 elements are read three times, an element at a time: 4000 x 32768 bfloat16 424 and 558 us, float32 288 and 695.
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

// A vector of a row on its way through shared memory.  Rows of 16-bit elements on addresses that 4 does not divide have no copy of their own: an element
// comes as the 4-byte word that it is a half of.
template <class T, int BYTES>
struct alignas(BYTES < 4 ? 4 : BYTES) Slot {
  Pack<T, (BYTES < 4 ? 4 : BYTES)> p;
  // `half`: the address's second bit
  __device__ __forceinline__ float get(int e, int half) const { return to_float(BYTES < 4 ? (half ? p.v[1] : p.v[0]) : p.v[e]); }
};
// ... from global to shared memory without a register.
// (`read`: the bytes that are read of 4, the others are zero.)
template <int BYTES>
__device__ __forceinline__ void fetch(uint32_t dst, const void* src, uint32_t read) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else if constexpr (BYTES == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(read) : "memory");
}
// For BYTES < 4, the same for all of a thread's elements of a row: where their words begin, and what is read of them.  Of a word whose first half is the
// element no more than that is read: the tensor may end there.  One whose second half it is begins inside the allocation, which begins on a larger
// boundary.
template <int BYTES, class T>
__device__ __forceinline__ uint32_t to_words(const T*& row) {
  if constexpr (BYTES >= 4) return 4;
  const uintptr_t at = reinterpret_cast<uintptr_t>(row);
  row = reinterpret_cast<const T*>(at & ~static_cast<uintptr_t>(3));
  return 2u + static_cast<uint32_t>(at & 2);
}
__device__ __forceinline__ int half_of(const void* p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 1; }
__device__ __forceinline__ void wait_for_row(int stages) {
  if (stages == 4)
    cp_async_wait<3>();
  else if (stages == 2)
    cp_async_wait<1>();
  else
    cp_async_wait<0>();
}

// Two 32-bit numbers that are worked on at once: what these kernels would otherwise be bound by is the number of their instructions.
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 parts_of(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float both(Pair p) {
  const float2 f = parts_of(p);
  return f.x + f.y;
}
// Of 16-bit elements, as they lie in a word.
template <class T>
__device__ __forceinline__ Pair unpack(uint32_t w);
template <>
__device__ __forceinline__ Pair unpack<__nv_bfloat16>(uint32_t w) {  // (a bfloat16 is the upper half of a 32-bit number)
  return pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ Pair unpack<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pair_of(f.x, f.y);
}
template <class T>
__device__ __forceinline__ uint32_t pack(Pair p);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(Pair p) {
  const float2 f = parts_of(p);
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(Pair p) {
  const float2 f = parts_of(p);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// How the elements of a row are dealt out: vectors of N elements, vector v to thread v % TH of the row's group of TH threads, NV to a thread.  What
// lies behind the row's end is never fetched and stays zero.
template <class T, int BYTES, int NV, int TH>
struct Deal {
  using P = Pack<T, BYTES>;
  static constexpr int N = P::N;
  // A thread's elements are worked on in chunks of pairs: a vector, or two of one element.
  static constexpr int kVectors = N == 1 ? 2 : 1, kPairs = N == 1 ? 1 : N / 2, kChunks = NV / kVectors;
  int vectors;       // of the row
  int left;          // from the thread's first one on
  int first_column;
  __device__ __forceinline__ Deal(int t, int width) : vectors(width / N), left(width / N - t), first_column(t * N) {}
  __device__ __forceinline__ bool has(int i) const { return left > i * TH; }
  __device__ __forceinline__ int column(int i) const { return first_column + i * TH * N; }
  __device__ __forceinline__ bool beyond(int c) const { return vectors <= c * kVectors * TH; }            // for all threads
  __device__ __forceinline__ bool whole(int c) const { return vectors >= (c + 1) * kVectors * TH; }       // for all threads

  // Chunk c of a row in shared memory, `pitch` slots from vector to vector.
  __device__ __forceinline__ void read(const Slot<T, BYTES>* ring, int pitch, int c, int half, Pair (&out)[kPairs]) const {
    if constexpr (N == 1) {
      out[0] = pair_of(ring[2 * c * pitch].get(0, half), ring[(2 * c + 1) * pitch].get(0, half));
    } else if constexpr (sizeof(T) == 2) {
      using U = Pack<uint32_t, BYTES>;
      const U u = *reinterpret_cast<const U*>(ring + c * pitch);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) out[k] = unpack<T>(u.v[k]);
    } else {
      const Slot<T, BYTES> x = ring[c * pitch];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) out[k] = pair_of(x.get(2 * k, 0), x.get(2 * k + 1, 0));
    }
  }
  // ... into a row of global memory; `row` is where the thread's first vector goes.
  __device__ __forceinline__ void write(T* row, int c, const Pair (&v)[kPairs]) const {
    if constexpr (N == 1) {
      const float2 f = parts_of(v[0]);
      if (has(2 * c)) row[2 * c * TH] = from_float<T>(f.x);
      if (has(2 * c + 1)) row[(2 * c + 1) * TH] = from_float<T>(f.y);
    } else if (has(c)) {
      if constexpr (sizeof(T) == 2) {
        Pack<uint32_t, BYTES> u;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) u.v[k] = pack<T>(v[k]);
        *reinterpret_cast<Pack<uint32_t, BYTES>*>(row + c * TH * N) = u;
      } else {
        P o;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          const float2 f = parts_of(v[k]);
          o.v[2 * k] = f.x;
          o.v[2 * k + 1] = f.y;
        }
        *reinterpret_cast<P*>(row + c * TH * N) = o;
      }
    }
  }
  // The column of the first or second number of pair k of chunk c.
  __device__ __forceinline__ int column(int c, int k, int second) const {
    return N == 1 ? column(2 * c + second) : column(c) + 2 * k + second;
  }
  __device__ __forceinline__ bool has(int c, int second) const { return N == 1 ? has(2 * c + second) : has(c); }
};

// The thread's weights, zeros behind the row's end; 16 bytes at a time where the vectors are that and begin on such a boundary.
template <class W, int N>
__device__ __forceinline__ void load_vector(const W* w, bool aligned, float (&out)[N]) {
  constexpr int BYTES = N * static_cast<int>(sizeof(W));
  if (BYTES % 16 == 0 && aligned) {
#pragma unroll
    for (int part = 0; part < BYTES / 16; ++part) {
      using P = Pack<W, 16>;
      const P v = reinterpret_cast<const P*>(w)[part];
#pragma unroll
      for (int e = 0; e < P::N; ++e) out[part * P::N + e] = to_float(v.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = to_float(w[e]);
  }
}
template <class T, class D, int NV>
__device__ __forceinline__ void load_weights(const D& d, const void* w, int weight32, float fill, Pair (&out)[NV * D::N / 2]) {
  const bool aligned = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  float f[NV][D::N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < D::N; ++e) f[i][e] = d.has(i) ? fill : 0.f;
    if (w != nullptr && d.has(i)) {
      if (weight32)
        load_vector(static_cast<const float*>(w) + d.column(i), aligned, f[i]);
      else
        load_vector(static_cast<const T*>(w) + d.column(i), aligned, f[i]);
    }
  }
#pragma unroll
  for (int k = 0; k < NV * D::N / 2; ++k) out[k] = pair_of(f[2 * k / D::N][2 * k % D::N], f[(2 * k + 1) / D::N][(2 * k + 1) % D::N]);
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
__global__ void __launch_bounds__(BLOCK, NV * Pack<T, BYTES>::N > 16 ? 1 : BLOCK == 512 ? 2 : 768 / BLOCK) norm_forward_kernel(const NormArgs p) {
  using D = Deal<T, BYTES, NV, TH>;
  constexpr int kGroups = BLOCK / TH;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part[2][BLOCK / 32];
  const int group = threadIdx.x / TH, t = threadIdx.x % TH;
  const D d(t, p.width);
  using S = Slot<T, BYTES>;
  S* const ring = reinterpret_cast<S*>(smem) + threadIdx.x;
  const uint32_t ring_at = smem_u32(ring);
  const float inv = 1.f / static_cast<float>(p.width);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group, step = static_cast<int64_t>(gridDim.x) * kGroups;
  auto ask = [&](int64_t row, int stage) {
    if (row < p.rows) {
      const T* x = static_cast<const T*>(p.x) + row * p.x_stride + d.first_column;
      const uint32_t x_read = to_words<BYTES>(x);
      const uint32_t at = ring_at + stage * (NV * BLOCK * static_cast<int>(sizeof(S)));
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (d.has(i)) fetch<BYTES>(at + i * BLOCK * static_cast<int>(sizeof(S)), x + i * TH * D::N, x_read);
    }
    cp_async_commit();
  };
  for (int s = 0; s < p.stages; ++s) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (!d.has(i)) ring[(s * NV + i) * BLOCK] = S{};
    ask(first + s * step, s);
  }
  Pair weight[D::kChunks * D::kPairs], bias[D::kChunks * D::kPairs];
  load_weights<T, D, NV>(d, p.weight, p.weight32, 1.f, weight);
  load_weights<T, D, NV>(d, p.bias, p.weight32, 0.f, bias);
  int stage = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    wait_for_row(p.stages);
    const int half = BYTES < 4 ? half_of(static_cast<const T*>(p.x) + row * p.x_stride + d.first_column) : 0;  // (the same for all i: TH is even)
    Pair v[D::kChunks][D::kPairs], sum = pair_of(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < D::kChunks; ++c) {
      if (d.beyond(c)) break;
      d.read(ring + stage * NV * BLOCK, BLOCK, c, half, v[c]);
#pragma unroll
      for (int k = 0; k < D::kPairs; ++k) sum = sum + v[c][k];
    }
    const float mean = group_sum<TH>(both(sum), part, group) * inv;
    ask(row + p.stages * step, stage);  // (the values are in registers: they are part of the sum)
    stage = stage + 1 == p.stages ? 0 : stage + 1;
    const Pair down = pair_of(-mean, -mean);
    Pair squares = pair_of(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < D::kChunks; ++c) {
      if (d.beyond(c)) break;
#pragma unroll
      for (int k = 0; k < D::kPairs; ++k) v[c][k] = v[c][k] + down;
      if (!d.whole(c)) {
#pragma unroll
        for (int k = 0; k < D::kPairs; ++k) {
          const float2 f = parts_of(v[c][k]);
          v[c][k] = pair_of(d.has(c, 0) ? f.x : 0.f, d.has(c, 1) ? f.y : 0.f);
        }
      }
#pragma unroll
      for (int k = 0; k < D::kPairs; ++k) squares = fma2(v[c][k], v[c][k], squares);
    }
    const float rstd = 1.f / sqrtf(fmaf(group_sum<TH>(both(squares), part + 1, group), inv, p.eps));
    if (t == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
    const Pair scale = pair_of(rstd, rstd);
    T* y = static_cast<T*>(p.y) + row * p.width + d.first_column;
#pragma unroll
    for (int c = 0; c < D::kChunks; ++c) {
      if (d.beyond(c)) break;
#pragma unroll
      for (int k = 0; k < D::kPairs; ++k) v[c][k] = fma2(v[c][k] * scale, weight[c * D::kPairs + k], bias[c * D::kPairs + k]);
      d.write(y, c, v[c]);
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
  constexpr int kGroups = kBack / TH;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part[2][2][kBack / 32];
  const int group = threadIdx.x / TH, t = threadIdx.x % TH;
  const D d(t, p.width);
  using S = Slot<T, BYTES>;
  S* const ring = reinterpret_cast<S*>(smem) + threadIdx.x;
  const uint32_t ring_at = smem_u32(ring);
  const float inv = 1.f / static_cast<float>(p.width);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group, step = static_cast<int64_t>(gridDim.x) * kGroups;
  auto ask = [&](int64_t row, int stage) {
    if (row < p.rows) {
      const T* x = static_cast<const T*>(p.x) + row * p.x_stride + d.first_column;
      const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride + d.first_column;
      const uint32_t x_read = to_words<BYTES>(x), dy_read = to_words<BYTES>(dy);
      const uint32_t at = ring_at + stage * (2 * NV * kBack * static_cast<int>(sizeof(S)));
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (d.has(i)) {
          fetch<BYTES>(at + i * kBack * static_cast<int>(sizeof(S)), x + i * TH * D::N, x_read);
          fetch<BYTES>(at + (NV + i) * kBack * static_cast<int>(sizeof(S)), dy + i * TH * D::N, dy_read);
        }
    }
    cp_async_commit();
  };
  for (int s = 0; s < p.stages; ++s) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (!d.has(i)) ring[(s * 2 * NV + i) * kBack] = ring[(s * 2 * NV + NV + i) * kBack] = S{};
    ask(first + s * step, s);
  }
  Pair weight[D::kChunks * D::kPairs];
  load_weights<T, D, NV>(d, p.weight, p.weight32, 1.f, weight);
  float mean = 0.f, rstd = 0.f;
  if (first < p.rows) {
    mean = p.mean[first];
    rstd = p.rstd[first];
  }
  Pair dw[D::kChunks][D::kPairs], db[D::kChunks][D::kPairs];
#pragma unroll
  for (int c = 0; c < D::kChunks; ++c)
#pragma unroll
    for (int k = 0; k < D::kPairs; ++k) dw[c][k] = db[c][k] = pair_of(0.f, 0.f);
  int stage = 0, odd = 0;
  for (int64_t row = first; row < p.rows; row += step, odd ^= 1) {
    float next_mean = 0.f, next_rstd = 0.f;
    if (row + step < p.rows) {
      next_mean = p.mean[row + step];
      next_rstd = p.rstd[row + step];
    }
    const int half_x = BYTES < 4 ? half_of(static_cast<const T*>(p.x) + row * p.x_stride + d.first_column) : 0;
    const int half_dy = BYTES < 4 ? half_of(static_cast<const T*>(p.dy) + row * p.dy_stride + d.first_column) : 0;
    wait_for_row(p.stages);
    const Pair down = pair_of(-mean, -mean), scale = pair_of(rstd, rstd);
    Pair sg = pair_of(0.f, 0.f), sgh = sg;
    const S* const x_row = ring + stage * 2 * NV * kBack;
    const S* const dy_row = x_row + NV * kBack;
#pragma unroll
    for (int c = 0; c < D::kChunks; ++c) {
      if (d.beyond(c)) break;
      Pair x[D::kPairs], dy[D::kPairs];
      d.read(x_row, kBack, c, half_x, x);
      d.read(dy_row, kBack, c, half_dy, dy);
#pragma unroll
      for (int k = 0; k < D::kPairs; ++k) {
        const Pair h = (x[k] + down) * scale, g = dy[k] * weight[c * D::kPairs + k];
        sg = sg + g;
        sgh = fma2(g, h, sgh);
        dw[c][k] = fma2(dy[k], h, dw[c][k]);
        db[c][k] = db[c][k] + dy[k];
      }
    }
    float sums_of[2] = {both(sg), both(sgh)};
    group_sums<TH>(sums_of, part[odd], group);
    const float mg = sums_of[0] * inv, mgh = sums_of[1] * inv;
    const Pair minus_mg = pair_of(-mg, -mg), minus_mgh = pair_of(-mgh, -mgh);
    T* dx = static_cast<T*>(p.y) + row * p.width + d.first_column;
#pragma unroll
    for (int c = 0; c < D::kChunks; ++c) {
      if (d.beyond(c)) break;
      Pair x[D::kPairs], dy[D::kPairs];
      d.read(x_row, kBack, c, half_x, x);
      d.read(dy_row, kBack, c, half_dy, dy);
#pragma unroll
      for (int k = 0; k < D::kPairs; ++k) {
        const Pair h = (x[k] + down) * scale;
        x[k] = scale * fma2(h, minus_mgh, fma2(dy[k], weight[c * D::kPairs + k], minus_mg));
      }
      d.write(dx, c, x);
    }
    ask(row + p.stages * step, stage);  // (what the stage held went into the stores)
    stage = stage + 1 == p.stages ? 0 : stage + 1;
    mean = next_mean;
    rstd = next_rstd;
  }
  pdl_launch_dependents();
  float* mine = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.width;
  auto each_sum = [&](const Pair (&sums)[D::kChunks][D::kPairs], float* to) {
#pragma unroll
    for (int c = 0; c < D::kChunks; ++c)
#pragma unroll
      for (int k = 0; k < D::kPairs; ++k) {
        const float2 f = parts_of(sums[c][k]);
        if (d.has(c, 0)) to[d.column(c, k, 0)] = f.x;
        if (d.has(c, 1)) to[d.column(c, k, 1)] = f.y;
      }
  };
  if constexpr (kGroups == 1) {
    each_sum(dw, mine);
    each_sum(db, mine + p.width);
  } else {  // the groups' shares, added in their order
    cp_async_wait<0>();
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      each_sum(which == 0 ? dw : db, sums + group * p.width);
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
  if (code_of(cudaGetDevice(&dev)) != TRITURUS_B200_OK || dev < 0 || dev >= 64) return 0;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (code_of(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared)) != TRITURUS_B200_OK) return 0;
    if (code_of(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem)) != TRITURUS_B200_OK || n <= 0) return 0;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Rows under way, of what shared memory holds; no more than a group has in all.
constexpr int stages_for(size_t row_bytes) {
  return 4 * row_bytes <= kMostShared ? 4 : 2 * row_bytes <= kMostShared ? 2 : 1;
}
int stages_of(int most, int64_t rows, int64_t groups) { return rows <= groups ? 1 : rows <= 2 * groups ? std::min(most, 2) : most; }

template <class T, int BYTES, int NV, int TH>
int run_forward(NormArgs p, cudaStream_t stream) {
  constexpr int BLOCK = TH < 128 ? 128 : TH, kGroups = BLOCK / TH;
  constexpr size_t row_bytes = static_cast<size_t>(BLOCK) * NV * sizeof(Slot<T, BYTES>);
  constexpr int stages = stages_for(row_bytes);
  static std::atomic<int> known[64];
  const auto kern = norm_forward_kernel<T, BYTES, NV, TH, BLOCK>;
  const int fit = blocks_of_sm(kern, known, BLOCK, stages * row_bytes);
  if (fit == 0) return TRITURUS_B200_ELAUNCH;
  const int64_t blocks = std::min<int64_t>((p.rows + kGroups - 1) / kGroups, static_cast<int64_t>(device_sms()) * fit);
  p.stages = stages_of(stages, p.rows, blocks * kGroups);
  return launch_of(kern, dim3(static_cast<unsigned>(blocks)), BLOCK, p.stages * row_bytes, stream, nullptr, p);
}

// Blocks of the backward pass: each has a share of dw and db to write and to be added.
int most_shares(int64_t rows) { return static_cast<int>(std::min<int64_t>(rows, device_sms())); }

template <class T, int BYTES, int NV, int TH>
int run_backward(NormArgs p, int* blocks, cudaStream_t stream) {
  constexpr int kGroups = kBack / TH;
  constexpr size_t row_bytes = static_cast<size_t>(kBack) * NV * sizeof(Slot<T, BYTES>) * 2;
  constexpr int stages = stages_for(row_bytes);
  constexpr size_t sums = kGroups > 1 ? static_cast<size_t>(kBack) * NV * BYTES / sizeof(T) * sizeof(float) : 0;
  static std::atomic<int> known[64];
  const auto kern = norm_backward_kernel<T, BYTES, NV, TH>;
  if (blocks_of_sm(kern, known, kBack, std::max(stages * row_bytes, sums)) == 0) return TRITURUS_B200_ELAUNCH;
  *blocks = static_cast<int>(std::min<int64_t>((p.rows + kGroups - 1) / kGroups, device_sms()));
  p.stages = stages_of(stages, p.rows, static_cast<int64_t>(*blocks) * kGroups);
  return launch_of(kern, dim3(static_cast<unsigned>(*blocks)), kBack, std::max(p.stages * row_bytes, sums), stream, nullptr, p);
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
    return launch_of(norm_forward_long_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(p.rows, device_sms() * 2))), 1024, 0, stream, nullptr, p);
  }
  const int bytes = std::min(vector_bytes(p.x, p.x_stride, p.rows, p.width, SIZE), vector_bytes(p.y, p.width, p.rows, p.width, SIZE));
  return by_bytes<T>(bytes, [&](auto b) {
    return by_width<T, b()>(p.width, [&](auto nv, auto th) { return run_forward<T, b(), nv(), th()>(p, stream); });
  });
}

template <class W>
int run_reduce(const NormArgs& p, void* dweight, void* dbias, int blocks, cudaStream_t stream) {
  const cudaLaunchAttribute dependent = dependent_launch();
  return launch_of(norm_reduce_kernel<W>, dim3(static_cast<unsigned>((p.width + 31) / 32), 2), 512, 0, stream, &dependent, p.part, static_cast<W*>(dweight),
                   static_cast<W*>(dbias), blocks, p.width);
}

template <class T>
int backward(const NormArgs& p, void* dweight, void* dbias, cudaStream_t stream) {
  constexpr int SIZE = static_cast<int>(sizeof(T));
  int blocks = 0, rc;
  if (p.width > kLongest) {
    blocks = most_shares(std::min<int64_t>(p.rows, 64));
    rc = launch_of(norm_backward_long_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(p.rows, device_sms() * 2))), 1024, 0, stream, nullptr, p);
    if (rc == TRITURUS_B200_OK)
      rc = launch_of(norm_backward_columns_kernel<T>, dim3(static_cast<unsigned>((p.width + 255) / 256), static_cast<unsigned>(blocks)), 256, 0, stream,
                     nullptr, p);
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
      if (d != nullptr) {
        const int rc = code_of(cudaMemsetAsync(d, 0, static_cast<size_t>(width) * size_of(weight_type), st));
        if (rc != TRITURUS_B200_OK) return rc;
      }
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
