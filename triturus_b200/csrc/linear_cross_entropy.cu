// Cross entropy of a linear layer over many symbols, in pieces of the symbols and without keeping the logits.
//
//   z = x W^T,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_i,t_i
//   d_iv = g_i (exp(z_iv - lse_i) - [v = t_i]),  dx = d W,  dW = d^T x
//
// Forward: one launch of products whose tiles go no further than registers (entropy_kernel.cuh), and one that joins what the spans
// of symbols gave.  Backward: for each piece of the symbols the logits once more, as d in 16 bits, which two products then read.  The pieces
// are as large as kMostLogits allows; what they add to dx is kept in 32 bits.  Bound by the tensor cores (8 N V D operations a training step,
// of which 2 N V D for the logits that were not kept), for few rows by reading W.
#include <algorithm>
#include <atomic>

#include "entropy_few_kernel.cuh"
#include "entropy_kernel.cuh"
#include "tensor_map.cuh"

namespace tb200 {
namespace {

constexpr int64_t kMostLogits = 1ll << 28;  // of a piece, times its planes
constexpr int64_t kPiece = 256;             // symbols of a piece: a multiple of these
constexpr int64_t kMostStats = 1ll << 26;   // bytes of the spans' maxima and sums, about

// ----------------------------------------------------------------------------- operands that TMA cannot read in place

__device__ __forceinline__ int64_t index_at(const void* a, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(a)[i] : static_cast<int64_t>(static_cast<const int32_t*>(a)[i]);
}

// Rows that are not copied but zero: those whose target (null: there are none) is `ignore`.
struct Mask {
  const void* target;
  int64_t ignore;
  int wide;
};

// Rows on 16-byte boundaries, as they are or (PLANES) as three planes of bfloat16.
template <class T, bool PLANES>
__global__ void __launch_bounds__(256) entropy_copy_kernel(const T* x, int64_t rows, int width, int64_t stride, void* out, int64_t pitch, int64_t plane, Mask mask) {
  using Eight = Pack<T, 8 * static_cast<int>(sizeof(T))>;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t all = rows * (pitch / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / (pitch / 8);
    const int c = static_cast<int>(i - row * (pitch / 8)) * 8;
    const T* src = x + row * stride + c;
    Eight v;
    if (mask.target != nullptr && index_at(mask.target, mask.wide, row) == mask.ignore) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.v[e] = from_float<T>(0.f);
    } else if (c + 8 <= width && reinterpret_cast<uintptr_t>(src) % sizeof(v) == 0) {
      v = *reinterpret_cast<const Eight*>(src);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.v[e] = c + e < width ? src[e] : from_float<T>(0.f);
    }
    if constexpr (!PLANES) {
      *reinterpret_cast<Eight*>(static_cast<T*>(out) + row * pitch + c) = v;
    } else {
      uint16_t* to = static_cast<uint16_t*>(out) + row * pitch + c;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = plane_bits(v.v[2 * e], v.v[2 * e + 1]);
          v.v[2 * e] = plane_rest(v.v[2 * e]);
          v.v[2 * e + 1] = plane_rest(v.v[2 * e + 1]);
        }
        *reinterpret_cast<uint4*>(to + p * plane) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// ----------------------------------------------------------------------------- small kernels around the products

struct JoinArgs {
  const float2* stats;  // [parts][rows]
  const float* picked;  // the logits of the rows' own symbols
  const void* target;
  float *loss, *lse;
  double2* sums;  // of each block: losses, and how many there are
  int* arrived;   // blocks whose sums are there (zero before)
  int64_t ignore, symbols;
  int rows, parts, target_wide, reduction;
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 32 rows to a block: their parts are read by a lane to a row and every 32nd part to a warp, and joined by a warp to a row.  The block that comes last
// adds the blocks' losses, always in the same order.  One block is all latency (16 rows of 512 and 2000 symbols in bfloat16, the whole call: 11.0 us, 12.6 with the loads one after the other), so what it reads is
// on its way at once: the targets, which are the caller's, before the launch before this one has ended, up to kHeld parts to a thread behind it.
__global__ void __launch_bounds__(1024) entropy_join_kernel(const JoinArgs p) {
  __shared__ float shared[32][33], top_of[32];
  __shared__ double loss_of[32];
  __shared__ int given_of[32], last;
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int row = static_cast<int>(blockIdx.x) * 32 + lane;
  const int64_t own = static_cast<int64_t>(blockIdx.x) * 32 + warp;  // the row of this warp in the end
  constexpr int kHeld = 8;
  const int64_t target = own < p.rows ? index_at(p.target, p.target_wide, own) : p.ignore;
  pdl_launch_dependents();
  pdl_wait();
  float2 held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int i = warp + 32 * u;
    held[u] = row < p.rows && i < p.parts ? p.stats[static_cast<int64_t>(i) * p.rows + row] : make_float2(-INFINITY, 0.f);
  }
  const bool known = target != p.ignore && target >= 0 && target < p.symbols;
  const float picked = known ? p.picked[own] : 0.f;
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < kHeld; ++u) top = fmaxf(top, held[u].x);
  if (row < p.rows) {
#pragma unroll 8
    for (int i = warp + 32 * kHeld; i < p.parts; i += 32) top = fmaxf(top, p.stats[static_cast<int64_t>(i) * p.rows + row].x);
  }
  shared[warp][lane] = top;
  __syncthreads();
  top = warp_max(shared[lane][warp]);
  if (lane == 0) top_of[warp] = top == -INFINITY ? 0.f : top;
  __syncthreads();
  const float base = top_of[lane];
  float total = 0.f;
#pragma unroll
  for (int u = 0; u < kHeld; ++u) total = fmaf(held[u].y, ex2_approx((held[u].x - base) * LOG2E_F), total);
  if (row < p.rows) {
#pragma unroll 8
    for (int i = warp + 32 * kHeld; i < p.parts; i += 32) {
      const float2 a = p.stats[static_cast<int64_t>(i) * p.rows + row];
      total = fmaf(a.y, ex2_approx((a.x - base) * LOG2E_F), total);
    }
  }
  shared[warp][lane] = total;
  __syncthreads();
  total = warp_sum(shared[lane][warp]);
  if (lane == 0) {
    const float lse = top_of[warp] + logf(total);
    const bool given = target != p.ignore;
    const float loss = !given ? 0.f : known ? lse - picked : __int_as_float(0x7fc00000);
    if (own < p.rows) {
      p.lse[own] = lse;
      if (p.reduction == TRITURUS_B200_REDUCTION_NONE) p.loss[own] = loss;
    }
    loss_of[warp] = loss;
    given_of[warp] = given ? 1 : 0;
  }
  if (p.reduction == TRITURUS_B200_REDUCTION_NONE) return;
  __syncthreads();
  if (warp != 0) return;
  double sum = loss_of[lane], count = given_of[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if (gridDim.x > 1) {
    if (lane == 0) {
      p.sums[blockIdx.x] = make_double2(sum, count);
      __threadfence();
      last = atomicAdd(p.arrived, 1) == static_cast<int>(gridDim.x) - 1;
    }
    __syncwarp();
    if (!last) return;
    __threadfence();
    sum = count = 0.0;
    for (int i = lane; i < static_cast<int>(gridDim.x); i += 32) {
      const double2 a = __ldcg(&p.sums[i]);
      sum += a.x;
      count += a.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      count += __shfl_xor_sync(0xffffffffu, count, o);
    }
  }
  if (lane == 0) *p.loss = static_cast<float>(p.reduction == TRITURUS_B200_REDUCTION_MEAN ? sum / fmax(count, 1.0) : sum);
}

// factors[0] and [1]: see entropy_factors.
__global__ void __launch_bounds__(1024) entropy_factors_kernel(const float* dloss, int per_row, const void* target, int target_wide, int64_t ignore, int rows,
                                                               int mean, float scale, float* factors) {
  __shared__ float top_of[32];
  __shared__ int count_of[32];
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  float top = 0.f;
  int count = 0;
  pdl_launch_dependents();
  pdl_wait();
#pragma unroll 8
  for (int i = static_cast<int>(threadIdx.x); i < rows; i += 1024) {
    const bool given = index_at(target, target_wide, i) != ignore;
    const float g = per_row ? fabsf(dloss[i]) : 0.f;
    count += given ? 1 : 0;
    if (given && g < INFINITY) top = fmaxf(top, g);
  }
  if (!per_row) {
    const float g = fabsf(dloss[0]);
    if (g < INFINITY) top = g;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if (lane == 0) {
    top_of[warp] = top;
    count_of[warp] = count;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  count = 0;
  for (int w = 0; w < 32; ++w) {
    top = fmaxf(top, top_of[w]);
    count += count_of[w];
  }
  const float2 f = entropy_factors(top, count, mean, scale);
  factors[0] = f.x;
  factors[1] = f.y;
}

// The parts of shared tiles added up, four elements to a thread, and what is done with whole tiles.
template <class T>
__global__ void __launch_bounds__(256) entropy_sum_kernel(const __grid_constant__ EntropyParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int vectors = p.tile_cols / 4;  // of a tile's row, and blocks to a tile
  const int s = static_cast<int>(blockIdx.x) / vectors;
  const int i = (static_cast<int>(blockIdx.x) - s * vectors) * 256 + static_cast<int>(threadIdx.x);
  const int in_tile = i / vectors, c = (i - in_tile * vectors) * 4;
  const int u = p.whole + s, of_group = p.group * p.units_n;
  const int g = u / of_group, r = u - g * of_group, rows_here = min(p.group, p.tiles_m - g * p.group);
  const int row = (g * p.group + r % rows_here) * 256 + in_tile, col = r / rows_here * p.unit_cols + c;
  if (row >= p.rows || col >= p.cols) return;
  const float* part = p.part + (static_cast<int64_t>(s) * p.splits * 256 + in_tile) * p.tile_cols + c;
  float4 x = *reinterpret_cast<const float4*>(part);
  for (int k = 1; k < p.splits; ++k) {
    const float4 y = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(k) * 256 * p.tile_cols);
    x.x += y.x;
    x.y += y.y;
    x.z += y.z;
    x.w += y.w;
  }
  if (p.dest != DEST_FINAL) {
    float4* sum = reinterpret_cast<float4*>(p.sum + static_cast<int64_t>(row) * p.sum_pitch + col);
    if (p.dest != DEST_SUM) {
      const float4 y = *sum;
      x.x += y.x;
      x.y += y.y;
      x.z += y.z;
      x.w += y.w;
    }
    if (p.dest != DEST_FINAL_ADD) {
      *sum = x;
      return;
    }
  }
  entropy_put<T>(p, row, col, x, p.cols);
}

// The parts of dx from few rows, [splits][rows][pitch], added up.
template <class T>
__global__ void __launch_bounds__(256) entropy_few_sum_kernel(const __grid_constant__ FewParams p, int width) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = static_cast<int>(blockIdx.y), col = (static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x));
  if (col >= width) return;
  const float* part = p.e.part + row * p.e.sum_pitch + col;
  float x = 0.f;
#pragma unroll 16
  for (int k = 0; k < p.splits; ++k) x += part[static_cast<int64_t>(k) * p.rows * p.e.sum_pitch];
  float* sum = p.e.sum + row * p.e.sum_pitch + col;
  if (p.e.dest == DEST_SUM_ADD || p.e.dest == DEST_FINAL_ADD) x += *sum;
  if (p.e.dest == DEST_SUM || p.e.dest == DEST_SUM_ADD)
    *sum = x;
  else
    static_cast<T*>(p.e.out)[row * p.e.out_pitch + col] = from_float<T>(x);
}

// ----------------------------------------------------------------------------- host

int size_of(int type) { return type == TRITURUS_B200_TYPE_F32 ? 4 : 2; }
bool sizes_ok(int64_t rows, int64_t symbols, int64_t width, int type) {
  const int64_t most = 1 << 30;
  return rows >= 0 && rows <= most && symbols > 0 && symbols <= most && width > 0 && width <= most && type >= TRITURUS_B200_TYPE_F32 &&
         type <= TRITURUS_B200_TYPE_F16;
}
int64_t up_to(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }
int64_t parts_of(int64_t n, int64_t unit) { return (n + unit - 1) / unit; }

// A matrix as TMA reads it: of 16-bit elements, or of 32-bit ones as they are (`raw`).
struct Matrix {
  const void* data;
  int64_t rows, width, pitch, plane;
  int planes;
  bool raw;
};
// How the operands are read: 32-bit ones as planes but for W with few rows of x.  With many rows 16-bit operands whose rows are off 128-byte lines are
// copied too: TMA fetches two lines for each row of a box (4096 x 50000 of width 1000: forward 497 -> 365 us and 31 us for the copy, gradients 1168 -> 915;
// at 1024 rows the copy takes what it saves).
constexpr int64_t kLines = 2048;
struct Reading {
  int type;
  bool raw, lines;
  Mask mask;  // x of the gradients: dW multiplies it with d, and what a position without a loss holds (it may be NaN) must not count
};
Reading reading_of(int64_t rows, int type, bool weight, Mask mask = {});
// Whether an operand is read where it lies: rows on 16-byte boundaries (or lines) that do not overlap, and 32-bit elements only as they are.
bool in_place(const void* data, int64_t rows, int64_t width, int64_t stride, const Reading& how) {
  if ((how.type == TRITURUS_B200_TYPE_F32 && !how.raw) || how.mask.target != nullptr) return false;
  const int64_t unit = how.lines ? 128 : 16;
  return aligned_to(data, unit) && (rows == 1 || (stride >= width && stride * size_of(how.type) % unit == 0 && stride < (1ll << 37)));
}
// A copy's rows are on lines.
int64_t copy_pitch(int64_t width, const Reading& how) { return up_to(width, how.raw ? 32 : 64); }
size_t copy_bytes(const void* data, int64_t rows, int64_t width, int64_t stride, const Reading& how) {
  if (in_place(data, rows, width, stride, how)) return 0;
  return static_cast<size_t>(rows) * static_cast<size_t>(copy_pitch(width, how)) * (how.raw ? 4 : how.type == TRITURUS_B200_TYPE_F32 ? 6 : 2);
}

int make_map(CUtensorMap* map, const Matrix& m, int box_x, int box_y, int type) {
  const EncodeTiledFn fn = get_encode_fn();
  if (fn == nullptr) return TRITURUS_B200_EDRIVER;
  const cuuint64_t size = m.raw ? 4 : 2;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(m.width), static_cast<cuuint64_t>(m.rows), static_cast<cuuint64_t>(m.planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(m.pitch) * size, static_cast<cuuint64_t>(m.plane) * size};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_x), static_cast<cuuint32_t>(box_y), 1}, step[3] = {1, 1, 1};
  const CUtensorMapDataType kind = m.raw                            ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : type == TRITURUS_B200_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult rc = fn(map, kind, 3, const_cast<void*>(m.data), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? TRITURUS_B200_OK : TRITURUS_B200_ETENSORMAP;
}

// The launches of a call: each but the first may begin while the one before it ends, whose results it waits for.
struct Launches {
  cudaStream_t stream;
  bool first = true;
  template <class... Params, class... Args>
  int operator()(void (*kern)(Params...), dim3 grid, int threads, size_t smem, Args&&... args) {
    const cudaLaunchAttribute dependent = dependent_launch();
    const int rc = launch_of(kern, grid, threads, smem, stream, first ? nullptr : &dependent, static_cast<Args&&>(args)...);
    first = false;
    return rc;
  }
  template <class... Params, class... Args>
  int operator()(void (*kern)(Params...), int64_t grid, int threads, size_t smem, Args&&... args) {
    return (*this)(kern, dim3(static_cast<unsigned>(grid)), threads, smem, static_cast<Args&&>(args)...);
  }
};

int copy_grid(int64_t items) { return static_cast<int>(std::min<int64_t>(parts_of(items, 256), static_cast<int64_t>(device_sms()) * 16)); }

// The operand itself or, copied to `space`, one that TMA can read.
int prepare(Matrix* m, const void* data, int64_t rows, int64_t width, int64_t stride, const Reading& how, void* space, Launches& launch) {
  const int type = how.type;
  const bool raw = how.raw;
  m->rows = rows;
  m->width = width;
  m->raw = raw && type == TRITURUS_B200_TYPE_F32;
  m->planes = type == TRITURUS_B200_TYPE_F32 && !raw ? 3 : 1;
  if (in_place(data, rows, width, stride, how)) {
    m->data = data;
    m->pitch = rows == 1 ? up_to(width, 8) : stride;
    m->plane = rows * m->pitch;
    return TRITURUS_B200_OK;
  }
  m->data = space;
  m->pitch = copy_pitch(width, how);
  m->plane = rows * m->pitch;
  const int grid = copy_grid(rows * (m->pitch / 8));
  const auto run = [&](auto kern, auto t) {
    return launch(kern, grid, 256, 0, static_cast<const decltype(t)*>(data), rows, static_cast<int>(width), stride, space, m->pitch, m->plane, how.mask);
  };
  if (type == TRITURUS_B200_TYPE_F32) return raw ? run(entropy_copy_kernel<float, false>, 0.f) : run(entropy_copy_kernel<float, true>, 0.f);
  if (type == TRITURUS_B200_TYPE_BF16) return run(entropy_copy_kernel<__nv_bfloat16, false>, __nv_bfloat16());
  return run(entropy_copy_kernel<__half, false>, __half());
}

// k-blocks of an accumulator of 16-bit products.  Logits: root mean square error of the losses of 8192 x 32768 of width 2048 in float16 and the time, 4: 1.5e-7, 805 us;
// 8: 2.8e-7, 753; 16: 5.8e-7, 749; 32 (all): 1.2e-6, 741 (sums of float32 products one after the other: 3.7e-7).
constexpr int kDrainLogits = 8;
constexpr int kDrainOut = 256;  // (of results that are rounded to 16 bits; 2^-14 of the sum is cut off by then)

// Up to so many k-blocks the 32-bit results of OUT_W leave through TMA: dW alone of 50000 x 2048 with 16 rows 208 -> 184 us, 64: 217 -> 201, 128: 367 -> 360.  (With more
// rows their planes take the shared memory; 16-bit results gain nothing, 112 and 116.)
constexpr int kBoxed = 2;

int pairs_in_all() { return std::max(1, device_sms() / 2); }

template <class Cfg>
int launch_products(const Matrix& a, const Matrix& b, EntropyParams p, int type, Launches& launch) {
  CUtensorMap ta, tb, to;
  int rc = Cfg::A_MN ? make_map(&ta, a, 64, Cfg::BK, type) : make_map(&ta, a, Cfg::BK, Cfg::BM, type);
  if (rc == TRITURUS_B200_OK) rc = Cfg::B_MN ? make_map(&tb, b, 64, Cfg::BK, type) : make_map(&tb, b, Cfg::BK, Cfg::BNH, type);
  if (rc != TRITURUS_B200_OK) return rc;
  to = ta;  // (not used)
  if (p.boxed) {
    const Matrix out = {p.out, p.rows, p.cols, p.out_pitch, p.rows * p.out_pitch, 1, true};
    rc = make_map(&to, out, 32, 32, type);
    if (rc != TRITURUS_B200_OK) return rc;
  }
  const auto kern = entropy_kernel<Cfg>;
  static std::atomic<bool> known[64];
  int dev = 0;
  if (code_of(cudaGetDevice(&dev)) != TRITURUS_B200_OK || dev < 0 || dev >= 64) return TRITURUS_B200_ELAUNCH;
  if (!known[dev].load(std::memory_order_relaxed)) {
    rc = code_of(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    if (rc != TRITURUS_B200_OK) return rc;
    cudaFuncAttributes about;
    rc = code_of(cudaFuncGetAttributes(&about, kern));
    if (rc != TRITURUS_B200_OK) return rc;
    if (!Cfg::WIDE && about.numRegs != 168) return TRITURUS_B200_EREGISTERS;  // (its warps would wait for registers that nobody has)
    known[dev].store(true, std::memory_order_relaxed);
  }
  p.half = type == TRITURUS_B200_TYPE_F16;
  p.drain = Cfg::MODE == ENTROPY_STATS || Cfg::MODE == ENTROPY_PROB ? kDrainLogits : kDrainOut;
  p.idesc = umma_idesc_16(2 * Cfg::BM, p.half != 0, Cfg::A_MN, Cfg::B_MN);
  const int64_t pairs = std::min<int64_t>(p.whole + static_cast<int64_t>(p.shared) * p.splits, pairs_in_all());
  return launch(kern, 2 * pairs, Cfg::NTHREADS, Cfg::SMEM_BYTES, ta, tb, to, p);
}
template <int MODE>
int run_products(const Matrix& a, const Matrix& b, const EntropyParams& p, int type, Launches& launch) {
  int rc = type == TRITURUS_B200_TYPE_F32 ? launch_products<EntropyCfg<MODE, true>>(a, b, p, type, launch) : launch_products<EntropyCfg<MODE, false>>(a, b, p, type, launch);
  if (rc != TRITURUS_B200_OK || p.shared == 0) return rc;
  EntropyParams q = p;
  q.half = type == TRITURUS_B200_TYPE_F16;
  const int64_t grid = static_cast<int64_t>(p.shared) * (p.tile_cols / 4);
  return type == TRITURUS_B200_TYPE_F32    ? launch(entropy_sum_kernel<float>, grid, 256, 0, q)
         : type == TRITURUS_B200_TYPE_BF16 ? launch(entropy_sum_kernel<__nv_bfloat16>, grid, 256, 0, q)
                                           : launch(entropy_sum_kernel<__half>, grid, 256, 0, q);
}

// ----------------------------------------------------------------------------- tiles for pairs

int widest(int type) { return type == TRITURUS_B200_TYPE_F32 ? EntropyCfg<0, true>::BN : EntropyCfg<0, false>::BN; }
// Cycles of a k-block of a tile of `cols` columns, by whichever takes longer: the MMAs, or what they and TMA move through 128 bytes a cycle of shared memory.
int64_t cycles_of(int64_t cols, int type) {
  return type == TRITURUS_B200_TYPE_F32 ? std::max(12 * cols, 1152 + 9 * cols / 2) : std::max(2 * cols, 256 + cols);
}
constexpr int64_t kTileCycles = 2500;    // of a tile beside its MMAs
constexpr int64_t kSumCycles = 6000;     // of a launch that adds parts
constexpr int64_t kBytesPerCycle = 3500;
constexpr int64_t kLeastUnits = 5;       // waves of tiles from which on their rounding up does not matter

EntropyParams product_of(int64_t rows, int64_t cols, int64_t k) {
  EntropyParams p = {};
  p.rows = static_cast<int>(rows);
  p.cols = static_cast<int>(cols);
  p.kblocks = static_cast<int>(parts_of(k, EntropyCfg<0, false>::BK));
  p.tiles_m = static_cast<int>(parts_of(rows, 256));
  p.group = 8;
  return p;
}
void set_units(EntropyParams& p, int64_t unit_cols, int64_t tile_cols) {
  p.unit_cols = static_cast<int>(unit_cols);
  p.tile_cols = static_cast<int>(tile_cols);
  p.units_n = static_cast<int>(parts_of(p.cols, unit_cols));
}
// All units but the shared ones are whole; false where they are too many.
bool set_whole(EntropyParams& p) {
  const int64_t units = static_cast<int64_t>(p.tiles_m) * p.units_n;
  if (units > INT32_MAX || static_cast<int64_t>(p.group) * p.units_n > INT32_MAX) return false;
  p.whole = static_cast<int>(units - p.shared);
  p.by_group = Divisor(p.group * p.units_n);
  p.by_rows = Divisor(p.group);
  p.by_last = Divisor(p.tiles_m % p.group != 0 ? p.tiles_m % p.group : p.group);
  p.by_shared = Divisor(std::max(p.shared, 1));
  return true;
}

// STATS: spans of columns, of any length, so that the pairs have about the same to do: a number of them for each row tile that makes 1 to 16 units to a
// pair.  Few long ones where there are few tiles, since each ends with an epilogue that nothing covers.
EntropyParams stats_of(int64_t rows, int64_t symbols, int64_t width, int type) {
  EntropyParams p = product_of(rows, symbols, width);
  const int64_t pairs = pairs_in_all(), wide = widest(type);
  const int64_t most = std::max<int64_t>(1, std::min(parts_of(symbols, 32), kMostStats / (rows * 2 * static_cast<int64_t>(sizeof(float2)))));
  int64_t best = INT64_MAX;
  for (int64_t k = 1; k <= 16; ++k) {
    const int64_t spans = std::clamp<int64_t>(k * pairs / p.tiles_m, 1, most);
    const int64_t cols = parts_of(symbols, spans), tiles = parts_of(cols, wide), tile = up_to(parts_of(cols, tiles), 32);
    const int64_t cost = parts_of(p.tiles_m * parts_of(symbols, cols), pairs) * (tiles * p.kblocks * cycles_of(tile, type) + kTileCycles);
    if (cost < best) {
      best = cost;
      set_units(p, cols, tile);
    }
  }
  return p;
}

// PROB: tiles of up to the widest, of fewer columns where that makes the waves of them even.
EntropyParams prob_of(int64_t rows, int64_t symbols, int64_t width, int type) {
  EntropyParams p = product_of(rows, symbols, width);
  const int64_t pairs = pairs_in_all();
  int64_t best = INT64_MAX;
  for (int64_t tile = widest(type); tile >= 96; tile -= 32) {
    const int64_t waves = parts_of(p.tiles_m * parts_of(symbols, tile), pairs);
    const int64_t cost = waves * (p.kblocks * cycles_of(tile, type) + kTileCycles);
    if (cost < best) {
      best = cost;
      set_units(p, tile, tile);
    }
    if (waves > kLeastUnits) break;
  }
  return p;
}

// OUT: the same, and the contraction of the tiles that are left over behind full waves is cut into parts where waves of those take less time.
EntropyParams out_of(int64_t rows, int64_t cols, int64_t k, int type) {
  EntropyParams p = product_of(rows, cols, k);
  const int64_t pairs = pairs_in_all();
  int64_t best = INT64_MAX;
  for (int64_t tile = widest(type); tile >= 96; tile -= 32) {
    const int64_t even = std::min<int64_t>(tile, up_to(parts_of(cols, parts_of(cols, tile)), 32));
    const int64_t units = p.tiles_m * parts_of(cols, even), full = units / pairs, left = units - full * pairs, cycles = cycles_of(even, type);
    // (few parts, and the most that 1 to 4 waves of them have)
    const int candidates = left == 0 ? 1 : 12;
    for (int i = 0; i < candidates; ++i) {
      const int64_t most = i < 8 ? i + 1 : (i - 7) * pairs / left;
      if (most > p.kblocks || (i >= 8 && most <= 8)) continue;
      const int64_t kb = parts_of(p.kblocks, most), splits = parts_of(p.kblocks, kb);
      const int64_t parts = left * splits * 256 * even * 2 * static_cast<int64_t>(sizeof(float)) / kBytesPerCycle;  // written and read
      const int64_t cost = full * (p.kblocks * cycles + kTileCycles) + parts_of(left * splits, pairs) * (kb * cycles + kTileCycles) +
                           (splits > 1 ? kSumCycles + parts : 0);
      if (cost < best) {
        best = cost;
        set_units(p, even, even);
        p.shared = splits > 1 ? static_cast<int>(left) : 0;
        p.splits = static_cast<int>(splits);
        p.kb_split = static_cast<int>(kb);
      }
    }
    if (full > kLeastUnits) break;
  }
  return p;
}
size_t part_bytes(const EntropyParams& p) {
  return static_cast<size_t>(p.shared) * static_cast<size_t>(p.splits) * 256 * static_cast<size_t>(p.tile_cols) * sizeof(float);
}

// ----------------------------------------------------------------------------- few rows

// Up to this many rows of x the exchanged forms are used.  Microseconds forwards / gradients, exchanged and not, of 50000 symbols of width 2048: bfloat16 64 rows
// 47 / 143 and 47 / 149, 96 rows (two tiles of 64) 68 / 184 and 48 / 151; float32 64 rows 100 / 312 and 376 / 714, 192 rows 239 / 774 and
// 406 / 885, 256 rows 356 / 1064 and 415 / 972.
bool few(int64_t rows, int type) { return rows <= (type == TRITURUS_B200_TYPE_F32 ? 192 : 64); }
Reading reading_of(int64_t rows, int type, bool weight, Mask mask) {
  return {type, type == TRITURUS_B200_TYPE_F32 && weight && few(rows, type), type != TRITURUS_B200_TYPE_F32 && rows >= kLines, mask};
}

FewParams few_of(int64_t rows, int64_t length, int64_t k) {
  FewParams p = {};
  p.rows = static_cast<int>(rows);
  p.length = static_cast<int>(length);
  p.kblocks = static_cast<int>(parts_of(k, 64));
  p.mma_n = static_cast<int>(std::min<int64_t>(64, up_to(rows, 16)));
  return p;
}
// STATS, PROB: an even span of the symbols for each SM.
FewParams few_symbols_of(int64_t rows, int64_t symbols, int64_t width) {
  FewParams p = few_of(rows, symbols, width);
  const int64_t row_tiles = parts_of(rows, 64);
  p.span = static_cast<int>(std::max<int64_t>(16, parts_of(symbols, std::max<int64_t>(1, device_sms() / row_tiles))));
  p.spans = static_cast<int>(parts_of(symbols, p.span));
  p.tile = static_cast<int>(parts_of(p.span, parts_of(p.span, 128)));
  p.splits = 1;
  p.kb_split = p.kblocks;
  p.units = static_cast<int>(p.spans * row_tiles);
  return p;
}
// OUT_X: tiles of 128 columns, the contraction cut into parts for the SMs.
FewParams few_columns_of(int64_t rows, int64_t width, int64_t symbols) {
  FewParams p = few_of(rows, width, symbols);
  const int64_t row_tiles = parts_of(rows, 64);
  p.span = p.tile = 128;
  p.spans = static_cast<int>(parts_of(width, 128));
  const int64_t splits = std::clamp<int64_t>(device_sms() / (p.spans * row_tiles), 1, parts_of(p.kblocks, 4));
  p.kb_split = static_cast<int>(parts_of(p.kblocks, splits));
  p.splits = static_cast<int>(parts_of(p.kblocks, p.kb_split));
  p.units = static_cast<int>(p.spans * p.splits * row_tiles);
  return p;
}

// W (a) and x or d (b).
template <class Cfg>
int launch_few(const Matrix& a, const Matrix& b, FewParams p, int type, Launches& launch) {
  CUtensorMap ta, tb;
  int rc = Cfg::A_MN ? make_map(&ta, a, Cfg::WIDE ? 32 : 64, Cfg::BK, type) : make_map(&ta, a, Cfg::WIDE ? 32 : 64, p.tile, type);
  if (rc == TRITURUS_B200_OK) rc = make_map(&tb, b, Cfg::BK, p.mma_n, type);
  if (rc != TRITURUS_B200_OK) return rc;
  const auto kern = entropy_few_kernel<Cfg>;
  static std::atomic<bool> known[64];
  int dev = 0;
  if (code_of(cudaGetDevice(&dev)) != TRITURUS_B200_OK || dev < 0 || dev >= 64) return TRITURUS_B200_ELAUNCH;
  if (!known[dev].load(std::memory_order_relaxed)) {
    rc = code_of(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    if (rc != TRITURUS_B200_OK) return rc;
    known[dev].store(true, std::memory_order_relaxed);
  }
  p.e.half = type == TRITURUS_B200_TYPE_F16;
  p.e.drain = Cfg::MODE == ENTROPY_OUT_X ? kDrainOut : kDrainLogits;
  p.a_bytes = Cfg::A_MN ? Cfg::A_TILE : p.tile * Cfg::BK * (Cfg::WIDE ? 4 : 2);
  p.b_bytes = Cfg::PLANES * p.mma_n * Cfg::BK * 2;
  p.idesc = umma_idesc_16(Cfg::BM, p.e.half != 0, Cfg::A_MN && !Cfg::WIDE, false) | static_cast<uint32_t>(p.mma_n >> 3) << 17;
  return launch(kern, std::min(p.units, device_sms()), Cfg::NTHREADS, Cfg::SMEM_BYTES, ta, tb, p);
}
template <int MODE>
int run_few(const Matrix& a, const Matrix& b, const FewParams& p, int type, Launches& launch) {
  return type == TRITURUS_B200_TYPE_F32 ? launch_few<FewCfg<MODE, true>>(a, b, p, type, launch) : launch_few<FewCfg<MODE, false>>(a, b, p, type, launch);
}

int sum_few(const FewParams& p, int64_t width, int type, Launches& launch) {
  const dim3 grid(static_cast<unsigned>(parts_of(width, 256)), static_cast<unsigned>(p.rows));
  const int w = static_cast<int>(width);
  return type == TRITURUS_B200_TYPE_F32    ? launch(entropy_few_sum_kernel<float>, grid, 256, 0, p, w)
         : type == TRITURUS_B200_TYPE_BF16 ? launch(entropy_few_sum_kernel<__nv_bfloat16>, grid, 256, 0, p, w)
                                           : launch(entropy_few_sum_kernel<__half>, grid, 256, 0, p, w);
}

struct Space {  // the workspace as it is handed out
  char* at;
  size_t used;
  void* take(size_t bytes) {
    void* p = at + used;
    used += (bytes + 255) & ~static_cast<size_t>(255);
    return p;
  }
};

struct ForwardSpace {
  void *x, *weight;
  float2* stats;
  float* picked;
  double2* sums;
  int* arrived;
  size_t bytes;
};
ForwardSpace forward_space(void* base, const void* x, const void* weight, int64_t rows, int64_t symbols, int64_t width, int64_t x_stride,
                           int64_t weight_stride, int type) {
  Space s = {static_cast<char*>(base), 0};
  ForwardSpace f;
  const bool is_few = few(rows, type);
  f.x = s.take(copy_bytes(x, rows, width, x_stride, reading_of(rows, type, false)));
  f.weight = s.take(copy_bytes(weight, symbols, width, weight_stride, reading_of(rows, type, true)));
  const int64_t parts = is_few ? few_symbols_of(rows, symbols, width).spans : stats_of(rows, symbols, width, type).units_n * 2;
  f.stats = static_cast<float2*>(s.take(static_cast<size_t>(parts) * static_cast<size_t>(rows) * sizeof(float2)));
  f.picked = static_cast<float*>(s.take(static_cast<size_t>(rows) * sizeof(float)));
  f.sums = static_cast<double2*>(s.take(static_cast<size_t>(parts_of(rows, 32)) * sizeof(double2)));
  f.arrived = static_cast<int*>(s.take(sizeof(int)));
  f.bytes = s.used;
  return f;
}

struct BackwardPlan {
  int64_t piece, pieces, last, d_pitch, sum_pitch;  // last: symbols of the last piece
  EntropyParams x[2], w[2];                         // OUT_X (not of few rows) and OUT_W, of a piece and of the last one
};
BackwardPlan backward_plan(int64_t rows, int64_t symbols, int64_t width, int type) {
  BackwardPlan b;
  const int planes = type == TRITURUS_B200_TYPE_F32 ? 3 : 1;
  const int64_t most = std::max(kPiece, kMostLogits / planes / rows / kPiece * kPiece);
  b.pieces = parts_of(symbols, most);
  b.piece = std::min(up_to(parts_of(symbols, b.pieces), kPiece), symbols);
  b.pieces = parts_of(symbols, b.piece);
  b.last = symbols - (b.pieces - 1) * b.piece;
  b.d_pitch = up_to(b.piece, 64);
  b.sum_pitch = up_to(width, 8);
  for (int i = 0; i < 2; ++i) {
    const int64_t piece = i == 0 ? b.piece : b.last;
    if (i == 1 && b.last == b.piece) {
      b.x[1] = b.x[0];
      b.w[1] = b.w[0];
    } else {
      b.x[i] = few(rows, type) ? EntropyParams{} : out_of(rows, width, piece, type);
      b.w[i] = out_of(piece, width, rows, type);
    }
  }
  return b;
}
struct BackwardSpace {
  void *x, *weight;
  float *factors, *sum, *part;
  uint16_t* d;
  size_t bytes;
};
BackwardSpace backward_space(void* base, const BackwardPlan& b, const void* x, const void* weight, int64_t rows, int64_t symbols, int64_t width,
                             int64_t x_stride, int64_t weight_stride, int type) {
  Space s = {static_cast<char*>(base), 0};
  BackwardSpace f;
  const bool is_few = few(rows, type);
  f.x = s.take(copy_bytes(x, rows, width, x_stride, reading_of(rows, type, false, {&f, 0, 0})));  // (room for a copy in any case)
  f.weight = s.take(copy_bytes(weight, symbols, width, weight_stride, reading_of(rows, type, true)));
  f.factors = static_cast<float*>(s.take(2 * sizeof(float)));
  f.d = static_cast<uint16_t*>(s.take(static_cast<size_t>(rows) * static_cast<size_t>(b.d_pitch) * 2 * (type == TRITURUS_B200_TYPE_F32 ? 3 : 1)));
  f.sum = static_cast<float*>(s.take(b.pieces > 1 ? static_cast<size_t>(rows) * static_cast<size_t>(b.sum_pitch) * sizeof(float) : 0));
  size_t parts = 0;  // (one product at a time uses them)
  for (int i = 0; i < 2; ++i) {
    const size_t of_x = is_few ? static_cast<size_t>(few_columns_of(rows, width, i == 0 ? b.piece : b.last).splits) * static_cast<size_t>(rows * b.sum_pitch) * sizeof(float)
                               : part_bytes(b.x[i]);
    parts = std::max({parts, of_x, part_bytes(b.w[i])});
  }
  f.part = static_cast<float*>(s.take(parts));
  f.bytes = s.used;
  return f;
}

bool reduction_ok(int r) { return r >= TRITURUS_B200_REDUCTION_NONE && r <= TRITURUS_B200_REDUCTION_SUM; }

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" {

size_t triturus_b200_linear_cross_entropy_workspace_bytes(const void* x, const void* weight, int64_t rows, int64_t symbols, int64_t width,
                                                          int64_t x_stride, int64_t weight_stride, int type) {
  if (!sizes_ok(rows, symbols, width, type) || rows == 0) return 0;
  return forward_space(nullptr, x, weight, rows, symbols, width, x_stride, weight_stride, type).bytes;
}

int triturus_b200_linear_cross_entropy(const void* x, const void* weight, const void* target, int target_bytes, float* loss, float* lse,
                                       int64_t rows, int64_t symbols, int64_t width, int64_t x_stride, int64_t weight_stride, int type,
                                       int reduction, int64_t ignore_index, void* workspace, size_t workspace_bytes, int32_t* status_dev, void* stream) {
  if (!sizes_ok(rows, symbols, width, type) || !reduction_ok(reduction) || (target_bytes != 4 && target_bytes != 8)) return TRITURUS_B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Launches launch = {st};
  if (rows == 0) {
    if (reduction == TRITURUS_B200_REDUCTION_NONE) return TRITURUS_B200_OK;
    if (loss == nullptr) return TRITURUS_B200_EINVAL;
    return aligned_to(loss, 4) ? code_of(cudaMemsetAsync(loss, 0, sizeof(float), st)) : TRITURUS_B200_EALIGN;
  }
  if (x == nullptr || weight == nullptr || target == nullptr || loss == nullptr || lse == nullptr || workspace == nullptr) return TRITURUS_B200_EINVAL;
  if (!aligned_to(x, size_of(type)) || !aligned_to(weight, size_of(type)) || !aligned_to(target, target_bytes) || !aligned_to(loss, 4) ||
      !aligned_to(lse, 4) || !aligned_to(workspace, 256))
    return TRITURUS_B200_EALIGN;
  const ForwardSpace space = forward_space(workspace, x, weight, rows, symbols, width, x_stride, weight_stride, type);
  if (workspace_bytes < space.bytes) return TRITURUS_B200_EWORKSPACE;

  Matrix a, b;
  const bool is_few = few(rows, type);
  int rc = prepare(&a, x, rows, width, x_stride, reading_of(rows, type, false), space.x, launch);
  if (rc == TRITURUS_B200_OK) rc = prepare(&b, weight, symbols, width, weight_stride, reading_of(rows, type, true), space.weight, launch);
  if (rc != TRITURUS_B200_OK) return rc;
  JoinArgs j = {};
  if (is_few) {
    FewParams p = few_symbols_of(rows, symbols, width);
    p.e.stats = space.stats;
    p.e.picked = space.picked;
    p.e.arrived = space.arrived;
    p.e.target = target;
    p.e.target_wide = target_bytes == 8;
    p.e.symbols = symbols;
    p.e.status = status_dev;
    p.x = x;
    p.weight = weight;
    p.x_stride = x_stride;
    p.weight_stride = weight_stride;
    p.width = static_cast<int>(width);
    rc = run_few<ENTROPY_STATS>(b, a, p, type, launch);
    j.parts = p.spans;
  } else {
    EntropyParams p = stats_of(rows, symbols, width, type);
    if (!set_whole(p)) return TRITURUS_B200_EINVAL;
    p.stats = space.stats;
    p.picked = space.picked;
    p.arrived = space.arrived;
    p.target = target;
    p.target_wide = target_bytes == 8;
    p.ignore = ignore_index;
    p.symbols = symbols;
    p.status = status_dev;
    rc = run_products<ENTROPY_STATS>(a, b, p, type, launch);
    j.parts = p.units_n * 2;
  }
  if (rc != TRITURUS_B200_OK) return rc;

  j.stats = space.stats;
  j.picked = space.picked;
  j.arrived = space.arrived;
  j.target = target;
  j.loss = loss;
  j.lse = lse;
  j.sums = space.sums;
  j.ignore = ignore_index;
  j.symbols = symbols;
  j.rows = static_cast<int>(rows);
  j.target_wide = target_bytes == 8;
  j.reduction = reduction;
  const int blocks = static_cast<int>(parts_of(rows, 32));
  return launch(entropy_join_kernel, blocks, 1024, 0, j);
}

size_t triturus_b200_linear_cross_entropy_backward_workspace_bytes(const void* x, const void* weight, int64_t rows, int64_t symbols, int64_t width,
                                                                   int64_t x_stride, int64_t weight_stride, int type) {
  if (!sizes_ok(rows, symbols, width, type) || rows == 0) return 0;
  return backward_space(nullptr, backward_plan(rows, symbols, width, type), x, weight, rows, symbols, width, x_stride, weight_stride, type).bytes;
}

int triturus_b200_linear_cross_entropy_backward(const float* dloss, const void* x, const void* weight, const void* target, int target_bytes,
                                                const float* lse, void* dx, void* dweight, int64_t rows, int64_t symbols, int64_t width,
                                                int64_t x_stride, int64_t weight_stride, int type, int reduction, int64_t ignore_index,
                                                void* workspace, size_t workspace_bytes, int32_t* status_dev, void* stream) {
  if (!sizes_ok(rows, symbols, width, type) || !reduction_ok(reduction) || (target_bytes != 4 && target_bytes != 8)) return TRITURUS_B200_EINVAL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int size = size_of(type);
  if (!aligned_to(dx, size) || !aligned_to(dweight, size)) return TRITURUS_B200_EALIGN;
  if (rows == 0) return dweight == nullptr ? TRITURUS_B200_OK : code_of(cudaMemsetAsync(dweight, 0, static_cast<size_t>(symbols) * static_cast<size_t>(width) * size, st));
  if (dloss == nullptr || x == nullptr || weight == nullptr || target == nullptr || lse == nullptr || workspace == nullptr) return TRITURUS_B200_EINVAL;
  if (!aligned_to(x, size) || !aligned_to(weight, size) || !aligned_to(target, target_bytes) || !aligned_to(dloss, 4) || !aligned_to(lse, 4) ||
      !aligned_to(workspace, 256))
    return TRITURUS_B200_EALIGN;
  const BackwardPlan plan = backward_plan(rows, symbols, width, type);
  const BackwardSpace space = backward_space(workspace, plan, x, weight, rows, symbols, width, x_stride, weight_stride, type);
  if (workspace_bytes < space.bytes) return TRITURUS_B200_EWORKSPACE;
  if (dx == nullptr && dweight == nullptr) return TRITURUS_B200_OK;

  Launches launch = {st};
  Matrix mx, mw;
  const bool is_few = few(rows, type);
  const Mask mask = {dweight != nullptr ? target : nullptr, ignore_index, target_bytes == 8};
  int rc = prepare(&mx, x, rows, width, x_stride, reading_of(rows, type, false, mask), space.x, launch);
  if (rc == TRITURUS_B200_OK) rc = prepare(&mw, weight, symbols, width, weight_stride, reading_of(rows, type, true), space.weight, launch);
  const int wide = target_bytes == 8;
  const int per_row = reduction == TRITURUS_B200_REDUCTION_NONE ? 1 : 0;
  if (rc == TRITURUS_B200_OK && !is_few)
    rc = launch(entropy_factors_kernel, 1, 1024, 0, dloss, per_row, target, wide, ignore_index, static_cast<int>(rows),
                reduction == TRITURUS_B200_REDUCTION_MEAN ? 1 : 0, entropy_scale(type == TRITURUS_B200_TYPE_F32, type == TRITURUS_B200_TYPE_F16 ? 1 : 0, per_row),
                space.factors);
  Matrix md = {};
  md.data = space.d;
  md.rows = rows;
  md.pitch = plan.d_pitch;
  md.plane = rows * plan.d_pitch;
  md.planes = type == TRITURUS_B200_TYPE_F32 ? 3 : 1;
  for (int64_t i = 0; i < plan.pieces && rc == TRITURUS_B200_OK; ++i) {
    const int64_t first = i * plan.piece, piece = i + 1 < plan.pieces ? plan.piece : plan.last;
    const int last = i + 1 == plan.pieces ? 1 : 0;
    EntropyParams p = is_few ? EntropyParams{} : prob_of(rows, piece, width, type);
    if (!is_few && !set_whole(p)) return TRITURUS_B200_EINVAL;
    p.b_row = static_cast<int>(first);
    p.target = target;
    p.target_wide = wide;
    p.ignore = ignore_index;
    p.symbols = symbols;
    p.lse = lse;
    p.dloss = dloss;
    p.per_row = per_row;
    p.factors = space.factors;
    p.d = space.d;
    p.d_pitch = md.pitch;
    p.d_plane = md.plane;
    p.status = status_dev;
    if (is_few) {
      FewParams f = few_symbols_of(rows, piece, width);
      f.e = p;
      f.mean = reduction == TRITURUS_B200_REDUCTION_MEAN;
      rc = run_few<ENTROPY_PROB>(mw, mx, f, type, launch);
    } else {
      rc = run_products<ENTROPY_PROB>(mx, mw, p, type, launch);
    }
    md.width = piece;
    const auto out = [&](EntropyParams q, void* to, int dest) {
      q.factors = space.factors;
      q.target = target;
      q.target_wide = wide;
      q.ignore = ignore_index;
      q.dest = dest;
      q.out = to;
      q.out_pitch = width;
      q.out_vec = width * size % 16 == 0 && aligned_to(to, 16);
      q.direct = width * size % 32 == 0 && aligned_to(to, 32);
      q.sum = space.sum;
      q.sum_pitch = plan.sum_pitch;
      q.part = space.part;
      q.status = status_dev;
      return q;
    };
    if (dx != nullptr && rc == TRITURUS_B200_OK) {
      const bool begin = i == 0, end = i + 1 == plan.pieces;
      EntropyParams q = out(plan.x[last], dx, begin ? end ? DEST_FINAL : DEST_SUM : end ? DEST_FINAL_ADD : DEST_SUM_ADD);
      q.b_k = static_cast<int>(first);
      if (is_few) {
        FewParams f = few_columns_of(rows, width, piece);
        f.e = q;
        rc = run_few<ENTROPY_OUT_X>(mw, md, f, type, launch);
        if (rc == TRITURUS_B200_OK) rc = sum_few(f, width, type, launch);
      } else {
        rc = set_whole(q) ? run_products<ENTROPY_OUT_X>(md, mw, q, type, launch) : TRITURUS_B200_EINVAL;
      }
    }
    if (dweight != nullptr && rc == TRITURUS_B200_OK) {
      EntropyParams q = out(plan.w[last], static_cast<char*>(dweight) + first * width * size, DEST_FINAL);
      q.boxed = size == 4 && q.out_vec && q.kblocks <= kBoxed;
      rc = set_whole(q) ? run_products<ENTROPY_OUT_W>(md, mx, q, type, launch) : TRITURUS_B200_EINVAL;
    }
  }
  return rc;
}

}  // extern "C"
