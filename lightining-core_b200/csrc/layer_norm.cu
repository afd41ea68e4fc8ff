// Layer norm with weights: forward with the row statistics a backward pass needs, and backward
// with the reduction of the weights' gradients.  (elementwise.cu has the reference's norm without
// weights.)
//
//   h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps),  y = h * gamma + beta
//   w = dy * gamma,  dx = rstd * (w - avg(w) - h * avg(w * h))
//   dgamma = sum over rows of dy * h,  dbeta = sum over rows of dy
//
// Both passes are bound by HBM: 8 and 14 operations for every value moved.  So a row is read once
// and held in registers (as fp32 sums of its own type's values), by one warp while it has at most
// 1024 columns and by up to eight warps (backward) or sixteen (forward) beyond that; every
// statistic, sum and gradient accumulates in fp32 and is rounded once, on the way out.
//
// Weights' gradients: a thread owns the same columns in every row its block walks, so dgamma and
// dbeta accumulate in its registers; a block adds its row groups in shared memory and writes one
// fp32 partial row, and a second kernel adds the blocks' partials in a fixed order -- no atomics, so
// the same call gives the same bits.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "lc_internal.hpp"

namespace lcb {
namespace {

// Loads VEC values of a row as fp32; VEC > 1 is one 16-byte access (the caller checked alignment).
template <typename T, int VEC>
struct Pack;
template <>
struct Pack<float, 1> {
  using Raw = float;
  static __device__ __forceinline__ void get(Raw r, float* f) { f[0] = r; }
  static __device__ __forceinline__ Raw put(const float* f) { return f[0]; }
};
template <>
struct Pack<float, 4> {
  using Raw = float4;
  static __device__ __forceinline__ void get(Raw r, float* f) { f[0] = r.x, f[1] = r.y, f[2] = r.z, f[3] = r.w; }
  static __device__ __forceinline__ Raw put(const float* f) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct Pack<__nv_bfloat16, 1> {
  using Raw = __nv_bfloat16;
  static __device__ __forceinline__ void get(Raw r, float* f) { f[0] = __bfloat162float(r); }
  static __device__ __forceinline__ Raw put(const float* f) { return __float2bfloat16_rn(f[0]); }
};
template <>
struct Pack<__nv_bfloat16, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ void get(Raw r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ Raw put(const float* f) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};

// A weight vector of either type (NULL: the given constant).
struct Weight {
  const void* p;
  int bf16;
  __device__ __forceinline__ float at(size_t c, float none) const {
    if (!p) return none;
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]) : static_cast<const float*>(p)[c];
  }
};
__device__ __forceinline__ void store_weight(void* p, int bf16, size_t c, float v) {
  if (bf16)
    static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(p)[c] = v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ void group_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Sum over the W warps of a row (W == 1: shuffles only).  `buf` is W floats that no one else uses
// until every warp of the group has passed another barrier.
template <int W>
__device__ __forceinline__ float row_sum(float v, float* buf, int warp_in_row, int lane, int bar_id) {
  v = warp_sum(v);
  if (W == 1) return v;
  if (lane == 0) buf[warp_in_row] = v;
  group_sync(bar_id, W * 32);
  float t = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) t += buf[i];
  return t;
}

struct LnFwd {
  const void* x;
  void* out;
  float *mean, *rstd;
  Weight gamma, beta;
  size_t rows, cols, x_stride, out_stride;
  float eps;
};

// One row per W warps, NV packs of VEC columns per lane in registers.
template <typename T, int VEC, int NV, int W>
__global__ void __launch_bounds__(W < 8 ? 256 : W * 32) ln_fwd_kernel(LnFwd a) {
  using P = Pack<T, VEC>;
  constexpr int THREADS = W < 8 ? 256 : W * 32;
  constexpr int GROUPS = THREADS / (W * 32);
  __shared__ float buf[GROUPS][2][W];
  const int lane = threadIdx.x & 31, group = threadIdx.x / (W * 32), wr = (threadIdx.x >> 5) % W;
  const size_t row = static_cast<size_t>(blockIdx.x) * GROUPS + group;
  if (row >= a.rows) return;  // whole groups leave: their barrier is their own
  const typename P::Raw* xr = reinterpret_cast<const typename P::Raw*>(static_cast<const T*>(a.x) + row * a.x_stride);
  typename P::Raw* orow = reinterpret_cast<typename P::Raw*>(static_cast<T*>(a.out) + row * a.out_stride);
  const size_t nvec = a.cols / VEC;
  const size_t t0 = static_cast<size_t>(wr) * 32 + lane;
  const float n = static_cast<float>(a.cols);
  float f[NV][VEC];
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const size_t c = u * (W * 32) + t0;
    if (c < nvec) {
      P::get(xr[c], f[u]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[u][e] = 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += f[u][e];
  const float mean = row_sum<W>(sum, buf[group][0], wr, lane, 1 + group) / n;
  float var = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (u * (W * 32) + t0 < nvec)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        f[u][e] -= mean;
        var = fmaf(f[u][e], f[u][e], var);
      }
  var = row_sum<W>(var, buf[group][1], wr, lane, 1 + group) / n;
  const float rstd = 1.0f / sqrtf(var + a.eps);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const size_t c = u * (W * 32) + t0;
    if (c < nvec) {
      float y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        y[e] = fmaf(f[u][e] * rstd, a.gamma.at(c * VEC + e, 1.0f), a.beta.at(c * VEC + e, 0.0f));
      orow[c] = P::put(y);
    }
  }
  if (wr == 0 && lane == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
}

template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* buf) {
  return row_sum<THREADS / 32>(v, buf, threadIdx.x >> 5, threadIdx.x & 31, 1);
}

// Rows too long for registers: one block streams the row three times (L2 serves the re-reads).
template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(LnFwd a) {
  __shared__ float buf[2][32];
  const size_t row = blockIdx.x;
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride;
  T* orow = static_cast<T*>(a.out) + row * a.out_stride;
  float sum = 0.0f, var = 0.0f, f;
  for (size_t c = threadIdx.x; c < a.cols; c += 1024) {
    Pack<T, 1>::get(xr[c], &f);
    sum += f;
  }
  const float mean = block_sum<1024>(sum, buf[0]) / static_cast<float>(a.cols);
  for (size_t c = threadIdx.x; c < a.cols; c += 1024) {
    Pack<T, 1>::get(xr[c], &f);
    f -= mean;
    var = fmaf(f, f, var);
  }
  var = block_sum<1024>(var, buf[1]) / static_cast<float>(a.cols);
  const float rstd = 1.0f / sqrtf(var + a.eps);
  for (size_t c = threadIdx.x; c < a.cols; c += 1024) {
    Pack<T, 1>::get(xr[c], &f);
    f = fmaf((f - mean) * rstd, a.gamma.at(c, 1.0f), a.beta.at(c, 0.0f));
    orow[c] = Pack<T, 1>::put(&f);
  }
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
}

struct LnBwd {
  const void *dout, *x;
  Weight gamma;
  const float *mean, *rstd;
  void* dx;
  float* part;  // [blocks][2][cols]: dgamma and dbeta partials (NULL: not wanted)
  size_t rows, cols, dout_stride, x_stride, dx_stride;
};

// Walks rows with W warps to a row; 8 / W rows of a block at a time.
template <typename T, int VEC, int NV, int W>
__global__ void __launch_bounds__(256) ln_bwd_kernel(LnBwd a) {
  using P = Pack<T, VEC>;
  constexpr int GROUPS = 8 / W;
  constexpr int OWN = NV * VEC;  // columns per thread
  extern __shared__ float acc[];  // [2][cols], used once at the end
  __shared__ float buf[GROUPS][2][2][W];
  const int lane = threadIdx.x & 31, group = threadIdx.x / (W * 32), wr = (threadIdx.x >> 5) % W;
  const int nvec = static_cast<int>(a.cols / VEC);
  const int t0 = wr * 32 + lane;
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  float dg[OWN], db[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) dg[i] = db[i] = 0.0f;
  int flip = 0;
  for (size_t row = static_cast<size_t>(blockIdx.x) * GROUPS + group; row < a.rows;
       row += static_cast<size_t>(gridDim.x) * GROUPS, flip ^= 1) {
    const typename P::Raw* xr = reinterpret_cast<const typename P::Raw*>(static_cast<const T*>(a.x) + row * a.x_stride);
    const typename P::Raw* gr =
        reinterpret_cast<const typename P::Raw*>(static_cast<const T*>(a.dout) + row * a.dout_stride);
    typename P::Raw xv[NV], gv[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = u * (W * 32) + t0;
      if (c < nvec) {
        xv[u] = xr[c];
        gv[u] = gr[c];
      }
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = u * (W * 32) + t0;
      if (c < nvec) {
        float x[VEC], g[VEC];
        P::get(xv[u], x);
        P::get(gv[u], g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = (x[e] - mean) * rstd;
          dg[u * VEC + e] = fmaf(g[e], h, dg[u * VEC + e]);
          db[u * VEC + e] += g[e];
          const float w = g[e] * a.gamma.at(c * VEC + e, 1.0f);
          s1 += w;
          s2 = fmaf(w, h, s2);
        }
      }
    }
    if (!a.dx) continue;
    // The two sums' buffers alternate from row to row, so one barrier a sum is enough.
    const float m1 = row_sum<W>(s1, buf[group][flip][0], wr, lane, 1 + group) * inv_n;
    const float m2 = row_sum<W>(s2, buf[group][flip][1], wr, lane, 1 + group) * inv_n;
    typename P::Raw* dr = reinterpret_cast<typename P::Raw*>(static_cast<T*>(a.dx) + row * a.dx_stride);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = u * (W * 32) + t0;
      if (c < nvec) {
        float x[VEC], g[VEC];
        P::get(xv[u], x);
        P::get(gv[u], g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = (x[e] - mean) * rstd;
          const float w = g[e] * a.gamma.at(c * VEC + e, 1.0f);
          g[e] = rstd * (w - m1 - h * m2);
        }
        dr[c] = P::put(g);
      }
    }
  }
  griddep_launch_dependents();
  if (!a.part) return;
  // Row groups add up in shared memory, one after the other.
  for (int gI = 0; gI < GROUPS; ++gI) {
    if (group == gI) {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int c = u * (W * 32) + t0;
        if (c < nvec)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float* p = acc + c * VEC + e;
            p[0] = (gI ? p[0] : 0.0f) + dg[u * VEC + e];
            p[a.cols] = (gI ? p[a.cols] : 0.0f) + db[u * VEC + e];
          }
      }
    }
    __syncthreads();
  }
  float* mine = a.part + static_cast<size_t>(blockIdx.x) * 2 * a.cols;
  for (size_t i = threadIdx.x; i < 2 * a.cols; i += 256) mine[i] = acc[i];
}

// Rows too long for registers: dx of one row per block, streamed twice.
template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(LnBwd a) {
  __shared__ float buf[2][32];
  const size_t row = blockIdx.x;
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* gr = static_cast<const T*>(a.dout) + row * a.dout_stride;
  T* dr = static_cast<T*>(a.dx) + row * a.dx_stride;
  const float mean = a.mean[row], rstd = a.rstd[row], inv_n = 1.0f / static_cast<float>(a.cols);
  float s1 = 0.0f, s2 = 0.0f, x, g;
  for (size_t c = threadIdx.x; c < a.cols; c += 1024) {
    Pack<T, 1>::get(xr[c], &x);
    Pack<T, 1>::get(gr[c], &g);
    const float w = g * a.gamma.at(c, 1.0f);
    s1 += w;
    s2 = fmaf(w, (x - mean) * rstd, s2);
  }
  const float m1 = block_sum<1024>(s1, buf[0]) * inv_n;
  const float m2 = block_sum<1024>(s2, buf[1]) * inv_n;
  for (size_t c = threadIdx.x; c < a.cols; c += 1024) {
    Pack<T, 1>::get(xr[c], &x);
    Pack<T, 1>::get(gr[c], &g);
    g = rstd * (g * a.gamma.at(c, 1.0f) - m1 - (x - mean) * rstd * m2);
    dr[c] = Pack<T, 1>::put(&g);
  }
}

// ... and their weights' gradients: a thread owns a column, a block row a slice of the rows.
template <typename T>
__global__ void __launch_bounds__(256) ln_bwd_long_part_kernel(LnBwd a) {
  const size_t c = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= a.cols) return;
  const size_t per = (a.rows + gridDim.y - 1) / gridDim.y;
  const size_t r0 = blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
  float dg = 0.0f, db = 0.0f, x, g;
  for (size_t r = r0; r < r1; ++r) {
    Pack<T, 1>::get(static_cast<const T*>(a.x)[r * a.x_stride + c], &x);
    Pack<T, 1>::get(static_cast<const T*>(a.dout)[r * a.dout_stride + c], &g);
    dg = fmaf(g, (x - a.mean[r]) * a.rstd[r], dg);
    db += g;
  }
  a.part[(static_cast<size_t>(blockIdx.y) * 2) * a.cols + c] = dg;
  a.part[(static_cast<size_t>(blockIdx.y) * 2 + 1) * a.cols + c] = db;
}

// Adds the partial rows: 32 columns by 16 slices of the partials to a block; blockIdx.y picks
// dgamma (0) or dbeta (1).
constexpr int kRedSlices = 16;
__global__ void __launch_bounds__(32 * kRedSlices) ln_reduce_kernel(const float* part, int nparts, size_t cols,
                                                                    void* dgamma, void* dbeta, int bf16) {
  __shared__ float buf[kRedSlices][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const size_t c = static_cast<size_t>(blockIdx.x) * 32 + lane;
  void* out = blockIdx.y == 0 ? dgamma : dbeta;
  griddep_wait();
  float s = 0.0f;
  if (c < cols && out)
    for (int i = slice; i < nparts; i += kRedSlices) s += part[(static_cast<size_t>(i) * 2 + blockIdx.y) * cols + c];
  buf[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && c < cols && out) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kRedSlices; ++i) t += buf[i][lane];
    store_weight(out, bf16, c, t);
  }
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

template <typename T, int VEC, int NV, int W>
cudaError_t run_fwd(const LnFwd& a, cudaStream_t s) {
  constexpr int THREADS = W < 8 ? 256 : W * 32;
  constexpr int GROUPS = THREADS / (W * 32);
  const size_t blocks = (a.rows + GROUPS - 1) / GROUPS;
  if (blocks > 0x7fffffffu) return cudaErrorNotSupported;
  ln_fwd_kernel<T, VEC, NV, W><<<static_cast<unsigned>(blocks), THREADS, 0, s>>>(a);
  return cudaGetLastError();
}

// The smallest register tile that holds the row: 8, 16 or 32 columns a lane of one warp, then more
// warps of 32 columns a lane.
template <typename T, int VEC>
cudaError_t pick_fwd(const LnFwd& a, cudaStream_t s) {
  const size_t c = a.cols;
  if (c <= 256) return run_fwd<T, VEC, 8 / VEC, 1>(a, s);
  if (c <= 512) return run_fwd<T, VEC, 16 / VEC, 1>(a, s);
  if (c <= 1024) return run_fwd<T, VEC, 32 / VEC, 1>(a, s);
  if (c <= 2048) return run_fwd<T, VEC, 32 / VEC, 2>(a, s);
  if (c <= 4096) return run_fwd<T, VEC, 32 / VEC, 4>(a, s);
  if (c <= 8192) return run_fwd<T, VEC, 32 / VEC, 8>(a, s);
  if (c <= 16384) return run_fwd<T, VEC, 32 / VEC, 16>(a, s);
  if (a.rows > 0x7fffffffu) return cudaErrorNotSupported;
  ln_fwd_long_kernel<T><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t ln_fwd(const LnFwd& a, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const bool vec = a.cols % E == 0 && a.x_stride % E == 0 && a.out_stride % E == 0 && aligned(a.x, 16) &&
                   aligned(a.out, 16);
  return vec ? pick_fwd<T, E>(a, s) : pick_fwd<T, 1>(a, s);
}

template <typename T, int VEC, int NV, int W>
cudaError_t run_bwd(const LnBwd& a, int blocks, cudaStream_t s) {
  const size_t smem = a.part ? 2 * a.cols * sizeof(float) : 0;
  if (smem > 48 * 1024) {
    static std::atomic<unsigned long long> attr_done{0};
    const cudaError_t e = once_per_device(attr_done, [&] {
      return cudaFuncSetAttribute(ln_bwd_kernel<T, VEC, NV, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  2 * 8192 * static_cast<int>(sizeof(float)));
    });
    if (e != cudaSuccess) return e;
  }
  ln_bwd_kernel<T, VEC, NV, W><<<blocks, 256, smem, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int VEC>
cudaError_t pick_bwd(const LnBwd& a, int blocks, cudaStream_t s) {
  const size_t c = a.cols;
  if (c <= 256) return run_bwd<T, VEC, 8 / VEC, 1>(a, blocks, s);
  if (c <= 512) return run_bwd<T, VEC, 16 / VEC, 1>(a, blocks, s);
  if (c <= 1024) return run_bwd<T, VEC, 32 / VEC, 1>(a, blocks, s);
  if (c <= 2048) return run_bwd<T, VEC, 32 / VEC, 2>(a, blocks, s);
  if (c <= 4096) return run_bwd<T, VEC, 32 / VEC, 4>(a, blocks, s);
  return run_bwd<T, VEC, 32 / VEC, 8>(a, blocks, s);
}

template <typename T>
cudaError_t ln_bwd(LnBwd a, void* dgamma, void* dbeta, int param_bf16, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const bool grads = dgamma || dbeta;
  const bool in_regs = a.cols <= 8192;
  // Blocks that hold partial rows: two to an SM, no more than there are groups of rows.
  const size_t per_block = in_regs ? (a.cols <= 1024 ? 8 : a.cols <= 2048 ? 4 : a.cols <= 4096 ? 2 : 1) : 64;
  const int blocks = static_cast<int>(
      std::min<size_t>((a.rows + per_block - 1) / per_block, static_cast<size_t>(ctx->sm_count) * 2));
  void* ws = nullptr;
  if (grads) {
    const cudaError_t e = workspace_alloc(ctx, &ws, static_cast<size_t>(blocks) * 2 * a.cols * sizeof(float), s);
    if (e != cudaSuccess) return e;
    a.part = static_cast<float*>(ws);
  }
  cudaError_t e = cudaSuccess;
  if (in_regs) {
    const bool vec = a.cols % E == 0 && a.x_stride % E == 0 && a.dout_stride % E == 0 && aligned(a.x, 16) &&
                     aligned(a.dout, 16) && (!a.dx || (a.dx_stride % E == 0 && aligned(a.dx, 16)));
    e = vec ? pick_bwd<T, E>(a, blocks, s) : pick_bwd<T, 1>(a, blocks, s);
  } else {
    // The partials first: dx may be written over dout or x.
    if (grads) {
      const size_t gx = (a.cols + 255) / 256;
      if (gx > 0x7fffffffu) e = cudaErrorNotSupported;
      if (e == cudaSuccess) {
        ln_bwd_long_part_kernel<T><<<dim3(static_cast<unsigned>(gx), blocks), 256, 0, s>>>(a);
        e = cudaGetLastError();
      }
    }
    if (e == cudaSuccess && a.dx) {
      if (a.rows > 0x7fffffffu) e = cudaErrorNotSupported;
      if (e == cudaSuccess) {
        ln_bwd_long_kernel<T><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
        e = cudaGetLastError();
      }
    }
  }
  if (e == cudaSuccess && grads) {
    const dim3 grid(static_cast<unsigned>((a.cols + 31) / 32), 2);
    if (in_regs) {
      e = launch_pdl(ln_reduce_kernel, grid, dim3(32 * kRedSlices), 0, s, static_cast<const float*>(a.part), blocks,
                     a.cols, dgamma, dbeta, param_bf16);
    } else {
      ln_reduce_kernel<<<grid, 32 * kRedSlices, 0, s>>>(a.part, blocks, a.cols, dgamma, dbeta, param_bf16);
      e = cudaGetLastError();
    }
  }
  const cudaError_t f = workspace_free(ws, s);
  return e != cudaSuccess ? e : f;
}

}  // namespace

cudaError_t layer_norm_forward(const LayerNormArgs& a, cudaStream_t s) {
  LnFwd f{a.x,    a.out,  a.mean,     a.rstd,       {a.gamma, a.param_bf16}, {a.beta, a.param_bf16},
          a.rows, a.cols, a.x_stride, a.out_stride, a.eps};
  return a.bf16 ? ln_fwd<__nv_bfloat16>(f, s) : ln_fwd<float>(f, s);
}

cudaError_t layer_norm_backward(const LayerNormGradArgs& a, cudaStream_t s) {
  LnBwd b{a.dout, a.x,    {a.gamma, a.param_bf16}, a.mean,     a.rstd,     a.dx,
          nullptr, a.rows, a.cols,                  a.dout_stride, a.x_stride, a.dx_stride};
  return a.bf16 ? ln_bwd<__nv_bfloat16>(b, a.dgamma, a.dbeta, a.param_bf16, s)
                : ln_bwd<float>(b, a.dgamma, a.dbeta, a.param_bf16, s);
}

}  // namespace lcb
