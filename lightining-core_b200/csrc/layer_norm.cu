// Layer norm with weights: forward with the row statistics a backward pass needs, and backward
// with the reduction of the weights' gradients.  (elementwise.cu has the reference's norm without
// weights.)
//
//   h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps),  y = h * gamma + beta
//   w = dy * gamma,  dx = rstd * (w - avg(w) - h * avg(w * h))
//   dgamma = sum over rows of dy * h,  dbeta = sum over rows of dy
//
// Both passes are bound by HBM: 8 and 14 operations for every value moved.  So a row is read once
// and held in registers, by as many warps as it has 1024 columns (forward) or 512 (backward), up to 8192
// columns; every statistic, sum and gradient accumulates in fp32 and is rounded once, on the way out.
//
// Weights' gradients: a thread owns the same columns in every row its block walks, so dgamma and
// dbeta accumulate in its registers; a block adds its row groups in shared memory and writes one
// fp32 partial row, and a second kernel adds the blocks' partials in a fixed order -- no atomics, so
// the same call gives the same bits.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "attention_math.cuh"
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
// VEC weights from column c on; VEC > 1: 16-byte aligned (the caller checked).
template <int VEC>
__device__ __forceinline__ void load_weights(const Weight& w, size_t c, float none, float* f) {
  if constexpr (VEC == 1) {
    f[0] = w.at(c, none);
  } else if (!w.p) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = none;
  } else if (w.bf16) {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w.p) + c + e));
      f[e] = __uint_as_float(v.x << 16);
      f[e + 1] = __uint_as_float(v.x & 0xffff0000u);
      f[e + 2] = __uint_as_float(v.y << 16);
      f[e + 3] = __uint_as_float(v.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(w.p) + c + e));
      f[e] = v.x, f[e + 1] = v.y, f[e + 2] = v.z, f[e + 3] = v.w;
    }
  }
}
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

// The backward kernel gives a row to W warps with kBwdOwn columns a lane, several such groups to a block, one block
// to an SM, and lets a group walk rows.  What bounds it is bytes in flight: a group's rows arrive
// through a ring of its own in shared memory, filled by bulk copies several rows ahead, so ~150 KB
// are under way to an SM whatever the registers hold, and the weights of a lane's columns and
// their gradients stay in registers.  A row's stage is read into registers at once and handed to
// the next copy at the row's first barrier.  Measured at [32768, 1024] bf16 (floor 31 us): 94 us
// with a warp to a row, weights re-read and no ring; 54 us with a one-row register prefetch at 8
// columns a lane, bound by issue slots; 45 us so, with 16 columns a lane and packed fp32 pairs.
// A copy starts on a 16-byte boundary: rows that do not are copied from the boundary before them to
// the one after them (never into another page; with dx over x or dout the bytes of a neighbouring row may be
// written meanwhile, and are not used) and read from there with scalar accesses: [5003, 1333] fp32 27 us (floor 12).
constexpr int kFwdOwn = 32, kBwdOwn = 16;     // columns a lane
constexpr int kBwdWarps = 16;                 // of a block
constexpr int kMaxCols = 8192;                // 16 warps to a row (backward)
constexpr int kMaxStages = 8;
constexpr size_t kRingBytes = 192 * 1024;

struct Rows {
  int warps;   // per row
  int groups;  // rows per block
  int stages;  // of a group's ring
  int pitch;   // bytes from one staged row to the next
};

// The ring of a row group, for NB tensors.  Rows are taken in turn: stage and phase, the row that the
// leader copies next and the shared-memory address of the row to read are stepped, not computed.
template <int NB, bool ALIGNED>
struct Ring {
  uint8_t* mem;
  uint64_t* full;
  int stages, pitch, cols_bytes;
  unsigned* err;
  volatile int* abort_flag;
  const uint8_t* next[NB];  // the next row to copy
  size_t hop[NB];           // bytes from a group's row to its next one
  size_t left;              // rows still to copy
  int s;                    // stage of the current row, and its phase
  uint32_t phase, lead[NB], lead_hop[NB];

  // One thread: the next row of the tensors into stage `to`.
  __device__ void load(int to) {
    uint32_t bytes[NB], total = 0;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t l = ALIGNED ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(next[i]) & 15u);
      bytes[i] = (l + cols_bytes + 15u) & ~15u;
      total += bytes[i];
    }
    mbar_arrive_expect_tx(&full[to], total);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t l = ALIGNED ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(next[i]) & 15u);
      bulk_load(mem + (to * NB + i) * pitch, next[i] - l, bytes[i], &full[to]);
      next[i] += hop[i];
    }
    --left;
  }
  // Every lane: waits for the current row; gives up after the common limit and records it (the row
  // is then wrong, the barriers of the group still meet).
  __device__ bool wait() { return warp_wait_poll(&full[s], phase, abort_flag, err, kErrNormLoadWait); }
  // The leader, when a wait has failed: the last copies land (0.1 s at most) before the block's sums take the ring's
  // place or the block ends.  `rows`: all of the group's.
  __device__ void drain(size_t rows) const {
    const uint64_t t0 = globaltimer_ns();
    const size_t issued = rows - left, n = stages;
    for (size_t k = issued > n ? issued - n : 0; k < issued; ++k)
      while (!mbar_try_wait(&full[k % n], (k / n) & 1) && globaltimer_ns() - t0 < 100000000ull) {
      }
  }
  __device__ const uint8_t* row(int i) const { return mem + (s * NB + i) * pitch + (ALIGNED ? 0u : lead[i]); }
  __device__ void step() {
    if (++s == stages) s = 0, phase ^= 1u;
    if (!ALIGNED)
#pragma unroll
      for (int i = 0; i < NB; ++i) lead[i] = (lead[i] + lead_hop[i]) & 15u;
  }
};

// A lane's columns of a staged row, as fp32 pairs; columns past the end are 0.
template <typename T, int VEC, bool FULL, int kOwn>
__device__ __forceinline__ void read_own(uint64_t (&v)[kOwn / 2], const uint8_t* row, int t, int step, int nvec) {
  const typename Pack<T, VEC>::Raw* r = reinterpret_cast<const typename Pack<T, VEC>::Raw*>(row);
  float f[kOwn];
#pragma unroll
  for (int u = 0; u < kOwn / VEC; ++u) {
    if (FULL || u * step + t < nvec) {
      Pack<T, VEC>::get(r[u * step + t], f + u * VEC);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[u * VEC + e] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kOwn / 2; ++i) v[i] = pk2(f[2 * i], f[2 * i + 1]);
}

template <typename T, int VEC, bool FULL, int kOwn>
__device__ __forceinline__ void write_own(T* row, const uint64_t (&v)[kOwn / 2], int t, int step, int nvec) {
  typename Pack<T, VEC>::Raw* r = reinterpret_cast<typename Pack<T, VEC>::Raw*>(row);
  float f[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn / 2; ++i) unpk2(v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int u = 0; u < kOwn / VEC; ++u)
    if (FULL || u * step + t < nvec) __stcs(r + u * step + t, Pack<T, VEC>::put(f + u * VEC));
}

__device__ __forceinline__ float pair_sum(const uint64_t (&v)[4]) {
  float a, b;
  unpk2(add2(add2(v[0], v[1]), add2(v[2], v[3])), a, b);
  return a + b;
}

// Adds a value over the W warps of a row; `buf` holds W of them and is not used
// again before another barrier of the group.
__device__ __forceinline__ float group_sum(float v, float* buf, int W, int wr, int lane, int bar) {
  v = warp_sum(v);
  if (W == 1) return v;
  if (lane == 0) buf[wr] = v;
  group_sync(bar, W * 32);
  v = 0.0f;
  for (int w = 0; w < W; ++w) v += buf[w];
  return v;
}

struct LnFwd {
  const void* x;
  void* out;
  float *mean, *rstd;
  Weight gamma, beta;
  size_t rows, cols, x_stride, out_stride;
  float eps;
};

struct NormTail {
  uint64_t full[kBwdWarps * kMaxStages];
  float2 sums[2][kBwdWarps];
  int abort_flag;
};

// Barriers of a block's rings and the first rows' copies (one thread to a group).
template <int NB, bool ALIGNED>
__device__ __forceinline__ Ring<NB, ALIGNED> open_ring(NormTail& tail, uint8_t* mem, const Rows& rw, int group, int es,
                                                       size_t cols, unsigned* err, const void* const (&base)[NB],
                                                       const size_t (&stride)[NB], size_t row, size_t rows, size_t hop,
                                                       bool leader) {
  Ring<NB, ALIGNED> ring;
  ring.mem = mem + static_cast<size_t>(group) * rw.stages * NB * rw.pitch;
  ring.full = tail.full + group * rw.stages;
  ring.stages = rw.stages;
  ring.pitch = rw.pitch;
  ring.cols_bytes = static_cast<int>(cols) * es;
  ring.err = err;
  ring.abort_flag = &tail.abort_flag;
  ring.left = row < rows ? (rows - row + hop - 1) / hop : 0;
  ring.s = 0;
  ring.phase = 0;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    ring.next[i] = static_cast<const uint8_t*>(base[i]) + row * stride[i] * es;
    ring.hop[i] = hop * stride[i] * es;
    ring.lead[i] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring.next[i]) & 15u);
    ring.lead_hop[i] = static_cast<uint32_t>(ring.hop[i] & 15u);
  }
  if (threadIdx.x == 0) tail.abort_flag = 0;
  if (leader)
    for (int s = 0; s < rw.stages; ++s) mbar_init(&ring.full[s], 1);
  fence_barrier_init();
  __syncthreads();
  if (leader)
    for (int s = 0; s < rw.stages && ring.left; ++s) ring.load(s);
  return ring;
}

// Forward: one row to W warps and done, so that blocks are dealt out as SMs get free.  (Rows walked by
// resident blocks through the backward kernel's rings took 98 us at [65536, 1024] fp32 where this takes
// 83 and a plain copy 84: the SMs do not see memory equally fast, and a fixed share of the rows each waits
// for the slowest.)
template <typename T, int VEC>
__global__ void __launch_bounds__(512) ln_fwd_kernel(LnFwd a, int W) {
  using P = Pack<T, VEC>;
  constexpr int NV = kFwdOwn / VEC;
  __shared__ float sums[2][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / W, wr = warp % W, step = W * 32, t = wr * 32 + lane;
  const size_t row = static_cast<size_t>(blockIdx.x) * (blockDim.x / step) + group;
  if (row >= a.rows) return;  // whole groups leave: their barrier is their own
  const int nvec = static_cast<int>(a.cols) / VEC;
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  const typename P::Raw* x = reinterpret_cast<const typename P::Raw*>(static_cast<const T*>(a.x) + row * a.x_stride) + t;
  typename P::Raw v[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (u * step + t < nvec) v[u] = __ldcs(x + u * step);
  float f[kFwdOwn], sum = 0.0f, sq = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    float* g = f + u * VEC;
    if (u * step + t < nvec) {
      P::get(v[u], g);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[e] = 0.0f;
    }
    float part = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) part += g[e];
    sum += part;
  }
  const float mean = group_sum(sum, sums[0] + group * W, W, wr, lane, 1 + group) * inv_n;
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (u * step + t < nvec) {
      float part = 0.0f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        f[u * VEC + e] -= mean;
        part = fmaf(f[u * VEC + e], f[u * VEC + e], part);
      }
      sq += part;
    }
  const float var = group_sum(sq, sums[1] + group * W, W, wr, lane, 1 + group) * inv_n;
  const float rstd = 1.0f / sqrtf(var + a.eps);
  typename P::Raw* out = reinterpret_cast<typename P::Raw*>(static_cast<T*>(a.out) + row * a.out_stride) + t;
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (u * step + t < nvec) {
      float g[VEC], b[VEC];
      load_weights<VEC>(a.gamma, static_cast<size_t>(u * step + t) * VEC, 1.0f, g);
      load_weights<VEC>(a.beta, static_cast<size_t>(u * step + t) * VEC, 0.0f, b);
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[e] = fmaf(f[u * VEC + e] * rstd, g[e], b[e]);
      __stcs(out + u * step, P::put(g));
    }
  if (t == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
}

// Sum over a block's warps; `buf` is a float for each that nothing else uses.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* buf) {
  return group_sum(v, buf, THREADS / 32, threadIdx.x >> 5, threadIdx.x & 31, 1);
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
  unsigned* err;
};

template <typename T, int VEC, bool FULL>
__global__ void __launch_bounds__(kBwdWarps * 32, 1) ln_bwd_kernel(LnBwd a, Rows rw) {
  constexpr int kOwn = kBwdOwn;
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ NormTail tail;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = rw.warps;
  const int group = warp / W, wr = warp % W, step = W * 32, t = wr * 32 + lane;
  const int nvec = static_cast<int>(a.cols) / VEC;
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  const size_t hop = static_cast<size_t>(gridDim.x) * rw.groups;
  size_t row = static_cast<size_t>(blockIdx.x) * rw.groups + group;
  const void* const base[2] = {a.x, a.dout};
  const size_t stride[2] = {a.x_stride, a.dout_stride};
  auto ring = open_ring<2, (VEC > 1)>(tail, ring_mem, rw, group, sizeof(T), a.cols, a.err, base, stride, row, a.rows, hop, t == 0);
  uint64_t gm[kOwn / 2], dg[kOwn / 2], db[kOwn / 2];
#pragma unroll
  for (int k = 0; k < kOwn; k += 2) {
    const auto one = [&](int j) {
      const int c = (j / VEC) * step + t;
      return c < nvec ? a.gamma.at(static_cast<size_t>(c) * VEC + j % VEC, 1.0f) : 0.0f;
    };
    gm[k / 2] = pk2(one(k), one(k + 1));
    dg[k / 2] = db[k / 2] = 0;
  }
  const float *mp = a.mean + row, *rp = a.rstd + row;
  float mean = 0.0f, rstd = 0.0f;
  if (row < a.rows) mean = *mp, rstd = *rp;
  bool ok = true;
  T* dx = static_cast<T*>(a.dx) + row * a.dx_stride;
  float2* sums = tail.sums[0] + group * W;  // alternates between the two sets
  int other = kBwdWarps;
  for (; row < a.rows; row += hop, dx += hop * a.dx_stride, sums += other, other = -other, ring.step()) {
    const float r = rstd;
    const uint64_t r2 = pk2(r, r), nm = pk2(-mean, -mean);
    if (row + hop < a.rows) mean = *(mp += hop), rstd = *(rp += hop);
    ok = ring.wait() && ok;
    uint64_t h[kOwn / 2], w[kOwn / 2], p1[4] = {0, 0, 0, 0}, p2[4] = {0, 0, 0, 0};
    read_own<T, VEC, FULL, kOwn>(h, ring.row(0), t, step, nvec);
    read_own<T, VEC, FULL, kOwn>(w, ring.row(1), t, step, nvec);
    // (Columns past the end have w = 0, and what h is there enters no sum.)
#pragma unroll
    for (int k = 0; k < kOwn / 2; ++k) {
      h[k] = mul2(add2(h[k], nm), r2);  // (the difference first: a row's offset cancels exactly)
      dg[k] = fma2(w[k], h[k], dg[k]);
      db[k] = add2(db[k], w[k]);
      w[k] = mul2(w[k], gm[k]);
      p1[k & 3] = add2(p1[k & 3], w[k]);
      p2[k & 3] = fma2(w[k], h[k], p2[k & 3]);
    }
    float s1 = warp_sum(pair_sum(p1)), s2 = warp_sum(pair_sum(p2));
    if (W > 1) {
      if (lane == 0) sums[wr] = make_float2(s1, s2);
      group_sync(1 + group, W * 32);
      float2 v = sums[0];
      s1 = v.x, s2 = v.y;
      for (int j = 1; j < W; ++j) {
        v = sums[j];
        s1 += v.x;
        s2 += v.y;
      }
    } else {
      __syncwarp();
    }
    // Every warp of the group has read the stage: it takes the row `stages` ahead.
    if (t == 0 && ok && ring.left) ring.load(ring.s);
    if (!a.dx) continue;
    const uint64_t c1 = pk2(-r * s1 * inv_n, -r * s1 * inv_n), c2 = pk2(-r * s2 * inv_n, -r * s2 * inv_n);
#pragma unroll
    for (int k = 0; k < kOwn / 2; ++k) w[k] = fma2(h[k], c2, fma2(w[k], r2, c1));
    write_own<T, VEC, FULL, kOwn>(dx, w, t, step, nvec);
  }
  if (!ok && t == 0) {  // (rows from this group's first one on)
    const size_t first = static_cast<size_t>(blockIdx.x) * rw.groups + group;
    ring.drain((a.rows - first + hop - 1) / hop);
  }
  griddep_launch_dependents();
  if (!a.part) return;
  // Every group puts its sums beside the others' over the rings (every copy has landed), then the block
  // adds them column by column.
  float* acc = reinterpret_cast<float*>(ring_mem);  // [groups][2][cols]
  __syncthreads();
  {
    float g[kOwn], d[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn / 2; ++k) {
      unpk2(dg[k], g[2 * k], g[2 * k + 1]);
      unpk2(db[k], d[2 * k], d[2 * k + 1]);
    }
    float* mine = acc + static_cast<size_t>(group) * 2 * a.cols;
#pragma unroll
    for (int u = 0; u < kOwn / VEC; ++u)
      if (u * step + t < nvec) {
        constexpr int V = VEC < 4 ? 1 : 4;  // (with VEC > 1 the columns are whole float4s)
#pragma unroll
        for (int e = 0; e < VEC; e += V) {
          float* p = mine + (u * step + t) * VEC + e;
          if constexpr (V == 4) {
            *reinterpret_cast<float4*>(p) =
                make_float4(g[u * VEC + e], g[u * VEC + e + 1], g[u * VEC + e + 2], g[u * VEC + e + 3]);
            *reinterpret_cast<float4*>(p + a.cols) =
                make_float4(d[u * VEC + e], d[u * VEC + e + 1], d[u * VEC + e + 2], d[u * VEC + e + 3]);
          } else {
            p[0] = g[u * VEC + e];
            p[a.cols] = d[u * VEC + e];
          }
        }
      }
  }
  __syncthreads();
  float* out = a.part + static_cast<size_t>(blockIdx.x) * 2 * a.cols;
  for (size_t i = threadIdx.x; i < 2 * a.cols; i += blockDim.x) {
    float v = acc[i];
    for (int g = 1; g < rw.groups; ++g) v += acc[g * 2 * a.cols + i];
    out[i] = v;
  }
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

// Adds the partial rows: 32 columns by 32 slices of the partials to a block; blockIdx.y picks
// dgamma (0) or dbeta (1).
constexpr int kRedSlices = 32;
__global__ void __launch_bounds__(32 * kRedSlices) ln_reduce_kernel(const float* part, int nparts, size_t cols,
                                                                    void* dgamma, void* dbeta, int bf16) {
  __shared__ float buf[kRedSlices][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const size_t c = static_cast<size_t>(blockIdx.x) * 32 + lane;
  void* out = blockIdx.y == 0 ? dgamma : dbeta;
  griddep_wait();
  float s = 0.0f;
  if (c < cols && out)
#pragma unroll 8
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

// The split of the backward pass over a block: as many rows to a block as 16 warps hold, but no more than spread
// the rows over all SMs; rings of up to 8 rows of x and dout.
Rows rows_of(size_t rows, size_t cols, int es, int sms) {
  Rows r;
  r.warps = static_cast<int>((cols + 32 * kBwdOwn - 1) / (32 * kBwdOwn));
  r.groups = static_cast<int>(std::min<size_t>(kBwdWarps / r.warps, (rows + sms - 1) / sms));
  r.pitch = static_cast<int>((cols * es + 30 + 15) / 16 * 16);
  const size_t row_bytes = static_cast<size_t>(r.pitch) * 2 * r.groups;
  r.stages = static_cast<int>(std::min<size_t>(kMaxStages, kRingBytes / row_bytes));
  return r;
}

template <class Kernel>
cudaError_t allow_ring(std::atomic<unsigned long long>& done, Kernel k) {
  return once_per_device(done, [&] {
    return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kRingBytes));
  });
}

template <typename T>
cudaError_t ln_fwd(const LnFwd& a, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  if (a.rows > 0x7fffffffu) return cudaErrorNotSupported;
  if (a.cols > static_cast<size_t>(kMaxCols)) {
    ln_fwd_long_kernel<T><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
    return cudaGetLastError();
  }
  const bool vec = a.cols % E == 0 && a.x_stride % E == 0 && a.out_stride % E == 0 && aligned(a.x, 16) &&
                   aligned(a.out, 16) && aligned(a.gamma.p, 16) && aligned(a.beta.p, 16);
  const int warps = static_cast<int>((a.cols + 32 * kFwdOwn - 1) / (32 * kFwdOwn));
  const int groups = std::max(1, 8 / warps);
  const unsigned blocks = static_cast<unsigned>((a.rows + groups - 1) / groups);
  if (vec)
    ln_fwd_kernel<T, E><<<blocks, warps * groups * 32, 0, s>>>(a, warps);
  else
    ln_fwd_kernel<T, 1><<<blocks, warps * groups * 32, 0, s>>>(a, warps);
  return cudaGetLastError();
}

template <typename T, int VEC, bool FULL = false>
cudaError_t run_bwd(const LnBwd& a, const Rows& rw, int blocks, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_ring(done, ln_bwd_kernel<T, VEC, FULL>);
  if (e != cudaSuccess) return e;
  // The groups' sums come together over the rings.
  const size_t ring = rw.groups * std::max(static_cast<size_t>(rw.stages) * 2 * rw.pitch, 2 * a.cols * sizeof(float));
  ln_bwd_kernel<T, VEC, FULL><<<blocks, rw.warps * rw.groups * 32, ring, s>>>(a, rw);
  return cudaGetLastError();
}

template <typename T>
cudaError_t ln_bwd(LnBwd a, void* dgamma, void* dbeta, int param_bf16, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const bool grads = dgamma || dbeta;
  a.err = ctx->err_word;
  const bool in_regs = a.cols <= static_cast<size_t>(kMaxCols);
  Rows rw{};
  if (in_regs) rw = rows_of(a.rows, a.cols, sizeof(T), ctx->sm_count);
  // Blocks, each with a partial row of sums.
  const size_t per_block = in_regs ? rw.groups : 64;
  const int blocks = static_cast<int>(
      std::min<size_t>((a.rows + per_block - 1) / per_block, static_cast<size_t>(ctx->sm_count)));
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
    const bool full = a.cols == static_cast<size_t>(rw.warps) * 32 * kBwdOwn;  // no lane runs past the row: 45 us at [32768, 1024] bf16, 49 with the checks
    e = vec ? full ? run_bwd<T, E, true>(a, rw, blocks, s) : run_bwd<T, E>(a, rw, blocks, s)
            : run_bwd<T, 1>(a, rw, blocks, s);
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
          nullptr, a.rows, a.cols,                  a.dout_stride, a.x_stride, a.dx_stride,
          nullptr};
  return a.bf16 ? ln_bwd<__nv_bfloat16>(b, a.dgamma, a.dbeta, a.param_bf16, s)
                : ln_bwd<float>(b, a.dgamma, a.dbeta, a.param_bf16, s);
}

}  // namespace lcb
