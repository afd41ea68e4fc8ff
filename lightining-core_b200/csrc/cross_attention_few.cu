// Cross attention of a few query rows in bf16 (single tokens with the heads that share a key head): head_dim 64
// or 128, at most 16 rows to a (batch, key head) pair.
//
// K and V are read once, 2 * head_dim * 2 bytes a key against 16 * 4 * head_dim operations, so HBM bounds it and
// what matters is bytes in flight: tiles of 64 keys arrive by TMA in a ring of 96 KB, two blocks to an SM, and four
// warps take 16 keys of each with the 16 x 8 x 16 matrix instruction:
//   S = Q K^T   the order of the columns inside a dot product is free, so lane c of a quad takes the 8
//               contiguous values 8c.. of every 32 as its share of two k-steps, of Q alike: 16-byte reads of K
//               as it lies
//   O += P V    lane (g, c) reads keys 2c, 2c+1, 2c+8, 2c+9 at columns 8g..8g+7 and pairs keys with byte
//               permutes; n-tile u then holds the columns 8g + u
// P enters the product as the sum of two bf16 numbers (what rounding the first leaves goes into a second
// product), so no precision is lost to it; scores, statistics and sums are fp32.
// A block's four warps take 64 keys in turn and join their (maximum, sum, O) in shared memory; the keys of a
// pair are split over a cluster of up to 8 blocks, which join theirs through distributed shared memory -- one
// launch, no workspace -- and over several clusters (and cross_combine) only when pairs are very few.
// B200, 64 sequences of 32 / 8 heads over 2048..4096 keys, head_dim 128 (811 MB, floor 126 us): loads straight
// into registers, three blocks to an SM, 226 us; the tiled tensor-core kernel 202 us (two stages of 64 KB do not cover
// the latency); this one 142 us (with 4 blocks to a pair instead of 2: 154, with 8: 195).
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "cross_attention.cuh"
#include "lc_internal.hpp"

namespace cg = cooperative_groups;

namespace lcb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int WARPS = 4, KEYS = 16 * WARPS;  // keys of a block's step
constexpr int ROWS = 16;
constexpr int BOX = KEYS * 128;  // [64 keys x 64 bf16], 128-byte swizzle
constexpr int THREADS = (WARPS + 1) * 32;

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

template <int D>
struct FewSmem {
  float o[WARPS][ROWS][D + 4];  // per warp; [0] ends as the block's sum
  float m[WARPS][ROWS], l[WARPS][ROWS];
  float bm[ROWS], bl[ROWS];     // the block's
};
template <int D>
struct FewRing {
  static constexpr int NW = D / 64, STAGE = 2 * NW * BOX, NS = 96 * 1024 / STAGE;
  static_assert(sizeof(FewSmem<D>) <= NS * STAGE, "the sums lie over the ring");
};
struct FewBars {
  uint64_t full[6], free_[6];
  int abort_flag;
};

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
    cross_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, CrossArgs a,
                     CrossSplit sp, int cluster, KvAxes ax, unsigned* err) {
  constexpr int NB = D / 32, NW = D / 64, NS = FewRing<D>::NS, STAGE = FewRing<D>::STAGE;
  extern __shared__ __align__(1024) uint8_t ring[];
  __shared__ FewBars bars;
  FewSmem<D>& sm = *reinterpret_cast<FewSmem<D>*>(ring);
  if ((smem_u32(ring) & 1023u) != 0) {  // the 128-byte swizzle atoms need 1 KB alignment
    if (threadIdx.x == 0) atomicCAS(err, 0u, static_cast<unsigned>(kErrCrossLoadWait) | 0x1000u);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int group = a.hq / a.hk, rows = group * a.q_len;
  const int rank = static_cast<int>(blockIdx.x) % cluster;
  const int pair = static_cast<int>(blockIdx.x) / cluster, b = pair / a.hk, hk = pair % a.hk;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  const auto live = [&](int r) { return r < rows && r % a.q_len < q_end; };
  // This block's keys: its share of this outer split's share, whole steps.
  const int steps = (kv_end + KEYS - 1) / KEYS;
  const int parts = cluster * sp.splits, part = static_cast<int>(blockIdx.y) * cluster + rank;
  const int per = (steps + parts - 1) / parts;
  const int t_lo = min(steps, part * per), n = min(steps, (part + 1) * per) - t_lo;  // tiles
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.free_[i], WARPS);
    }
    bars.abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncthreads();
  volatile int* abort_flag = &bars.abort_flag;
  float o[NW * 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  if (warp == WARPS) {
    if (lane == 0) {
      bool ok = true;
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % NS;
        if (i >= NS && !mbar_wait_bounded(&bars.free_[s], (i / NS - 1) & 1, abort_flag, err, kErrCrossLoadWait)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&bars.full[s], STAGE);
        for (int w = 0; w < NW; ++w) {
          tma_load_4d(ring + s * STAGE + w * BOX, &map_k, w * 64, (t_lo + i) * KEYS, ax.k_head ? hk : 0,
                      ax.k_batch ? b : 0, &bars.full[s]);
          tma_load_4d(ring + s * STAGE + (NW + w) * BOX, &map_v, w * 64, (t_lo + i) * KEYS, ax.v_head ? hk : 0,
                      ax.v_batch ? b : 0, &bars.full[s]);
        }
      }
      // Every copy has landed before the sums take the ring's place, whatever became of its readers.
      const uint64_t t0 = globaltimer_ns();
      for (int k = max(0, i - NS); !ok && k < i; ++k)
        while (!mbar_try_wait(&bars.full[k % NS], (k / NS) & 1) && globaltimer_ns() - t0 < 100000000ull) {
        }
    }
  } else {
  // Q fragments: rows g and g + 8, the 8 values 8c.. of every 32.
  uint4 q[NB][2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = g + 8 * r;
    const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) + b * a.qs.b +
                               (hk * group + row / a.q_len) * a.qs.h + row % a.q_len * a.qs.t + c * 8;
#pragma unroll
    for (int n = 0; n < NB; ++n) q[n][r] = live(row) ? __ldg(reinterpret_cast<const uint4*>(src + n * 32)) : make_uint4(0, 0, 0, 0);
  }
  const float sc = a.scale * kLog2e;
  const auto seen = [&](int key) { return key < kv_end && (!mask || mask[key]); };
  // Piece k of 16 bytes of this warp's key r in a box.
  const auto piece = [&](const uint8_t* box, int r, int k) {
    return *reinterpret_cast<const uint4*>(box + (warp * 16 + r) * 128 + ((k ^ (r & 7)) << 4));
  };
#pragma unroll
  for (int n8 = 0; n8 < NW * 8; ++n8) o[n8][0] = o[n8][1] = o[n8][2] = o[n8][3] = 0.0f;
  for (int i = 0; i < n; ++i) {
    const int st = i % NS, k0 = (t_lo + i) * KEYS + warp * 16;
    // The mask bytes of a step are asked for before the wait for its keys.
    bool vis[2][2] = {{true, true}, {true, true}}, vis_v[4] = {true, true, true, true};
    const bool partial = mask || k0 + 16 > kv_end;
    if (partial) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) vis_v[t * 2 + e] = vis[t][e] = seen(k0 + t * 8 + 2 * c + e);
    }
    if (!warp_wait_poll(&bars.full[st], (i / NS) & 1, abort_flag, err, kErrCrossSoftmaxWait)) break;
    const uint8_t *kbox = ring + st * STAGE, *vbox = kbox + NW * BOX;
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
      for (int n32 = 0; n32 < NB; ++n32) {
        const uint4 k = piece(kbox + (n32 >> 1) * BOX, t * 8 + g, (n32 & 1) * 4 + c);
        mma16816(s[t], q[n32][0].x, q[n32][1].x, q[n32][0].y, q[n32][1].y, k.x, k.y);
        mma16816(s[t], q[n32][0].z, q[n32][1].z, q[n32][0].w, q[n32][1].w, k.z, k.w);
      }
    }
    if (partial)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (!vis[t][e]) s[t][e] = s[t][2 + e] = -INFINITY;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float top = quad_max(fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]))) * sc;
      const float mx = fmaxf(m[r], top), base = mx == -INFINITY ? 0.0f : mx;
      const float keep = exp2f(m[r] - base);
      m[r] = mx;
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float p0 = exp2f(fmaf(s[t][2 * r], sc, -base)), p1 = exp2f(fmaf(s[t][2 * r + 1], sc, -base));
        sum += p0 + p1;
        const uint32_t h = pack_bf16x2(p0, p1);
        hi[t * 2 + r] = h;
        lo[t * 2 + r] = pack_bf16x2(p0 - __uint_as_float(h << 16), p1 - __uint_as_float(h & 0xffff0000u));
      }
      l[r] = fmaf(l[r], keep, sum);
      if (__any_sync(0xffffffffu, keep != 1.0f))
#pragma unroll
        for (int n8 = 0; n8 < NW * 8; ++n8) {
          o[n8][2 * r] *= keep;
          o[n8][2 * r + 1] *= keep;
        }
    }
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      uint4 vf[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        vf[k] = piece(vbox + w * BOX, 2 * c + (k & 1) + (k >> 1) * 8, g);
        // A masked value would enter the sum: a weight of 0 does not hide a NaN.
        if (partial && !vis_v[k]) vf[k] = make_uint4(0, 0, 0, 0);
      }
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vf[0]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vf[1]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vf[2]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vf[3]);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t sel = (u & 1) ? 0x7632 : 0x5410;
        const uint32_t b0 = __byte_perm(v0[u >> 1], v1[u >> 1], sel), b1 = __byte_perm(v2[u >> 1], v3[u >> 1], sel);
        mma16816(o[w * 8 + u], hi[0], hi[1], hi[2], hi[3], b0, b1);
        mma16816(o[w * 8 + u], lo[0], lo[1], lo[2], lo[3], b0, b1);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.free_[st]);
  }
  }

  // The block's sums, over the ring (all its copies have landed and been read): every warp scales its own to the
  // common maximum.
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] = quad_sum(l[r]);
    if (c == 0 && warp < WARPS) {
      sm.m[warp][g + 8 * r] = m[r];
      sm.l[warp][g + 8 * r] = l[r];
    }
  }
  __syncthreads();
  if (warp < WARPS)
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = g + 8 * r;
    float mx = sm.m[0][row];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) mx = fmaxf(mx, sm.m[w][row]);
    const float f = exp2f(m[r] - (mx == -INFINITY ? 0.0f : mx));
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v[8];  // columns 64 w + 8 (2c + e) + u
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = o[w * 8 + u][2 * r + e] * f;
        float4* dst = reinterpret_cast<float4*>(&sm.o[warp][row][w * 64 + (2 * c + e) * 8]);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    if (warp == 0 && c == 0) {
      const float base = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) sum = fmaf(sm.l[w][row], exp2f(sm.m[w][row] - base), sum);
      sm.bm[row] = mx;
      sm.bl[row] = sum;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += THREADS) {
    const int row = i / (D / 4), col = i % (D / 4) * 4;
    float4 t = *reinterpret_cast<float4*>(&sm.o[0][row][col]);
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
      const float4 v = *reinterpret_cast<float4*>(&sm.o[w][row][col]);
      t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
    *reinterpret_cast<float4*>(&sm.o[0][row][col]) = t;
  }
  cg::cluster_group cl = cg::this_cluster();
  if (cluster > 1)
    cl.sync();
  else
    __syncthreads();
  // The cluster's: a block takes rows rank, rank + cluster, ...; a warp half a row's columns at a time.
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += THREADS) {
    const int row = i / (D / 4), col = i % (D / 4) * 4;
    if (row % cluster != rank || !live(row)) continue;
    float mx = -INFINITY;
    for (int n = 0; n < cluster; ++n) mx = fmaxf(mx, *(cluster > 1 ? cl.map_shared_rank(&sm.bm[row], n) : &sm.bm[row]));
    const float base = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int n = 0; n < cluster; ++n) {
      const float bm = *(cluster > 1 ? cl.map_shared_rank(&sm.bm[row], n) : &sm.bm[row]);
      const float f = exp2f(bm - base);
      sum = fmaf(*(cluster > 1 ? cl.map_shared_rank(&sm.bl[row], n) : &sm.bl[row]), f, sum);
      const float4 v = *reinterpret_cast<const float4*>(cluster > 1 ? cl.map_shared_rank(&sm.o[0][row][col], n) : &sm.o[0][row][col]);
      t.x = fmaf(v.x, f, t.x), t.y = fmaf(v.y, f, t.y), t.z = fmaf(v.z, f, t.z), t.w = fmaf(v.w, f, t.w);
    }
    const int h = hk * group + row / a.q_len, tok = row % a.q_len;
    const long long at = (static_cast<long long>(b) * a.hq + h) * a.q_len + tok;  // dense row
    if (sp.splits > 1) {
      const long long part_row = static_cast<long long>(blockIdx.y) * sp.rows + at;
      *reinterpret_cast<float4*>(sp.o + part_row * a.d + col) = t;
      if (col == 0) sp.ml[part_row] = make_float2(mx, sum);
      continue;
    }
    const float inv = mx == -INFINITY ? 0.0f : 1.0f / sum;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + b * a.os.b + h * a.os.h + tok * a.os.t + col;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(t.x * inv, t.y * inv), pack_bf16x2(t.z * inv, t.w * inv));
    if (col == 0 && a.lse) a.lse[at] = mx == -INFINITY ? -INFINITY : (mx + log2f(sum)) * kLn2;
  }
  if (cluster > 1) cl.sync();  // no block leaves while another reads its sums
}

template <int D>
cudaError_t run_few(const CrossArgs& a, cudaStream_t s) {
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const long long pairs = static_cast<long long>(a.batch) * a.hk, steps = (a.kv_len + KEYS - 1) / KEYS;
  const long long slots = 2LL * ctx->sm_count;
  // Blocks to a pair: enough to fill the SMs twice (the lengths differ, and a block that ends makes room for the
  // next; every block has a fill and a drain of its own to pay), at least one step of keys each.
  int cluster = 1;
  while (cluster < 8 && pairs * cluster < 2 * slots && 2 * cluster <= steps) cluster *= 2;
  if (pairs * cluster > 0x7fffffffLL) return cudaErrorNotSupported;
  CUtensorMap mk, mv;
  KvAxes ax;
  if (!cross_kv_maps(a, KEYS, &mk, &mv, &ax)) return cudaErrorInvalidValue;
  constexpr size_t SMEM = static_cast<size_t>(FewRing<D>::NS) * FewRing<D>::STAGE;
  static std::atomic<unsigned long long> attr_done{0};
  const cudaError_t ea = once_per_device(attr_done, [] {
    return cudaFuncSetAttribute(cross_few_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  });
  if (ea != cudaSuccess) return ea;
  CrossSplitWork w;
  // Very few pairs over very many keys: several clusters, at least eight steps to a block.
  cudaError_t e = w.begin_parts(a, std::min<long long>({slots / (pairs * cluster), steps / (8 * cluster), 64}), s);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs * cluster), w.sp.splits);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return w.end(a, cudaLaunchKernelEx(&cfg, cross_few_kernel<D>, mk, mv, a, w.sp, cluster, ax, ctx->err_word), s);
}

}  // namespace

bool cross_few_supported(const CrossArgs& a) {
  return cross_tc_supported(a) && (a.d == 64 || a.d == 128) && a.hq / a.hk * a.q_len <= ROWS;
}

cudaError_t cross_forward_few(const CrossArgs& a, cudaStream_t s) {
  return a.d == 64 ? run_few<64>(a, s) : run_few<128>(a, s);
}

}  // namespace lcb
