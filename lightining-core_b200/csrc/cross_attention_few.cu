// Cross attention of a few query rows (single tokens with the heads that share a key head).
//
// K and V are read once against a few operations a byte, so HBM bounds it and what matters is bytes in flight: tiles
// of keys arrive by TMA in a ring of 96 KB, two blocks to an SM, and four warps share each tile's keys.
// bf16, at most 16 rows, head_dim 64 or 128: 16 keys a warp with the 16 x 8 x 16 matrix instruction:
//   S = Q K^T   the order of the columns inside a dot product is free, so lane c of a quad takes the 8
//               contiguous values 8c.. of every 32 as its share of two k-steps, of Q alike: 16-byte reads of K
//               as it lies
//   O += P V    lane (g, c) reads keys 2c, 2c+1, 2c+8, 2c+9 at columns 8g..8g+7 and pairs keys with byte
//               permutes; n-tile u then holds the columns 8g + u
// P enters the product as the sum of two bf16 numbers: its upper half, and what that leaves, rounded (by 2^-15 of P
// at most), in a second product; scores, statistics and sums are fp32.  The second part is 2^-126 at least, which no
// sum of finite values sees, so that both have P's sign and an infinite value gives an infinity in both products.
// fp32, at most 8 rows, head_dim <= 128 (tiles of 4096 / D keys): the CUDA cores, 2 * D * rows FMAs a key against 8 * D
// bytes, are faster than the bytes.  A quad takes a key's dot products (the rows of Q in shared memory), then every
// lane four columns of O.
// A block's warps join their (maximum, sum, O) in shared memory; the keys of a pair are split over a cluster of up to
// 8 blocks, which join theirs through distributed shared memory -- one launch, no workspace -- and over several
// clusters (and the join of parts) only when pairs are very few.
// B200, 64 sequences of 32 / 8 heads over 2048..4096 keys, head_dim 128 (811 MB, floor 126 us): loads straight
// into registers, three blocks to an SM, 226 us; the tiled tensor-core kernel 202 us (two stages of 64 KB do not cover
// the latency); this one 142 us (with 4 blocks to a pair instead of 2: 154, with 8: 195).
// fp32, all 4096 keys (2.1 GB, floor 315 us): 346 us, on 64 x 64 tiles of the CUDA-core kernel 4114; with 8 rows to a
// pair 540 (its FMAs and its 164 registers then show), from 9 on the tensor cores take over.
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
constexpr float kLeast = 1.17549435e-38f;  // 2^-126
constexpr int WARPS = 4;
constexpr int ROWS = 16, ROWS_F32 = 8;
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

template <int D, int R>
struct FewSmem {
  float o[WARPS][R][D + 4];  // per warp; [0] ends as the block's sum
  float m[WARPS][R], l[WARPS][R];
  float bm[R], bl[R];        // the block's
};
// A ring of 96 KB: stages of KEYS keys, K's boxes of 128 bytes of columns, then V's.
template <typename T, int D, int R>
struct FewRing {
  static constexpr int ES = sizeof(T), KEYS = ES == 2 ? 64 : 4096 / D, NW = D * ES / 128, BOX = KEYS * 128;
  static constexpr int STAGE = 2 * NW * BOX, NS = 96 * 1024 / STAGE;
  static_assert(sizeof(FewSmem<D, R>) <= NS * STAGE, "the sums lie over the ring");
};
struct FewBars {
  uint64_t full[6], free_[6];
  int abort_flag;
};

// Which keys a block takes: its share of this outer split's share, whole tiles.
template <typename L>
struct FewJob {
  int pair, b, hk, rank, group, rows, q_end, kv_end, t_lo, n;
  const unsigned char* mask;
  __device__ FewJob(const CrossArgs& a, const CrossSplit& sp, int cluster) {
    group = a.hq / a.hk, rows = group * a.q_len;
    rank = static_cast<int>(blockIdx.x) % cluster;
    pair = static_cast<int>(blockIdx.x) / cluster, b = pair / a.hk, hk = pair % a.hk;
    q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
    mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
    const int steps = (kv_end + L::KEYS - 1) / L::KEYS;
    const int parts = cluster * sp.splits, part = static_cast<int>(blockIdx.y) * cluster + rank;
    const int per = (steps + parts - 1) / parts;
    t_lo = min(steps, part * per), n = min(steps, (part + 1) * per) - t_lo;
  }
  __device__ bool live(const CrossArgs& a, int r) const { return r < rows && r % a.q_len < q_end; }
  __device__ bool seen(int key) const { return key < kv_end && (!mask || mask[key]); }
};

template <typename L>
__device__ __forceinline__ void few_init(FewBars& bars, const CUtensorMap* mk, const CUtensorMap* mv) {
  for (int i = 0; i < L::NS; ++i) {
    mbar_init(&bars.full[i], 1);
    mbar_init(&bars.free_[i], WARPS);
  }
  bars.abort_flag = 0;
  fence_barrier_init();
  tma_prefetch_desc(mk);
  tma_prefetch_desc(mv);
}

// The loading thread.
template <typename L, typename T>
__device__ __forceinline__ void few_load(uint8_t* ring, FewBars& bars, const CUtensorMap* mk, const CUtensorMap* mv,
                                         const FewJob<L>& job, const KvAxes& ax, unsigned* err) {
  bool ok = true;
  int i = 0;
  for (; i < job.n; ++i) {
    const int s = i % L::NS;
    if (i >= L::NS && !mbar_wait_bounded(&bars.free_[s], (i / L::NS - 1) & 1, &bars.abort_flag, err, kErrCrossLoadWait)) {
      ok = false;
      break;
    }
    mbar_arrive_expect_tx(&bars.full[s], L::STAGE);
    const int key = (job.t_lo + i) * L::KEYS;
    for (int w = 0; w < L::NW; ++w) {
      uint8_t* at = ring + s * L::STAGE + w * L::BOX;
      constexpr int COLS = 128 / sizeof(T);
      tma_load_4d(at, mk, w * COLS, key, ax.k_head ? job.hk : 0, ax.k_batch ? job.b : 0, &bars.full[s]);
      tma_load_4d(at + L::NW * L::BOX, mv, w * COLS, key, ax.v_head ? job.hk : 0, ax.v_batch ? job.b : 0, &bars.full[s]);
    }
  }
  // Every copy has landed before the sums take the ring's place, whatever became of its readers.
  const uint64_t t0 = globaltimer_ns();
  for (int k = max(0, i - L::NS); !ok && k < i; ++k)
    while (!mbar_try_wait(&bars.full[k % L::NS], (k / L::NS) & 1) && globaltimer_ns() - t0 < 100000000ull) {
    }
}

// The maximum of a row over the block's warps, and (one thread) the block's own statistics.
template <int D, int R>
__device__ __forceinline__ float few_block_max(FewSmem<D, R>& sm, int row, bool write) {
  float mx = sm.m[0][row];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) mx = fmaxf(mx, sm.m[w][row]);
  if (write) {
    const float base = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum = fmaf(sm.l[w][row], exp2f(sm.m[w][row] - base), sum);
    sm.bm[row] = mx;
    sm.bl[row] = sum;
  }
  return mx;
}

__device__ __forceinline__ void put4(__nv_bfloat16* out, float4 t, float f) {
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(t.x * f, t.y * f), pack_bf16x2(t.z * f, t.w * f));
}
__device__ __forceinline__ void put4(float* out, float4 t, float f) {
  *reinterpret_cast<float4*>(out) = make_float4(t.x * f, t.y * f, t.z * f, t.w * f);
}

// From the warps' sums (scaled to the block's maximum) to the result: the block's, then the cluster's.
template <typename T, int D, int R, typename L>
__device__ __forceinline__ void few_join(FewSmem<D, R>& sm, const CrossArgs& a, const CrossSplit& sp, int cluster,
                                         const FewJob<L>& job) {
  for (int i = threadIdx.x; i < R * (D / 4); i += THREADS) {
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
  // A block takes rows rank, rank + cluster, ...
  for (int i = threadIdx.x; i < R * (D / 4); i += THREADS) {
    const int row = i / (D / 4), col = i % (D / 4) * 4;
    if (row % cluster != job.rank || !job.live(a, row) || col >= a.d) continue;
    const auto of = [&](float* p, int n) { return cluster > 1 ? cl.map_shared_rank(p, n) : p; };
    float mx = -INFINITY;
    for (int n = 0; n < cluster; ++n) mx = fmaxf(mx, *of(&sm.bm[row], n));
    const float base = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f;
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int n = 0; n < cluster; ++n) {
      const float f = exp2f(*of(&sm.bm[row], n) - base);
      sum = fmaf(*of(&sm.bl[row], n), f, sum);
      const float4 v = *reinterpret_cast<const float4*>(of(&sm.o[0][row][col], n));
      t.x = fmaf(v.x, f, t.x), t.y = fmaf(v.y, f, t.y), t.z = fmaf(v.z, f, t.z), t.w = fmaf(v.w, f, t.w);
    }
    const int h = job.hk * job.group + row / a.q_len, tok = row % a.q_len;
    const long long at = (static_cast<long long>(job.b) * a.hq + h) * a.q_len + tok;  // dense row
    if (sp.splits > 1) {
      const long long part_row = static_cast<long long>(blockIdx.y) * sp.rows + at;
      *reinterpret_cast<float4*>(sp.o + part_row * a.d + col) = t;
      if (col == 0) sp.ml[part_row] = make_float2(mx, sum);
      continue;
    }
    put4(static_cast<T*>(a.out) + job.b * a.os.b + h * a.os.h + tok * a.os.t + col, t, cross_inverse(mx, sum));
    if (col == 0 && a.lse) a.lse[at] = cross_lse(mx, sum);
  }
  if (cluster > 1) cl.sync();  // no block leaves while another reads its sums
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
    cross_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, CrossArgs a,
                     CrossSplit sp, int cluster, KvAxes ax, unsigned* err) {
  using L = FewRing<__nv_bfloat16, D, ROWS>;
  constexpr int NB = D / 32, NW = L::NW, NS = L::NS, STAGE = L::STAGE, KEYS = L::KEYS, BOX = L::BOX;
  extern __shared__ __align__(1024) uint8_t ring[];
  __shared__ FewBars bars;
  FewSmem<D, ROWS>& sm = *reinterpret_cast<FewSmem<D, ROWS>*>(ring);
  if ((smem_u32(ring) & 1023u) != 0) {  // the 128-byte swizzle atoms need 1 KB alignment
    if (threadIdx.x == 0) atomicCAS(err, 0u, static_cast<unsigned>(kErrCrossLoadWait) | 0x1000u);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  griddep_launch_dependents();  // the parts' join waits for the end of this grid
  const FewJob<L> job(a, sp, cluster);
  if (threadIdx.x == 0) few_init<L>(bars, &map_k, &map_v);
  __syncthreads();
  float o[NW * 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  bool saw = false;  // a visible key
  if (warp == WARPS) {
    if (lane == 0) few_load<L, __nv_bfloat16>(ring, bars, &map_k, &map_v, job, ax, err);
  } else {
    // Q fragments: rows g and g + 8, the 8 values 8c.. of every 32.
    uint4 q[NB][2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) + job.b * a.qs.b +
                                 (job.hk * job.group + row / a.q_len) * a.qs.h + row % a.q_len * a.qs.t + c * 8;
#pragma unroll
      for (int n = 0; n < NB; ++n)
        q[n][r] = job.live(a, row) ? __ldg(reinterpret_cast<const uint4*>(src + n * 32)) : make_uint4(0, 0, 0, 0);
    }
    const float sc = a.scale * kLog2e;
    // Piece k of 16 bytes of this warp's key r in a box.
    const auto piece = [&](const uint8_t* box, int r, int k) {
      return *reinterpret_cast<const uint4*>(box + (warp * 16 + r) * 128 + ((k ^ (r & 7)) << 4));
    };
#pragma unroll
    for (int n8 = 0; n8 < NW * 8; ++n8) o[n8][0] = o[n8][1] = o[n8][2] = o[n8][3] = 0.0f;
    for (int i = 0; i < job.n; ++i) {
      const int st = i % NS, k0 = (job.t_lo + i) * KEYS + warp * 16;
      // The mask bytes of a step are asked for before the wait for its keys.
      bool vis[2][2] = {{true, true}, {true, true}}, vis_v[4] = {true, true, true, true};
      const bool partial = job.mask || k0 + 16 > job.kv_end;
      if (partial) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) vis_v[t * 2 + e] = vis[t][e] = job.seen(k0 + t * 8 + 2 * c + e);
      }
      saw |= vis[0][0] | vis[0][1] | vis[1][0] | vis[1][1];
      if (!warp_wait_poll(&bars.full[st], (i / NS) & 1, &bars.abort_flag, err, kErrCrossSoftmaxWait)) break;
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
          const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
          hi[t * 2 + r] = __byte_perm(u0, u1, 0x7632);
          lo[t * 2 + r] = pack_bf16x2(fmaxf(p0 - __uint_as_float(u0 & 0xffff0000u), kLeast),
                                      fmaxf(p1 - __uint_as_float(u1 & 0xffff0000u), kLeast));
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
  saw = __any_sync(0xffffffffu, saw);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (saw) m[r] = fmaxf(m[r], kCrossLowest);
    l[r] = quad_sum(l[r]);
    if (c == 0 && warp < WARPS) {
      sm.m[warp][g + 8 * r] = m[r];
      sm.l[warp][g + 8 * r] = l[r];
    }
  }
  __syncthreads();
  if (warp < WARPS) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r;
      const float mx = few_block_max(sm, row, warp == 0 && c == 0);
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
    }
  }
  __syncthreads();
  few_join<__nv_bfloat16>(sm, a, sp, cluster, job);
}

template <int D, int R>
__global__ void __launch_bounds__(THREADS, 2)
    cross_few_f32_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, CrossArgs a,
                         CrossSplit sp, int cluster, KvAxes ax, unsigned* err) {
  using L = FewRing<float, D, R>;
  constexpr int NW = L::NW, NS = L::NS, STAGE = L::STAGE, BOX = L::BOX;
  constexpr int KW = L::KEYS / WARPS, KG = KW / 8;  // a warp's keys of a tile, in groups of 8
  constexpr int CL = D / 4;                         // lanes that hold a row of O; 32 / CL groups share the keys
  extern __shared__ __align__(1024) uint8_t ring[];
  __shared__ FewBars bars;
  __shared__ __align__(16) float sq[R][D], sp_w[WARPS][R][KW];
  FewSmem<D, R>& sm = *reinterpret_cast<FewSmem<D, R>*>(ring);
  if ((smem_u32(ring) & 1023u) != 0) {  // the 128-byte swizzle atoms need 1 KB alignment
    if (threadIdx.x == 0) atomicCAS(err, 0u, static_cast<unsigned>(kErrCrossLoadWait) | 0x1000u);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  griddep_launch_dependents();  // the parts' join waits for the end of this grid
  const FewJob<L> job(a, sp, cluster);
  if (threadIdx.x == 0) few_init<L>(bars, &map_k, &map_v);
  for (int i = threadIdx.x; i < R * D / 4; i += THREADS) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (job.live(a, r) && col < a.d)
      f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + job.b * a.qs.b +
                                                (job.hk * job.group + r / a.q_len) * a.qs.h + r % a.q_len * a.qs.t + col));
    *reinterpret_cast<float4*>(&sq[r][col]) = f;
  }
  __syncthreads();
  float4 o[R];
  float m[R], l[R];
  bool saw = false;  // a visible key
#pragma unroll
  for (int r = 0; r < R; ++r) {
    o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    m[r] = -INFINITY;
    l[r] = 0.0f;
  }
  if (warp == WARPS) {
    if (lane == 0) few_load<L, float>(ring, bars, &map_k, &map_v, job, ax, err);
  } else {
    const float sc = a.scale * kLog2e;
    const auto piece = [&](const uint8_t* box, int r, int k) {
      return *reinterpret_cast<const float4*>(box + (warp * KW + r) * 128 + ((k ^ (r & 7)) << 4));
    };
    for (int i = 0; i < job.n; ++i) {
      const int st = i % NS, k0 = (job.t_lo + i) * L::KEYS + warp * KW;
      const bool partial = job.mask || k0 + KW > job.kv_end;
      unsigned vis[KG];  // bit 4 n: key n of the group
      bool mine[KG];
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        mine[k] = !partial || job.seen(k0 + k * 8 + g);
        vis[k] = __ballot_sync(0xffffffffu, mine[k]);
        saw |= vis[k] != 0;
      }
      if (!warp_wait_poll(&bars.full[st], (i / NS) & 1, &bars.abort_flag, err, kErrCrossSoftmaxWait)) break;
      const uint8_t *kbox = ring + st * STAGE, *vbox = kbox + NW * BOX;
      float s[KG][R];
#pragma unroll
      for (int k = 0; k < KG; ++k)
#pragma unroll
        for (int r = 0; r < R; ++r) s[k][r] = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int p = c + 4 * ((h ^ g) & 1);  // neighbouring keys read different halves of a box's rows: other banks
          float4 kv[KG];
#pragma unroll
          for (int k = 0; k < KG; ++k) kv[k] = piece(kbox + w * BOX, k * 8 + g, p);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float4 q = *reinterpret_cast<const float4*>(&sq[r][w * 32 + p * 4]);
#pragma unroll
            for (int k = 0; k < KG; ++k)
              s[k][r] = fmaf(q.w, kv[k].w, fmaf(q.z, kv[k].z, fmaf(q.y, kv[k].y, fmaf(q.x, kv[k].x, s[k][r]))));
          }
        }
      bool rescale = false;
      float keep[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < KG; ++k) {
          s[k][r] = quad_sum(s[k][r]);
          if (!mine[k]) s[k][r] = -INFINITY;
          top = fmaxf(top, s[k][r]);
        }
#pragma unroll
        for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float mx = fmaxf(m[r], top * sc), base = mx == -INFINITY ? 0.0f : mx;
        keep[r] = exp2f(m[r] - base);
        rescale |= keep[r] != 1.0f;
        m[r] = mx;
        l[r] *= keep[r];
#pragma unroll
        for (int k = 0; k < KG; ++k) {
          const float p = exp2f(fmaf(s[k][r], sc, -base));
          l[r] += p;
          if (c == (r & 3)) sp_w[warp][r][k * 8 + g] = p;
        }
      }
      __syncwarp();
      if (rescale) {
#pragma unroll
        for (int r = 0; r < R; ++r) o[r].x *= keep[r], o[r].y *= keep[r], o[r].z *= keep[r], o[r].w *= keep[r];
      }
      const int part = lane / CL, col = lane % CL;  // keys part * 8 .. + 8, columns col * 4 .. + 4
#pragma unroll
      for (int k4 = 0; k4 < 8; k4 += 4) {
        float4 v[4], p[R];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = piece(vbox + (col >> 3) * BOX, part * 8 + k4 + e, col & 7);
          // A masked value would enter the sum: a weight of 0 does not hide a NaN.
          if (partial && !(((part ? vis[KG - 1] : vis[0]) >> (4 * (k4 + e))) & 1u)) v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) p[r] = *reinterpret_cast<const float4*>(&sp_w[warp][r][part * 8 + k4]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          o[r].x = fmaf(p[r].w, v[3].x, fmaf(p[r].z, v[2].x, fmaf(p[r].y, v[1].x, fmaf(p[r].x, v[0].x, o[r].x))));
          o[r].y = fmaf(p[r].w, v[3].y, fmaf(p[r].z, v[2].y, fmaf(p[r].y, v[1].y, fmaf(p[r].x, v[0].y, o[r].y))));
          o[r].z = fmaf(p[r].w, v[3].z, fmaf(p[r].z, v[2].z, fmaf(p[r].y, v[1].z, fmaf(p[r].x, v[0].z, o[r].z))));
          o[r].w = fmaf(p[r].w, v[3].w, fmaf(p[r].z, v[2].w, fmaf(p[r].y, v[1].w, fmaf(p[r].x, v[0].w, o[r].w))));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.free_[st]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (saw) m[r] = fmaxf(m[r], kCrossLowest);
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
      if constexpr (CL == 16) {
        o[r].x += __shfl_xor_sync(0xffffffffu, o[r].x, 16);
        o[r].y += __shfl_xor_sync(0xffffffffu, o[r].y, 16);
        o[r].z += __shfl_xor_sync(0xffffffffu, o[r].z, 16);
        o[r].w += __shfl_xor_sync(0xffffffffu, o[r].w, 16);
      }
    }
  }

  // The block's sums, over the ring (all its copies have landed and been read).
  __syncthreads();
  if (warp < WARPS && lane == 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sm.m[warp][r] = m[r];
      sm.l[warp][r] = l[r];
    }
  }
  __syncthreads();
  if (warp < WARPS) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mx = few_block_max(sm, r, warp == 0 && lane == 0);
      const float f = exp2f(m[r] - (mx == -INFINITY ? 0.0f : mx));
      if (lane < CL) put4(&sm.o[warp][r][lane * 4], o[r], f);
    }
  }
  __syncthreads();
  few_join<float>(sm, a, sp, cluster, job);
}

using FewKernel = void (*)(CUtensorMap, CUtensorMap, CrossArgs, CrossSplit, int, KvAxes, unsigned*);

template <typename L, FewKernel kernel>
cudaError_t run_few(const CrossArgs& a, cudaStream_t s) {
  constexpr int KEYS = L::KEYS;
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
  constexpr size_t SMEM = static_cast<size_t>(L::NS) * L::STAGE;
  static std::atomic<unsigned long long> attr_done{0};
  const cudaError_t ea = once_per_device(attr_done, [] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
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
  return w.end(a, cudaLaunchKernelEx(&cfg, kernel, mk, mv, a, w.sp, cluster, ax, ctx->err_word), s);
}

// The kernel's rows: 2, 4 or 8 (64 sequences of 4096 keys, 8 key heads of head_dim 128, 4 rows: 532 us
// with 8, 346 with 4).
template <int D>
cudaError_t run_few_f32(const CrossArgs& a, cudaStream_t s) {
  const int rows = a.hq / a.hk * a.q_len;
  if (rows <= 2) return run_few<FewRing<float, D, 2>, cross_few_f32_kernel<D, 2>>(a, s);
  if (rows <= 4) return run_few<FewRing<float, D, 4>, cross_few_f32_kernel<D, 4>>(a, s);
  return run_few<FewRing<float, D, ROWS_F32>, cross_few_f32_kernel<D, ROWS_F32>>(a, s);
}

}  // namespace

bool cross_few_supported(const CrossArgs& a) {
  const int rows = a.hq / a.hk * a.q_len;
  return a.bf16 ? cross_tc_supported(a) && (a.d == 64 || a.d == 128) && rows <= ROWS
                : a.d <= 128 && rows <= ROWS_F32 && cross_rows16(a);
}

cudaError_t cross_forward_few(const CrossArgs& a, cudaStream_t s) {
  if (a.bf16)
    return a.d == 64 ? run_few<FewRing<__nv_bfloat16, 64, ROWS>, cross_few_kernel<64>>(a, s)
                     : run_few<FewRing<__nv_bfloat16, 128, ROWS>, cross_few_kernel<128>>(a, s);
  return a.d <= 64 ? run_few_f32<64>(a, s) : run_few_f32<128>(a, s);
}

}  // namespace lcb
