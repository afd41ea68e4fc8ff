// Cross attention in bf16 on the 5th-generation tensor cores: forward and backward for head_dim <= 128
// (a multiple of 8; columns up to 64 or 128 are zeros that TMA fills in).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "attention_math.cuh"
#include "common.cuh"
#include "cross_attention.cuh"
#include "lc_internal.hpp"

namespace lcb {

void* tensor_map_encoder();

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int TILE = 128;               // rows and keys of a tile
constexpr int CH = 128 * 128;           // one [128 rows x 64 bf16] box, 128-byte swizzle: 16 KB

// ---- shared by forward and backward -----------------------------------------------------------
// A K, V, Q or dout tensor as TMA sees it: [batch, heads, tokens, d] with any strides.  An axis that is
// not stepped over (stride 0, or a single entry) is described as one entry and its coordinate is 0.
struct HeadMap {
  CUtensorMap map;
  int by_head, by_batch;
};

__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, int nch, int token, int h, int b,
                                          uint64_t* bar) {
  for (int c = 0; c < nch; ++c) tma_load_4d(dst + c * CH, map, c * 64, token, h, b, bar);
}

// Bounded drain of a copy already issued, so that no block leaves with TMA writes in flight.
__device__ __forceinline__ void drain_bar(uint64_t* bar, uint32_t ph) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, ph) && globaltimer_ns() - t0 < 100000000ull) {
  }
}

// Zeroes the rows of a staged tile for which keep(row) is false (one warp).  Swizzling permutes
// inside a row only.  The matrix unit multiplies a masked row by a weight of 0, which would keep a
// NaN or an infinity that memory holds there.
template <int NCH, class Keep>
__device__ __forceinline__ void scrub_rows(uint8_t* tile, Keep keep) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 32 + lane;
    if (!keep(row))
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(tile + c * CH + row * 128 + e * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Visible keys of the tile at kv0 as four words of 32 (bit e of word i: key kv0 + 32 i + e).  `byte`
// are this lane's four mask bytes (loaded early); without a mask only the end of the keys counts.
__device__ __forceinline__ void load_mask_bytes(const unsigned char* mask, int kv0, int kv_end, int lane,
                                                unsigned char (&byte)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = kv0 + i * 32 + lane;
    byte[i] = k < kv_end && (!mask || mask[k]);
  }
}

// ---- forward ----------------------------------------------------------------------------------
// One block per SM owns two tiles of 128 rows (A and B) of a (batch, key head) pair, which share every
// K and V tile of 128 keys.  A row is (head in the group, token), so short queries of a group fill a
// tile together.  Roles (10 warps):
//   warp 0      TMA: K_j and V_j into rings of NS stages
//   warp 1      MMA: S_h = Q_h K_j^T, O_h += P_h V_j for h = A, B, in the order PV_A(j), S_A(j+1),
//               PV_B(j), S_B(j+1), so that one tile's softmax runs beside the other's products;
//               it also zeroes the masked rows of V_j
//   warps 2..5  rows of A (warps 6..9: of B): the Q rows into shared memory, then softmax -- a
//               thread owns a row (one TMEM lane) -- and the epilogue
// TMEM: S_A 0, S_B 128, O_A 256, O_B 384; P_h is written as bf16 pairs over the first half of S_h
// and read from there as the A operand.  O is rescaled only when a row's maximum grows by more than
// 2^8 (the final division makes up for it).
template <int D>
struct Fwd {
  static constexpr int NCH = D / 64;
  static constexpr int BYTES = NCH * CH;     // a Q, K or V tile
  static constexpr int NS = D == 64 ? 4 : 2; // ring stages
  static constexpr int K_OFF = 2 * BYTES;
  static constexpr int V_OFF = K_OFF + NS * BYTES;
  static constexpr int TAIL_OFF = V_OFF + NS * BYTES;
  static constexpr int THREADS = 320;
  struct Tail {
    uint64_t q_full[2];             // 4 warp arrivals
    uint64_t k_full[NS], v_full[NS];
    uint64_t k_free[NS], v_free[NS];
    uint64_t s_full[2], p_full[2], o_done[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t SMEM = 1024 + TAIL_OFF + sizeof(Tail);
};
constexpr float kRescale = 8.0f;

struct FwdParams {
  CrossArgs a;
  CrossSplit sp;
  int k_head, k_batch, v_head, v_batch;  // 1: the tensor map has that axis
  float scale_log2;
  unsigned* err;
};

template <int D>
__global__ void __launch_bounds__(Fwd<D>::THREADS, 1)
    cross_fwd_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const FwdParams p) {
  using F = Fwd<D>;
  constexpr int NS = F::NS;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  typename F::Tail* st = reinterpret_cast<typename F::Tail*>(smem + F::TAIL_OFF);
  const auto sQ = [&](int h) { return smem + h * F::BYTES; };
  const auto sK = [&](int s) { return smem + F::K_OFF + s * F::BYTES; };
  const auto sV = [&](int s) { return smem + F::V_OFF + s * F::BYTES; };
  const CrossArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int group = a.hq / a.hk, rows = group * a.q_len;
  const int pairs = (rows + 2 * TILE - 1) / (2 * TILE);
  const int bh = blockIdx.x / pairs, b = bh / a.hk, hk = bh % a.hk;
  const int r0 = (blockIdx.x % pairs) * 2 * TILE;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const int tiles = (kv_end + TILE - 1) / TILE;
  const int per = (tiles + p.sp.splits - 1) / p.sp.splits;
  const int t_lo = min(tiles, static_cast<int>(blockIdx.y) * per);
  const int n = min(tiles, t_lo + per) - t_lo;  // KV tiles of this block
  // Whether a tile has a row to compute: its first row's token is one, or another head starts in it.
  const auto live = [&](int h) {
    const int r = r0 + h * TILE;
    if (r >= rows || q_end == 0) return false;
    const int t = r % a.q_len;
    return t < q_end || r + a.q_len - t < min(r + TILE, rows);
  };
  const bool act[2] = {live(0), live(1)};
  if (!act[0] && !act[1]) return;
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&st->k_full[s], 1);
      mbar_init(&st->v_full[s], 1);
      mbar_init(&st->k_free[s], 1);
      mbar_init(&st->v_free[s], 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&st->q_full[h], 4);
      mbar_init(&st->s_full[h], 1);
      mbar_init(&st->p_full[h], 4);
      mbar_init(&st->o_done[h], 1);
    }
    mbar_init(&st->drain, 1);
    st->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 0) {
    tmem_alloc(&st->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = st->tmem_base;
  volatile int* abort_flag = &st->abort_flag;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      bool ok = true;
      int k_issued = 0, v_issued = 0;
      for (int j = 0; j < n && ok; ++j) {
        const int s = j % NS, ph = (j / NS - 1) & 1;
        // A stage's next completion of k_free / v_free needs the tile loaded here, so each parity
        // wait is unambiguous.
        if (j >= NS && !mbar_wait_bounded(&st->k_free[s], ph, abort_flag, p.err, kErrCrossLoadWait)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&st->k_full[s], F::BYTES);
        load_tile(sK(s), &map_k, F::NCH, (t_lo + j) * TILE, p.k_head ? hk : 0, p.k_batch ? b : 0, &st->k_full[s]);
        ++k_issued;
        if (j >= NS && !mbar_wait_bounded(&st->v_free[s], ph, abort_flag, p.err, kErrCrossLoadWait)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&st->v_full[s], F::BYTES);
        load_tile(sV(s), &map_v, F::NCH, (t_lo + j) * TILE, p.v_head ? hk : 0, p.v_batch ? b : 0, &st->v_full[s]);
        ++v_issued;
      }
      if (!ok) {
        for (int j = max(0, k_issued - NS); j < k_issued; ++j) drain_bar(&st->k_full[j % NS], (j / NS) & 1);
        for (int j = max(0, v_issued - NS); j < v_issued; ++j) drain_bar(&st->v_full[j % NS], (j / NS) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (whole warp)
    constexpr uint32_t IDESC_S = idesc_bf16_f32(TILE, TILE, 0, 0);  // Q and K K-major
    constexpr uint32_t IDESC_O = idesc_bf16_f32(TILE, D, 0, 1);     // P in TMEM, V MN-major
    bool ok = true, issued = false;
    const auto wait = [&](uint64_t* bar, uint32_t ph) {
      return warp_wait_poll(bar, ph, abort_flag, p.err, kErrCrossMmaWait);
    };
    const auto issue_s = [&](int h, int j) {
      const uint64_t qd = smem_desc_sw128(smem_u32(sQ(h)), 16, 1024);
      const uint64_t kd = smem_desc_sw128(smem_u32(sK(j % NS)), 16, 1024);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t o16 = ((kk >> 2) * CH + (kk & 3) * 32) >> 4;
        umma_f16_ss_w(tmem + h * 128, qd + o16, kd + o16, IDESC_S, kk > 0 ? 1u : 0u);
      }
      issued = true;
      umma_commit_w(&st->s_full[h]);
    };
    const auto issue_pv = [&](int h, int j) {
      const uint64_t vd = smem_desc_sw128(smem_u32(sV(j % NS)), CH, 1024);
#pragma unroll
      for (int kk = 0; kk < TILE / 16; ++kk)
        umma_f16_ts_w(tmem + 256 + h * 128, tmem + h * 128 + kk * 8, vd + (kk * 2048 >> 4), IDESC_O,
                      (j > 0 || kk > 0) ? 1u : 0u);
      umma_commit_w(&st->o_done[h]);
    };
    if (n > 0) {
      for (int h = 0; h < 2 && ok; ++h)
        if (act[h]) {
          ok = wait(&st->q_full[h], 0) && wait(&st->k_full[0], 0);
          if (ok) {
            tc_fence_after();
            issue_s(h, 0);
          }
        }
      if (ok && NS < n) umma_commit_w(&st->k_free[0]);
    }
    for (int j = 0; j < n && ok; ++j) {
      const int s = j % NS, kv0 = (t_lo + j) * TILE;
      if (!(ok = wait(&st->v_full[s], (j / NS) & 1))) break;
      // Masked rows of V: keys past kv_end that memory holds (TMA zero-fills past kv_len), and holes.
      if (mask || (kv0 + TILE > kv_end && kv_end < a.kv_len))
        scrub_rows<F::NCH>(sV(s), [&](int r) { return kv0 + r < kv_end && (!mask || mask[kv0 + r]); });
      for (int h = 0; h < 2 && ok; ++h) {
        if (!act[h]) continue;
        // p_full[h] next completes for P_h(j+1), which needs S_h(j+1), issued after this wait.
        if (!(ok = wait(&st->p_full[h], j & 1))) break;
        tc_fence_after();
        issue_pv(h, j);
        if (j + 1 < n) {
          if (!(ok = wait(&st->k_full[(j + 1) % NS], ((j + 1) / NS) & 1))) break;
          tc_fence_after();
          issue_s(h, j + 1);
        }
      }
      if (!ok) break;
      // Both commits cover everything issued so far: the last readers of V_j and of K_{j+1}.  Only
      // stages that are loaded again are handed back, so no arrival is left in flight at the end.
      if (j + NS < n) umma_commit_w(&st->v_free[s]);
      if (j + 1 + NS < n) umma_commit_w(&st->k_free[(j + 1) % NS]);
    }
    if (!ok && issued) {
      umma_commit_w(&st->drain);
      drain_bar(&st->drain, 0);
    }
  } else {
    // ------------------------------------------------------------ rows of tile h
    const int h = warp >= 6 ? 1 : 0;
    const int quarter = warp & 3;  // TMEM lanes a warp may read
    const int base = r0 + h * TILE;
    if (act[h]) {
      // Q rows into shared memory: D/8 lanes to a row, 16 bytes each, chunk k of row r at k ^ (r & 7).
      constexpr int LPR = D / 8, RPI = 32 / LPR;
      uint8_t* q = sQ(h);
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) + b * a.qs.b;
#pragma unroll 4
      for (int i = 0; i < 32 / RPI; ++i) {
        const int r = quarter * 32 + i * RPI + lane / LPR, c = lane % LPR;
        const int g = (base + r) / a.q_len, t = (base + r) % a.q_len;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (base + r < rows && t < q_end && c * 8 < a.d)
          w = __ldg(reinterpret_cast<const uint4*>(src + (hk * group + g) * a.qs.h + t * a.qs.t + c * 8));
        *reinterpret_cast<uint4*>(q + (c >> 3) * CH + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = w;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->q_full[h]);

      const int row = quarter * 32 + lane;  // = TMEM lane
      const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
      const uint32_t s_tmem = tmem + lane_base + static_cast<uint32_t>(h * 128);
      const uint32_t o_tmem = s_tmem + 256;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      unsigned char byte[4];
      for (int j = 0; j < n; ++j) {
        const int kv0 = (t_lo + j) * TILE;
        const bool partial = mask || kv0 + TILE > kv_end;
        if (partial) load_mask_bytes(mask, kv0, kv_end, lane, byte);
        // s_full[h] next completes for S_h(j+1), which needs P_h(j) from these warps first.
        if (!(ok = warp_wait_poll(&st->s_full[h], j & 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
        tc_fence_after();
        uint32_t r[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, r[c]);
        if (partial) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const unsigned w = __ballot_sync(0xffffffffu, byte[c]);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((w >> e) & 1u)) r[c][e] = __float_as_uint(-INFINITY);
          }
        }
        float pm[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pm[i] = __uint_as_float(r[0][i]);
#pragma unroll
        for (int e = 8; e < TILE; e += 2)
          pm[(e >> 1) & 7] = max3(pm[(e >> 1) & 7], __uint_as_float(r[e >> 5][e & 31]),
                                  __uint_as_float(r[(e + 1) >> 5][(e + 1) & 31]));
        const float mx =
            max3(max3(pm[0], pm[1], pm[2]), max3(pm[3], pm[4], pm[5]), fmaxf(pm[6], pm[7])) * p.scale_log2;
        const bool need = mx > m + kRescale;
        float factor = 1.0f;
        if (need) {
          factor = m == -INFINITY ? 0.0f : exp2f(m - mx);
          l *= factor;
          m = mx;
        }
        if (j > 0 && __any_sync(0xffffffffu, need)) {
          // O_h is rescaled in place: PV_h(j-1) must have landed (o_done[h] next completes for
          // PV_h(j), which needs this tile's P).
          if (!(ok = warp_wait_poll(&st->o_done[h], (j - 1) & 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_tmem + c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st16(o_tmem + c, o);
          }
          tmem_wait_st();
        }
        // A row that has seen no key yet has m = -inf: every score is -inf too and its weights are 0
        // (or 2^-125 where the polynomial serves, times rows of V that are zeros).
        const float mu = m == -INFINITY ? 0.0f : m;
        const uint64_t sc2 = pk2(p.scale_log2, p.scale_log2), nm2 = pk2(-mu, -mu);
        uint64_t ps2[4] = {0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < TILE / 32; ++g) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x0, x1, e0, e1;
            unpk2(fma2(pk2(__uint_as_float(r[g][2 * i]), __uint_as_float(r[g][2 * i + 1])), sc2, nm2), x0, x1);
            if ((i & 7) < 2) {
              exp2_poly_pair(x0, x1, e0, e1);
            } else {
              e0 = fast_exp2(x0);
              e1 = fast_exp2(x1);
            }
            ps2[i & 3] = add2(ps2[i & 3], pk2(e0, e1));
            w[i] = pack_bf16x2(e0, e1);
          }
          tmem_st16(s_tmem + g * 16, w);
        }
        float x, y;
        unpk2(add2(add2(ps2[0], ps2[1]), add2(ps2[2], ps2[3])), x, y);
        l += x + y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&st->p_full[h]);
      }
      if (ok && n > 0)
        ok = warp_wait_poll(&st->o_done[h], (n - 1) & 1, abort_flag, p.err, kErrCrossSoftmaxWait);
      if (ok) {
        tc_fence_after();
        const int rr = base + row, g = rr / a.q_len, t = rr % a.q_len;
        const bool store = rr < rows && t < q_end;
        const bool empty = m == -INFINITY;
        const long long at = (static_cast<long long>(b) * a.hq + hk * group) * a.q_len + rr;  // dense row
        const bool split = p.sp.splits > 1;
        const float inv = split ? 1.0f : empty ? 0.0f : 1.0f / l;
        if (store && split) p.sp.ml[static_cast<long long>(blockIdx.y) * p.sp.rows + at] = make_float2(m, empty ? 0.0f : l);
        if (store && !split && a.lse) a.lse[at] = empty ? -INFINITY : (m + log2f(l)) * kLn2;
        float* part = p.sp.o + (static_cast<long long>(blockIdx.y) * p.sp.rows + at) * a.d;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + b * a.os.b + (hk * group + g) * a.os.h + t * a.os.t;
        // tcgen05.ld is warp-collective: every lane loads, only live rows store.
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_tmem + c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = empty ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
          if (store && split) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (c + e < a.d) *reinterpret_cast<uint4*>(part + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          } else if (store) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (c + e < a.d) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  w[i] = pack_bf16x2(__uint_as_float(o[e + 2 * i]), __uint_as_float(o[e + 2 * i + 1]));
                *reinterpret_cast<uint4*>(out + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
              }
          }
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- host -------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool head_map(HeadMap* m, const void* base, const HeadStrides& s, int batch, int heads, int len, int d) {
  auto enc = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!enc) return false;
  m->by_head = heads > 1 && s.h != 0;
  m->by_batch = batch > 1 && s.b != 0;
  const cuuint64_t row = static_cast<cuuint64_t>(len > 1 ? s.t : d) * 2;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(len),
                              static_cast<cuuint64_t>(m->by_head ? heads : 1),
                              static_cast<cuuint64_t>(m->by_batch ? batch : 1)};
  const cuuint64_t strides[3] = {row, m->by_head ? static_cast<cuuint64_t>(s.h) * 2 : row,
                                 m->by_batch ? static_cast<cuuint64_t>(s.b) * 2 : row};
  const cuuint32_t box[4] = {64, TILE, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(&m->map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 16-byte rows and strides that a tensor map can hold (below 2^40 bytes).
bool rows16(const void* p, const HeadStrides& s, int len) {
  const auto ok = [](long long x) { return x % 8 == 0 && x < (1LL << 38); };
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ok(s.b) && ok(s.h) && ok(s.t) && (len == 1 || s.t != 0);
}

template <int D>
cudaError_t fwd_tc(const CrossArgs& a, cudaStream_t s) {
  using F = Fwd<D>;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  HeadMap mk, mv;
  if (!head_map(&mk, a.k, a.ks, a.batch, a.hk, a.kv_len, a.d) ||
      !head_map(&mv, a.v, a.vs, a.batch, a.hk, a.kv_len, a.d))
    return cudaErrorInvalidValue;
  static std::atomic<unsigned long long> attr{0};
  cudaError_t e = once_per_device(attr, [] {
    return cudaFuncSetAttribute(cross_fwd_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(F::SMEM));
  });
  if (e != cudaSuccess) return e;
  const long long rows = static_cast<long long>(a.hq / a.hk) * a.q_len;
  const long long blocks = (rows + 2 * TILE - 1) / (2 * TILE) * a.batch * a.hk;
  if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
  CrossSplitWork w;
  if ((e = w.begin(a, blocks, TILE, 1, s)) != cudaSuccess) return e;
  const FwdParams p{a, w.sp, mk.by_head, mk.by_batch, mv.by_head, mv.by_batch, a.scale * kLog2e, ctx->err_word};
  cross_fwd_tc_kernel<D>
      <<<dim3(static_cast<unsigned>(blocks), w.sp.splits), F::THREADS, F::SMEM, s>>>(mk.map, mv.map, p);
  return w.end(a, cudaGetLastError(), s);
}

}  // namespace

bool cross_tc_supported(const CrossArgs& a) {
  return a.bf16 && a.d <= 128 && a.d % 8 == 0 && rows16(a.q, a.qs, a.q_len) && rows16(a.k, a.ks, a.kv_len) &&
         rows16(a.v, a.vs, a.kv_len) && rows16(a.out, a.os, a.q_len) && tensor_map_encoder() != nullptr;
}

cudaError_t cross_forward_tc(const CrossArgs& a, cudaStream_t s) {
  return a.d <= 64 ? fwd_tc<64>(a, s) : fwd_tc<128>(a, s);
}

}  // namespace lcb
