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

// ---- backward: dk and dv ------------------------------------------------------------------------
// One block per SM owns a tile of 128 keys of a (batch, key head) pair and walks the tiles of 128
// queries of the group's heads ("items"; of every batch entry in turn when k and v are shared by
// them).  Keys are the rows: S^T = K Q^T and dP^T = V dout^T arrive with a key per TMEM lane, so
// P^T and dS^T go straight back to TMEM as the A operands of dV += P^T dout and dK += dS^T Q, whose B
// operands are the same dout and Q tiles read MN-major.  Nothing is transposed or passed through
// shared memory, and both gradients accumulate in TMEM: no atomics, one order of summation.
//   warp 0      TMA: K and V once; Q, dout and the row terms of each item into NS stages
//   warp 1      MMA, in the order S(0) dP(0) | dV(i) S(i+1) dK(i) dP(i+1): while the other warps form
//               dS(i) the products dV(i) and S(i+1) run, while they form P(i+1) dK(i) and dP(i+1) do
//   warps 2..9  P and dS: a thread owns a key (lane) and half of the item's queries
// TMEM columns: S^T / P^T 0 (P of query half h over the first 32 columns of that half's scores),
// dP^T / dS^T 128 (likewise), dV 256, dK 256 + D.
template <int D>
struct Dkv {
  static constexpr int NCH = D / 64;
  static constexpr int BYTES = NCH * CH;
  static constexpr int NS = D == 64 ? 4 : 2;
  static constexpr int STAGE = 2 * BYTES;   // Q, dout
  static constexpr int STAGE_OFF = 2 * BYTES;
  static constexpr int TERM_OFF = STAGE_OFF + NS * STAGE;  // [NS][2][128] floats
  static constexpr int TAIL_OFF = TERM_OFF + NS * 1024;
  static constexpr int THREADS = 320;
  struct Tail {
    uint64_t kv_full;
    uint64_t q_full[NS], g_full[NS], free_[NS];
    uint64_t s_full, dp_full, p_full, ds_full, done;
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t SMEM = 1024 + TAIL_OFF + sizeof(Tail);
};

struct GradParams {
  CrossGradArgs g;
  const float *neg_lse2, *neg_d;
  int q_pad;
  int q_head, q_batch, g_head, g_batch, k_head, k_batch, v_head, v_batch;  // 1: the map has that axis
  float scale_log2;
  unsigned* err;
};

// The items of a key tile, in order: batch entries that see a key of it, heads of the group, tiles of
// their queries.
struct Items {
  const CrossArgs& a;
  int k0, b_hi, group;
  int b, g, qt, q_end, kv_end;  // the current item, and its batch entry's lengths
  __device__ Items(const CrossArgs& a_, int k0_, int b_lo, int b_hi_)
      : a(a_), k0(k0_), b_hi(b_hi_), group(a_.hq / a_.hk), b(b_lo), g(0), qt(0), q_end(0), kv_end(0) {
    settle();
  }
  // Moves to the first batch entry from b on that has an item; b == b_hi: none left.
  __device__ void settle() {
    for (; b < b_hi; ++b) {
      q_end = cross_len(a.q_lens, b, a.q_len);
      kv_end = cross_len(a.kv_lens, b, a.kv_len);
      if (k0 < kv_end && q_end > 0) return;
    }
  }
  __device__ bool valid() const { return b < b_hi; }
  __device__ void next() {
    if ((qt + 1) * TILE < q_end) {
      ++qt;
      return;
    }
    qt = 0;
    if (++g < group) return;
    g = 0;
    ++b;
    settle();
  }
};

template <int D>
__global__ void __launch_bounds__(Dkv<D>::THREADS, 1)
    cross_dkv_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_g,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const GradParams p) {
  using L = Dkv<D>;
  constexpr int NS = L::NS;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  typename L::Tail* st = reinterpret_cast<typename L::Tail*>(smem + L::TAIL_OFF);
  uint8_t *sK = smem, *sV = smem + L::BYTES;
  const auto sQ = [&](int s) { return smem + L::STAGE_OFF + s * L::STAGE; };
  const auto sG = [&](int s) { return smem + L::STAGE_OFF + s * L::STAGE + L::BYTES; };
  const auto terms = [&](int s) { return reinterpret_cast<float*>(smem + L::TERM_OFF + s * 1024); };
  const CrossArgs& a = p.g.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int key_tiles = (a.kv_len + TILE - 1) / TILE;
  const int bh = blockIdx.x / key_tiles, b0 = bh / a.hk, hk = bh % a.hk;
  const int k0 = (blockIdx.x % key_tiles) * TILE;
  const int b_hi = p.g.kv_shared ? a.batch : b0 + 1;
  const int group = a.hq / a.hk;

  if (threadIdx.x == 0) {
    mbar_init(&st->kv_full, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&st->q_full[s], 1);
      mbar_init(&st->g_full[s], 1);
      mbar_init(&st->free_[s], 1);
    }
    mbar_init(&st->s_full, 1);
    mbar_init(&st->dp_full, 1);
    mbar_init(&st->p_full, 8);
    mbar_init(&st->ds_full, 8);
    mbar_init(&st->done, 1);
    mbar_init(&st->drain, 1);
    st->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_g);
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
  Items it(a, k0, b0, b_hi);
  const bool any = it.valid();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && any) {
      bool ok = true;
      int q_issued = 0, g_issued = 0;
      mbar_arrive_expect_tx(&st->kv_full, 2 * L::BYTES);
      load_tile(sK, &map_k, L::NCH, k0, p.k_head ? hk : 0, p.k_batch ? b0 : 0, &st->kv_full);
      load_tile(sV, &map_v, L::NCH, k0, p.v_head ? hk : 0, p.v_batch ? b0 : 0, &st->kv_full);
      for (int i = 0; it.valid(); it.next(), ++i) {
        const int s = i % NS;
        // free_[s] next completes for the item loaded here, so the parity wait is unambiguous.
        if (i >= NS && !mbar_wait_bounded(&st->free_[s], (i / NS - 1) & 1, abort_flag, p.err, kErrCrossLoadWait)) {
          ok = false;
          break;
        }
        const int h = hk * group + it.g;
        const long long term = (static_cast<long long>(it.b) * a.hq + h) * p.q_pad + it.qt * TILE;
        mbar_arrive_expect_tx(&st->q_full[s], L::BYTES + 512);
        load_tile(sQ(s), &map_q, L::NCH, it.qt * TILE, p.q_head ? h : 0, p.q_batch ? it.b : 0, &st->q_full[s]);
        bulk_load(terms(s), p.neg_lse2 + term, 512, &st->q_full[s]);
        ++q_issued;
        mbar_arrive_expect_tx(&st->g_full[s], L::BYTES + 512);
        load_tile(sG(s), &map_g, L::NCH, it.qt * TILE, p.g_head ? h : 0, p.g_batch ? it.b : 0, &st->g_full[s]);
        bulk_load(terms(s) + 128, p.neg_d + term, 512, &st->g_full[s]);
        ++g_issued;
      }
      if (!ok) {
        drain_bar(&st->kv_full, 0);
        for (int i = max(0, q_issued - NS); i < q_issued; ++i) drain_bar(&st->q_full[i % NS], (i / NS) & 1);
        for (int i = max(0, g_issued - NS); i < g_issued; ++i) drain_bar(&st->g_full[i % NS], (i / NS) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (whole warp)
    constexpr uint32_t IDESC_S = idesc_bf16_f32(TILE, TILE, 0, 0);
    constexpr uint32_t IDESC_G = idesc_bf16_f32(TILE, D, 0, 1);  // A in TMEM, B MN-major
    bool ok = true, issued = false;
    const auto wait = [&](uint64_t* bar, uint32_t ph) {
      return warp_wait_poll(bar, ph, abort_flag, p.err, kErrCrossMmaWait);
    };
    // [128 keys x 128 queries] = A (keys) B^T (queries), both K-major, into column `col`.
    const auto scores = [&](uint32_t col, const uint8_t* keys, const uint8_t* queries, uint64_t* bar) {
      const uint64_t ad = smem_desc_sw128(smem_u32(keys), 16, 1024), bd = smem_desc_sw128(smem_u32(queries), 16, 1024);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t o16 = ((kk >> 2) * CH + (kk & 3) * 32) >> 4;
        umma_f16_ss_w(tmem + col, ad + o16, bd + o16, IDESC_S, kk > 0 ? 1u : 0u);
      }
      issued = true;
      umma_commit_w(bar);
    };
    // [128 keys x D] (+)= A (weights in TMEM at `col`) B (the item's rows, MN-major).
    const auto grads = [&](uint32_t dst, uint32_t col, const uint8_t* queries, bool first) {
      const uint64_t bd = smem_desc_sw128(smem_u32(queries), CH, 1024);
#pragma unroll
      for (int kk = 0; kk < TILE / 16; ++kk)
        umma_f16_ts_w(tmem + dst, tmem + col + (kk >> 2) * 64 + (kk & 3) * 8, bd + (kk * 2048 >> 4), IDESC_G,
                      (first && kk == 0) ? 0u : 1u);
    };
    // Rows past q_lens that memory holds are zeroed: they would enter both gradients' sums.
    const auto ready = [&](uint64_t* bar, int i, uint8_t* tile, const Items& x) {
      if (!wait(bar, (i / NS) & 1)) return false;
      if (x.qt * TILE + TILE > x.q_end && x.q_end < a.q_len)
        scrub_rows<L::NCH>(tile, [&](int r) { return x.qt * TILE + r < x.q_end; });
      tc_fence_after();
      return true;
    };
    if (any) {
      ok = wait(&st->kv_full, 0) && ready(&st->q_full[0], 0, sQ(0), it);
      if (ok) scores(0, sK, sQ(0), &st->s_full);
      if (ok) ok = ready(&st->g_full[0], 0, sG(0), it);
      if (ok) scores(128, sV, sG(0), &st->dp_full);
      for (int i = 0; ok; ++i) {
        const int s = i % NS, sn = (i + 1) % NS;
        Items nx = it;
        nx.next();
        const bool more = nx.valid();
        // p_full next completes for P(i+1), which needs S(i+1), issued after this wait.
        if (!(ok = wait(&st->p_full, i & 1))) break;
        tc_fence_after();
        grads(256, 0, sG(s), i == 0);
        if (more) {
          if (!(ok = ready(&st->q_full[sn], i + 1, sQ(sn), nx))) break;
          scores(0, sK, sQ(sn), &st->s_full);
        }
        // ds_full next completes for dS(i+1), which needs dP(i+1), issued after this wait.
        if (!(ok = wait(&st->ds_full, i & 1))) break;
        tc_fence_after();
        grads(256 + D, 128, sQ(s), i == 0);
        if (!more) {
          umma_commit_w(&st->done);
          break;
        }
        umma_commit_w(&st->free_[s]);
        if (!(ok = ready(&st->g_full[sn], i + 1, sG(sn), nx))) break;
        scores(128, sV, sG(sn), &st->dp_full);
        it.next();
      }
    }
    if (!ok && issued) {
      umma_commit_w(&st->drain);
      drain_bar(&st->drain, 0);
    }
  } else {
    // ------------------------------------------------------------ P and dS
    const int half = warp >= 6 ? 1 : 0, quarter = warp & 3;
    const int row = quarter * 32 + lane, key = k0 + row;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + lane_base + half * 64, dp_tmem = s_tmem + 128;
    bool ok = true, vis = false, ever = false;
    int vis_b = -1;
    const uint64_t sc2 = pk2(p.scale_log2, p.scale_log2);
    for (int i = 0; it.valid(); it.next(), ++i) {
      const int s = i % NS;
      if (it.b != vis_b) {
        vis_b = it.b;
        vis = key < it.kv_end && (!a.key_mask || a.key_mask[static_cast<long long>(it.b) * a.kv_len + key]);
        ever |= vis;
      }
      // The stage is refilled only after dS(i) of these very warps.
      if (!(ok = warp_wait_poll(&st->q_full[s], (i / NS) & 1, abort_flag, p.err, kErrCrossSoftmaxWait) &&
                 warp_wait_poll(&st->s_full, i & 1, abort_flag, p.err, kErrCrossSoftmaxWait)))
        break;
      tc_fence_after();
      const float4* nl = reinterpret_cast<const float4*>(terms(s) + half * 64);
      uint64_t pr[32];  // this key's weights of 64 queries
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t r[32], w[16];
        tmem_ld32(s_tmem + c * 32, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float4 t = nl[c * 8 + e];
          float x0, x1, x2, x3;
          unpk2(fma2(pk2(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1])), sc2, pk2(t.x, t.y)), x0, x1);
          unpk2(fma2(pk2(__uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3])), sc2, pk2(t.z, t.w)), x2, x3);
          x0 = fast_exp2(x0);
          x1 = fast_exp2(x1);
          x2 = fast_exp2(x2);
          x3 = fast_exp2(x3);
          pr[c * 16 + 2 * e] = vis ? pk2(x0, x1) : 0;
          pr[c * 16 + 2 * e + 1] = vis ? pk2(x2, x3) : 0;
          w[2 * e] = vis ? pack_bf16x2(x0, x1) : 0u;
          w[2 * e + 1] = vis ? pack_bf16x2(x2, x3) : 0u;
        }
        tmem_st16(s_tmem + c * 16, w);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->p_full);
      if (!(ok = warp_wait_poll(&st->g_full[s], (i / NS) & 1, abort_flag, p.err, kErrCrossSoftmaxWait) &&
                 warp_wait_poll(&st->dp_full, i & 1, abort_flag, p.err, kErrCrossSoftmaxWait)))
        break;
      tc_fence_after();
      const float4* nd = reinterpret_cast<const float4*>(terms(s) + 128 + half * 64);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t r[32], w[16];
        tmem_ld32(dp_tmem + c * 32, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float4 t = nd[c * 8 + e];
          float x0, x1, x2, x3;
          unpk2(mul2(pr[c * 16 + 2 * e], add2(pk2(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1])), pk2(t.x, t.y))),
                x0, x1);
          unpk2(mul2(pr[c * 16 + 2 * e + 1],
                     add2(pk2(__uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3])), pk2(t.z, t.w))),
                x2, x3);
          w[2 * e] = vis ? pack_bf16x2(x0, x1) : 0u;  // (a masked value may hold a NaN)
          w[2 * e + 1] = vis ? pack_bf16x2(x2, x3) : 0u;
        }
        tmem_st16(dp_tmem + c * 16, w);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->ds_full);
    }
    if (ok && any) ok = warp_wait_poll(&st->done, 0, abort_flag, p.err, kErrCrossSoftmaxWait);
    if (ok) {
      tc_fence_after();
      // Warps 2..5 store dv, 6..9 dk; a masked key's gradient is 0 whatever its row holds.
      const HeadStrides& gs = half ? a.ks : a.vs;
      const float f = half ? a.scale : 1.0f;
      __nv_bfloat16* out =
          static_cast<__nv_bfloat16*>(half ? p.g.dk : p.g.dv) + b0 * gs.b + hk * gs.h + static_cast<long long>(key) * gs.t;
      const bool store = key < a.kv_len;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld32(tmem + lane_base + 256 + half * D + c, o);
        if (store) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (c + e < a.d) {
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                w[q] = ever ? pack_bf16x2(__uint_as_float(o[e + 2 * q]) * f, __uint_as_float(o[e + 2 * q + 1]) * f) : 0u;
              *reinterpret_cast<uint4*>(out + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        __syncwarp();
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

// ---- backward: dq -------------------------------------------------------------------------------
// One block per SM owns a tile of 128 rows of a (batch, key head) pair (rows as in the forward pass) and
// walks the key tiles: S = Q K^T and dP = dout V^T again, dS back to TMEM as the A operand of
// dQ += dS K (K read MN-major).  Forming S and dP a second time costs two products, 7 instead of 5 in
// the whole backward pass; adding dQ tiles from the kernel above would need either atomics, whose order
// changes the result, or fp32 partial rows of every key tile in memory.
//   warp 0      TMA: K_j and V_j into rings
//   warp 1      MMA: S(0) dP(0) | S(j+1) dQ(j) dP(j+1): S alternates between two TMEM buffers, so it
//               runs ahead while dS(j) is formed; masked rows of K_j are zeroed here
//   warps 2..9  the Q and dout rows into shared memory, then dS: a thread owns a row and half the keys
// TMEM columns: S 0 and 128, dP / dS 256, dQ 384.
template <int D>
struct Dq {
  static constexpr int NCH = D / 64;
  static constexpr int BYTES = NCH * CH;
  static constexpr int NK = D == 64 ? 4 : 3;  // K stages: S(j+1) is issued while K_j serves dQ(j)
  static constexpr int NV = D == 64 ? 4 : 2;
  static constexpr int K_OFF = 2 * BYTES;  // after Q and dout
  static constexpr int V_OFF = K_OFF + NK * BYTES;
  static constexpr int TAIL_OFF = V_OFF + NV * BYTES;
  static constexpr int THREADS = 320;
  struct Tail {
    uint64_t rows_full;  // 8 warp arrivals
    uint64_t k_full[NK], k_free[NK], v_full[NV], v_free[NV];
    uint64_t s_full[2], dp_full, ds_full, done;
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t SMEM = 1024 + TAIL_OFF + sizeof(Tail);
};

template <int D>
__global__ void __launch_bounds__(Dq<D>::THREADS, 1)
    cross_dq_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const GradParams p) {
  using L = Dq<D>;
  constexpr int NK = L::NK, NV = L::NV;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  typename L::Tail* st = reinterpret_cast<typename L::Tail*>(smem + L::TAIL_OFF);
  uint8_t *sQ = smem, *sG = smem + L::BYTES;
  const auto sK = [&](int s) { return smem + L::K_OFF + s * L::BYTES; };
  const auto sV = [&](int s) { return smem + L::V_OFF + s * L::BYTES; };
  const CrossArgs& a = p.g.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.hq / a.hk, rows = group * a.q_len;
  const int row_tiles = (rows + TILE - 1) / TILE;
  const int bh = blockIdx.x / row_tiles, b = bh / a.hk, hk = bh % a.hk;
  const int r0 = (blockIdx.x % row_tiles) * TILE;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const int n = (kv_end + TILE - 1) / TILE;
  {
    const int t = r0 % a.q_len;  // no row of the tile is computed: leave (uniform over the block)
    if (q_end == 0 || (t >= q_end && r0 + a.q_len - t >= min(r0 + TILE, rows))) return;
  }
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;

  if (threadIdx.x == 0) {
    mbar_init(&st->rows_full, 8);
    for (int s = 0; s < NK; ++s) {
      mbar_init(&st->k_full[s], 1);
      mbar_init(&st->k_free[s], 1);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(&st->v_full[s], 1);
      mbar_init(&st->v_free[s], 1);
    }
    mbar_init(&st->s_full[0], 1);
    mbar_init(&st->s_full[1], 1);
    mbar_init(&st->dp_full, 1);
    mbar_init(&st->ds_full, 8);
    mbar_init(&st->done, 1);
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
      for (int j = 0; j < n; ++j) {
        const int s = j % NK, sv = j % NV;
        if (j >= NK && !mbar_wait_bounded(&st->k_free[s], (j / NK - 1) & 1, abort_flag, p.err, kErrCrossLoadWait)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&st->k_full[s], L::BYTES);
        load_tile(sK(s), &map_k, L::NCH, j * TILE, p.k_head ? hk : 0, p.k_batch ? b : 0, &st->k_full[s]);
        ++k_issued;
        if (j >= NV && !mbar_wait_bounded(&st->v_free[sv], (j / NV - 1) & 1, abort_flag, p.err, kErrCrossLoadWait)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&st->v_full[sv], L::BYTES);
        load_tile(sV(sv), &map_v, L::NCH, j * TILE, p.v_head ? hk : 0, p.v_batch ? b : 0, &st->v_full[sv]);
        ++v_issued;
      }
      if (!ok) {
        for (int j = max(0, k_issued - NK); j < k_issued; ++j) drain_bar(&st->k_full[j % NK], (j / NK) & 1);
        for (int j = max(0, v_issued - NV); j < v_issued; ++j) drain_bar(&st->v_full[j % NV], (j / NV) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (whole warp)
    constexpr uint32_t IDESC_S = idesc_bf16_f32(TILE, TILE, 0, 0);
    constexpr uint32_t IDESC_G = idesc_bf16_f32(TILE, D, 0, 1);
    bool ok = true, issued = false;
    const auto wait = [&](uint64_t* bar, uint32_t ph) {
      return warp_wait_poll(bar, ph, abort_flag, p.err, kErrCrossMmaWait);
    };
    const auto scores = [&](uint32_t col, const uint8_t* queries, const uint8_t* keys, uint64_t* bar) {
      const uint64_t ad = smem_desc_sw128(smem_u32(queries), 16, 1024), bd = smem_desc_sw128(smem_u32(keys), 16, 1024);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t o16 = ((kk >> 2) * CH + (kk & 3) * 32) >> 4;
        umma_f16_ss_w(tmem + col, ad + o16, bd + o16, IDESC_S, kk > 0 ? 1u : 0u);
      }
      issued = true;
      umma_commit_w(bar);
    };
    const auto k_ready = [&](int j) {
      if (!wait(&st->k_full[j % NK], (j / NK) & 1)) return false;
      const int kv0 = j * TILE;
      // Masked rows of K enter the sum of dQ with a weight of 0: zeroed, in case they hold a NaN.
      if (mask || (kv0 + TILE > kv_end && kv_end < a.kv_len))
        scrub_rows<L::NCH>(sK(j % NK), [&](int r) { return kv0 + r < kv_end && (!mask || mask[kv0 + r]); });
      tc_fence_after();
      return true;
    };
    if (n > 0) {
      ok = wait(&st->rows_full, 0) && k_ready(0);
      if (ok) scores(0, sQ, sK(0), &st->s_full[0]);
      if (ok) ok = wait(&st->v_full[0], 0);
      if (ok) {
        tc_fence_after();
        scores(256, sG, sV(0), &st->dp_full);
        if (NV < n) umma_commit_w(&st->v_free[0]);
      }
    }
    for (int j = 0; j < n && ok; ++j) {
      if (j + 1 < n) {
        // Buffer (j+1)&1 held S(j-1), which those warps had read before ds_full(j-1).
        if (!(ok = k_ready(j + 1))) break;
        scores(((j + 1) & 1) * 128, sQ, sK((j + 1) % NK), &st->s_full[(j + 1) & 1]);
      }
      // ds_full next completes for dS(j+1), which needs dP(j+1), issued after this wait.
      if (!(ok = wait(&st->ds_full, j & 1))) break;
      tc_fence_after();
      const uint64_t bd = smem_desc_sw128(smem_u32(sK(j % NK)), CH, 1024);
#pragma unroll
      for (int kk = 0; kk < TILE / 16; ++kk)
        umma_f16_ts_w(tmem + 384, tmem + 256 + (kk >> 2) * 64 + (kk & 3) * 8, bd + (kk * 2048 >> 4), IDESC_G,
                      (j == 0 && kk == 0) ? 0u : 1u);
      if (j + 1 == n) {
        umma_commit_w(&st->done);
        break;
      }
      if (j + NK < n) umma_commit_w(&st->k_free[j % NK]);
      if (!(ok = wait(&st->v_full[(j + 1) % NV], ((j + 1) / NV) & 1))) break;
      tc_fence_after();
      scores(256, sG, sV((j + 1) % NV), &st->dp_full);
      if (j + 1 + NV < n) umma_commit_w(&st->v_free[(j + 1) % NV]);
    }
    if (!ok && issued) {
      umma_commit_w(&st->drain);
      drain_bar(&st->drain, 0);
    }
  } else {
    // ------------------------------------------------------------ rows: Q and dout in, dS, dq out
    const int half = warp >= 6 ? 1 : 0, quarter = warp & 3;
    {
      // Warps 2..5 stage Q, 6..9 dout: D/8 lanes to a row, chunk k of row r at k ^ (r & 7).
      constexpr int LPR = D / 8, RPI = 32 / LPR;
      uint8_t* dst = half ? sG : sQ;
      const HeadStrides& ss = half ? a.os : a.qs;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(half ? p.g.dout : a.q) + b * ss.b;
#pragma unroll 4
      for (int i = 0; i < 32 / RPI; ++i) {
        const int r = quarter * 32 + i * RPI + lane / LPR, c = lane % LPR;
        const int g = (r0 + r) / a.q_len, t = (r0 + r) % a.q_len;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (r0 + r < rows && t < q_end && c * 8 < a.d)
          w = __ldg(reinterpret_cast<const uint4*>(src + (hk * group + g) * ss.h + t * ss.t + c * 8));
        *reinterpret_cast<uint4*>(dst + (c >> 3) * CH + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = w;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->rows_full);
    }
    const int row = quarter * 32 + lane, rr = r0 + row;
    const int g = rr / a.q_len, t = rr % a.q_len;
    const bool store = rr < rows && t < q_end;
    const long long term = (static_cast<long long>(b) * a.hq + hk * group + g) * p.q_pad + t;
    const float nl = store ? p.neg_lse2[term] : -INFINITY, nd = store ? p.neg_d[term] : 0.0f;
    const uint64_t sc2 = pk2(p.scale_log2, p.scale_log2), nl2 = pk2(nl, nl), nd2 = pk2(nd, nd);
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t dp_tmem = tmem + lane_base + 256 + half * 64;
    bool ok = true;
    unsigned char byte[4];
    for (int j = 0; j < n; ++j) {
      const int kv0 = j * TILE;
      const bool partial = mask || kv0 + TILE > kv_end;
      if (partial) load_mask_bytes(mask, kv0, kv_end, lane, byte);
      if (!(ok = warp_wait_poll(&st->s_full[j & 1], (j >> 1) & 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
      tc_fence_after();
      unsigned word[2] = {~0u, ~0u};
      if (partial) {
        const unsigned w0 = __ballot_sync(0xffffffffu, byte[0]), w1 = __ballot_sync(0xffffffffu, byte[1]);
        const unsigned w2 = __ballot_sync(0xffffffffu, byte[2]), w3 = __ballot_sync(0xffffffffu, byte[3]);
        word[0] = half ? w2 : w0;
        word[1] = half ? w3 : w1;
      }
      uint64_t pr[32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t r[32];
        tmem_ld32(tmem + lane_base + (j & 1) * 128 + half * 64 + c * 32, r);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          unpk2(fma2(pk2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), sc2, nl2), x0, x1);
          pr[c * 16 + e] = pk2(fast_exp2(x0), fast_exp2(x1));
        }
      }
      if (!(ok = warp_wait_poll(&st->dp_full, j & 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t r[32], w[16];
        tmem_ld32(dp_tmem + c * 32, r);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          unpk2(mul2(pr[c * 16 + e], add2(pk2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), nd2)), x0, x1);
          w[e] = pack_bf16x2(x0, x1);
        }
        if (partial) {  // a masked key's score or value may hold a NaN
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (!((word[c] >> (2 * e)) & 1u)) w[e] &= 0xffff0000u;
            if (!((word[c] >> (2 * e + 1)) & 1u)) w[e] &= 0x0000ffffu;
          }
        }
        tmem_st16(dp_tmem + c * 16, w);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->ds_full);
    }
    if (ok && n > 0) ok = warp_wait_poll(&st->done, 0, abort_flag, p.err, kErrCrossSoftmaxWait);
    if (ok) {
      tc_fence_after();
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.g.dq) + b * a.qs.b + (hk * group + g) * a.qs.h + t * a.qs.t;
#pragma unroll
      for (int c0 = 0; c0 < D / 2; c0 += 32) {
        const int c = half * (D / 2) + c0;  // each half stores half of the columns
        uint32_t o[32];
        tmem_ld32(tmem + lane_base + 384 + c, o);
        if (store) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (c + e < a.d) {
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                w[q] = n > 0 ? pack_bf16x2(__uint_as_float(o[e + 2 * q]) * a.scale,
                                           __uint_as_float(o[e + 2 * q + 1]) * a.scale)
                             : 0u;
              *reinterpret_cast<uint4*>(out + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        __syncwarp();
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

template <class Kernel>
cudaError_t allow_smem(std::atomic<unsigned long long>& done, Kernel k, size_t bytes) {
  return once_per_device(done, [&] {
    return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  });
}

template <int D>
cudaError_t bwd_tc(const CrossGradArgs& g, const float* neg_lse2, const float* neg_d, int q_pad, cudaStream_t s) {
  const CrossArgs& a = g.f;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  HeadMap mq, mg, mk, mv;
  if (!head_map(&mq, a.q, a.qs, a.batch, a.hq, a.q_len, a.d) ||
      !head_map(&mg, g.dout, a.os, a.batch, a.hq, a.q_len, a.d) ||
      !head_map(&mk, a.k, a.ks, a.batch, a.hk, a.kv_len, a.d) ||
      !head_map(&mv, a.v, a.vs, a.batch, a.hk, a.kv_len, a.d))
    return cudaErrorInvalidValue;
  const GradParams p{g,           neg_lse2,   neg_d,       q_pad,      mq.by_head,  mq.by_batch,         mg.by_head,
                     mg.by_batch, mk.by_head, mk.by_batch, mv.by_head, mv.by_batch, a.scale * kLog2e, ctx->err_word};
  if (g.dk) {
    static std::atomic<unsigned long long> attr{0};
    cudaError_t e = allow_smem(attr, cross_dkv_tc_kernel<D>, Dkv<D>::SMEM);
    if (e != cudaSuccess) return e;
    const long long blocks = static_cast<long long>((a.kv_len + TILE - 1) / TILE) * (g.kv_shared ? 1 : a.batch) * a.hk;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    cross_dkv_tc_kernel<D><<<static_cast<unsigned>(blocks), Dkv<D>::THREADS, Dkv<D>::SMEM, s>>>(mq.map, mg.map, mk.map,
                                                                                              mv.map, p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if (g.dq) {
    static std::atomic<unsigned long long> attr{0};
    cudaError_t e = allow_smem(attr, cross_dq_tc_kernel<D>, Dq<D>::SMEM);
    if (e != cudaSuccess) return e;
    const long long rows = static_cast<long long>(a.hq / a.hk) * a.q_len;
    const long long blocks = (rows + TILE - 1) / TILE * a.batch * a.hk;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    cross_dq_tc_kernel<D><<<static_cast<unsigned>(blocks), Dq<D>::THREADS, Dq<D>::SMEM, s>>>(mk.map, mv.map, p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

bool cross_tc_supported(const CrossArgs& a) {
  return a.bf16 && a.d <= 128 && a.d % 8 == 0 && rows16(a.q, a.qs, a.q_len) && rows16(a.k, a.ks, a.kv_len) &&
         rows16(a.v, a.vs, a.kv_len) && rows16(a.out, a.os, a.q_len) && tensor_map_encoder() != nullptr;
}

cudaError_t cross_forward_tc(const CrossArgs& a, cudaStream_t s) {
  return a.d <= 64 ? fwd_tc<64>(a, s) : fwd_tc<128>(a, s);
}

bool cross_grad_tc_supported(const CrossGradArgs& g) {
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  return cross_tc_supported(g.f) && aligned(g.dout) && aligned(g.dq) && aligned(g.dk) && aligned(g.dv);
}

cudaError_t cross_backward_tc(const CrossGradArgs& g, const float* neg_lse2, const float* neg_d, int q_pad,
                              cudaStream_t s) {
  return g.f.d <= 64 ? bwd_tc<64>(g, neg_lse2, neg_d, q_pad, s) : bwd_tc<128>(g, neg_lse2, neg_d, q_pad, s);
}

}  // namespace lcb
