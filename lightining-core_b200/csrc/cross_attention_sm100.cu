// Cross attention in bf16 on the 5th-generation tensor cores: forward and backward for head_dim <= 128
// (a multiple of 8; columns up to 64 or 128 are zeros that TMA fills in).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attention_math.cuh"
#include "common.cuh"
#include "cross_attention.cuh"
#include "lc_internal.hpp"

namespace lcb {

void* tensor_map_encoder();

namespace {

constexpr float kLog2e = 1.4426950408889634f;
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

// Zeroes the rows of a staged tile for which keep(row) is false (one warp).  Swizzling permutes
// inside a row only.  The matrix unit multiplies a masked row by a weight of 0, which would keep a
// NaN or an infinity that memory holds there.
template <int NCH, int ROWS, class Keep>
__device__ __forceinline__ void scrub_rows(uint8_t* tile, Keep keep) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < ROWS / 32; ++i) {
    const int row = i * 32 + lane;
    if (!keep(row))
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(tile + (c * ROWS + row) * 128 + e * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Whether this lane's keys of the tile at kv0 (kv0 + 64 i + lane) are visible; a ballot of byte[i]
// gives every lane the word of those 32 keys.  Loaded ahead of the wait for the scores.
template <int N>
__device__ __forceinline__ void load_mask_bytes(const unsigned char* mask, int kv0, int kv_end, int lane,
                                                unsigned char (&byte)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = kv0 + i * 64 + lane;
    byte[i] = k < kv_end && (!mask || mask[k]);
  }
}

// ---- forward ----------------------------------------------------------------------------------
// One block per SM owns two tiles of 128 rows (A and B) of a (batch, key head) pair, which share every
// K and V tile of 128 keys.  A row is (head in the group, token), so short queries of a group fill a
// tile together.  Roles (19 warps):
//   warp 0      TMA: K_j and V_j into rings of NS stages
//   warp 1      MMA: S_h = Q_h K_j^T, O_h += P_h V_j for h = A, B (at head_dim 128 in the order PV_A(j), S_A(j+1),
//               PV_B(j), S_B(j+1)), so that one tile's softmax runs beside the other's products; the warp
//               of the products with V also zeroes the masked rows of V_j
//   warps 2..9  rows of A (warps 10..17: of B): the Q rows into shared memory, then softmax -- two threads
//               to a row (one TMEM lane), 32 of every 64 keys of a tile and half of the output columns each,
//               which swap the row's maximum through tagged words in shared memory -- and the epilogue
//   warp 18     at head_dim 64: the products with V, while warp 1 issues the scores
// TMEM: S_A 0, S_B 128.  At head_dim 64 P_A 256, P_B 320, O_A 384, O_B 448, and S_h(j+1) is issued when S_h(j)
// is in the softmax warps' registers; at 128 O_A 256, O_B 384 leave P_h (bf16 pairs) to lie over the first half
// of S_h.  The products with the first 64 weights of a step start while the other 64 are formed (at 128 509 us
// instead of 527 over the same inputs).  O is rescaled only when a row's maximum grows by more than
// 2^8 (the final division makes up for it).  P is rounded to bf16 for the second product, 2^-8 of a weight at most and
// unbiased; the row's sum takes the unrounded weights.
// Bound by the issue slots and dependent steps of the softmax warps: about 3500 cycles a pair of tiles at head_dim 64
// (MUFU 2048 of them, the products 1130) and 4300 at 128, where S, P and the sums of a tile follow one another (2200).
// B200, inputs not in L2: [16, 16, 512 x 2048 ragged, 64] 112 us, [8, 16/4, 2048 x 4096, 128] 585 us (0.94 PFLOP/s;
// called again and again on the same inputs 517); the CUDA cores took 1937 us and 22.6 ms.  At 64, where this took 111, one
// issuing warp and P over S took 127; one thread to a row (8 warps fewer) 116; a fourth of the exponentials by a
// polynomial on the FMA pipes, which pays in the self attention kernel, 113.
template <int D>
struct Fwd {
  static constexpr int NCH = D / 64;
  static constexpr int BYTES = NCH * CH;     // a Q, K or V tile
  static constexpr int NS = D == 64 ? 4 : 2; // ring stages
  static constexpr int K_OFF = 2 * BYTES;
  static constexpr int V_OFF = K_OFF + NS * BYTES;
  static constexpr int TAIL_OFF = V_OFF + NS * BYTES;
  static constexpr int THREADS = 608;
  struct Tail {
    unsigned long long swap[2][2][2][TILE];  // [tile][step & 1][half][row], tagged with the step
    uint64_t q_full[2];             // 8 warp arrivals
    uint64_t k_full[NS], v_full[NS];
    uint64_t k_free[NS], v_free[NS];
    uint64_t s_full[2], s_read[2], p_half[2], p_full[2], o_done[2];  // p_half: weights of 64 keys
    uint64_t drain[2];
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t SMEM = 1024 + TAIL_OFF + sizeof(Tail);
  static constexpr bool OWN_P = D == 64;  // P has columns of its own
  static constexpr uint32_t P_COL = OWN_P ? 256 : 0, P_STEP = OWN_P ? 64 : 128, O_COL = OWN_P ? 384 : 256, O_STEP = D;
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
  griddep_launch_dependents();  // the parts' join waits for the end of this grid
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
      mbar_init(&st->q_full[h], 8);
      mbar_init(&st->s_full[h], 1);
      mbar_init(&st->s_read[h], 8);
      mbar_init(&st->p_half[h], 8);
      mbar_init(&st->p_full[h], 8);
      mbar_init(&st->o_done[h], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&st->drain[i], 1);
    st->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  for (int i = threadIdx.x; i < 8 * TILE; i += F::THREADS) (&st->swap[0][0][0][0])[i] = ~0ull;
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
  } else if (warp == 1 || warp == 18) {
    // ------------------------------------------------------------ MMA issuers (whole warps)
    constexpr uint32_t IDESC_S = idesc_bf16_f32(TILE, TILE, 0, 0);  // Q and K K-major
    constexpr uint32_t IDESC_O = idesc_bf16_f32(TILE, D, 0, 1);     // P in TMEM, V MN-major
    bool ok = true, issued = false;
    const auto wait = [&](uint64_t* bar, uint32_t ph) {
      return warp_wait_ready(bar, ph, abort_flag, p.err, kErrCrossMmaWait);
    };
    const auto issue_s = [&](int h, int j) {
      const uint64_t qd = smem_desc_sw128(smem_u32(sQ(h)), 16, 1024);
      const uint64_t kd = smem_desc_sw128(smem_u32(sK(j % NS)), 16, 1024);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        umma_f16_ss4_w(tmem + h * 128, qd + (c * CH >> 4), kd + (c * CH >> 4), IDESC_S, c > 0 ? 1u : 0u);
      issued = true;
      umma_commit_w(&st->s_full[h]);
    };
    const auto issue_pv = [&](int h, int j, int part) {
      const uint64_t vd = smem_desc_sw128(smem_u32(sV(j % NS)), CH, 1024);
      const uint32_t o = tmem + F::O_COL + h * F::O_STEP, pr = tmem + F::P_COL + h * F::P_STEP;
      umma_f16_ts4_w(o, pr + part * 32, vd + part * (4 * 2048 >> 4), IDESC_O, j > 0 || part > 0 ? 1u : 0u);
    };
    // Scores of step j (their K tile has been waited for).
    const auto scores = [&](int h, int j) {
      tc_fence_after();
      issue_s(h, j);
    };
    // Weights of step j times V, 64 keys at a time; p_half[h] and p_full[h] next complete for P_h(j+1), which needs
    // what is issued after these waits.
    const auto sums = [&](int h, int j) {
      if (!wait(&st->p_half[h], j & 1)) return false;
      tc_fence_after();
      issue_pv(h, j, 0);
      issued = true;
      if (!wait(&st->p_full[h], j & 1)) return false;
      tc_fence_after();
      issue_pv(h, j, 1);
      umma_commit_w(&st->o_done[h]);
      return true;
    };
    // V of step j, its masked rows zeroed: keys past kv_end that memory holds (TMA zero-fills past kv_len), and holes.
    const auto values = [&](int j) {
      const int s = j % NS, kv0 = (t_lo + j) * TILE;
      if (!wait(&st->v_full[s], (j / NS) & 1)) return false;
      if (mask || (kv0 + TILE > kv_end && kv_end < a.kv_len))
        scrub_rows<F::NCH, TILE>(sV(s), [&](int r) { return kv0 + r < kv_end && (!mask || mask[kv0 + r]); });
      return true;
    };
    if (n > 0 && warp == 1) {
      for (int h = 0; h < 2 && ok; ++h) {
        if (!act[h]) continue;
        if (F::OWN_P && h == 1 && act[0]) ok = wait(&st->p_half[0], 0);
        if (ok && (ok = wait(&st->q_full[h], 0) && wait(&st->k_full[0], 0))) scores(h, 0);
      }
      if (ok && NS < n) umma_commit_w(&st->k_free[0]);
    }
    // Commits cover everything issued so far, so one after both tiles' last product with a stage hands it back.
    // Only stages that are loaded again are, so no arrival is left in flight at the end.
    for (int j = 0; j < n && ok && (F::OWN_P || warp == 1); ++j) {
      const auto k_used = [&] {
        if (j + 1 + NS < n) umma_commit_w(&st->k_free[(j + 1) % NS]);
      };
      const auto next_keys = [&] { return j + 1 >= n || wait(&st->k_full[(j + 1) % NS], ((j + 1) / NS) & 1); };
      if constexpr (F::OWN_P) {
        // Tile B is half a step behind A (its first scores wait for A's first weights): one tile's exponentials
        // run beside the rest of the other's softmax.
        if (warp == 1) {
          if (j + 1 == n || !(ok = next_keys())) break;
          for (int h = 0; h < 2 && ok; ++h)  // s_read[h] next completes for S_h(j+1)
            if (act[h] && (ok = wait(&st->s_read[h], j & 1))) scores(h, j + 1);
          if (ok) k_used();
        } else {
          ok = values(j);
          for (int h = 0; h < 2 && ok; ++h)
            if (act[h]) ok = sums(h, j);
          if (ok && j + NS < n) umma_commit_w(&st->v_free[j % NS]);
        }
      } else {
        if (!(ok = values(j))) break;
        for (int h = 0; h < 2 && ok; ++h) {
          if (!act[h]) continue;
          if (!(ok = sums(h, j) && next_keys())) break;
          if (j + 1 < n) scores(h, j + 1);
        }
        if (!ok) break;
        if (j + NS < n) umma_commit_w(&st->v_free[j % NS]);
        k_used();
      }
    }
    if (!ok && issued) {
      umma_commit_w(&st->drain[warp & 1]);
      drain_bar(&st->drain[warp & 1], 0);
    }
  } else {
    // ------------------------------------------------------------ rows of tile h
    const int h = warp >= 10 ? 1 : 0, half = ((warp - 2) >> 2) & 1;
    const int quarter = warp & 3;  // TMEM lanes a warp may read
    const int base = r0 + h * TILE;
    if (act[h]) {
      // Q rows into shared memory: D/8 lanes to a row, 16 bytes each, chunk k of row r at k ^ (r & 7).
      constexpr int LPR = D / 8, RPI = 32 / LPR;
      uint8_t* q = sQ(h);
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) + b * a.qs.b;
#pragma unroll 4
      for (int i = 0; i < 16 / RPI; ++i) {
        const int r = quarter * 32 + half * 16 + i * RPI + lane / LPR, c = lane % LPR;
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
      const uint32_t p_tmem = tmem + lane_base + F::P_COL + h * F::P_STEP + half * 16;
      const uint32_t o_tmem = tmem + lane_base + F::O_COL + h * F::O_STEP;
      constexpr int OC = D / 2;
      const float floor = cross_floor(p.scale_log2);
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      unsigned char byte[2];
      // Publishes v under `tag` and fetches the other half's value of the same tag.  A slot is written again
      // two steps later, when the partner, which has published the step between, has read it.  Both
      // halves' scores are in registers by then: P may be written over them.
      const auto swap = [&](uint32_t tag, float v, float* other) {
        *reinterpret_cast<volatile unsigned long long*>(&st->swap[h][tag & 1][half][row]) =
            (static_cast<unsigned long long>(tag) << 32) | __float_as_uint(v);
        volatile unsigned long long* theirs = &st->swap[h][tag & 1][half ^ 1][row];
        unsigned long long x = *theirs;
        bool got = static_cast<uint32_t>(x >> 32) == tag;
        if (!got) {
          const uint64_t t0 = globaltimer_ns();
          uint32_t spins = 0;
          while (!(got = static_cast<uint32_t>((x = *theirs) >> 32) == tag)) {
            if (*abort_flag) break;
            if ((++spins & 63u) == 0 && globaltimer_ns() - t0 > LC_WAIT_TIMEOUT_NS) {
              *abort_flag = 1;
              atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCrossSoftmaxWait));
              break;
            }
          }
        }
        *other = __uint_as_float(static_cast<uint32_t>(x));
        return __all_sync(0xffffffffu, got) != 0;
      };
      for (int j = 0; j < n; ++j) {
        const int kv0 = (t_lo + j) * TILE;
        const bool partial = mask || kv0 + TILE > kv_end;
        if (partial) load_mask_bytes(mask, kv0 + half * 32, kv_end, lane, byte);
        // s_full[h] next completes for S_h(j+1), which needs P_h(j) from these warps first.
        if (!(ok = warp_wait_ready(&st->s_full[h], j & 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
        tc_fence_after();
        uint32_t r[2][32];  // keys half * 32.. and 64 + half * 32..
        tmem_ld32(s_tmem + half * 32, r[0]);
        tmem_ld32(s_tmem + 64 + half * 32, r[1]);
        if (F::OWN_P) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&st->s_read[h]);
        }
        float lowest = floor;  // of the maximum, unless this half sees no key
        if (partial) {
          lowest = -INFINITY;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const unsigned w = __ballot_sync(0xffffffffu, byte[c]);
            if (w) lowest = floor;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((w >> e) & 1u)) r[c][e] = __float_as_uint(-INFINITY);
          }
        }
        float pm[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pm[i] = __uint_as_float(r[0][i]);
#pragma unroll
        for (int e = 8; e < 64; e += 2)
          pm[(e >> 1) & 7] = max3(pm[(e >> 1) & 7], __uint_as_float(r[e >> 5][e & 31]), __uint_as_float(r[e >> 5][(e & 31) + 1]));
        float mx = max3(max3(pm[0], pm[1], pm[2]), max3(pm[3], pm[4], pm[5]), max3(pm[6], pm[7], lowest)), mo;
        if (!(ok = swap(static_cast<uint32_t>(j), mx, &mo))) break;
        mx = fmaxf(mx, mo) * p.scale_log2;
        const bool need = mx > m + kRescale;
        float factor = 1.0f;
        if (need) {
          factor = m == -INFINITY ? 0.0f : exp2f(m - mx);
          l *= factor;
          m = mx;
        }
        const bool rescale = __any_sync(0xffffffffu, need);
        if (j > 0 && (rescale || F::OWN_P)) {
          // O_h is rescaled in place, and columns of P's own are read by PV_h(j-1): it must have landed (o_done[h]
          // next completes for PV_h(j), which needs this tile's P).
          if (!(ok = warp_wait_ready(&st->o_done[h], (j - 1) & 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
          tc_fence_after();
        }
        if (j > 0 && rescale) {
#pragma unroll 1
          for (int c = half * OC; c < half * OC + OC; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_tmem + c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st16(o_tmem + c, o);
          }
          tmem_wait_st();
        }
        // A row that has seen no key yet has m = -inf: every score is -inf too and its weights are 0 (cross_floor).
        const float mu = m == -INFINITY ? 0.0f : m;
        const uint64_t sc2 = pk2(p.scale_log2, p.scale_log2), nm2 = pk2(-mu, -mu);
        uint64_t ps2[4] = {0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x0, x1, e0, e1;
            unpk2(fma2(pk2(__uint_as_float(r[g][2 * i]), __uint_as_float(r[g][2 * i + 1])), sc2, nm2), x0, x1);
            e0 = fast_exp2(x0);
            e1 = fast_exp2(x1);
            ps2[i & 3] = add2(ps2[i & 3], pk2(e0, e1));
            w[i] = pack_bf16x2(e0, e1);
          }
          tmem_st16(p_tmem + g * 32, w);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(g == 0 ? &st->p_half[h] : &st->p_full[h]);
        }
        float x, y;
        unpk2(add2(add2(ps2[0], ps2[1]), add2(ps2[2], ps2[3])), x, y);
        l += x + y;
      }
      if (ok && n > 0)
        ok = warp_wait_ready(&st->o_done[h], (n - 1) & 1, abort_flag, p.err, kErrCrossSoftmaxWait);
      float other = 0.0f;
      if (ok && n > 0) ok = swap(static_cast<uint32_t>(n), l, &other);
      if (ok) {
        l = half == 0 ? l + other : other + l;  // the same sum in both
        tc_fence_after();
        const int rr = base + row, g = rr / a.q_len, t = rr % a.q_len;
        const bool store = rr < rows && t < q_end;
        const bool empty = m == -INFINITY;  // no visible key
        const long long at = (static_cast<long long>(b) * a.hq + hk * group) * a.q_len + rr;  // dense row
        const bool split = p.sp.splits > 1;
        const float inv = split ? 1.0f : cross_inverse(m, l);
        if (store && half == 0) {
          if (split)
            p.sp.ml[static_cast<long long>(blockIdx.y) * p.sp.rows + at] = make_float2(m, empty ? 0.0f : l);
          else if (a.lse)
            a.lse[at] = cross_lse(m, l);
        }
        float* part = p.sp.o + (static_cast<long long>(blockIdx.y) * p.sp.rows + at) * a.d;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + b * a.os.b + (hk * group + g) * a.os.h + t * a.os.t;
        // tcgen05.ld is warp-collective: every lane loads, only live rows store.
#pragma unroll
        for (int cc = 0; cc < OC; cc += 32) {
          const int c = half * OC + cc;
          uint32_t o[32];
          __syncwarp();
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

// ---- backward -----------------------------------------------------------------------------------
// One kernel walks both ways over the score matrix.  A job keeps 128 rows of one side and streams tiles of
// 64 rows of the other ("items"):
//   KV    rows are keys (X1 = K, X2 = V), items are queries of the group's heads, and of every batch
//         entry in turn when k and v are shared by them (Y1 = Q, Y2 = dout): writes dk and dv
//   else  rows are queries as in the forward pass (X1 = Q, X2 = dout), items are keys (Y1 = K, Y2 = V):
//         writes dq
// With S = X1 Y1^T, P = exp(S - lse), dP = X2 Y2^T, dS = P (dP - D), the sums over the items are
// A1 += P Y2 (dv) and A2 += dS Y1 (dk or dq), both kept in TMEM.  P and dS are formed with a row per TMEM
// lane, rounded to bf16 as the forward pass rounds its weights (the matrix unit's type; sums stay fp32), and go
// back into TMEM columns of their own as the A operands; Y1 and Y2 are read as they lie, MN-major: nothing is
// transposed.  Forming S and dP once for each side costs two products, 7 instead of 5; taking dq from the
// walk that yields dk and dv would need atomics, whose order changes the result, or fp32 partial rows of
// every key tile in memory.
// What bounds it is keeping three things busy at once that depend on each other: the tensor pipe (64-row
// items: 650 cycles at head_dim 64, 1120 at 128), MUFU (512 cycles) and the issue slots of the warps that
// form P and dS; a wait and a commit cost the issuing warp some 100 cycles each.  Hence
//   * X1 and X2 in TMEM as A operands: an N = 64 product then takes 36 cycles a step instead of 53 (its
//     operands in shared memory are what binds it), and shared memory holds more items
//   * P and dS in columns of their own, so the score columns are free as soon as they have been read, and the
//     next item's products run while this one's weights are formed (through shared memory instead, each warp's
//     fence towards the matrix unit cost 600 cycles an item)
//   * two groups of eight warps that take the items in turn
//   * three issuing warps, for S, dP and the sums, which order each other by barriers only
//   * resident blocks that go from job to job: four more warps load the next job's rows and store
//     the last one's sums meanwhile (two sets of TMEM columns where they fit)
// B200, row terms included: [16, 16, 512 x 2048 ragged, 64] 296 us with inputs that are not in L2, 261 called again and
// again on the same (blocks of one job with one chain of products: 471), [4, 16/4, 1024 x 2048 ragged, 128] 213 and 189
// (266).  The times of single steps below and in the launches are such repeated calls'.
constexpr int QT = 64;         // rows of an item
constexpr int QCH = QT * 128;  // one [64 rows x 64 bf16] box
template <int D, bool KV>
struct Grad {
  static constexpr int NCH = D / 64;
  static constexpr int BYTES = NCH * QCH;    // a Y tile
  static constexpr int STAGE = 2 * BYTES;
  static constexpr bool X_SMEM = KV && D == 128;     // rows in shared memory, the TMEM columns are taken
  static constexpr int NS = D == 64 ? 8 : 4;
  static constexpr int NX = D == 64 ? 2 : 1;         // sets of rows
  static constexpr int NA = D == 64 && !KV ? 2 : 1;  // sets of sums
  static constexpr int X_OFF = NS * STAGE;           // [2][128 x D] bf16
  static constexpr int TERM_OFF = X_OFF + (X_SMEM ? 2 * NCH * CH : 0);  // [NS][2][64] floats (KV)
  // Boxes of [128 rows x 64 bf16]: next rows on their way to TMEM, and sums on their way to memory (as many
  // as fit), a quarter to each of the four warps that move rows.
  static constexpr int IN_OFF = TERM_OFF + (KV ? NS * 512 : 0);
  static constexpr int OUT_OFF = IN_OFF + (X_SMEM ? 0 : 2 * NCH * CH);
  static constexpr int OUTS = X_SMEM ? 1 : (KV ? 2 : 1) * NCH;
  static constexpr int TAIL_OFF = OUT_OFF + OUTS * CH;
  static constexpr int THREADS = 24 * 32;
  // TMEM columns: rows, S, dP, P and dS of the two groups, sums.
  static constexpr uint32_t X = 0, XW = X_SMEM ? 0 : D, S = NX * XW, DP = S + 64, P = DP + 64, DS = P + (KV ? 64 : 0),
                            A = DS + 64, AW = KV ? 2 * D : D;
  static_assert(A + NA * AW <= 512, "TMEM");
  struct Tail {
    uint64_t full[NS], free_[NS];
    uint64_t x_full[NX], done[NA], sums_free[NA], in_full, in_free;
    uint64_t s_full[2], dp_full[2], p_full[2], ds_full[2], used[2];  // by group
    uint64_t s_read, dp_read;
    uint64_t drain[3];
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t SMEM = TAIL_OFF + sizeof(Tail);
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct GradParams {
  CrossGradArgs g;
  const float *neg_lse2, *neg_d;
  int q_pad;
  int y1_head, y1_batch, y2_head, y2_batch;  // 1: the map of the streamed tensor has that axis
  int x1_head, x1_batch, x2_head, x2_batch;  // KV: the same of k and v, and of their gradients
  int jobs, tiles;                           // tiles of rows of a (batch, key head) pair
  int group, step_tile, step_hk, step_b;     // rows' heads to a key head; the grid's size in jobs' digits
  int beside;                                // the dq walk may run beside the other
  float scale_log2;
  unsigned* err;
};

// A job's rows.  Its items are, in order: the batch entries [b, b_hi) with span() > 0, `heads` heads each, tiles
// of 64 rows up to span().
// A block goes from job to job by adding the grid's size in (batch entry, key head, tile) digits (with divisions
// 270 and 188 us below, without 267 and 185).
template <bool KV>
struct Job {
  int job, b, hk, tile;
  __device__ explicit Job(const GradParams& p) {
    job = blockIdx.x;
    tile = job % p.tiles;
    hk = job / p.tiles % p.g.f.hk;
    b = job / p.tiles / p.g.f.hk;
  }
  __device__ void step(const GradParams& p) {
    job += gridDim.x;
    tile += p.step_tile;
    hk += p.step_hk;
    b += p.step_b;
    if (tile >= p.tiles) tile -= p.tiles, ++hk;
    if (hk >= p.g.f.hk) hk -= p.g.f.hk, ++b;
  }
  __device__ int r0() const { return tile * TILE; }
  __device__ int b_hi(const GradParams& p) const { return KV && p.g.kv_shared ? p.g.f.batch : b + 1; }
  __device__ int heads(const GradParams& p) const { return KV ? p.group : 1; }
  // Rows of batch entry yb to walk (0: none), for KV the queries if the tile has a key to see, else the keys if
  // the tile has a query to compute: its first row's token is one, or another head starts in it.
  __device__ int span(const GradParams& p, int yb) const {
    const CrossArgs& a = p.g.f;
    const int q_end = cross_len(a.q_lens, yb, a.q_len), kv_end = cross_len(a.kv_lens, yb, a.kv_len);
    if (KV) return r0() < kv_end ? q_end : 0;
    if (q_end == a.q_len) return kv_end;
    const int t = r0() % a.q_len;
    return q_end > 0 && (t < q_end || r0() + a.q_len - t < min(r0() + TILE, p.group * a.q_len)) ? kv_end : 0;
  }
  __device__ int count(const GradParams& p) const {
    int n = 0;
    for (int yb = b; yb < b_hi(p); ++yb) n += heads(p) * ((span(p, yb) + QT - 1) / QT);
    return n;
  }
};

template <int D, bool KV>
__global__ void __launch_bounds__(Grad<D, KV>::THREADS, 1)
    cross_grad_tc_kernel(const __grid_constant__ CUtensorMap map_y1, const __grid_constant__ CUtensorMap map_y2,
                         const __grid_constant__ CUtensorMap map_x1, const __grid_constant__ CUtensorMap map_x2,
                         const __grid_constant__ CUtensorMap map_dk, const __grid_constant__ CUtensorMap map_dv,
                         const GradParams p) {
  using L = Grad<D, KV>;
  constexpr int NS = L::NS, NX = L::NX, NA = L::NA;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {  // the 128-byte swizzle atoms need 1 KB alignment
    if (threadIdx.x == 0) atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCrossLoadWait) | 0x1000u);
    return;
  }
  typename L::Tail* st = reinterpret_cast<typename L::Tail*>(smem + L::TAIL_OFF);
  const auto sY1 = [&](int s) { return smem + s * L::STAGE; };
  const auto sY2 = [&](int s) { return smem + s * L::STAGE + L::BYTES; };
  const auto terms = [&](int s) { return reinterpret_cast<float*>(smem + L::TERM_OFF + s * 512); };
  const CrossArgs& a = p.g.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&st->full[s], 1);
      mbar_init(&st->free_[s], 1);
    }
    for (int x = 0; x < NX; ++x) mbar_init(&st->x_full[x], L::X_SMEM ? 1 : 4);
    mbar_init(&st->in_full, 1);
    mbar_init(&st->in_free, 4);
    for (int x = 0; x < NA; ++x) {
      mbar_init(&st->done[x], 1);
      mbar_init(&st->sums_free[x], 4);
    }
    for (int c = 0; c < 2; ++c) {
      mbar_init(&st->s_full[c], 1);
      mbar_init(&st->dp_full[c], 1);
      mbar_init(&st->p_full[c], 8);
      mbar_init(&st->ds_full[c], 8);
      mbar_init(&st->used[c], 1);
    }
    for (int c = 0; c < 3; ++c) mbar_init(&st->drain[c], 1);
    mbar_init(&st->s_read, 8);
    mbar_init(&st->dp_read, 8);
    st->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_y1);
    tma_prefetch_desc(&map_y2);
    if (KV) {
      tma_prefetch_desc(&map_x1);
      tma_prefetch_desc(&map_x2);
      tma_prefetch_desc(&map_dk);
      tma_prefetch_desc(&map_dv);
    }
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
  // The row terms, and whatever ran before.  The dq walk may start once every block of the other one has passed
  // here, and takes the SMs that its last jobs leave idle; it is not over before the other is (see the end).
  if (KV || !p.beside) griddep_wait();
  if (KV) griddep_launch_dependents();
  // Every role counts the items it has passed (i) and the jobs that have some (x); item i belongs to group
  // i & 1 and stage i % NS, job x to columns x % NX and x % NA.  Each barrier's next completion needs
  // what its waiters do after this one, so no parity wait is ambiguous.

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    bool ok = true;
    int i = 0, x = 0;
    for (Job<KV> j(p); j.job < p.jobs && ok; j.step(p)) {
      if (KV) {
        if (j.count(p) == 0) {
          // No query sees a key of this tile: zeros, a row's pieces to neighbouring lanes.
          const int vecs = a.d / 8;
          __nv_bfloat16* dk = static_cast<__nv_bfloat16*>(p.g.dk) + j.b * a.ks.b + j.hk * a.ks.h;
          __nv_bfloat16* dv = static_cast<__nv_bfloat16*>(p.g.dv) + j.b * a.vs.b + j.hk * a.vs.h;
          for (int k = lane; k < TILE * vecs; k += 32) {
            const int key = j.r0() + k / vecs, c = k % vecs * 8;
            if (key >= a.kv_len) break;
            *reinterpret_cast<uint4*>(dk + key * a.ks.t + c) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(dv + key * a.vs.t + c) = make_uint4(0, 0, 0, 0);
          }
          __syncwarp();
          continue;
        }
        // The job's rows: into their boxes once the last ones have left them, or (X_SMEM) to where they stay once
        // the last job is done.
        uint64_t *const bar = L::X_SMEM ? &st->x_full[0] : &st->in_full, *const before = L::X_SMEM ? &st->done[0] : &st->in_free;
        if (lane == 0) {
          ok = x == 0 || mbar_wait_bounded_backoff(before, (x - 1) & 1, abort_flag, p.err, kErrCrossLoadWait, 32);
          if (ok) {
            uint8_t* box = smem + (L::X_SMEM ? L::X_OFF : L::IN_OFF);
            mbar_arrive_expect_tx(bar, 2 * L::NCH * CH);
            load_tile(box, &map_x1, L::NCH, j.r0(), p.x1_head ? j.hk : 0, p.x1_batch ? j.b : 0, bar);
            load_tile(box + L::NCH * CH, &map_x2, L::NCH, j.r0(), p.x2_head ? j.hk : 0, p.x2_batch ? j.b : 0, bar);
          }
        }
        ++x;
      }
      if (lane == 0)
        for (int yb = j.b; yb < j.b_hi(p) && ok; ++yb) {
          const int y_end = j.span(p, yb);
          for (int g = 0; g < j.heads(p) && ok; ++g)
            for (int t0 = 0; t0 < y_end; t0 += QT, ++i) {
              const int s = i % NS;
              if (i >= NS &&
                  !mbar_wait_bounded_backoff(&st->free_[s], (i / NS - 1) & 1, abort_flag, p.err, kErrCrossLoadWait, 32)) {
                ok = false;
                break;
              }
              const int h = KV ? j.hk * p.group + g : j.hk;
              mbar_arrive_expect_tx(&st->full[s], L::STAGE + (KV ? 512 : 0));
              for (int c = 0; c < L::NCH; ++c)
                tma_load_4d(sY1(s) + c * QCH, &map_y1, c * 64, t0, p.y1_head ? h : 0, p.y1_batch ? yb : 0, &st->full[s]);
              for (int c = 0; c < L::NCH; ++c)
                tma_load_4d(sY2(s) + c * QCH, &map_y2, c * 64, t0, p.y2_head ? h : 0, p.y2_batch ? yb : 0, &st->full[s]);
              if (KV) {
                const long long term = (static_cast<long long>(yb) * a.hq + h) * p.q_pad + t0;
                bulk_load(terms(s), p.neg_lse2 + term, 256, &st->full[s]);
                bulk_load(terms(s) + 64, p.neg_d + term, 256, &st->full[s]);
              }
            }
        }
      ok = __all_sync(0xffffffffu, ok);
    }
    if (!ok && lane == 0) {
      for (int k = max(0, i - NS); k < i; ++k) drain_bar(&st->full[k % NS], (k / NS) & 1);
      if (KV && x > 0) drain_bar(L::X_SMEM ? &st->x_full[0] : &st->in_full, (x - 1) & 1);
    }
  } else if (warp < 3) {
    // ------------------------------------------------------------ S (warp 1) and dP (warp 2), whole warps
    constexpr uint32_t IDESC = idesc_bf16_f32(TILE, QT, 0, 0);
    const int which = warp - 1;
    uint64_t *const read = which ? &st->dp_read : &st->s_read, *const ready = which ? st->dp_full : st->s_full;
    const uint32_t col = tmem + (which ? L::DP : L::S);
    bool ok = true;
    const auto wait = [&](uint64_t* bar, uint32_t ph) {
      return warp_wait_ready(bar, ph, abort_flag, p.err, kErrCrossMmaWait);
    };
    int i = 0, x = 0;
    for (Job<KV> j(p); j.job < p.jobs && ok; j.step(p)) {
      const uint32_t rows = tmem + L::X + (x % NX) * L::XW + which * (D / 2);
      bool first = true;
      for (int yb = j.b; yb < j.b_hi(p) && ok; ++yb) {
        const int y_end = j.span(p, yb), y_len = KV ? a.q_len : a.kv_len;
        const unsigned char* mask = !KV && a.key_mask ? a.key_mask + static_cast<long long>(yb) * a.kv_len : nullptr;
        for (int g = 0; g < j.heads(p) && ok; ++g)
          for (int t0 = 0; t0 < y_end; t0 += QT, ++i) {
            const int s = i % NS;
            uint8_t* y = which ? sY2(s) : sY1(s);
            if (first && !(ok = wait(&st->x_full[x % NX], (x / NX) & 1))) break;
            first = false;
            if (!(ok = wait(&st->full[s], (i / NS) & 1))) break;
            // Rows that memory holds but that do not count are zeroed: their weights are 0, but a NaN
            // would enter the sums all the same (Y2 of the dq walk, V, enters none).
            if ((KV || !which) && (mask || (t0 + QT > y_end && y_end < y_len))) {
              const auto keep = [&](int r) { return t0 + r < y_end && (!mask || mask[t0 + r]); };
              scrub_rows<L::NCH, QT>(y, keep);
              // dv reads Y2 as soon as P is there, which waits for S and not for dP: here too, whoever comes first.
              if (KV && !which) scrub_rows<L::NCH, QT>(sY2(s), keep);
            }
            if (i > 0 && !(ok = wait(read, (i - 1) & 1))) break;
            tc_fence_after();
            const uint64_t bd = smem_desc_sw128(smem_u32(y), 16, 1024);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              if constexpr (L::X_SMEM)
                umma_f16_ss4_w(col, smem_desc_sw128(smem_u32(smem + L::X_OFF + (which * L::NCH + c) * CH), 16, 1024),
                               bd + (c * QCH >> 4), IDESC, c > 0 ? 1u : 0u);
              else
                umma_f16_ts4k_w(col, rows + c * 32, bd + (c * QCH >> 4), IDESC, c > 0 ? 1u : 0u);
            umma_commit_w(&ready[i & 1]);
          }
      }
      if (!first) ++x;
    }
    if (!ok) {
      umma_commit_w(&st->drain[which]);
      drain_bar(&st->drain[which], 0);
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ the sums (whole warp)
    constexpr uint32_t IDESC = idesc_bf16_f32(TILE, D, 0, 1);  // Y MN-major
    bool ok = true;
    const auto wait = [&](uint64_t* bar, uint32_t ph) {
      return warp_wait_ready(bar, ph, abort_flag, p.err, kErrCrossMmaWait);
    };
    int i = 0, x = 0;
    for (Job<KV> j(p); j.job < p.jobs && ok; j.step(p)) {
      const int n = j.count(p);
      if (n == 0) continue;
      const uint32_t sums = tmem + L::A + (x % NA) * L::AW;
      if (x >= NA && !(ok = wait(&st->sums_free[x % NA], (x / NA - 1) & 1))) break;
      for (int k = 0; k < n; ++k, ++i) {
        const int s = i % NS, c = i & 1;
        const uint32_t ph = (i >> 1) & 1, add = k > 0 ? 1u : 0u;
        if (KV) {
          if (!(ok = wait(&st->p_full[c], ph))) break;
          tc_fence_after();
          umma_f16_ts4_w(sums, tmem + L::P + c * 32, smem_desc_sw128(smem_u32(sY2(s)), QCH, 1024), IDESC, add);
        }
        if (!(ok = wait(&st->ds_full[c], ph))) break;
        tc_fence_after();
        umma_f16_ts4_w(sums + (KV ? D : 0), tmem + L::DS + c * 32, smem_desc_sw128(smem_u32(sY1(s)), QCH, 1024), IDESC, add);
        umma_commit_w(&st->used[c]);
        umma_commit_w(&st->free_[s]);
      }
      if (ok) umma_commit_w(&st->done[x % NA]);
      ++x;
    }
    // No arrival may be in flight when the block ends: the last commits have landed when these have.
    umma_commit_w(&st->drain[2]);
    drain_bar(&st->drain[2], 0);
  } else if (warp < 20) {
    // ------------------------------------------------------------ P and dS
    const int c = (warp - 4) >> 3, part = ((warp - 4) >> 2) & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint64_t sc2 = pk2(p.scale_log2, p.scale_log2);
    bool ok = true;
    int i0 = 0;  // items passed before this batch entry
    for (Job<KV> j(p); j.job < p.jobs && ok; j.step(p)) {
      uint64_t nl2 = 0, nd2 = 0;
      if (!KV) {
        const int rr = j.r0() + row, t = rr % a.q_len;
        const bool in = rr < p.group * a.q_len && t < cross_len(a.q_lens, j.b, a.q_len);
        const long long term = (static_cast<long long>(j.b) * a.hq + j.hk * p.group + rr / a.q_len) * p.q_pad + t;
        const float nl = in ? p.neg_lse2[term] : -INFINITY, nd = in ? p.neg_d[term] : 0.0f;
        nl2 = pk2(nl, nl);
        nd2 = pk2(nd, nd);
      }
      for (int yb = j.b; yb < j.b_hi(p) && ok; ++yb) {
        const int y_end = j.span(p, yb), n = j.heads(p) * ((y_end + QT - 1) / QT);
        const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(yb) * a.kv_len : nullptr;
        bool zero = false;  // KV: this row's key is masked
        if (KV && n > 0) {
          const int key = j.r0() + row;
          zero = key >= cross_len(a.kv_lens, yb, a.kv_len) || (mask && !mask[key]);
        }
        for (int k = (i0 ^ c) & 1; k < n; k += 2) {
          const int i = i0 + k, s = i % NS;
          const uint32_t ph = (i >> 1) & 1;
          const bool partial = !KV && (mask || k * QT + QT > y_end);
          bool byte = true;  // of key k * 64 + part * 32 + lane
          if (partial) {
            const int key = k * QT + part * 32 + lane;
            byte = key < y_end && (!mask || mask[key]);
          }
          if (KV && !(ok = warp_wait_ready(&st->full[s], (i / NS) & 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
          if (!(ok = warp_wait_ready(&st->s_full[c], ph, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
          tc_fence_after();
          const float4* nl = reinterpret_cast<const float4*>(terms(s)) + part * 8;
          uint32_t r[32], w[16];
          uint64_t pr[16];  // this row's weights of 32 of the item's rows
          tmem_ld32(lanes + L::S + part * 32, r);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&st->s_read);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint64_t l0 = nl2, l1 = nl2;
            if (KV) {
              const float4 t = nl[e];
              l0 = pk2(t.x, t.y);
              l1 = pk2(t.z, t.w);
            }
            float x0, x1, x2, x3;
            unpk2(fma2(pk2(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1])), sc2, l0), x0, x1);
            unpk2(fma2(pk2(__uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3])), sc2, l1), x2, x3);
            x0 = fast_exp2(x0);
            x1 = fast_exp2(x1);
            x2 = fast_exp2(x2);
            x3 = fast_exp2(x3);
            pr[2 * e] = pk2(x0, x1);
            pr[2 * e + 1] = pk2(x2, x3);
            if (KV) {
              w[2 * e] = zero ? 0u : pack_bf16x2(x0, x1);  // a masked key's scores may be anything
              w[2 * e + 1] = zero ? 0u : pack_bf16x2(x2, x3);
            }
          }
          // This group's P and dS of two items ago have been used.
          if (i >= 2 && !(ok = warp_wait_ready(&st->used[c], ph ^ 1, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
          if (KV) {
            tmem_st16(lanes + L::P + c * 32 + part * 16, w);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&st->p_full[c]);
          }
          if (!(ok = warp_wait_ready(&st->dp_full[c], ph, abort_flag, p.err, kErrCrossSoftmaxWait))) break;
          tc_fence_after();
          tmem_ld32(lanes + L::DP + part * 32, r);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&st->dp_read);
          const float4* nd = nl + 16;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint64_t d0 = nd2, d1 = nd2;
            if (KV) {
              const float4 t = nd[e];
              d0 = pk2(t.x, t.y);
              d1 = pk2(t.z, t.w);
            }
            float x0, x1, x2, x3;
            unpk2(mul2(pr[2 * e], add2(pk2(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1])), d0)), x0, x1);
            unpk2(mul2(pr[2 * e + 1], add2(pk2(__uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3])), d1)), x2, x3);
            w[2 * e] = zero ? 0u : pack_bf16x2(x0, x1);
            w[2 * e + 1] = zero ? 0u : pack_bf16x2(x2, x3);
          }
          if (partial) {  // a masked key's score or value may hold a NaN
            const unsigned word = __ballot_sync(0xffffffffu, byte);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (!((word >> (2 * e)) & 1u)) w[e] &= 0xffff0000u;
              if (!((word >> (2 * e + 1)) & 1u)) w[e] &= 0x0000ffffu;
            }
          }
          tmem_st16(lanes + L::DS + c * 32 + part * 16, w);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&st->ds_full[c]);
        }
        i0 += n;
      }
    }
  } else {
    // ------------------------------------------------------------ rows in, sums out
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    bool ok = true;
    // This thread's row of a job: offsets in X1 and X2, and in the gradients; false: there is no such row.
    const auto row_at = [&](const Job<KV>& j, long long& o1, long long& o2) {
      const int r = j.r0() + row;
      if (KV) {
        o1 = j.b * a.ks.b + j.hk * a.ks.h + r * a.ks.t;
        o2 = j.b * a.vs.b + j.hk * a.vs.h + r * a.vs.t;
        return r < a.kv_len;
      }
      const int h = j.hk * p.group + r / a.q_len, t = r % a.q_len;
      o1 = j.b * a.qs.b + h * a.qs.h + t * a.qs.t;
      o2 = j.b * a.os.b + h * a.os.h + t * a.os.t;
      return r < p.group * a.q_len && t < cross_len(a.q_lens, j.b, a.q_len);
    };
    // Rows go through shared memory, so that eight lanes move 128 bytes of one: a lane to a row in global
    // memory costs 32 transactions an access, and the warps that form P and dS wait behind them.
    uint8_t *const in_box = smem + L::IN_OFF + quarter * 4096, *const out_box = smem + L::OUT_OFF + quarter * 4096;
    const int sub = lane >> 3, piece = lane & 7;
    const auto slot = [](uint8_t* box, int r, int k) {  // piece k of row r of a 128-byte-swizzled box
      return reinterpret_cast<uint4*>(box + r * 128 + ((k ^ (r & 7)) << 4));
    };
    // Starts the copies of a job's rows into their boxes.  (Of keys' rows the TMA producer does.)
    const auto fetch_rows = [&](const Job<KV>& j) {
      if (KV) return;
      long long o[2];
      const bool in = row_at(j, o[0], o[1]);
      const __nv_bfloat16* src[2] = {static_cast<const __nv_bfloat16*>(a.q), static_cast<const __nv_bfloat16*>(p.g.dout)};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const long long at = __shfl_sync(0xffffffffu, in ? o[t] : -1, i * 4 + sub);
#pragma unroll
          for (int c = 0; c < D; c += 64) {
            const int k = c + piece * 8;
            const bool ok = at >= 0 && k < a.d;
            cp_async16(slot(in_box + (t * L::NCH + c / 64) * CH, i * 4 + sub, piece), src[t] + (ok ? at + k : 0), ok);
          }
        }
    };
    // ... and puts them where the products read them: columns x % NX.
    const auto place_rows = [&](int x) {
      if constexpr (!L::X_SMEM) {
        if (KV) {
          if (!warp_wait_ready(&st->in_full, x & 1, abort_flag, p.err, kErrCrossLoadWait)) return;
        } else {
          cp_async_wait_all();
          __syncwarp();
        }
#pragma unroll
        for (int t = 0; t < 2 * L::NCH; ++t)
#pragma unroll
          for (int k = 0; k < 8; k += 4) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint4 u = *slot(in_box + t * CH, lane, k + e);
              w[4 * e] = u.x, w[4 * e + 1] = u.y, w[4 * e + 2] = u.z, w[4 * e + 3] = u.w;
            }
            tmem_st16(lanes + L::X + (x % NX) * L::XW + t * 32 + k * 4, w);
          }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&st->x_full[x % NX]);
          if (KV) mbar_arrive(&st->in_free);
        }
      }
    };
    // Zeros for rows whose sums are empty.  (Of keys' rows the TMA producer does.)
    const auto store_zeros = [&](const Job<KV>& j) {
      if (KV) return;
      long long at, other;
      const bool in = row_at(j, at, other);
      for (int r = 0; r < 32; r += 4) {
        const long long o = __shfl_sync(0xffffffffu, in ? at : -1, r + sub);
        for (int c = piece * 8; o >= 0 && c < a.d; c += 64)
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.g.dq) + o + c) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
    };
    const auto next_job_quiet = [&](Job<KV>& j) {  // to the next job with items
      while (j.job < p.jobs && j.count(p) == 0) j.step(p);
    };
    const auto next_job = [&](Job<KV>& j) {  // ... with zeros for those without
      for (; j.job < p.jobs && j.count(p) == 0; j.step(p)) store_zeros(j);
    };
    // The rows of the first NX jobs, then each time a job is done those of the one that takes its columns,
    // fetched while it runs.
    int x = 0;
    Job<KV> j(p);
    next_job(j);
    Job<KV> ahead = j;  // the next job to fetch
    const auto advance = [&] {
      ahead.step(p);
      next_job(ahead);
    };
    for (int k = 0; k < NX && ahead.job < p.jobs; ++k) {
      fetch_rows(ahead);
      place_rows(k);
      advance();
    }
    while (j.job < p.jobs) {
      if (!L::X_SMEM && ahead.job < p.jobs) fetch_rows(ahead);
      long long o[2];
      const bool in = !KV && row_at(j, o[0], o[1]);
      bool seen = true;
      if (KV && (a.kv_lens || a.key_mask)) {  // a masked key's gradient is 0 whatever its row holds
        seen = false;
        for (int b = j.b; b < j.b_hi(p); ++b)
          seen |= j.r0() + row < cross_len(a.kv_lens, b, a.kv_len) &&
                  (!a.key_mask || a.key_mask[static_cast<long long>(b) * a.kv_len + min(j.r0() + row, a.kv_len - 1)]);
      }
      // These warps wait for a whole job: they sleep between polls and leave the issue slots to the others, and have a
      // millisecond more for each item (0.8 us; a job of a shared source walks the rows of the whole batch).
      const uint64_t limit = LC_WAIT_TIMEOUT_NS + 1000000ull * static_cast<unsigned>(j.count(p));
      ok = mbar_wait_bounded_backoff(&st->done[x % NA], (x / NA) & 1, abort_flag, p.err, kErrCrossSoftmaxWait, 40, limit);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      if (NX == 1 && ahead.job < p.jobs) place_rows(x + 1);
      // Sums: through the boxes, as many as there are at a time.
      constexpr int SUMS = (KV ? 2 : 1) * L::NCH;  // chunks of 64 columns: dv, then dk; or dq
#pragma unroll
      for (int h0 = 0; h0 < SUMS; h0 += L::OUTS) {
        if (KV && lane == 0) bulk_wait_group_read0();  // the boxes' last contents are on their way
        __syncwarp();
#pragma unroll
        for (int h = h0; h < h0 + L::OUTS; ++h) {
          const float f = KV && h < L::NCH ? 1.0f : a.scale;  // dv has no scale
#pragma unroll
          for (int k = 0; k < 8; k += 4) {
            uint32_t v[32];
            __syncwarp();  // tcgen05.ld is warp-collective
            tmem_ld32(lanes + L::A + (x % NA) * L::AW + h * 64 + k * 8, v);
            if (h == SUMS - 1 && k == 4) {  // the last read: the columns take another job
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&st->sums_free[x % NA]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                w[q] = seen ? pack_bf16x2(__uint_as_float(v[8 * e + 2 * q]) * f, __uint_as_float(v[8 * e + 2 * q + 1]) * f)
                            : 0u;
              *slot(out_box + (h - h0) * CH, lane, k + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (KV) {
          // 32 rows a box; the tensor maps end at kv_len and head_dim.
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && j.r0() + quarter * 32 < a.kv_len) {  // (no store starts past the tensor)
            for (int h = h0; h < h0 + L::OUTS; ++h) {
              const bool v = h < L::NCH;
              tma_store_4d(v ? &map_dv : &map_dk, out_box + (h - h0) * CH, h % L::NCH * 64, j.r0() + quarter * 32,
                           (v ? p.x2_head : p.x1_head) ? j.hk : 0, (v ? p.x2_batch : p.x1_batch) ? j.b : 0);
            }
            bulk_commit_group();
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int h = h0; h < h0 + L::OUTS; ++h) {
            const int c = h * 64 + piece * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const long long at = __shfl_sync(0xffffffffu, in ? o[0] : -1, i * 4 + sub);
              if (at >= 0 && c < a.d)
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.g.dq) + at + c) =
                    *slot(out_box + (h - h0) * CH, i * 4 + sub, piece);
            }
          }
          __syncwarp();
        }
      }
      if (NX > 1 && ahead.job < p.jobs) place_rows(x + NX);
      if (ahead.job < p.jobs) advance();
      j.step(p);
      next_job_quiet(j);
      ++x;
    }
    if (KV && lane == 0) bulk_wait_group0();  // shared memory outlives the stores' reads
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (!KV) griddep_wait();
}

// ---- host -------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Boxes of 128 bytes (64 bf16 or, es = 4, 32 fp32 values) of box_rows tokens.
bool head_map(HeadMap* m, const void* base, const HeadStrides& s, int batch, int heads, int len, int d, int box_rows,
              int es = 2) {
  auto enc = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!enc) return false;
  m->by_head = heads > 1 && s.h != 0;
  m->by_batch = batch > 1 && s.b != 0;
  const cuuint64_t row = static_cast<cuuint64_t>(len > 1 ? s.t : d) * es;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(len),
                              static_cast<cuuint64_t>(m->by_head ? heads : 1),
                              static_cast<cuuint64_t>(m->by_batch ? batch : 1)};
  const cuuint64_t strides[3] = {row, m->by_head ? static_cast<cuuint64_t>(s.h) * es : row,
                                 m->by_batch ? static_cast<cuuint64_t>(s.b) * es : row};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / es), static_cast<cuuint32_t>(box_rows), 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(&m->map, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4,
             const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t fwd_tc(const CrossArgs& a, cudaStream_t s) {
  using F = Fwd<D>;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  HeadMap mk, mv;
  if (!head_map(&mk, a.k, a.ks, a.batch, a.hk, a.kv_len, a.d, TILE) ||
      !head_map(&mv, a.v, a.vs, a.batch, a.hk, a.kv_len, a.d, TILE))
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
  if ((e = w.begin(a, blocks, TILE, 3, 1, s)) != cudaSuccess) return e;
  const FwdParams p{a, w.sp, mk.by_head, mk.by_batch, mv.by_head, mv.by_batch, a.scale * kLog2e, ctx->err_word};
  cross_fwd_tc_kernel<D>
      <<<dim3(static_cast<unsigned>(blocks), w.sp.splits), F::THREADS, F::SMEM, s>>>(mk.map, mv.map, p);
  return w.end(a, cudaGetLastError(), s);
}

template <class Kernel>
cudaError_t allow_smem(std::atomic<unsigned long long>& done, Kernel k, size_t bytes) {
  return once_per_device(done, [&] {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    return e != cudaSuccess ? e : cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  });
}

template <int D>
cudaError_t bwd_tc(const CrossGradArgs& g, const float* neg_lse2, const float* neg_d, int q_pad, cudaStream_t s) {
  const CrossArgs& a = g.f;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  // One walk: resident blocks, one to an SM.  (The dq walk beside the other's last jobs: [4, 16/4, 1024 x 2048 ragged,
  // 128] 188 us, one after the other 210; with two or four blocks to an SM, dealt out as they get free, 191 and
  // 197.)
  const auto walk = [&](auto kv, const HeadMap& y1, const HeadMap& y2, const HeadMap& x1, const HeadMap& x2,
                        const HeadMap& dk, const HeadMap& dv, int tiles, int entries) -> cudaError_t {
    constexpr bool KV = decltype(kv)::value;
    using L = Grad<D, KV>;
    static std::atomic<unsigned long long> attr{0};
    const cudaError_t e = allow_smem(attr, cross_grad_tc_kernel<D, KV>, L::SMEM);
    if (e != cudaSuccess) return e;
    const long long jobs = static_cast<long long>(tiles) * entries * a.hk;
    if (jobs > 0x7fffffffLL - ctx->sm_count) return cudaErrorNotSupported;
    const int blocks = static_cast<int>(std::min<long long>(jobs, ctx->sm_count));
    const GradParams p{g,           neg_lse2,   neg_d,       q_pad,      y1.by_head,  y1.by_batch,
                       y2.by_head,  y2.by_batch, x1.by_head, x1.by_batch, x2.by_head, x2.by_batch,
                       static_cast<int>(jobs), tiles, a.hq / a.hk, blocks % tiles, blocks / tiles % a.hk, blocks / tiles / a.hk,
                       !KV && g.dk, a.scale * kLog2e, ctx->err_word};
    return launch_pdl(cross_grad_tc_kernel<D, KV>, dim3(blocks), dim3(L::THREADS), L::SMEM, s, y1.map, y2.map, x1.map, x2.map,
                      dk.map, dv.map, p);
  };
  HeadMap m1, m2, x1{}, x2{}, dk{}, dv{};
  if (g.dk) {
    const int entries = g.kv_shared ? 1 : a.batch;
    if (!head_map(&m1, a.q, a.qs, a.batch, a.hq, a.q_len, a.d, QT) ||
        !head_map(&m2, g.dout, a.os, a.batch, a.hq, a.q_len, a.d, QT) ||
        !head_map(&x1, a.k, a.ks, entries, a.hk, a.kv_len, a.d, TILE) ||
        !head_map(&x2, a.v, a.vs, entries, a.hk, a.kv_len, a.d, TILE) ||
        !head_map(&dk, g.dk, a.ks, entries, a.hk, a.kv_len, a.d, 32) ||
        !head_map(&dv, g.dv, a.vs, entries, a.hk, a.kv_len, a.d, 32))
      return cudaErrorInvalidValue;
    const cudaError_t e = walk(std::true_type{}, m1, m2, x1, x2, dk, dv, (a.kv_len + TILE - 1) / TILE, entries);
    if (e != cudaSuccess) return e;
  }
  if (g.dq) {
    if (!head_map(&m1, a.k, a.ks, a.batch, a.hk, a.kv_len, a.d, QT) ||
        !head_map(&m2, a.v, a.vs, a.batch, a.hk, a.kv_len, a.d, QT))
      return cudaErrorInvalidValue;
    const cudaError_t e = walk(std::false_type{}, m1, m2, x1, x2, dk, dv, (a.hq / a.hk * a.q_len + TILE - 1) / TILE, a.batch);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

// 16-byte rows and strides that a tensor map can hold (below 2^40 bytes).
bool cross_rows16(const CrossArgs& a) {
  const int per = a.bf16 ? 8 : 4;  // values in 16 bytes
  const auto ok = [&](const void* p, const HeadStrides& s, int len) {
    const auto in = [&](long long x) { return x % per == 0 && x < (1LL << 37); };
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && in(s.b) && in(s.h) && in(s.t) && (len == 1 || s.t != 0);
  };
  return a.d % per == 0 && ok(a.q, a.qs, a.q_len) && ok(a.k, a.ks, a.kv_len) && ok(a.v, a.vs, a.kv_len) &&
         ok(a.out, a.os, a.q_len) && tensor_map_encoder() != nullptr;
}

bool cross_tc_supported(const CrossArgs& a) { return a.bf16 && a.d <= 128 && cross_rows16(a); }

bool cross_kv_maps(const CrossArgs& a, int rows, CUtensorMap* k, CUtensorMap* v, KvAxes* ax) {
  HeadMap mk, mv;
  const int es = a.bf16 ? 2 : 4;
  if (!head_map(&mk, a.k, a.ks, a.batch, a.hk, a.kv_len, a.d, rows, es) ||
      !head_map(&mv, a.v, a.vs, a.batch, a.hk, a.kv_len, a.d, rows, es))
    return false;
  *k = mk.map;
  *v = mv.map;
  *ax = {mk.by_head, mk.by_batch, mv.by_head, mv.by_batch};
  return true;
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
