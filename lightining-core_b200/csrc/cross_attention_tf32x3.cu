// Cross attention forward in strict fp32 on the tensor cores, head_dim <= 64.
//
// Every product by the 3xTF32 split: x = x_hi + x_lo with x_hi rounded to tf32, x.y ~= x_hi.y_hi + x_hi.y_lo +
// x_lo.y_hi (what is dropped is 2^-22 |x y|).  A pre-pass writes the hi and lo planes: Q's rows packed by key head
// (row = head in the group * q_len + token), K's rows, and V transposed so that every operand is K-major; rows that
// are not computed and masked keys are written as zeros, so what memory holds there never enters a product.
// One block = 128 rows, one block to an SM:
//   warp 0      TMA: Q once, K tiles of 64 keys into two stages freed by S_j; warp 6: V^T tiles, freed by P.V_j
//   warp 1      MMA: S_j into one of two TMEM buffers (24 steps of K = 8), O_j = P_j V_j with P from TMEM into
//               one of two buffers, a fresh partial per tile
//   warps 2..5, 7..10   softmax, two warps to a row (32 score and output columns each) that swap the row's
//               maximum through tagged shared-memory words; P_hi over S_j's columns, P_lo in a buffer of its own;
//               the previous tile's partial is folded into fp32 registers (O * alpha + O_j, rounded to
//               nearest: long accumulations in the tensor core drift)
// The tensor pipe bounds it: 1536 cycles a tile of 64 keys.  B200, [4, 16, 333 x 1000, 64] with holes: 89 us,
// planes included (14 GFLOP: 153 TFLOP/s; 370 us on the CUDA cores, whose peak would allow 190).
#include <cuda.h>
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
constexpr int D = 64, TILE = 128, TK = 64;
constexpr int THREADS = 352;
constexpr int QCH = TILE * 128;  // one [128 rows x 32 fp32] swizzled box
constexpr int KCH = TK * 128;    // [64 keys x 32 fp32], and [64 columns x 32 keys] of V^T
constexpr int Q_PLANE = 2 * QCH, K_PLANE = 2 * KCH;
constexpr int K_OFF = 2 * Q_PLANE;                 // two stages of (hi, lo)
constexpr int V_OFF = K_OFF + 2 * 2 * K_PLANE;
constexpr int TAIL_OFF = V_OFF + 2 * 2 * K_PLANE;
constexpr uint32_t S_COL = 0, PL_COL = 128, O_COL = 256;
constexpr float kRescale = 8.0f;
constexpr uint32_t IDESC = idesc_tf32_f32(TILE, 64, 0, 0);

struct Tail {
  uint64_t q_full, k_full[2], v_full[2], s_full[2], p_full[2], o_full[2], o_free[2], drain;
  unsigned long long xmax[2][2][TILE];  // [tile & 1][half][row]: running maxima, tagged with the tile
  unsigned long long xsum[2][TILE];     // [half][row]: final sums
  uint32_t tmem_base;
  int abort_flag;
};
constexpr size_t SMEM = 1024 + TAIL_OFF + sizeof(Tail);

struct Planes {
  float *qh, *ql, *kh, *kl, *vh, *vl;
  int rows, kv_pad;  // rows of a pair; keys rounded up to 4
};

// One block: 64 rows of Q or K, or 64 keys of V^T, of pair blockIdx.y.
__global__ void __launch_bounds__(256) cross_split_kernel(CrossArgs a, Planes pl, int q_blocks, int k_blocks, int vec) {
  griddep_launch_dependents();  // the attention may take its SMs now; it waits for the planes itself
  __shared__ float tile[64][65];
  const int pair = blockIdx.y, b = pair / a.hk, hk = pair % a.hk;
  const int group = a.hq / a.hk;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  const int part = blockIdx.x < q_blocks ? 0 : blockIdx.x < q_blocks + k_blocks ? 1 : 2;
  const int r0 = (blockIdx.x - (part == 0 ? 0 : part == 1 ? q_blocks : q_blocks + k_blocks)) * 64;
  const float* src = static_cast<const float*>(part == 0 ? a.q : part == 1 ? a.k : a.v);
  const HeadStrides& st = part == 0 ? a.qs : part == 1 ? a.ks : a.vs;
  const int n = part == 0 ? pl.rows : a.kv_len;
  const int c = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int lr = i * 16 + (threadIdx.x >> 4), r = r0 + lr;
    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    bool in = r < n;
    long long at = 0;
    if (part == 0) {
      const int t = r % a.q_len;
      in = in && t < q_end;
      at = b * st.b + (hk * group + r / a.q_len) * st.h + t * st.t;
    } else {
      in = in && r < kv_end && (!mask || mask[r]);
      at = b * st.b + hk * st.h + r * st.t;
    }
    if (in) {
      if (vec && c < a.d) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(src + at + c));
        f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < a.d) f[e] = src[at + c + e];
      }
    }
    if (part == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[lr][c + e] = f[e];
    } else if (r < n) {
      float h[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = tf32_round(f[e]), l[e] = f[e] - h[e];
      const long long o = (static_cast<long long>(pair) * n + r) * D + c;
      *reinterpret_cast<float4*>((part == 0 ? pl.qh : pl.kh) + o) = make_float4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<float4*>((part == 0 ? pl.ql : pl.kl) + o) = make_float4(l[0], l[1], l[2], l[3]);
    }
  }
  if (part < 2) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int d = i / 64, k = i % 64;
    if (r0 + k >= pl.kv_pad) continue;
    const float x = tile[k][d], h = tf32_round(x);
    const long long o = (static_cast<long long>(pair) * D + d) * pl.kv_pad + r0 + k;
    pl.vh[o] = h;
    pl.vl[o] = x - h;
  }
}

__global__ void __launch_bounds__(THREADS, 1)
    cross_f32_tc_kernel(const __grid_constant__ CUtensorMap map_qh, const __grid_constant__ CUtensorMap map_ql,
                        const __grid_constant__ CUtensorMap map_kh, const __grid_constant__ CUtensorMap map_kl,
                        const __grid_constant__ CUtensorMap map_vh, const __grid_constant__ CUtensorMap map_vl,
                        const CrossArgs a, const CrossSplit sp, float scale_log2, int vec_out, unsigned* err) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Tail* st = reinterpret_cast<Tail*>(smem + TAIL_OFF);
  uint8_t *sQh = smem, *sQl = smem + Q_PLANE;
  const auto sK = [&](int s, int lo) { return smem + K_OFF + (s * 2 + lo) * K_PLANE; };
  const auto sV = [&](int s, int lo) { return smem + V_OFF + (s * 2 + lo) * K_PLANE; };
  griddep_wait();  // the planes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.hq / a.hk, rows = group * a.q_len, row_tiles = (rows + TILE - 1) / TILE;
  const int pair = blockIdx.x / row_tiles, b = pair / a.hk, hk = pair % a.hk;
  const int r0 = (blockIdx.x % row_tiles) * TILE;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  const int tiles = (kv_end + TK - 1) / TK, per = (tiles + sp.splits - 1) / sp.splits;
  const int t_lo = min(tiles, static_cast<int>(blockIdx.y) * per), n = min(tiles, t_lo + per) - t_lo;

  if (threadIdx.x == 0) {
    mbar_init(&st->q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&st->k_full[i], 1);
      mbar_init(&st->v_full[i], 1);
      mbar_init(&st->s_full[i], 1);
      mbar_init(&st->p_full[i], 8);
      mbar_init(&st->o_full[i], 1);
      mbar_init(&st->o_free[i], 8);
    }
    mbar_init(&st->drain, 1);
    st->abort_flag = 0;
    fence_barrier_init();
    if (n > 0) {
      mbar_arrive_expect_tx(&st->q_full, 2 * Q_PLANE);
      for (int c = 0; c < 2; ++c) {
        tma_load_3d(sQh + c * QCH, &map_qh, c * 32, r0, pair, &st->q_full);
        tma_load_3d(sQl + c * QCH, &map_ql, c * 32, r0, pair, &st->q_full);
      }
    }
  }
  for (int i = threadIdx.x; i < 2 * 2 * TILE; i += THREADS) (&st->xmax[0][0][0])[i] = ~0ull;
  for (int i = threadIdx.x; i < 2 * TILE; i += THREADS) (&st->xsum[0][0])[i] = ~0ull;
  if (warp == 0) {
    tmem_alloc(&st->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = st->tmem_base;
  volatile int* abort_flag = &st->abort_flag;
  const auto drain = [](uint64_t* bar, uint32_t ph) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, ph) && globaltimer_ns() - t0 < 100000000ull) {
    }
  };

  if (warp == 0 || warp == 6) {
    // ------------------------------------------------------------ K loads (warp 0) and V^T loads (warp 6)
    if (lane == 0) {
      const bool v = warp == 6;
      uint64_t *full = v ? st->v_full : st->k_full, *used = v ? st->o_full : st->s_full;
      const CUtensorMap *mh = v ? &map_vh : &map_kh, *ml = v ? &map_vl : &map_kl;
      bool ok = true;
      int issued = 0;
      for (int j = 0; j < n; ++j, ++issued) {
        const int s = j & 1;
        // The stage's last tile has been read (the one commit of its products); its barrier's next
        // completion needs this load, so the parity wait is unambiguous.
        if (j >= 2 && !mbar_wait_bounded(&used[s], ((j - 2) >> 1) & 1, abort_flag, err, kErrCrossLoadWait)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[s], 2 * K_PLANE);
        for (int c = 0; c < 2; ++c) {
          const int k0 = (t_lo + j) * TK;
          tma_load_3d((v ? sV(s, 0) : sK(s, 0)) + c * KCH, mh, v ? k0 + c * 32 : c * 32, v ? 0 : k0, pair, &full[s]);
          tma_load_3d((v ? sV(s, 1) : sK(s, 1)) + c * KCH, ml, v ? k0 + c * 32 : c * 32, v ? 0 : k0, pair, &full[s]);
        }
      }
      if (!ok) {
        if (!v) drain(&st->q_full, 0);
        for (int j = issued > 2 ? issued - 2 : 0; j < issued; ++j) drain(&full[j & 1], (j >> 1) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA (whole warp)
    bool ok = n > 0, issued = false;
    const auto wait = [&](uint64_t* bar, uint32_t ph) { return warp_wait_poll(bar, ph, abort_flag, err, kErrCrossMmaWait); };
    const auto issue_s = [&](int j) {
      const int s = j & 1;
      if (!wait(&st->k_full[s], (j >> 1) & 1)) return false;
      tc_fence_after();
      const uint32_t d = tmem + S_COL + static_cast<uint32_t>(s * TK);
      const uint64_t qh = smem_desc_sw128(smem_u32(sQh), 16, 1024), ql = smem_desc_sw128(smem_u32(sQl), 16, 1024);
      const uint64_t kh = smem_desc_sw128(smem_u32(sK(s, 0)), 16, 1024), kl = smem_desc_sw128(smem_u32(sK(s, 1)), 16, 1024);
#pragma unroll
      for (int kk = 0; kk < D / 8; ++kk) {
        const uint32_t qo = ((kk >> 2) * QCH + (kk & 3) * 32) >> 4, ko = ((kk >> 2) * KCH + (kk & 3) * 32) >> 4;
        umma_tf32_ss_w(d, ql + qo, kh + ko, IDESC, kk > 0 ? 1u : 0u);
        umma_tf32_ss_w(d, qh + qo, kl + ko, IDESC, 1u);
        umma_tf32_ss_w(d, qh + qo, kh + ko, IDESC, 1u);
      }
      issued = true;
      umma_commit_w(&st->s_full[s]);
      return true;
    };
    if (ok) ok = wait(&st->q_full, 0) && issue_s(0);
    for (int j = 0; j < n && ok; ++j) {
      const int s = j & 1;
      if (j + 1 < n && !(ok = issue_s(j + 1))) break;
      // Each barrier's next completion needs what is issued after these waits.
      if (!(ok = wait(&st->p_full[s], (j >> 1) & 1) && wait(&st->v_full[s], (j >> 1) & 1) &&
                 (j < 2 || wait(&st->o_free[s], ((j - 2) >> 1) & 1))))
        break;
      tc_fence_after();
      const uint32_t o = tmem + O_COL + static_cast<uint32_t>(s * D);
      const uint32_t ph = tmem + S_COL + static_cast<uint32_t>(s * TK), pl = tmem + PL_COL + static_cast<uint32_t>(s * TK);
      const uint64_t vh = smem_desc_sw128(smem_u32(sV(s, 0)), 16, 1024), vl = smem_desc_sw128(smem_u32(sV(s, 1)), 16, 1024);
#pragma unroll
      for (int kk = 0; kk < TK / 8; ++kk) {
        const uint32_t vo = ((kk >> 2) * KCH + (kk & 3) * 32) >> 4;
        umma_tf32_ts_w(o, pl + kk * 8, vh + vo, IDESC, kk > 0 ? 1u : 0u);
        umma_tf32_ts_w(o, ph + kk * 8, vl + vo, IDESC, 1u);
        umma_tf32_ts_w(o, ph + kk * 8, vh + vo, IDESC, 1u);
      }
      umma_commit_w(&st->o_full[s]);
    }
    if (!ok && issued) {
      umma_commit_w(&st->drain);
      drain(&st->drain, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax, fold, epilogue
    const int quarter = warp & 3, half = warp >= 7 ? 1 : 0;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16), hc = static_cast<uint32_t>(half * 32);
    float m = -INFINITY, l = 0.0f, alpha_prev = 1.0f, o_acc[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) o_acc[e] = 0.0f;
    bool ok = true;
    // Publishes v under `tag` and returns the partner's value under the same tag.
    const auto swap = [&](unsigned long long* mine, unsigned long long* theirs, uint32_t tag, float v, float* out) {
      *reinterpret_cast<volatile unsigned long long*>(mine) = (static_cast<unsigned long long>(tag) << 32) | __float_as_uint(v);
      volatile unsigned long long* t = theirs;
      unsigned long long x = *t;
      if (static_cast<uint32_t>(x >> 32) != tag) {
        const uint64_t t0 = globaltimer_ns();
        uint32_t spins = 0;
        while (static_cast<uint32_t>((x = *t) >> 32) != tag) {
          if (*abort_flag) return false;
          if ((++spins & 63u) == 0 && globaltimer_ns() - t0 > LC_WAIT_TIMEOUT_NS) {
            *abort_flag = 1;
            atomicCAS(err, 0u, static_cast<unsigned>(kErrCrossSoftmaxWait));
            return false;
          }
        }
      }
      *out = __uint_as_float(static_cast<uint32_t>(x));
      return true;
    };
    const auto fold = [&](int t, float alpha) {
      if (!warp_wait_poll(&st->o_full[t & 1], (t >> 1) & 1, abort_flag, err, kErrCrossSoftmaxWait)) return false;
      tc_fence_after();
      uint32_t r[32];
      tmem_ld32(lanes + O_COL + static_cast<uint32_t>((t & 1) * D) + hc, r);
#pragma unroll
      for (int e = 0; e < 32; ++e) o_acc[e] = __fmaf_rn(o_acc[e], alpha, __uint_as_float(r[e]));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->o_free[t & 1]);
      return true;
    };
    for (int j = 0; j < n; ++j) {
      const int s = j & 1, kv0 = (t_lo + j) * TK + half * 32;
      const bool partial = mask || kv0 + 32 > kv_end;
      bool seen = true;
      if (partial) seen = kv0 + lane < kv_end && (!mask || mask[kv0 + lane]);
      if (!(ok = warp_wait_poll(&st->s_full[s], (j >> 1) & 1, abort_flag, err, kErrCrossSoftmaxWait))) break;
      tc_fence_after();
      const uint32_t sb = lanes + S_COL + static_cast<uint32_t>(s * TK) + hc;
      uint32_t r[32];
      tmem_ld32(sb, r);
      if (partial) {
        const unsigned w = __ballot_sync(0xffffffffu, seen);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!((w >> e) & 1u)) r[e] = __float_as_uint(-INFINITY);
      }
      float mx4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) mx4[i] = __uint_as_float(r[i]);
#pragma unroll
      for (int e = 4; e < 32; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(r[e]));
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), mo;
      // Slot [j & 1] is written again for tile j + 2 only after the partner published tile j + 1, which it does
      // after reading this one.  The verdict is made uniform: the tcgen05 accesses are warp-collective.
      if (!(ok = __all_sync(0xffffffffu, swap(&st->xmax[s][half][row], &st->xmax[s][half ^ 1][row],
                                              static_cast<uint32_t>(j), mx, &mo))))
        break;
      mx = fmaxf(mx, mo) * scale_log2;
      float alpha = 1.0f;
      if (mx > m + kRescale) {
        alpha = m == -INFINITY ? 0.0f : exp2f(m - mx);
        l *= alpha;
        m = mx;
      }
      const float mu = m == -INFINITY ? 0.0f : m;  // nothing seen yet: every weight is 0
      float ls4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t wh[16], wl[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float pv = exp2_acc(__fmaf_rn(__uint_as_float(r[g * 16 + i]), scale_log2, -mu));
          const float ph = __uint_as_float((__float_as_uint(pv) + 0x1000u) & 0xffffe000u);
          ls4[i & 3] += pv;
          wh[i] = __float_as_uint(ph);
          wl[i] = __float_as_uint(pv - ph);
        }
        tmem_st16(sb + g * 16, wh);
        tmem_st16(lanes + PL_COL + static_cast<uint32_t>(s * TK) + hc + g * 16, wl);
      }
      l += (ls4[0] + ls4[1]) + (ls4[2] + ls4[3]);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->p_full[s]);
      // The previous tile's partial (formed with the previous maximum), then this tile's factor for its own.
      if (j > 0 && !(ok = fold(j - 1, alpha_prev))) break;
      alpha_prev = alpha;
    }
    float other = 0.0f;
    if (ok && n > 0) ok = fold(n - 1, alpha_prev);
    if (ok && n > 0) ok = swap(&st->xsum[half][row], &st->xsum[half ^ 1][row], static_cast<uint32_t>(n), l, &other);
    l = half == 0 ? l + other : other + l;
    const int rr = r0 + row, g = rr / a.q_len, t = rr % a.q_len;
    if (ok && rr < rows && t < q_end) {
      const bool empty = m == -INFINITY;
      const long long at = (static_cast<long long>(b) * a.hq + hk * group) * a.q_len + rr;  // dense row
      const bool split = sp.splits > 1;
      const float f = empty ? 0.0f : split ? 1.0f : 1.0f / l;
      if (half == 0) {
        if (split)
          sp.ml[static_cast<long long>(blockIdx.y) * sp.rows + at] = make_float2(m, empty ? 0.0f : l);
        else if (a.lse)
          a.lse[at] = empty ? -INFINITY : (m + log2f(l)) * kLn2;
      }
      float* out = split ? sp.o + (static_cast<long long>(blockIdx.y) * sp.rows + at) * a.d
                         : static_cast<float*>(a.out) + b * a.os.b + (hk * group + g) * a.os.h + t * a.os.t;
      const bool vec = vec_out || (split && a.d % 4 == 0);
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const int c = half * 32 + e;
        if (vec) {
          if (c < a.d)
            *reinterpret_cast<float4*>(out + c) =
                make_float4(o_acc[e] * f, o_acc[e + 1] * f, o_acc[e + 2] * f, o_acc[e + 3] * f);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i < a.d) out[c + i] = o_acc[e + i] * f;
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

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// fp32 [pairs, rows, cols], box [1, box_rows, 32], 128-byte swizzle, zeros outside.
bool plane_map(CUtensorMap* map, const void* base, int pairs, int rows, int cols, int box_rows) {
  auto enc = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!enc) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(pairs)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 4, static_cast<cuuint64_t>(rows) * cols * 4};
  const cuuint32_t box[3] = {32, static_cast<cuuint32_t>(box_rows), 1}, estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool rows4(const void* p, const HeadStrides& s, int d) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && d % 4 == 0 && s.b % 4 == 0 && s.h % 4 == 0 && s.t % 4 == 0;
}

}  // namespace

bool cross_f32_tc_supported(const CrossArgs& a) {
  const long long rows = static_cast<long long>(a.hq / a.hk) * a.q_len, pairs = static_cast<long long>(a.batch) * a.hk;
  // From 8 rows a pair on this beats the CUDA cores although most of the tile is padding: [4, 16, R x 1000, 64]
  // takes 45 / 50 us for R = 8 / 128 here and 52 / 92 there; [16, 16, 512 x 16, 64] 77 and 94; one 64 x 64 tile 12.5
  // both.  A grid's second axis ends at 65535.
  return !a.bf16 && a.d <= D && rows >= 8 && pairs <= 65535 && tensor_map_encoder() != nullptr;
}

cudaError_t cross_forward_f32_tc(const CrossArgs& a, cudaStream_t s) {
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const int rows = a.hq / a.hk * a.q_len, pairs = a.batch * a.hk, kv_pad = (a.kv_len + 3) / 4 * 4;
  const size_t nq = static_cast<size_t>(pairs) * rows * D, nk = static_cast<size_t>(pairs) * a.kv_len * D,
               nv = static_cast<size_t>(pairs) * kv_pad * D;
  const long long blocks = static_cast<long long>((rows + TILE - 1) / TILE) * pairs;
  if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
  static std::atomic<unsigned long long> attr{0};
  cudaError_t e = once_per_device(attr, [] {
    return cudaFuncSetAttribute(cross_f32_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM));
  });
  if (e != cudaSuccess) return e;
  void* ws = nullptr;
  if ((e = workspace_alloc(ctx, &ws, 2 * (nq + nk + nv) * sizeof(float), s)) != cudaSuccess) return e;
  Planes pl{};
  pl.qh = static_cast<float*>(ws);
  pl.ql = pl.qh + nq;
  pl.kh = pl.ql + nq;
  pl.kl = pl.kh + nk;
  pl.vh = pl.kl + nk;
  pl.vl = pl.vh + nv;
  pl.rows = rows;
  pl.kv_pad = kv_pad;
  CUtensorMap mqh, mql, mkh, mkl, mvh, mvl;
  if (!plane_map(&mqh, pl.qh, pairs, rows, D, TILE) || !plane_map(&mql, pl.ql, pairs, rows, D, TILE) ||
      !plane_map(&mkh, pl.kh, pairs, a.kv_len, D, TK) || !plane_map(&mkl, pl.kl, pairs, a.kv_len, D, TK) ||
      !plane_map(&mvh, pl.vh, pairs, D, kv_pad, D) || !plane_map(&mvl, pl.vl, pairs, D, kv_pad, D))
    e = cudaErrorInvalidValue;
  if (e == cudaSuccess) {
    CrossSplitWork w;
    e = w.begin(a, blocks, TK, 1, s);
    if (e == cudaSuccess) {
      const int qb = (rows + 63) / 64, kb = (a.kv_len + 63) / 64;
      const int vec = rows4(a.q, a.qs, a.d) && rows4(a.k, a.ks, a.d) && rows4(a.v, a.vs, a.d);
      cross_split_kernel<<<dim3(qb + 2 * kb, pairs), 256, 0, s>>>(a, pl, qb, kb, vec);
      e = cudaGetLastError();
      if (e == cudaSuccess)
        e = launch_pdl(cross_f32_tc_kernel, dim3(static_cast<unsigned>(blocks), w.sp.splits), dim3(THREADS), SMEM, s, mqh,
                       mql, mkh, mkl, mvh, mvl, a, w.sp, a.scale * kLog2e, static_cast<int>(rows4(a.out, a.os, a.d)),
                       ctx->err_word);
      e = w.end(a, e, s);
    }
  }
  const cudaError_t f = workspace_free(ws, s);
  return e != cudaSuccess ? e : f;
}

}  // namespace lcb
