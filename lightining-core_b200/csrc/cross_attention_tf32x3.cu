// Cross attention in strict fp32 on the tensor cores, head_dim <= 128: forward and backward.
//
// Every product by the 3xTF32 split: x = x_hi + x_lo, both rounded to tf32 (x_lo is off by 2^-22 |x| at most), x.y ~=
// x_hi.y_hi + x_hi.y_lo + x_lo.y_hi (what is dropped is 2^-22 |x y|, so a product is off by 3 * 2^-22 |x y| at most).
// A pre-pass writes the operands' hi and lo planes, dense by (batch, key head) pair and padded to D columns: rows (of
// the group: head in the group * q_len + token; or keys), and where a product sums over rows or keys their transpose, so
// that every operand is K-major (tf32 has no other form).  Rows that are not computed and masked keys are written as
// zeros: what memory holds there never enters a product.  (The planes of k and v are a batch entry's own, as its mask is,
// broadcast or not.)
// Blocks own 128 rows or keys, one block to an SM, and stream tiles of T = 4096 / D of the other side: a tile's hi and
// lo planes are always 32 KB.  Long accumulations in the tensor core drift (it truncates), so a tile's sums are
// folded into fp32 registers, rounded to nearest.  Visible infinities give NaN (inf - inf in the split).
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
constexpr int TILE = 128;
constexpr int PIECE = 32768;     // hi and lo planes of a streamed tile
constexpr int ACH = TILE * 128;  // one [128 rows x 32 fp32] swizzled chunk
constexpr float kRescale = 8.0f;

// ---- planes ---------------------------------------------------------------------------------
// An operand: its rows (of the group, or keys) as [2][pairs][n][D] at `rows` and / or transposed as
// [2][pairs][D][pad] at `cols`; hi planes first.
struct PlanePart {
  const float* src;
  HeadStrides st;
  int keys;    // rows are keys, else the group's rows
  int blocks;  // of 64 rows
  float *rows, *cols;
  int terms;  // also the rows' terms of the backward pass (src is dout)
};
struct PlaneJob {
  PlanePart part[4];
  int rows, rows_pad, kv_pad, pairs;  // padded to 64
  const float *out, *lse;
  float2* terms;  // [pairs][rows_pad]: -lse in the log2 domain, -(dout . out)
};

// One block: 64 rows of one operand of pair blockIdx.y.
template <int D>
__global__ void __launch_bounds__(256)
    cross_split_kernel(const __grid_constant__ CrossArgs a, const __grid_constant__ PlaneJob job, int vec) {
  griddep_launch_dependents();  // the attention may take its SMs now; it waits for the planes itself
  constexpr int V = D / 4, RP = 256 / V;
  __shared__ float tile[64][D + 1];
  int blk = blockIdx.x, pi = 0;
  while (blk >= job.part[pi].blocks) blk -= job.part[pi++].blocks;
  const PlanePart& part = job.part[pi];
  const int pair = blockIdx.y, b = pair / a.hk, hk = pair % a.hk, group = a.hq / a.hk, r0 = blk * 64;
  const int end = part.keys ? cross_len(a.kv_lens, b, a.kv_len) : cross_len(a.q_lens, b, a.q_len);
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  const int n = part.keys ? a.kv_len : job.rows, c = (threadIdx.x % V) * 4;
#pragma unroll
  for (int i = 0; i < 64 / RP; ++i) {
    const int lr = i * RP + threadIdx.x / V, r = r0 + lr;
    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int t = part.keys ? r : r % a.q_len, h = part.keys ? hk : hk * group + r / a.q_len;
    const bool in = r < n && t < end && (!part.keys || !mask || mask[r]);
    const long long at = b * part.st.b + h * part.st.h + t * part.st.t + c;
    const auto read = [&](const float* src, float (&x)[4]) {
      if (vec && c < a.d) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(src + at));
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < a.d) x[e] = src[at + e];
      }
    };
    if (in) read(part.src, f);
    if (part.terms) {
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, lse = -INFINITY;
      if (in) {
        lse = job.lse[(static_cast<long long>(b) * a.hq + h) * a.q_len + t];
        read(job.out, o);
      }
      float sum = fmaf(f[0], o[0], fmaf(f[1], o[1], fmaf(f[2], o[2], f[3] * o[3])));
#pragma unroll
      for (int s = V / 2; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      // Rows that are not computed or see no key: every weight exp2(s - inf) is 0.
      if (c == 0)
        job.terms[static_cast<long long>(pair) * job.rows_pad + r] =
            lse == -INFINITY ? make_float2(-INFINITY, 0.0f) : make_float2(-lse * kLog2e, -sum);
    }
    if (part.cols) {
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[lr][c + e] = f[e];
    }
    if (part.rows && r < n) {
      float hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) hi[e] = tf32_round(f[e]), lo[e] = tf32_round(f[e] - hi[e]);
      float* o = part.rows + (static_cast<long long>(pair) * n + r) * D + c;
      *reinterpret_cast<float4*>(o) = make_float4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<float4*>(o + static_cast<long long>(job.pairs) * n * D) = make_float4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
  if (!part.cols) return;
  __syncthreads();
  const int pad = part.keys ? job.kv_pad : job.rows_pad;
  float* o = part.cols + static_cast<long long>(pair) * D * pad + r0;
  const long long lo = static_cast<long long>(job.pairs) * D * pad;
  for (int i = threadIdx.x; i < 64 * D; i += 256) {
    const int d = i / 64, k = i % 64;
    const float x = tile[k][d], h = tf32_round(x);
    o[static_cast<long long>(d) * pad + k] = h;
    o[static_cast<long long>(d) * pad + k + lo] = tf32_round(x - h);
  }
}

// ---- building blocks ------------------------------------------------------------------------
// A streamed tile: T rows of a row plane from row0 (`dst` + lo * 16 KB + chunk of 32 columns), or T columns of a
// transposed plane from row0.
template <int D, bool COLS>
__device__ __forceinline__ void load_piece(uint8_t* dst, const CUtensorMap* map, int row0, int pair, int pairs,
                                           uint64_t* bar) {
  constexpr int T = 4096 / D, CH = (COLS ? T : D) / 32, BYTES = (COLS ? D : T) * 128;
#pragma unroll
  for (int lo = 0; lo < 2; ++lo)
#pragma unroll
    for (int c = 0; c < CH; ++c)
      tma_load_3d(dst + lo * (PIECE / 2) + c * BYTES, map, COLS ? row0 + c * 32 : c * 32, COLS ? 0 : row0,
                  pair + lo * pairs, bar);
}
// 128 rows of a row plane (boxes of T rows): hi at dst, lo behind it.
template <int D>
__device__ __forceinline__ void load_rows(uint8_t* dst, const CUtensorMap* map, int row0, int pair, int pairs, uint64_t* bar) {
  constexpr int T = 4096 / D;
  for (int lo = 0; lo < 2; ++lo)
    for (int c = 0; c < D / 32; ++c)
      for (int i = 0; i < TILE / T; ++i)
        tma_load_3d(dst + (lo * (D / 32) + c) * ACH + i * T * 128, map, c * 32, row0 + i * T, pair + lo * pairs, bar);
}
// The small products first: the tensor core truncates after each step, by 2^-24 of what has been summed so far.
// d[128 x T] = A[128 x D] . piece[T x D]^T, A in shared memory.
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d, const uint8_t* a, const uint8_t* piece) {
  constexpr int T = 4096 / D;
  constexpr uint32_t IDESC = idesc_tf32_f32(TILE, T, 0, 0);
  const uint64_t ah = smem_desc_sw128(smem_u32(a), 16, 1024), al = smem_desc_sw128(smem_u32(a + D / 32 * ACH), 16, 1024);
  const uint64_t bh = smem_desc_sw128(smem_u32(piece), 16, 1024), bl = smem_desc_sw128(smem_u32(piece + PIECE / 2), 16, 1024);
  // (Chunks of 32 values, four steps each.)
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const uint32_t ao = c * ACH >> 4, bo = c * T * 128 >> 4;
    umma_tf32_ss4_w(d, al + ao, bh + bo, IDESC, c > 0 ? 1u : 0u);
    umma_tf32_ss4_w(d, ah + ao, bl + bo, IDESC, 1u);
  }
#pragma unroll
  for (int c = 0; c < D / 32; ++c) umma_tf32_ss4_w(d, ah + (c * ACH >> 4), bh + (c * T * 128 >> 4), IDESC, 1u);
}
// d[128 x N] = A[128 x K] . piece[N x K]^T, A's hi and lo columns in TMEM.
template <int N, int K>
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t ah, uint32_t al, const uint8_t* piece) {
  constexpr uint32_t IDESC = idesc_tf32_f32(TILE, N, 0, 0);
  const uint64_t bh = smem_desc_sw128(smem_u32(piece), 16, 1024), bl = smem_desc_sw128(smem_u32(piece + PIECE / 2), 16, 1024);
#pragma unroll
  for (int c = 0; c < K / 32; ++c) {
    umma_tf32_ts4k_w(d, al + c * 32, bh + (c * N * 128 >> 4), IDESC, c > 0 ? 1u : 0u);
    umma_tf32_ts4k_w(d, ah + c * 32, bl + (c * N * 128 >> 4), IDESC, 1u);
  }
#pragma unroll
  for (int c = 0; c < K / 32; ++c) umma_tf32_ts4k_w(d, ah + c * 32, bh + (c * N * 128 >> 4), IDESC, 1u);
}
template <int N>
__device__ __forceinline__ void tmem_read(uint32_t at, uint32_t (&r)[N]) {
  if constexpr (N == 32)
    tmem_ld32(at, r);
  else
    tmem_ld16(at, r);
}
// Hi and lo parts of 16 values into two groups of 16 columns (the tensor core ignores the 13 low bits: half a unit is
// added to the bits of hi, and 2^-11 of itself, half a unit to one, to lo: off by 2^-11 of lo at most either way).
// The hi part of a NaN may be anything, as the carry reaches its sign; the lo part of a NaN and of an infinity is
// NaN, which adding to the bits would lose and the multiplication keeps.
__device__ __forceinline__ void put_split(uint32_t hi_at, uint32_t lo_at, const float* v) {
  uint32_t wh[16], wl[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float h = __uint_as_float((__float_as_uint(v[i]) + 0x1000u) & 0xffffe000u);
    wh[i] = __float_as_uint(h);
    wl[i] = __float_as_uint((v[i] - h) * 1.00048828125f);
  }
  tmem_st16(hi_at, wh);
  tmem_st16(lo_at, wl);
}
// Stores N columns from column c0 of one row, scaled.
template <int N>
__device__ __forceinline__ void store_cols(float* out, const float* v, float f, int c0, int d, bool vec) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const int c = c0 + e;
    if (vec) {
      if (c < d) *reinterpret_cast<float4*>(out + c) = make_float4(v[e] * f, v[e + 1] * f, v[e + 2] * f, v[e + 3] * f);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < d) out[c + i] = v[e + i] * f;
    }
  }
}

// ---- forward --------------------------------------------------------------------------------
//   warp 0      TMA: Q once, K tiles into two stages freed by S_j; warp 6: V^T tiles, freed by P.V_j (two stages;
//               one at D = 128, where Q takes 128 KB)
//   warp 1      MMA: S_j into one of two TMEM buffers, O_j = P_j V_j with P from TMEM into one of two buffers, a
//               fresh partial per tile
//   warps 2..5, 7..10   softmax, two warps to a row, half of its score and output columns each; the previous tile's
//               partial is folded into registers (O * alpha + O_j).  At D = 64 they swap the row's maximum through
//               tagged shared-memory words and P_hi lies over S_j's columns; at D = 128 a tile has 32 keys, each
//               warp reads them all and P_hi has columns of its own.
// The tensor pipe bounds it: 1536 cycles a tile of 64 keys at D = 64.
// B200, [4, 16, 333 x 1000, 64] with holes: 82 us, planes included (370 us on the CUDA cores); D = 128: 174 (698).
template <int D>
struct Fwd {
  static constexpr int T = 4096 / D, VS = D == 64 ? 2 : 1, OC = D / 2;
  static constexpr uint32_t S_COL = 0, PH_COL = D == 64 ? 0 : 2 * T, PL_COL = D == 64 ? 2 * T : 4 * T, O_COL = 256;
  static constexpr int K_OFF = D / 32 * ACH * 2, V_OFF = K_OFF + 2 * PIECE, TAIL_OFF = V_OFF + VS * PIECE;
  struct Tail {
    uint64_t q_full, k_full[2], v_full[2], s_full[2], p_full[2], o_full[2], o_free[2], drain;
    unsigned long long xmax[D == 64 ? 2 : 1][D == 64 ? 2 : 1][D == 64 ? TILE : 1];  // [tile & 1][half][row], tagged with the tile
    unsigned long long xsum[D == 64 ? 2 : 1][D == 64 ? TILE : 1];                   // [half][row]: final sums
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t SMEM = 1024 + TAIL_OFF + sizeof(Tail);
  static_assert(SMEM <= 232448);
};

constexpr int FWD_THREADS = 352;

template <int D>
__global__ void __launch_bounds__(FWD_THREADS, 1)
    cross_f32_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const CrossArgs a, const CrossSplit sp, int pairs,
                        float scale_log2, int vec_out, unsigned* err) {
  using F = Fwd<D>;
  constexpr int T = F::T, OC = F::OC;
  griddep_launch_dependents();  // the parts' join waits for the end of this grid
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  typename F::Tail* st = reinterpret_cast<typename F::Tail*>(smem + F::TAIL_OFF);
  const auto sK = [&](int j) { return smem + F::K_OFF + (j & 1) * PIECE; };
  const auto sV = [&](int j) { return smem + F::V_OFF + (j % F::VS) * PIECE; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.hq / a.hk, rows = group * a.q_len, row_tiles = (rows + TILE - 1) / TILE;
  const int pair = blockIdx.x / row_tiles, b = pair / a.hk, hk = pair % a.hk;
  const int r0 = (blockIdx.x % row_tiles) * TILE;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  const int tiles = (kv_end + T - 1) / T, per = (tiles + sp.splits - 1) / sp.splits;
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
  }
  if constexpr (D == 64) {
    for (int i = threadIdx.x; i < 2 * 2 * TILE; i += FWD_THREADS) (&st->xmax[0][0][0])[i] = ~0ull;
    for (int i = threadIdx.x; i < 2 * TILE; i += FWD_THREADS) (&st->xsum[0][0])[i] = ~0ull;
  }
  if (warp == 0) {
    tmem_alloc(&st->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_wait();  // the planes
  const uint32_t tmem = st->tmem_base;
  volatile int* abort_flag = &st->abort_flag;

  if (warp == 0 || warp == 6) {
    // ------------------------------------------------------------ Q and K loads (warp 0), V^T loads (warp 6)
    if (lane == 0) {
      const bool v = warp == 6;
      if (!v && n > 0) {
        mbar_arrive_expect_tx(&st->q_full, D / 32 * ACH * 2);
        load_rows<D>(smem, &map_q, r0, pair, pairs, &st->q_full);
      }
      const int stages = v ? F::VS : 2;
      uint64_t *full = v ? st->v_full : st->k_full, *used = v ? st->o_full : st->s_full;
      int j = 0;
      for (; j < n; ++j) {
        uint64_t* bar = &full[j % stages];
        // The stage's last tile has been read (the one commit of its products); its barrier's next
        // completion needs this load, so the parity wait is unambiguous.
        if (j >= stages && !mbar_wait_bounded(&used[(j - stages) & 1], ((j - stages) >> 1) & 1, abort_flag, err, kErrCrossLoadWait))
          break;
        mbar_arrive_expect_tx(bar, PIECE);
        if (v)
          load_piece<D, true>(sV(j), &map_v, (t_lo + j) * T, pair, pairs, bar);
        else
          load_piece<D, false>(sK(j), &map_k, (t_lo + j) * T, pair, pairs, bar);
      }
      if (j < n) {
        if (!v) drain_bar(&st->q_full, 0);
        for (int i = max(0, j - stages); i < j; ++i) drain_bar(&full[i % stages], (i / stages) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA (whole warp)
    bool ok = n > 0, issued = false;
    const auto wait = [&](uint64_t* bar, uint32_t ph) { return warp_wait_ready(bar, ph, abort_flag, err, kErrCrossMmaWait); };
    const auto issue_s = [&](int j) {
      if (!wait(&st->k_full[j & 1], (j >> 1) & 1)) return false;
      tc_fence_after();
      mma_scores<D>(tmem + F::S_COL + static_cast<uint32_t>((j & 1) * T), smem, sK(j));
      issued = true;
      umma_commit_w(&st->s_full[j & 1]);
      return true;
    };
    if (ok) ok = wait(&st->q_full, 0) && issue_s(0);
    for (int j = 0; j < n && ok; ++j) {
      const int s = j & 1;
      if (j + 1 < n && !(ok = issue_s(j + 1))) break;
      // Each barrier's next completion needs what is issued after these waits.
      if (!(ok = wait(&st->p_full[s], (j >> 1) & 1) && wait(&st->v_full[j % F::VS], (j / F::VS) & 1) &&
                 (j < 2 || wait(&st->o_free[s], ((j - 2) >> 1) & 1))))
        break;
      tc_fence_after();
      mma_tmem<D, T>(tmem + F::O_COL + static_cast<uint32_t>(s * D), tmem + F::PH_COL + static_cast<uint32_t>(s * T),
                     tmem + F::PL_COL + static_cast<uint32_t>(s * T), sV(j));
      umma_commit_w(&st->o_full[s]);
    }
    if (!ok && issued) {
      umma_commit_w(&st->drain);
      drain_bar(&st->drain, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax, fold, epilogue
    const int quarter = warp & 3, half = warp >= 7 ? 1 : 0;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const float floor = cross_floor(scale_log2);
    float m = -INFINITY, l = 0.0f, alpha_prev = 1.0f, o_acc[OC];
#pragma unroll
    for (int e = 0; e < OC; ++e) o_acc[e] = 0.0f;
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
      if (!warp_wait_ready(&st->o_full[t & 1], (t >> 1) & 1, abort_flag, err, kErrCrossSoftmaxWait)) return false;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < OC; c += 32) {
        uint32_t r[32];
        tmem_ld32(lanes + F::O_COL + static_cast<uint32_t>((t & 1) * D + half * OC + c), r);
#pragma unroll
        for (int e = 0; e < 32; ++e) o_acc[c + e] = __fmaf_rn(o_acc[c + e], alpha, __uint_as_float(r[e]));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->o_free[t & 1]);
      return true;
    };
    for (int j = 0; j < n; ++j) {
      const int s = j & 1, own = D == 64 ? half * 32 : 0, kv0 = (t_lo + j) * T + own;  // first key of the 32 read here
      const bool partial = mask || kv0 + 32 > kv_end;
      bool seen = true;
      if (partial) seen = kv0 + lane < kv_end && (!mask || mask[kv0 + lane]);
      if (!(ok = warp_wait_ready(&st->s_full[s], (j >> 1) & 1, abort_flag, err, kErrCrossSoftmaxWait))) break;
      tc_fence_after();
      uint32_t r[32];
      tmem_ld32(lanes + F::S_COL + static_cast<uint32_t>(s * T + own), r);
      float lowest = floor;  // of the maximum, unless none of these keys is visible
      if (partial) {
        const unsigned w = __ballot_sync(0xffffffffu, seen);
        if (!w) lowest = -INFINITY;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!((w >> e) & 1u)) r[e] = __float_as_uint(-INFINITY);
      }
      float mx4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) mx4[i] = __uint_as_float(r[i]);
#pragma unroll
      for (int e = 4; e < 32; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(r[e]));
      float mx = fmaxf(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), lowest);
      if constexpr (D == 64) {
        // Slot [j & 1] is written again for tile j + 2 only after the partner published tile j + 1, which it does
        // after reading this one.  The verdict is made uniform: the tcgen05 accesses are warp-collective.
        float mo;
        if (!(ok = __all_sync(0xffffffffu, swap(&st->xmax[s][half][row], &st->xmax[s][half ^ 1][row],
                                                static_cast<uint32_t>(j), mx, &mo))))
          break;
        mx = fmaxf(mx, mo);
      }
      mx *= scale_log2;
      float alpha = 1.0f;
      if (mx > m + kRescale) {
        alpha = m == -INFINITY ? 0.0f : exp2f(m - mx);
        l *= alpha;
        m = mx;
      }
      const float mu = m == -INFINITY ? 0.0f : m;  // nothing seen yet: every weight is 0
      float p[32], ls4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        p[e] = fast_exp2(__fmaf_rn(__uint_as_float(r[e]), scale_log2, -mu));
        ls4[e & 3] += p[e];
      }
      l += (ls4[0] + ls4[1]) + (ls4[2] + ls4[3]);
      const uint32_t ph = lanes + F::PH_COL + static_cast<uint32_t>(s * T), pl = lanes + F::PL_COL + static_cast<uint32_t>(s * T);
      if constexpr (D == 64) {
        put_split(ph + own, pl + own, p);
        put_split(ph + own + 16, pl + own + 16, p + 16);
      } else if (half == 0) {
        put_split(ph, pl, p);
      } else {
        put_split(ph + 16, pl + 16, p + 16);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st->p_full[s]);
      // The previous tile's partial (formed with the previous maximum), then this tile's factor for its own.
      if (j > 0 && !(ok = fold(j - 1, alpha_prev))) break;
      alpha_prev = alpha;
    }
    if (ok && n > 0) ok = fold(n - 1, alpha_prev);
    if constexpr (D == 64) {
      float other = 0.0f;
      if (ok && n > 0) ok = swap(&st->xsum[half][row], &st->xsum[half ^ 1][row], static_cast<uint32_t>(n), l, &other);
      l = half == 0 ? l + other : other + l;
    }
    const int rr = r0 + row, g = rr / a.q_len, t = rr % a.q_len;
    if (ok && rr < rows && t < q_end) {
      const bool empty = m == -INFINITY, split = sp.splits > 1;
      const long long at = (static_cast<long long>(b) * a.hq + hk * group) * a.q_len + rr;  // dense row
      const float f = split ? 1.0f : cross_inverse(m, l);  // (without a key the sums are 0)
      if (half == 0) {
        if (split)
          sp.ml[static_cast<long long>(blockIdx.y) * sp.rows + at] = make_float2(m, empty ? 0.0f : l);
        else if (a.lse)
          a.lse[at] = cross_lse(m, l);
      }
      float* out = split ? sp.o + (static_cast<long long>(blockIdx.y) * sp.rows + at) * a.d
                         : static_cast<float*>(a.out) + b * a.os.b + (hk * group + g) * a.os.h + t * a.os.t;
      store_cols<OC>(out, o_acc, f, half * OC, a.d, vec_out || (split && a.d % 4 == 0));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- backward -------------------------------------------------------------------------------
// One launch, a block to 128 keys or 128 rows of a pair and a pass:
//   dk, dv   A = K in shared memory, X = V in TMEM; streams Q, dO and their transposes.
//            S^T = K Q^T, dP^T = V dO^T; dv += P^T dO, dk += dS^T Q.  (D = 128: a pass each, for TMEM's sake.)
//   dq       A = Q, X = dO; streams K, V, K^T.  S = Q K^T, dP = dO V^T; dq += dS K.
//   warp 0  TMA: A once, then the pieces of 32 KB of tile after tile through a ring
//   warp 1  MMA: S, dP, then the sums with P and dS (hi and lo) from TMEM; the next tile's S and dP run while the
//           sums are folded
//   warps 2..9  X into TMEM, then two warps to a row: P, dS, and a tile's sums folded into registers
// The tensor pipe bounds it: 96 steps of 32 cycles a tile of 64 rows for dk and dv at D = 64, 72 for dq.
// B200, [4, 16, 333 x 1000, 64]: 232 us, planes included (782 on the CUDA cores), D = 128: 559 (1852); one row a pair
// 112 (226); [2, 8, 77 x 300, 64] 27 (84).
enum GradPass { kGradDq, kGradDkv, kGradDk, kGradDv };

template <int D>
struct Grad {
  static constexpr int T = 4096 / D, NP = D == 64 ? 5 : 3, SC = T / 2;
  static constexpr uint32_t S_COL = 0, PL_COL = T, DP_COL = 2 * T, DL_COL = 3 * T, X_COL = 4 * T, O_COL = 384;
  static constexpr int R_OFF = D / 32 * ACH * 2, TAIL_OFF = R_OFF + NP * PIECE;
  struct Tail {
    float2 terms[2][T];
    uint64_t a_full, x_full, full[NP], used[NP], t_full[2], s_full, dp_full, p_full, ds_full, o_full, o_free, drain;
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t SMEM = 1024 + TAIL_OFF + sizeof(Tail);
  static_assert(SMEM <= 232448);
};

struct GradParams {
  CUtensorMap qr, gr, kr, vr, qt, gt, kt;
  CrossGradArgs g;
  const float *g_rows, *v_rows;
  const float2* terms;
  int pairs, rows_pad, key_tiles, row_tiles, key_jobs;  // key_jobs: of a pass over the keys
  float scale_log2;
  int vec_q, vec_k, vec_v;
  unsigned* err;
};

constexpr int GRAD_THREADS = 320;

template <int D>
__global__ void __launch_bounds__(GRAD_THREADS, 1) cross_grad_f32_tc_kernel(const __grid_constant__ GradParams p) {
  using G = Grad<D>;
  constexpr int T = G::T, SC = G::SC, NP = G::NP;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  typename G::Tail* st = reinterpret_cast<typename G::Tail*>(smem + G::TAIL_OFF);
  const CrossArgs& a = p.g.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.hq / a.hk, rows = group * a.q_len;
  int job = blockIdx.x;
  GradPass pass = kGradDq;
  if constexpr (D == 64) {
    if (job < p.key_jobs)
      pass = kGradDkv;
    else
      job -= p.key_jobs;
  } else {
    if (job < p.key_jobs)
      pass = kGradDk;
    else if ((job -= p.key_jobs) < p.key_jobs)
      pass = kGradDv;
    else
      job -= p.key_jobs;
  }
  const bool keys = pass != kGradDq, with_p = pass == kGradDkv || pass == kGradDv, with_ds = pass != kGradDv;
  const int per_pair = keys ? p.key_tiles : p.row_tiles;
  const int pair = job / per_pair, b = pair / a.hk, hk = pair % a.hk, r0 = (job % per_pair) * TILE;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  // The streamed extent.  Rows of a group of one head end at q_end; those of several lie behind one another.
  const int row_end = q_end == 0 ? 0 : group == 1 ? q_end : rows;
  const bool idle = keys ? r0 >= kv_end : r0 >= row_end;
  const int n = idle ? 0 : ((keys ? row_end : kv_end) + T - 1) / T;

  if (threadIdx.x == 0) {
    mbar_init(&st->a_full, 1);
    mbar_init(&st->x_full, 8);
    for (int i = 0; i < NP; ++i) {
      mbar_init(&st->full[i], 1);
      mbar_init(&st->used[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&st->t_full[i], 1);
    mbar_init(&st->s_full, 1);
    mbar_init(&st->dp_full, 1);
    mbar_init(&st->p_full, 8);
    mbar_init(&st->ds_full, 8);
    mbar_init(&st->o_full, 1);
    mbar_init(&st->o_free, 8);
    mbar_init(&st->drain, 1);
    st->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(&st->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_wait();  // the planes
  const uint32_t tmem = st->tmem_base;
  volatile int* abort_flag = &st->abort_flag;
  const auto slot = [&](int i) { return smem + G::R_OFF + (i % NP) * PIECE; };

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(&st->a_full, D / 32 * ACH * 2);
      load_rows<D>(smem, keys ? &p.kr : &p.qr, r0, pair, p.pairs, &st->a_full);
      int i = 0;
      // Room for the next piece: the commit of the slot's last reader, whose barrier completes again only after
      // this load.
      const auto room = [&](uint32_t bytes) {
        if (i >= NP &&
            !mbar_wait_bounded(&st->used[i % NP], (i / NP - 1) & 1, abort_flag, p.err, kErrCrossLoadWait))
          return false;
        mbar_arrive_expect_tx(&st->full[i % NP], bytes);
        return true;
      };
      bool ok = true;
      int terms = 0;
      for (int j = 0; j < n && ok; ++j) {
        const int t0 = j * T;
        if (!(ok = room(PIECE))) break;
        load_piece<D, false>(slot(i), keys ? &p.qr : &p.kr, t0, pair, p.pairs, &st->full[i % NP]);
        // (A buffer of terms is written two tiles later, when pieces behind its tile's last product were read.)
        if (keys) {
          mbar_arrive_expect_tx(&st->t_full[j & 1], T * sizeof(float2));
          bulk_load(st->terms[j & 1], p.terms + static_cast<long long>(pair) * p.rows_pad + t0, T * sizeof(float2),
                    &st->t_full[j & 1]);
          ++terms;
        }
        ++i;
        if (with_ds) {
          if (!(ok = room(PIECE))) break;
          load_piece<D, false>(slot(i), keys ? &p.gr : &p.vr, t0, pair, p.pairs, &st->full[i % NP]);
          ++i;
        }
        if (with_p) {
          if (!(ok = room(PIECE))) break;
          load_piece<D, true>(slot(i), &p.gt, t0, pair, p.pairs, &st->full[i % NP]);
          ++i;
        }
        if (with_ds) {
          if (!(ok = room(PIECE))) break;
          load_piece<D, true>(slot(i), keys ? &p.qt : &p.kt, t0, pair, p.pairs, &st->full[i % NP]);
          ++i;
        }
      }
      if (!ok) {
        drain_bar(&st->a_full, 0);
        for (int k = max(0, i - NP); k < i; ++k) drain_bar(&st->full[k % NP], (k / NP) & 1);
        for (int k = max(0, terms - 2); k < terms; ++k) drain_bar(&st->t_full[k & 1], (k >> 1) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA (whole warp)
    const auto wait = [&](uint64_t* bar, uint32_t ph) { return warp_wait_ready(bar, ph, abort_flag, p.err, kErrCrossMmaWait); };
    bool issued = false, ok = n > 0;
    int i = 0;
    const auto piece = [&] { return wait(&st->full[i % NP], (i / NP) & 1); };
    const auto done = [&] { umma_commit_w(&st->used[i++ % NP]); };
    if (ok) ok = wait(&st->a_full, 0) && (!with_ds || wait(&st->x_full, 0));
    for (int j = 0; j < n && ok; ++j) {
      const uint32_t ph = j & 1;
      if (!(ok = piece())) break;
      tc_fence_after();
      mma_scores<D>(tmem + G::S_COL, smem, slot(i));
      issued = true;
      umma_commit_w(&st->s_full);
      done();
      if (with_ds) {
        if (!(ok = piece())) break;
        tc_fence_after();
        mma_tmem<T, D>(tmem + G::DP_COL, tmem + G::X_COL, tmem + G::X_COL + D, slot(i));
        umma_commit_w(&st->dp_full);
        done();
      }
      // The last tile's sums have been folded (the barrier's next completion needs this tile's sums).
      if (j > 0 && !(ok = wait(&st->o_free, ph ^ 1))) break;
      if (with_p) {
        if (!(ok = wait(&st->p_full, ph) && piece())) break;
        tc_fence_after();
        mma_tmem<D, T>(tmem + G::O_COL, tmem + G::S_COL, tmem + G::PL_COL, slot(i));
        if (!with_ds) umma_commit_w(&st->o_full);
        done();
      }
      if (with_ds) {
        if (!(ok = wait(&st->ds_full, ph) && piece())) break;
        tc_fence_after();
        mma_tmem<D, T>(tmem + G::O_COL + (D == 64 ? 64 : 0), tmem + G::DP_COL, tmem + G::DL_COL, slot(i));
        umma_commit_w(&st->o_full);
        done();
      }
    }
    if (!ok && issued) {
      umma_commit_w(&st->drain);
      drain_bar(&st->drain, 0);
    }
  } else {
    // ------------------------------------------------------------ weights, their gradient, fold, epilogue
    const int quarter = warp & 3, half = warp >= 6 ? 1 : 0;
    const int row = quarter * 32 + lane, r = r0 + row;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16), hc = static_cast<uint32_t>(half * SC);
    const auto wait = [&](uint64_t* bar, uint32_t ph) { return warp_wait_ready(bar, ph, abort_flag, p.err, kErrCrossSoftmaxWait); };
    const auto arrive = [&](uint64_t* bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    float acc[64];  // D = 64: 32 columns of dv, 32 of dk or dq; D = 128: 64 columns of one of them
#pragma unroll
    for (int e = 0; e < 64; ++e) acc[e] = 0.0f;
    bool ok = true, seen = true;
    float2 mine = make_float2(-INFINITY, 0.0f);
    if (n > 0) {
      if (with_ds) {
        const int most = keys ? a.kv_len : rows;
        const float* x = (keys ? p.v_rows : p.g_rows) + (static_cast<long long>(pair + half * p.pairs) * most + r) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 v = r < most ? *reinterpret_cast<const float4*>(x + c + e) : make_float4(0.f, 0.f, 0.f, 0.f);
            w[e] = __float_as_uint(v.x), w[e + 1] = __float_as_uint(v.y);
            w[e + 2] = __float_as_uint(v.z), w[e + 3] = __float_as_uint(v.w);
          }
          tmem_st16(lanes + G::X_COL + static_cast<uint32_t>(half * D + c), w);
        }
        tmem_wait_st();
        arrive(&st->x_full);
      }
      if (keys)
        seen = r < kv_end && (!mask || mask[r]);
      else if (r < rows)
        mine = p.terms[static_cast<long long>(pair) * p.rows_pad + r];
    }
    for (int j = 0; j < n; ++j) {
      const uint32_t ph = j & 1;
      unsigned vis = 0xffffffffu;
      if (!keys) {
        const int k = j * T + half * SC + lane;
        if (mask || (j + 1) * T > kv_end) vis = __ballot_sync(0xffffffffu, lane < SC && k < kv_end && (!mask || mask[k]));
      }
      if (keys && !(ok = wait(&st->t_full[ph], (j >> 1) & 1))) break;
      if (!(ok = wait(&st->s_full, ph))) break;
      tc_fence_after();
      uint32_t w[SC];
      float pr[SC];
      tmem_read<SC>(lanes + G::S_COL + hc, w);
      const float2* tm = st->terms[ph] + half * SC;
#pragma unroll
      for (int e = 0; e < SC; ++e) {
        const float x = fast_exp2(__fmaf_rn(__uint_as_float(w[e]), p.scale_log2, keys ? tm[e].x : mine.x));
        pr[e] = (keys ? seen : ((vis >> e) & 1u) != 0) ? x : 0.0f;
      }
      if (with_p) {
#pragma unroll
        for (int c = 0; c < SC; c += 16) put_split(lanes + G::S_COL + hc + c, lanes + G::PL_COL + hc + c, pr + c);
        tmem_wait_st();
        arrive(&st->p_full);
      }
      if (with_ds) {
        if (!(ok = wait(&st->dp_full, ph))) break;
        tc_fence_after();
        tmem_read<SC>(lanes + G::DP_COL + hc, w);
#pragma unroll
        for (int e = 0; e < SC; ++e) pr[e] *= __uint_as_float(w[e]) + (keys ? tm[e].y : mine.y);
#pragma unroll
        for (int c = 0; c < SC; c += 16) put_split(lanes + G::DP_COL + hc + c, lanes + G::DL_COL + hc + c, pr + c);
        tmem_wait_st();
        arrive(&st->ds_full);
      }
      if (!(ok = wait(&st->o_full, ph))) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        if (D == 64 && c == 0 && !with_p) continue;
        uint32_t o[32];
        tmem_ld32(lanes + G::O_COL + static_cast<uint32_t>(D == 64 ? c * 2 + half * 32 : half * 64 + c), o);
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[c + e] += __uint_as_float(o[e]);
      }
      arrive(&st->o_free);
    }
    // A masked key's sums, and those of a row that sees no key, hold weights of 0 times rows that may be NaN or infinite.
    if (keys ? !seen : mine.x == -INFINITY) {
#pragma unroll
      for (int e = 0; e < 64; ++e) acc[e] = 0.0f;
    }
    if (ok && keys && r < a.kv_len) {
      float* dk = static_cast<float*>(p.g.dk) + b * a.ks.b + hk * a.ks.h + r * a.ks.t;
      float* dv = static_cast<float*>(p.g.dv) + b * a.vs.b + hk * a.vs.h + r * a.vs.t;
      if constexpr (D == 64) {
        store_cols<32>(dv, acc, 1.0f, half * 32, a.d, p.vec_v);
        store_cols<32>(dk, acc + 32, a.scale, half * 32, a.d, p.vec_k);
      } else if (with_p) {
        store_cols<64>(dv, acc, 1.0f, half * 64, a.d, p.vec_v);
      } else {
        store_cols<64>(dk, acc, a.scale, half * 64, a.d, p.vec_k);
      }
    }
    if (ok && !keys && r < rows && r % a.q_len < q_end) {
      float* dq = static_cast<float*>(p.g.dq) + b * a.qs.b + (hk * group + r / a.q_len) * a.qs.h + (r % a.q_len) * a.qs.t;
      if constexpr (D == 64)
        store_cols<32>(dq, acc + 32, a.scale, half * 32, a.d, p.vec_q);
      else
        store_cols<64>(dq, acc, a.scale, half * 64, a.d, p.vec_q);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- host -----------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// fp32 [2 * pairs, rows, cols], box [1, box_rows, 32], 128-byte swizzle, zeros outside.
bool plane_map(CUtensorMap* map, const void* base, int pairs, int rows, int cols, int box_rows) {
  auto enc = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!enc) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), 2 * static_cast<cuuint64_t>(pairs)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 4, static_cast<cuuint64_t>(rows) * cols * 4};
  const cuuint32_t box[3] = {32, static_cast<cuuint32_t>(box_rows), 1}, estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool rows4(const void* p, const HeadStrides& s, int d) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && d % 4 == 0 && s.b % 4 == 0 && s.h % 4 == 0 && s.t % 4 == 0;
}

struct PlaneSizes {
  int rows, pairs, rows_pad, kv_pad, q_blocks, k_blocks;
  long long q, k, qt, kt;  // floats of hi and lo planes
  PlaneSizes(const CrossArgs& a, int D) {
    rows = a.hq / a.hk * a.q_len;
    pairs = a.batch * a.hk;
    q_blocks = (rows + 63) / 64;
    k_blocks = (a.kv_len + 63) / 64;
    rows_pad = q_blocks * 64;
    kv_pad = k_blocks * 64;
    const long long n = 2LL * pairs * D;
    q = n * rows, k = n * a.kv_len, qt = n * rows_pad, kt = n * kv_pad;
  }
};

template <int D>
cudaError_t fwd_f32(const CrossArgs& a, cudaStream_t s) {
  using F = Fwd<D>;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const PlaneSizes z(a, D);
  const long long blocks = static_cast<long long>((z.rows + TILE - 1) / TILE) * z.pairs;
  if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
  static std::atomic<unsigned long long> attr{0};
  cudaError_t e = once_per_device(attr, [] {
    return cudaFuncSetAttribute(cross_f32_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(F::SMEM));
  });
  if (e != cudaSuccess) return e;
  void* ws = nullptr;
  if ((e = workspace_alloc(ctx, &ws, (z.q + z.k + z.kt) * sizeof(float), s)) != cudaSuccess) return e;
  float *q = static_cast<float*>(ws), *k = q + z.q, *vt = k + z.k;
  PlaneJob job{};
  job.part[0] = {static_cast<const float*>(a.q), a.qs, 0, z.q_blocks, q, nullptr, 0};
  job.part[1] = {static_cast<const float*>(a.k), a.ks, 1, z.k_blocks, k, nullptr, 0};
  job.part[2] = {static_cast<const float*>(a.v), a.vs, 1, z.k_blocks, nullptr, vt, 0};
  job.rows = z.rows, job.rows_pad = z.rows_pad, job.kv_pad = z.kv_pad, job.pairs = z.pairs;
  CUtensorMap mq, mk, mv;
  if (!plane_map(&mq, q, z.pairs, z.rows, D, F::T) || !plane_map(&mk, k, z.pairs, a.kv_len, D, F::T) ||
      !plane_map(&mv, vt, z.pairs, D, z.kv_pad, D))
    e = cudaErrorInvalidValue;
  if (e == cudaSuccess) {
    CrossSplitWork w;
    e = w.begin(a, blocks, F::T, 2, 1, s);
    if (e == cudaSuccess) {
      const int vec = rows4(a.q, a.qs, a.d) && rows4(a.k, a.ks, a.d) && rows4(a.v, a.vs, a.d);
      cross_split_kernel<D><<<dim3(z.q_blocks + 2 * z.k_blocks, z.pairs), 256, 0, s>>>(a, job, vec);
      e = cudaGetLastError();
      if (e == cudaSuccess)
        e = launch_pdl(cross_f32_tc_kernel<D>, dim3(static_cast<unsigned>(blocks), w.sp.splits), dim3(FWD_THREADS), F::SMEM,
                       s, mq, mk, mv, a, w.sp, z.pairs, a.scale * kLog2e, static_cast<int>(rows4(a.out, a.os, a.d)),
                       ctx->err_word);
      e = w.end(a, e, s);
    }
  }
  const cudaError_t f = workspace_free(ws, s);
  return e != cudaSuccess ? e : f;
}

template <int D>
cudaError_t bwd_f32(const CrossGradArgs& g, cudaStream_t s) {
  using G = Grad<D>;
  const CrossArgs& a = g.f;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const PlaneSizes z(a, D);
  GradParams p{};
  p.key_tiles = (a.kv_len + TILE - 1) / TILE;
  p.row_tiles = (z.rows + TILE - 1) / TILE;
  const long long key_jobs = g.dk ? static_cast<long long>(p.key_tiles) * z.pairs : 0;
  const long long blocks = key_jobs * (D == 64 ? 1 : 2) + (g.dq ? static_cast<long long>(p.row_tiles) * z.pairs : 0);
  if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
  static std::atomic<unsigned long long> attr{0};
  cudaError_t e = once_per_device(attr, [] {
    return cudaFuncSetAttribute(cross_grad_f32_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(G::SMEM));
  });
  if (e != cudaSuccess) return e;
  // Transposes only for the sums that are asked for.
  const long long qt = g.dk ? z.qt : 0, kt = g.dq ? z.kt : 0;
  const long long n_terms = static_cast<long long>(z.pairs) * z.rows_pad;
  void* ws = nullptr;
  e = workspace_alloc(ctx, &ws, (2 * z.q + 2 * z.k + 2 * qt + kt) * sizeof(float) + n_terms * sizeof(float2), s);
  if (e != cudaSuccess) return e;
  float *q = static_cast<float*>(ws), *go = q + z.q, *k = go + z.q, *v = k + z.k, *q_t = v + z.k, *g_t = q_t + qt, *k_t = g_t + qt;
  float2* terms = reinterpret_cast<float2*>(k_t + kt);
  PlaneJob job{};
  job.part[0] = {static_cast<const float*>(a.q), a.qs, 0, z.q_blocks, q, g.dk ? q_t : nullptr, 0};
  job.part[1] = {static_cast<const float*>(g.dout), a.os, 0, z.q_blocks, go, g.dk ? g_t : nullptr, 1};
  job.part[2] = {static_cast<const float*>(a.k), a.ks, 1, z.k_blocks, k, g.dq ? k_t : nullptr, 0};
  job.part[3] = {static_cast<const float*>(a.v), a.vs, 1, z.k_blocks, v, nullptr, 0};
  job.rows = z.rows, job.rows_pad = z.rows_pad, job.kv_pad = z.kv_pad, job.pairs = z.pairs;
  job.out = static_cast<const float*>(a.out), job.lse = a.lse, job.terms = terms;
  // A transpose that no pass reads has no plane; its map then stays unused.
  if (!plane_map(&p.qr, q, z.pairs, z.rows, D, G::T) || !plane_map(&p.gr, go, z.pairs, z.rows, D, G::T) ||
      !plane_map(&p.kr, k, z.pairs, a.kv_len, D, G::T) || !plane_map(&p.vr, v, z.pairs, a.kv_len, D, G::T) ||
      (g.dk && (!plane_map(&p.qt, q_t, z.pairs, D, z.rows_pad, D) || !plane_map(&p.gt, g_t, z.pairs, D, z.rows_pad, D))) ||
      (g.dq && !plane_map(&p.kt, k_t, z.pairs, D, z.kv_pad, D)))
    e = cudaErrorInvalidValue;
  if (e == cudaSuccess) {
    p.g = g;
    p.g_rows = go, p.v_rows = v, p.terms = terms;
    p.pairs = z.pairs, p.rows_pad = z.rows_pad, p.key_jobs = static_cast<int>(key_jobs);
    p.scale_log2 = a.scale * kLog2e;
    p.vec_q = rows4(g.dq, a.qs, a.d), p.vec_k = rows4(g.dk, a.ks, a.d), p.vec_v = rows4(g.dv, a.vs, a.d);
    p.err = ctx->err_word;
    const int vec = rows4(a.q, a.qs, a.d) && rows4(a.k, a.ks, a.d) && rows4(a.v, a.vs, a.d) && rows4(g.dout, a.os, a.d) &&
                    rows4(a.out, a.os, a.d);
    cross_split_kernel<D><<<dim3(2 * z.q_blocks + 2 * z.k_blocks, z.pairs), 256, 0, s>>>(a, job, vec);
    e = cudaGetLastError();
    if (e == cudaSuccess)
      e = launch_pdl(cross_grad_f32_tc_kernel<D>, dim3(static_cast<unsigned>(blocks)), dim3(GRAD_THREADS), G::SMEM, s, p);
  }
  const cudaError_t f = workspace_free(ws, s);
  return e != cudaSuccess ? e : f;
}

}  // namespace

// (A grid's second axis ends at 65535.)
bool cross_f32_tc_supported(const CrossArgs& a) {
  const long long rows = static_cast<long long>(a.hq / a.hk) * a.q_len, pairs = static_cast<long long>(a.batch) * a.hk;
  // From 8 rows a pair on (fewer go to the kernel of few rows, where their strides allow it) this beats the CUDA
  // cores although most of the tile is padding: [4, 16, R x 1000, 64] takes 45 / 50 us for R = 8 / 128 here and
  // 52 / 92 there, at 128 columns and R = 8 85 and 109; [16, 16, 512 x 16, 64] 77 and 94; one 64 x 64 tile 12.5 both.
  return !a.bf16 && a.d <= 128 && rows >= 8 && pairs <= 65535 && tensor_map_encoder() != nullptr;
}

cudaError_t cross_forward_f32_tc(const CrossArgs& a, cudaStream_t s) {
  return a.d <= 64 ? fwd_f32<64>(a, s) : fwd_f32<128>(a, s);
}

bool cross_grad_f32_tc_supported(const CrossGradArgs& g) {
  const CrossArgs& a = g.f;
  const long long pairs = static_cast<long long>(a.batch) * a.hk;
  // (Keys that all batch entries share have one gradient: a sum over the batch, left to the CUDA cores.)
  return !a.bf16 && a.d <= 128 && !(g.kv_shared && g.dk) && pairs <= 65535 && tensor_map_encoder() != nullptr;
}

cudaError_t cross_backward_f32_tc(const CrossGradArgs& g, cudaStream_t s) {
  return g.f.d <= 64 ? bwd_f32<64>(g, s) : bwd_f32<128>(g, s);
}

}  // namespace lcb
