// Cross attention (queries and keys of different lengths, shared key heads, strides, key masks) on
// CUDA cores: forward and backward for every type and head_dim <= 256, the combination of
// forward parts that were split along the keys, and the dispatch.
//
//   s_tj = scale * q_t . k_j over the visible keys j,  p = softmax_j(s),  out_t = sum_j p_tj v_j
//   D_t = dout_t . out_t,  ds_tj = p_tj (dout_t . v_j - D_t)
//   dq_t = scale * sum_j ds_tj k_j,  dk_j = scale * sum_t ds_tj q_t,  dv_j = sum_t p_tj dout_t
//
// Tiles of TT x TT rows and keys with TT/4 x TT/4 threads: a thread owns rows rg + i*GL and keys
// cg + j*GL (i, j < 4), so a row's statistics are xor-shuffles over the GL lanes that share rg.  All
// operands are staged as fp32, row-major with 4 floats of padding: then the lanes' float4 reads of
// K rows (stride DP + 4 words) fall on different banks, every global read is contiguous, and the
// two inner products read 8 float4 for 64 FMAs.  Masked keys and rows past the end are staged as
// zeros and their scores replaced, so what memory holds there never enters a sum.
// Bound by shared-memory reads and issue slots.  B200, fp32: [4, 16, 333 x 1000, 64] 370 us (15 TFLOP/s), backward 782;
// [4, 16, 333 x 1000, 200] 1500 us, backward 4480 (with tiles of 32 rows, 64 threads, 3560 and 16253: hence one buffer
// for two operands above 128 columns, which leaves room for tiles of 64).
// Rows of the heads that share a key head form one list (row = head-in-group * q_len + token), so
// a tile of few queries is filled by its group.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "cross_attention.cuh"
#include "lc_internal.hpp"

namespace lcb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
__device__ __forceinline__ float to_f(T v) { return static_cast<float>(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return static_cast<T>(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int DP, int TT>
struct Tile {
  static constexpr int LD = DP + 4;          // row stride in floats
  static constexpr int LP = TT + 4;          // row stride of a [TT][TT] tile
  static constexpr int GL = TT / 4;          // lanes that share a row, and row groups
  static constexpr int NT = GL * GL;         // threads
  static constexpr int CPT = DP / GL;        // output columns per thread: cg*4 + n*4*GL + e
  static constexpr int NC = CPT / 4;         // ... in float4s
  static constexpr int ROWS = TT * LD;       // floats of an operand tile
  static constexpr int SQ = TT * LP;         // floats of a score tile
};

// Stages TT rows of d values: row i of the tile is at src + off(i) (off < 0: zeros).
template <typename T, int DP, int TT, class Off>
__device__ __forceinline__ void stage(float* dst, const T* src, int d, bool vec, Off off) {
  using L = Tile<DP, TT>;
  if (vec) {
    constexpr int V = DP / 4;
    for (int i = threadIdx.x; i < TT * V; i += L::NT) {
      const int r = i / V, c = (i % V) * 4;
      const long long o = off(r);
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (o >= 0 && c < d) {
        if constexpr (sizeof(T) == 4) {
          f = *reinterpret_cast<const float4*>(src + o + c);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(src + o + c);
          f = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                          __uint_as_float(w.y & 0xffff0000u));
        }
      }
      *reinterpret_cast<float4*>(dst + r * L::LD + c) = f;
    }
  } else {
    for (int i = threadIdx.x; i < TT * DP; i += L::NT) {
      const int r = i / DP, c = i % DP;
      const long long o = off(r);
      dst[r * L::LD + c] = (o >= 0 && c < d) ? to_f(src[o + c]) : 0.0f;
    }
  }
}

// s[i][j] = X[rg + i*GL] . Y[cg + j*GL] over DP columns.
template <int DP, int TT>
__device__ __forceinline__ void dot_tile(const float* x, const float* y, int rg, int cg, float (&s)[4][4]) {
  using L = Tile<DP, TT>;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll 4
  for (int c = 0; c < DP; c += 4) {
    float4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(x + (rg + i * L::GL) * L::LD + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(y + (cg + j * L::GL) * L::LD + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s[i][j] = fmaf(a[i].w, b[j].w, fmaf(a[i].z, b[j].z, fmaf(a[i].y, b[j].y, fmaf(a[i].x, b[j].x, s[i][j]))));
  }
}

// o[i][.] += sum_k P[rg + i*GL][k] * V[k][this thread's columns].
template <int DP, int TT>
__device__ __forceinline__ void acc_tile(const float* p, const float* v, int rg, int cg,
                                         float (&o)[4][Tile<DP, TT>::CPT]) {
  using L = Tile<DP, TT>;
#pragma unroll 2
  for (int k = 0; k < TT; k += 4) {
    float4 pr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) pr[i] = *reinterpret_cast<const float4*>(p + (rg + i * L::GL) * L::LP + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int n = 0; n < L::NC; ++n) {
        const float4 b = *reinterpret_cast<const float4*>(v + (k + kk) * L::LD + cg * 4 + n * 4 * L::GL);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = kk == 0 ? pr[i].x : kk == 1 ? pr[i].y : kk == 2 ? pr[i].z : pr[i].w;
          o[i][n * 4 + 0] = fmaf(w, b.x, o[i][n * 4 + 0]);
          o[i][n * 4 + 1] = fmaf(w, b.y, o[i][n * 4 + 1]);
          o[i][n * 4 + 2] = fmaf(w, b.z, o[i][n * 4 + 2]);
          o[i][n * 4 + 3] = fmaf(w, b.w, o[i][n * 4 + 3]);
        }
      }
  }
}

template <int GL>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = GL / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int GL>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = GL / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Scales this thread's rows by f[i] and stores them: row i at out + off(i) (off < 0: not stored).
template <typename T, int DP, int TT, class Off>
__device__ __forceinline__ void store_rows(T* out, const float (&o)[4][Tile<DP, TT>::CPT], const float (&f)[4], int d,
                                           int rg, int cg, Off off) {
  using L = Tile<DP, TT>;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long at = off(rg + i * L::GL);
    if (at < 0) continue;
#pragma unroll
    for (int n = 0; n < L::NC; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = cg * 4 + n * 4 * L::GL + e;
        if (c < d) out[at + c] = from_f<T>(o[i][n * 4 + e] * f[i]);
      }
  }
}

// One tile of TT rows of a (batch, key head) pair over the key tiles of split blockIdx.y.
template <typename T, int DP, int TT>
__global__ void __launch_bounds__(Tile<DP, TT>::NT) cross_fwd_simt_kernel(CrossArgs a, CrossSplit sp, int vec) {
  using L = Tile<DP, TT>;
  griddep_launch_dependents();  // the parts' join waits for the end of this grid
  extern __shared__ __align__(16) float smem[];
  float *Q = smem, *K = Q + L::ROWS, *V = K + L::ROWS, *P = V + L::ROWS;
  __shared__ unsigned char seen[TT];
  const int tid = threadIdx.x, rg = tid / L::GL, cg = tid % L::GL;
  const int group = a.hq / a.hk, rows = group * a.q_len;
  const int row_tiles = (rows + TT - 1) / TT;
  const int pair = blockIdx.x / row_tiles, r0 = (blockIdx.x % row_tiles) * TT;
  const int b = pair / a.hk, hk = pair % a.hk;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  // A row of the group's list: its head and token; computed rows only.
  const auto at = [&](int r, int& h, int& t) {
    r += r0;
    h = hk * group + r / a.q_len;
    t = r % a.q_len;
    return r < rows && t < q_end;
  };
  stage<T, DP, TT>(Q, static_cast<const T*>(a.q), a.d, vec, [&](int r) -> long long {
    int h, t;
    return at(r, h, t) ? b * a.qs.b + h * a.qs.h + t * a.qs.t : -1;
  });
  float o[4][L::CPT], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < L::CPT; ++c) o[i][c] = 0.0f;
  }
  const float sc = a.scale * kLog2e, floor = cross_floor(sc);
  const T* kp = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vp = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  const int tiles = (kv_end + TT - 1) / TT;
  const int per = (tiles + sp.splits - 1) / sp.splits;
  const int t_lo = static_cast<int>(blockIdx.y) * per, t_hi = min(tiles, t_lo + per);
  for (int t = t_lo; t < t_hi; ++t) {
    const int k0 = t * TT;
    __syncthreads();  // the previous tile is used up
    const auto visible = [&](int j) { return k0 + j < kv_end && (!mask || mask[k0 + j]); };
    if (tid < TT) seen[tid] = visible(tid);
    stage<T, DP, TT>(K, kp, a.d, vec, [&](int j) -> long long { return visible(j) ? (k0 + j) * a.ks.t : -1; });
    stage<T, DP, TT>(V, vp, a.d, vec, [&](int j) -> long long { return visible(j) ? (k0 + j) * a.vs.t : -1; });
    __syncthreads();
    float s[4][4];
    dot_tile<DP, TT>(Q, K, rg, cg, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (seen[cg + j * L::GL])
          mx = fmaxf(mx, fmaxf(s[i][j], floor));
        else
          s[i][j] = -INFINITY;
      }
      mx = fmaxf(m[i], lanes_max<L::GL>(mx) * sc);
      const float base = mx == -INFINITY ? 0.0f : mx;  // nothing visible yet: every weight is 0
      const float keep = exp2f(m[i] - base);
      m[i] = mx;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(fmaf(s[i][j], sc, -base));
        sum += s[i][j];
        P[(rg + i * L::GL) * L::LP + cg + j * L::GL] = s[i][j];
      }
      l[i] = fmaf(l[i], keep, lanes_sum<L::GL>(sum));
#pragma unroll
      for (int c = 0; c < L::CPT; ++c) o[i][c] *= keep;
    }
    __syncthreads();
    acc_tile<DP, TT>(P, V, rg, cg, o);
  }
  float f[4];
  const long long row_of = (static_cast<long long>(b) * a.hq + hk * group) * a.q_len + r0;  // + r: dense row index
  if (sp.splits > 1) {
    // Unnormalised parts; cross_combine adds them.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = 1.0f;
      int h, tt;
      const int r = rg + i * L::GL;
      if (cg == 0 && at(r, h, tt))
        sp.ml[static_cast<long long>(blockIdx.y) * sp.rows + row_of + r] = make_float2(m[i], l[i]);
    }
    store_rows<float, DP, TT>(sp.o + static_cast<long long>(blockIdx.y) * sp.rows * a.d, o, f, a.d, rg, cg,
                              [&](int r) -> long long {
                                int h, t;
                                return at(r, h, t) ? (row_of + r) * a.d : -1;
                              });
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = cross_inverse(m[i], l[i]);
    int h, tt;
    const int r = rg + i * L::GL;
    if (cg == 0 && a.lse && at(r, h, tt)) a.lse[row_of + r] = cross_lse(m[i], l[i]);
  }
  store_rows<T, DP, TT>(static_cast<T*>(a.out), o, f, a.d, rg, cg, [&](int r) -> long long {
    int h, t;
    return at(r, h, t) ? b * a.os.b + h * a.os.h + t * a.os.t : -1;
  });
}

// Adds the parts of rows split along the keys: one warp to a row.
template <typename T>
__global__ void __launch_bounds__(256) cross_combine_kernel(CrossArgs a, CrossSplit sp) {
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  griddep_wait();
  if (row >= sp.rows) return;
  const int t = static_cast<int>(row % a.q_len);
  const long long bh = row / a.q_len;
  const int h = static_cast<int>(bh % a.hq), b = static_cast<int>(bh / a.hq);
  if (t >= cross_len(a.q_lens, b, a.q_len)) return;
  float m = -INFINITY;
  for (int i = lane; i < sp.splits; i += 32) m = fmaxf(m, sp.ml[i * sp.rows + row].x);
  m = lanes_max<32>(m);
  const float base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (int i = lane; i < sp.splits; i += 32) {
    const float2 ml = sp.ml[i * sp.rows + row];
    l = fmaf(ml.y, exp2f(ml.x - base), l);
  }
  l = lanes_sum<32>(l);
  const float inv = cross_inverse(m, l);
  T* out = static_cast<T*>(a.out) + b * a.os.b + h * a.os.h + t * a.os.t;
  float acc[8];  // head_dim <= 256
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = 0.0f;
  for (int i = 0; i < sp.splits; ++i) {
    const float mi = sp.ml[i * sp.rows + row].x, w = exp2f(mi - base);
    if (mi == -INFINITY) continue;  // a part without a visible key
    const float* o = sp.o + (static_cast<long long>(i) * sp.rows + row) * a.d;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c * 32 + lane < a.d) acc[c] = fmaf(w, o[c * 32 + lane], acc[c]);
  }
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (c * 32 + lane < a.d) out[c * 32 + lane] = from_f<T>(acc[c] * inv);
  if (lane == 0 && a.lse) a.lse[row] = cross_lse(m, l);
}

// ---- backward -------------------------------------------------------------------------------
// Row terms, negated so that they are addends: -D with D = dout . out, and minus the row's
// log-sum-exp in the log2 domain.  Rows that are not computed or see no key get -infinity and 0:
// every weight exp2(s - inf) is 0.  One warp to a row; rows of the workspace are padded to whole
// tiles of 128 tokens (the walks load 64 at a time).  (The walks' blocks do not come in beside these kernels' last ones:
// they took 8 us from them that way.)
template <typename T>
__global__ void __launch_bounds__(256) cross_row_terms_kernel(CrossGradArgs g, float* neg_lse2, float* neg_d, int q_pad,
                                                              long long rows) {
  const CrossArgs& a = g.f;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int t = static_cast<int>(row % q_pad);
  const long long bh = row / q_pad;
  const int h = static_cast<int>(bh % a.hq), b = static_cast<int>(bh / a.hq);
  float sum = 0.0f, lse = -INFINITY;
  if (t < cross_len(a.q_lens, b, a.q_len)) {
    const float x = a.lse[bh * a.q_len + t];
    if (x != -INFINITY) {
      lse = -x * kLog2e;
      const long long at = b * a.os.b + h * a.os.h + t * a.os.t;
      const T *o = static_cast<const T*>(a.out) + at, *d = static_cast<const T*>(g.dout) + at;
      for (int c = lane; c < a.d; c += 32) sum = fmaf(to_f(o[c]), to_f(d[c]), sum);
    }
  }
  sum = lanes_sum<32>(sum);
  if (lane == 0) {
    neg_lse2[row] = lse;
    neg_d[row] = -sum;
  }
}

// The same for rows of 16-byte pieces, LPR lanes to a row: 128 rows of a (batch, head) to a block, the loads of
// a warp's 16 rows in flight together.  (A warp to a row with 2-byte loads and two divisions each took 45 us
// for the 131072 rows of [16, 16, 512, 64], whose 33.5 MB take 5.)
template <typename T, int LPR>
__global__ void __launch_bounds__(256) cross_row_terms_vec_kernel(CrossGradArgs g, float* neg_lse2, float* neg_d,
                                                                  int q_pad) {
  constexpr int E = 16 / sizeof(T), RPI = 32 / LPR, N = 16 / RPI;
  const CrossArgs& a = g.f;
  const int tiles = q_pad / 128;
  const int bh = blockIdx.x / tiles, b = bh / a.hq, h = bh % a.hq;
  const int t0 = (blockIdx.x % tiles) * 128 + (threadIdx.x >> 5) * 16 + (threadIdx.x & 31) / LPR;
  const int c = (threadIdx.x & 31) % LPR * E;
  const int q_end = cross_len(a.q_lens, b, a.q_len);
  const long long at = b * a.os.b + h * a.os.h + c;
  const T *o = static_cast<const T*>(a.out) + at, *d = static_cast<const T*>(g.dout) + at;
  uint4 x[N], y[N];
  float lse[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = t0 + i * RPI;
    x[i] = y[i] = make_uint4(0, 0, 0, 0);
    lse[i] = -INFINITY;
    if (t < q_end) {
      lse[i] = a.lse[static_cast<long long>(bh) * a.q_len + t];
      if (c < a.d) {
        x[i] = __ldg(reinterpret_cast<const uint4*>(o + t * a.os.t));
        y[i] = __ldg(reinterpret_cast<const uint4*>(d + t * a.os.t));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const T *xs = reinterpret_cast<const T*>(&x[i]), *ys = reinterpret_cast<const T*>(&y[i]);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum = fmaf(to_f(xs[e]), to_f(ys[e]), sum);
    sum = lanes_sum<LPR>(sum);
    if (c == 0) {
      const long long row = static_cast<long long>(bh) * q_pad + t0 + i * RPI;
      const bool none = lse[i] == -INFINITY;
      neg_lse2[row] = none ? -INFINITY : -lse[i] * kLog2e;
      neg_d[row] = none ? 0.0f : -sum;
    }
  }
}

// dq of one tile of TT rows of a (batch, key head) pair.
template <typename T, int DP, int TT>
__global__ void __launch_bounds__(Tile<DP, TT>::NT) cross_dq_simt_kernel(CrossGradArgs g, const float* neg_lse2,
                                                                         const float* neg_d, int q_pad, int vec) {
  using L = Tile<DP, TT>;
  constexpr bool ONE = DP > 128;  // one buffer for K and V
  const CrossArgs& a = g.f;
  extern __shared__ __align__(16) float smem[];
  float *Q = smem, *G = Q + L::ROWS, *K = G + L::ROWS, *V = ONE ? K : K + L::ROWS, *P = V + L::ROWS;
  __shared__ unsigned char seen[TT];
  const int tid = threadIdx.x, rg = tid / L::GL, cg = tid % L::GL;
  const int group = a.hq / a.hk, rows = group * a.q_len;
  const int row_tiles = (rows + TT - 1) / TT;
  const int pair = blockIdx.x / row_tiles, r0 = (blockIdx.x % row_tiles) * TT;
  const int b = pair / a.hk, hk = pair % a.hk;
  const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
  const auto at = [&](int r, int& h, int& t) {
    r += r0;
    h = hk * group + r / a.q_len;
    t = r % a.q_len;
    return r < rows && t < q_end;
  };
  const auto q_off = [&](int r) -> long long {
    int h, t;
    return at(r, h, t) ? b * a.qs.b + h * a.qs.h + t * a.qs.t : -1;
  };
  stage<T, DP, TT>(Q, static_cast<const T*>(a.q), a.d, vec, q_off);
  stage<T, DP, TT>(G, static_cast<const T*>(g.dout), a.d, vec, [&](int r) -> long long {
    int h, t;
    return at(r, h, t) ? b * a.os.b + h * a.os.h + t * a.os.t : -1;
  });
  float o[4][L::CPT], lse[4], del[4], f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int h, t;
    const bool in = at(rg + i * L::GL, h, t);
    const long long w = (static_cast<long long>(b) * a.hq + h) * q_pad + t;
    lse[i] = in ? neg_lse2[w] : -INFINITY;
    del[i] = in ? neg_d[w] : 0.0f;
    f[i] = a.scale;
#pragma unroll
    for (int c = 0; c < L::CPT; ++c) o[i][c] = 0.0f;
  }
  const float sc = a.scale * kLog2e;
  const T* kp = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vp = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
  for (int k0 = 0; k0 < kv_end; k0 += TT) {
    __syncthreads();
    const auto visible = [&](int j) { return k0 + j < kv_end && (!mask || mask[k0 + j]); };
    if (tid < TT) seen[tid] = visible(tid);
    const auto k_off = [&](int j) -> long long { return visible(j) ? (k0 + j) * a.ks.t : -1; };
    if (!ONE) stage<T, DP, TT>(K, kp, a.d, vec, k_off);
    stage<T, DP, TT>(V, vp, a.d, vec, [&](int j) -> long long { return visible(j) ? (k0 + j) * a.vs.t : -1; });
    __syncthreads();
    float s[4][4], dp[4][4];
    dot_tile<DP, TT>(G, V, rg, cg, dp);
    if (ONE) {
      __syncthreads();
      stage<T, DP, TT>(K, kp, a.d, vec, k_off);
      __syncthreads();
    }
    dot_tile<DP, TT>(Q, K, rg, cg, s);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(fmaf(s[i][j], sc, lse[i]));
        P[(rg + i * L::GL) * L::LP + cg + j * L::GL] = seen[cg + j * L::GL] ? p * (dp[i][j] + del[i]) : 0.0f;
      }
    __syncthreads();
    acc_tile<DP, TT>(P, K, rg, cg, o);
  }
  store_rows<T, DP, TT>(static_cast<T*>(g.dq), o, f, a.d, rg, cg, q_off);
}

// dk and / or dv of one tile of TT keys of a (batch, key head) pair: the group's rows, one tile after
// the other, and every batch entry in turn when k and v are shared by them.
template <typename T, int DP, int TT, bool DK, bool DV>
__global__ void __launch_bounds__(Tile<DP, TT>::NT) cross_dkv_simt_kernel(CrossGradArgs g, const float* neg_lse2,
                                                                          const float* neg_d, int q_pad, int vec) {
  using L = Tile<DP, TT>;
  constexpr bool ONE = DP > 128;  // one buffer for Q and dout
  static_assert(!ONE || DK != DV);
  const CrossArgs& a = g.f;
  extern __shared__ __align__(16) float smem[];
  float *Q = smem, *G = ONE ? Q : Q + L::ROWS, *K = G + L::ROWS, *V = K + L::ROWS, *P = V + L::ROWS;
  __shared__ float row_lse[TT], row_del[TT];
  __shared__ unsigned char seen[TT];
  const int tid = threadIdx.x, rg = tid / L::GL, cg = tid % L::GL;
  const int group = a.hq / a.hk, rows = group * a.q_len;
  const int key_tiles = (a.kv_len + TT - 1) / TT;
  const int pair = blockIdx.x / key_tiles, k0 = (blockIdx.x % key_tiles) * TT;
  const int b0 = pair / a.hk, hk = pair % a.hk;
  const float sc = a.scale * kLog2e;
  float dk[DK ? 4 : 1][L::CPT], dv[DV ? 4 : 1][L::CPT];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < L::CPT; ++c) {
      if constexpr (DK) dk[i][c] = 0.0f;
      if constexpr (DV) dv[i][c] = 0.0f;
    }
  const int b_hi = g.kv_shared ? a.batch : b0 + 1;
  unsigned any = 0;  // bit i: an entry sees key rg + i * GL
  for (int b = b0; b < b_hi; ++b) {
    const int q_end = cross_len(a.q_lens, b, a.q_len), kv_end = cross_len(a.kv_lens, b, a.kv_len);
    if (k0 >= kv_end) continue;
    const unsigned char* mask = a.key_mask ? a.key_mask + static_cast<long long>(b) * a.kv_len : nullptr;
    const auto visible = [&](int j) { return k0 + j < kv_end && (!mask || mask[k0 + j]); };
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= static_cast<unsigned>(visible(rg + i * L::GL)) << i;
    __syncthreads();
    if (tid < TT) seen[tid] = visible(tid);
    stage<T, DP, TT>(K, static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h, a.d, vec,
                     [&](int j) -> long long { return visible(j) ? (k0 + j) * a.ks.t : -1; });
    stage<T, DP, TT>(V, static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h, a.d, vec,
                     [&](int j) -> long long { return visible(j) ? (k0 + j) * a.vs.t : -1; });
    for (int r0 = 0; r0 < rows; r0 += TT) {
      const auto at = [&](int r, int& h, int& t) {
        r += r0;
        h = hk * group + r / a.q_len;
        t = r % a.q_len;
        return r < rows && t < q_end;
      };
      const auto stage_q = [&] {
        stage<T, DP, TT>(Q, static_cast<const T*>(a.q), a.d, vec, [&](int r) -> long long {
          int h, t;
          return at(r, h, t) ? b * a.qs.b + h * a.qs.h + t * a.qs.t : -1;
        });
      };
      const auto stage_g = [&] {
        stage<T, DP, TT>(G, static_cast<const T*>(g.dout), a.d, vec, [&](int r) -> long long {
          int h, t;
          return at(r, h, t) ? b * a.os.b + h * a.os.h + t * a.os.t : -1;
        });
      };
      float s[4][4], dp[4][4];
      __syncthreads();
      if (tid < TT) {
        int h, t;
        const bool in = at(tid, h, t);
        const long long w = (static_cast<long long>(b) * a.hq + h) * q_pad + t;
        row_lse[tid] = in ? neg_lse2[w] : -INFINITY;
        row_del[tid] = in ? neg_d[w] : 0.0f;
      }
      if (!ONE || DK) stage_g();
      if (!ONE) stage_q();
      if (ONE && DK) {  // dout gives way to Q
        __syncthreads();
        dot_tile<DP, TT>(V, G, rg, cg, dp);
        __syncthreads();
      }
      if (ONE) stage_q();
      __syncthreads();
      dot_tile<DP, TT>(K, Q, rg, cg, s);  // rows are keys here
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = seen[rg + i * L::GL] ? exp2f(fmaf(s[i][j], sc, row_lse[cg + j * L::GL])) : 0.0f;
      if constexpr (DV) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) P[(rg + i * L::GL) * L::LP + cg + j * L::GL] = s[i][j];
        if (ONE) {  // Q gives way to dout
          __syncthreads();
          stage_g();
        }
        __syncthreads();
        acc_tile<DP, TT>(P, G, rg, cg, dv);
      }
      if constexpr (DK) {
        if (!ONE) {
          dot_tile<DP, TT>(V, G, rg, cg, dp);
          __syncthreads();  // the weights are used up
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            P[(rg + i * L::GL) * L::LP + cg + j * L::GL] = s[i][j] * (dp[i][j] + row_del[cg + j * L::GL]);
        __syncthreads();
        acc_tile<DP, TT>(P, Q, rg, cg, dk);
      }
    }
  }
  // A masked key's sums hold weights of 0 times rows that may be NaN or infinite.
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < L::CPT; ++c) {
      if constexpr (DK) dk[i][c] = (any >> i) & 1u ? dk[i][c] : 0.0f;
      if constexpr (DV) dv[i][c] = (any >> i) & 1u ? dv[i][c] : 0.0f;
    }
  const float one[4] = {1.0f, 1.0f, 1.0f, 1.0f}, scale[4] = {a.scale, a.scale, a.scale, a.scale};
  if constexpr (DK)
    store_rows<T, DP, TT>(static_cast<T*>(g.dk) + b0 * a.ks.b + hk * a.ks.h, dk, scale, a.d, rg, cg,
                          [&](int j) -> long long { return k0 + j < a.kv_len ? (k0 + j) * a.ks.t : -1; });
  if constexpr (DV)
    store_rows<T, DP, TT>(static_cast<T*>(g.dv) + b0 * a.vs.b + hk * a.vs.h, dv, one, a.d, rg, cg,
                          [&](int j) -> long long { return k0 + j < a.kv_len ? (k0 + j) * a.vs.t : -1; });
}

template <class Kernel>
cudaError_t allow_smem(std::atomic<unsigned long long>& done, Kernel k, size_t bytes) {
  return once_per_device(done, [&] {
    return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  });
}

// Whether a tensor's rows can be read four values at a time.
bool vec4(const void* p, const HeadStrides& s, int d, int es) {
  return reinterpret_cast<uintptr_t>(p) % (4 * es) == 0 && d % 4 == 0 && s.b % 4 == 0 && s.h % 4 == 0 && s.t % 4 == 0;
}

template <typename T, int DP, int TT>
cudaError_t fwd_simt(const CrossArgs& a, cudaStream_t s) {
  using L = Tile<DP, TT>;
  constexpr size_t SMEM = (3 * L::ROWS + L::SQ) * sizeof(float);
  static std::atomic<unsigned long long> attr{0};
  cudaError_t e = allow_smem(attr, cross_fwd_simt_kernel<T, DP, TT>, SMEM);
  if (e != cudaSuccess) return e;
  const long long rows = static_cast<long long>(a.hq / a.hk) * a.q_len;
  const long long blocks = (rows + TT - 1) / TT * a.batch * a.hk;
  if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
  CrossSplitWork w;
  e = w.begin(a, blocks, TT, 1, 2, s);
  if (e != cudaSuccess) return e;
  const int vec = vec4(a.q, a.qs, a.d, sizeof(T)) && vec4(a.k, a.ks, a.d, sizeof(T)) && vec4(a.v, a.vs, a.d, sizeof(T));
  cross_fwd_simt_kernel<T, DP, TT>
      <<<dim3(static_cast<unsigned>(blocks), w.sp.splits), L::NT, SMEM, s>>>(a, w.sp, vec);
  return w.end(a, cudaGetLastError(), s);
}

template <typename T>
cudaError_t fwd_simt_any(const CrossArgs& a, cudaStream_t s) {
  if (a.d <= 64) return fwd_simt<T, 64, 64>(a, s);
  if (a.d <= 128) return fwd_simt<T, 128, 64>(a, s);
  return fwd_simt<T, 256, 64>(a, s);
}

template <typename T, int DP, int TT>
cudaError_t bwd_simt(const CrossGradArgs& g, const float* neg_lse2, const float* neg_d, int q_pad, cudaStream_t s) {
  using L = Tile<DP, TT>;
  const CrossArgs& a = g.f;
  constexpr size_t SMEM = ((DP > 128 ? 3 : 4) * L::ROWS + L::SQ) * sizeof(float);
  static_assert(SMEM <= 227 * 1024 - 1024);
  const int vec = vec4(a.q, a.qs, a.d, sizeof(T)) && vec4(a.k, a.ks, a.d, sizeof(T)) &&
                  vec4(a.v, a.vs, a.d, sizeof(T)) && vec4(g.dout, a.os, a.d, sizeof(T));
  cudaError_t e = cudaSuccess;
  if (g.dq) {
    static std::atomic<unsigned long long> attr{0};
    e = allow_smem(attr, cross_dq_simt_kernel<T, DP, TT>, SMEM);
    if (e != cudaSuccess) return e;
    const long long rows = static_cast<long long>(a.hq / a.hk) * a.q_len;
    const long long blocks = (rows + TT - 1) / TT * a.batch * a.hk;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    cross_dq_simt_kernel<T, DP, TT><<<static_cast<unsigned>(blocks), L::NT, SMEM, s>>>(g, neg_lse2, neg_d, q_pad, vec);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if (g.dk) {
    const long long blocks =
        static_cast<long long>((a.kv_len + TT - 1) / TT) * (g.kv_shared ? 1 : a.batch) * a.hk;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    const unsigned n = static_cast<unsigned>(blocks);
    if constexpr (DP <= 128) {
      static std::atomic<unsigned long long> attr{0};
      e = allow_smem(attr, cross_dkv_simt_kernel<T, DP, TT, true, true>, SMEM);
      if (e != cudaSuccess) return e;
      cross_dkv_simt_kernel<T, DP, TT, true, true><<<n, L::NT, SMEM, s>>>(g, neg_lse2, neg_d, q_pad, vec);
    } else {
      // Two passes: both gradients' sums of 256 columns would not fit the registers.
      static std::atomic<unsigned long long> attr_k{0}, attr_v{0};
      if ((e = allow_smem(attr_k, cross_dkv_simt_kernel<T, DP, TT, true, false>, SMEM)) != cudaSuccess) return e;
      if ((e = allow_smem(attr_v, cross_dkv_simt_kernel<T, DP, TT, false, true>, SMEM)) != cudaSuccess) return e;
      cross_dkv_simt_kernel<T, DP, TT, true, false><<<n, L::NT, SMEM, s>>>(g, neg_lse2, neg_d, q_pad, vec);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
      cross_dkv_simt_kernel<T, DP, TT, false, true><<<n, L::NT, SMEM, s>>>(g, neg_lse2, neg_d, q_pad, vec);
    }
    e = cudaGetLastError();
  }
  return e;
}

template <typename T>
cudaError_t bwd_any(const CrossGradArgs& g, cudaStream_t s) {
  const CrossArgs& a = g.f;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const int q_pad = (a.q_len + 127) / 128 * 128;
  const long long rows = static_cast<long long>(a.batch) * a.hq * q_pad;
  const long long blocks = (rows + 7) / 8;
  if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
  void* ws = nullptr;
  cudaError_t e = workspace_alloc(ctx, &ws, static_cast<size_t>(rows) * 2 * sizeof(float), s);
  if (e != cudaSuccess) return e;
  float *neg_lse2 = static_cast<float*>(ws), *neg_d = neg_lse2 + rows;
  const auto aligned16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  constexpr int E = 16 / sizeof(T);
  const bool vec = aligned16(a.out) && aligned16(g.dout) && a.d % E == 0 && a.d <= 32 * E && a.os.b % E == 0 &&
                   a.os.h % E == 0 && a.os.t % E == 0;
  const unsigned tiles = static_cast<unsigned>(rows / 128);
  if (!vec)
    cross_row_terms_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, s>>>(g, neg_lse2, neg_d, q_pad, rows);
  else if (a.d <= 8 * E)
    cross_row_terms_vec_kernel<T, 8><<<tiles, 256, 0, s>>>(g, neg_lse2, neg_d, q_pad);
  else if (a.d <= 16 * E)
    cross_row_terms_vec_kernel<T, 16><<<tiles, 256, 0, s>>>(g, neg_lse2, neg_d, q_pad);
  else
    cross_row_terms_vec_kernel<T, 32><<<tiles, 256, 0, s>>>(g, neg_lse2, neg_d, q_pad);
  e = cudaGetLastError();
  if (e == cudaSuccess && cross_grad_tc_supported(g))
    e = cross_backward_tc(g, neg_lse2, neg_d, q_pad, s);
  else if (e == cudaSuccess)
    e = a.d <= 64    ? bwd_simt<T, 64, 64>(g, neg_lse2, neg_d, q_pad, s)
        : a.d <= 128 ? bwd_simt<T, 128, 64>(g, neg_lse2, neg_d, q_pad, s)
                     : bwd_simt<T, 256, 64>(g, neg_lse2, neg_d, q_pad, s);
  const cudaError_t f = workspace_free(ws, s);
  return e != cudaSuccess ? e : f;
}

}  // namespace

// Splits a problem of `blocks` row tiles along its key tiles (of `tile` keys) when the blocks alone leave SMs idle: as
// many parts as fill `per_sm` blocks to an SM, at least `least` key tiles each -- a part's fill, drain and join must
// not cost more than it saves.  B200, bf16 (128 keys a tile): [1, 8, 64 x 4000, 128] 25 us split, 59 not; [2, 8, 512 x
// 512, 64] 23 in parts of one tile, 15.4 whole.  fp32 (64 keys): [1, 8, 100 x 1000, 64] 21 us, 25 in parts of one tile,
// 34 whole; on the CUDA cores [1, 8, 100 x 1000, 200] 78 in parts of one tile, 361 whole.
cudaError_t CrossSplitWork::begin(const CrossArgs& a, long long blocks, int tile, int least, int per_sm, cudaStream_t s) {
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  const long long tiles = (a.kv_len + tile - 1) / tile, room = static_cast<long long>(per_sm) * ctx->sm_count;
  return begin_parts(a, std::min<long long>({room / blocks, tiles / least, 64}), s);
}

cudaError_t CrossSplitWork::begin_parts(const CrossArgs& a, long long n, cudaStream_t s) {
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return cudaErrorNoDevice;
  n = std::max(1LL, n);
  sp.splits = static_cast<int>(n);
  sp.rows = static_cast<long long>(a.batch) * a.hq * a.q_len;
  sp.o = nullptr;
  sp.ml = nullptr;
  if (n <= 1) return cudaSuccess;
  const size_t stats = (static_cast<size_t>(n) * sp.rows + 1) / 2 * 2;  // the sums start on a 16-byte boundary
  const cudaError_t e = workspace_alloc(
      ctx, &ws, stats * sizeof(float2) + static_cast<size_t>(n) * sp.rows * a.d * sizeof(float), s);
  if (e == cudaErrorMemoryAllocation) {  // no room: in one part, which needs none
    cudaGetLastError();
    sp.splits = 1;
    return cudaSuccess;
  }
  if (e != cudaSuccess) return e;
  sp.ml = static_cast<float2*>(ws);
  sp.o = reinterpret_cast<float*>(sp.ml + stats);
  return cudaSuccess;
}

// After the split launch: the combination, and the workspace back to its pool.
cudaError_t CrossSplitWork::end(const CrossArgs& a, cudaError_t e, cudaStream_t s) {
  if (sp.splits <= 1) return e;
  if (e == cudaSuccess) {
    const long long blocks = (sp.rows + 7) / 8;
    const auto kernel = a.bf16 ? cross_combine_kernel<__nv_bfloat16> : cross_combine_kernel<float>;
    e = launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a, sp);
  }
  const cudaError_t f = workspace_free(ws, s);
  return e != cudaSuccess ? e : f;
}

cudaError_t cross_attention_forward(const CrossArgs& a, cudaStream_t s) {
  if (cross_few_supported(a)) return cross_forward_few(a, s);
  if (cross_tc_supported(a)) return cross_forward_tc(a, s);
  if (cross_f32_tc_supported(a)) {
    const cudaError_t e = cross_forward_f32_tc(a, s);
    if (e != cudaErrorMemoryAllocation) return e;
    cudaGetLastError();  // no room for the split operands: the CUDA cores need none
  }
  return a.bf16 ? fwd_simt_any<__nv_bfloat16>(a, s) : fwd_simt_any<float>(a, s);
}

cudaError_t cross_attention_backward(const CrossGradArgs& g, cudaStream_t s) {
  if (cross_grad_f32_tc_supported(g)) {
    const cudaError_t e = cross_backward_f32_tc(g, s);
    if (e != cudaErrorMemoryAllocation) return e;
    cudaGetLastError();
  }
  return g.f.bf16 ? bwd_any<__nv_bfloat16>(g, s) : bwd_any<float>(g, s);
}

}  // namespace lcb
