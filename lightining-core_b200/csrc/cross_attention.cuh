// What the cross-attention kernels share.
#pragma once

#include <cuda.h>
#include <math.h>

#include "lc_internal.hpp"

namespace lcb {

// Length of a batch entry, clamped to what the tensors hold.
__device__ __forceinline__ int cross_len(const int* lens, int b, int most) {
  return lens ? min(max(__ldg(lens + b), 0), most) : most;
}

// A row's maximum (log2 domain) is -infinity if it has seen no key, and kCrossLowest at least if it has.  The maximum
// itself drops NaN, so a row whose scores are all NaN would look like one without a key; with this floor its sum,
// which is NaN, reaches the result.  cross_floor: the same floor in scores, before the scale `sc`.
constexpr float kCrossLowest = -3.4e38f;
__device__ __forceinline__ float cross_floor(float sc) { return kCrossLowest / fmaxf(sc, 1.0f); }

// A row's factor and log-sum-exp from its maximum and sum.  A sum of 0 below a maximum that is not -infinity means
// visible scores that are all -infinity: no softmax, NaN.
__device__ __forceinline__ float cross_inverse(float m, float l) {
  if (m == -INFINITY) return 0.0f;
  return l == 0.0f ? NAN : 1.0f / l;
}
__device__ __forceinline__ float cross_lse(float m, float l) {
  if (m == -INFINITY) return -INFINITY;
  return l == 0.0f ? NAN : (m + log2f(l)) * 0.6931471805599453f;
}

// Parts of a forward pass that is split along the keys: part i of row r (rows are dense
// [batch, q_heads, q_len]) holds the unnormalised sum o[i][r][.] of exp2(s - m) v over its keys and
// ml[i][r] = (m, sum of exp2(s - m)), m the part's maximum of the scores in the log2 domain (-infinity: no visible
// key; the sums are 0 then).
struct CrossSplit {
  int splits;
  long long rows;
  float* o;
  float2* ml;
};

struct CrossSplitWork {
  CrossSplit sp{};
  void* ws = nullptr;
  cudaError_t begin(const CrossArgs& a, long long blocks, int tile, int least, int per_sm, cudaStream_t s);
  cudaError_t begin_parts(const CrossArgs& a, long long n, cudaStream_t s);  // n parts (at most 1: none)
  cudaError_t end(const CrossArgs& a, cudaError_t launched, cudaStream_t s);
};

// bf16 on the tensor cores (cross_attention_sm100.cu): head_dim <= 128 and a multiple of 8, rows of 16-byte
// alignment.
bool cross_tc_supported(const CrossArgs& a);
cudaError_t cross_forward_tc(const CrossArgs& a, cudaStream_t s);
// fp32 on the tensor cores by the 3xTF32 split (cross_attention_tf32x3.cu): head_dim <= 128; forward from 8 rows a
// pair on, backward where every batch entry has keys of its own.
bool cross_f32_tc_supported(const CrossArgs& a);
cudaError_t cross_forward_f32_tc(const CrossArgs& a, cudaStream_t s);
bool cross_grad_f32_tc_supported(const CrossGradArgs& g);
cudaError_t cross_backward_f32_tc(const CrossGradArgs& g, cudaStream_t s);
bool cross_rows16(const CrossArgs& a);
// Tensor maps of k and v in tiles of `rows` keys and 128 bytes of columns (128-byte swizzle), and which axes they have
// (an axis that is not stepped over is one entry, its coordinate 0).
struct KvAxes {
  int k_head, k_batch, v_head, v_batch;
};
bool cross_kv_maps(const CrossArgs& a, int rows, CUtensorMap* k, CUtensorMap* v, KvAxes* ax);
// Few rows to a (batch, key head) pair (cross_attention_few.cu): bf16 at most 16, head_dim 64 or 128; fp32 at most 8,
// head_dim <= 128.
bool cross_few_supported(const CrossArgs& a);
cudaError_t cross_forward_few(const CrossArgs& a, cudaStream_t s);
// neg_lse2, neg_d: the row terms, [batch * q_heads][q_pad], q_pad whole tiles of 128 tokens.
bool cross_grad_tc_supported(const CrossGradArgs& g);
cudaError_t cross_backward_tc(const CrossGradArgs& g, const float* neg_lse2, const float* neg_d, int q_pad,
                              cudaStream_t s);

}  // namespace lcb
