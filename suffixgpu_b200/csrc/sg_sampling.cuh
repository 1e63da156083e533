// Shared pieces of the draft-verification kernels (verify.cu,
// target_probs.cu): where a row of logits or probabilities lies, how its
// values are read and ordered, and a token's weight under a temperature.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "sg_common.cuh"

namespace sg {

// One row's sampling statistics, written per (request, position) by the
// statistics kernels and read by the kernels that pick or write.
struct RowStat {
  double z;       // sum of the kept weights, relative to the largest value
  float m;        // largest value of the row (-inf: no mass)
  int32_t arg;    // its lowest index (-1: no mass)
  uint32_t tkey;  // order key of the smallest kept value
  int32_t accept; // 1: this position's draft is accepted
};

// Row `j` of request `b`, or null when the request has no such row.
template <class T>
__device__ __forceinline__ const T* row_ptr(const sg_rows& r, int b, int j) {
  if (r.row_start != nullptr) {
    const int64_t at = static_cast<int64_t>(r.row_start[b]) + j;
    if (at < 0 || at >= r.n_rows) return nullptr;
    return static_cast<const T*>(r.data) + at * r.stride_b;
  }
  return static_cast<const T*>(r.data) + b * r.stride_b + j * r.stride_j;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

// NaN reads as -inf (a masked token) and -0 as +0, so that equal values
// have equal order keys.
__device__ __forceinline__ float canon(float x) {
  return x == x ? x + 0.0f : -CUDART_INF_F;
}

// Unsigned key with the order of the (canonical) values.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// exp((l - m) / T) in 64 bits; inv_t = 1 / T. A row with +inf entries gives
// them equal shares; -inf has no weight under any temperature.
__device__ __forceinline__ double weight64(float l, float m, double inv_t) {
  if (l == m) return 1.0;
  if (l == -CUDART_INF_F || m == CUDART_INF_F) return 0.0;
  return exp((static_cast<double>(l) - static_cast<double>(m)) * inv_t);
}

// Probabilities read from memory: NaN, infinities and negative values
// count as 0.
__device__ __forceinline__ float clean_prob(float p) {
  return (p > 0.0f && p < CUDART_INF_F) ? p : 0.0f;
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(SG_FULL_MASK, v, o);
  return v;
}

// Sum over the block, the same in every thread; `red` holds a value per
// warp. The order of additions is fixed.
__device__ __forceinline__ double block_sum64(double v, double* red) {
  v = warp_sum64(v);
  __syncthreads();
  if (lane_id() == 0) red[warp_id()] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  return warp_sum64(lane_id() < warps ? red[lane_id()] : 0.0);
}

// Drafted tokens of request b that count: -1 for an inactive request.
__device__ __forceinline__ int valid_drafts(const int32_t* num_valid, int b,
                                            int k) {
  if (num_valid == nullptr) return k;
  const int n = num_valid[b];
  return n < 0 ? -1 : min(n, k);
}

// A request's sampling settings.
struct Setting {
  float t;    // temperature; not > 0: greedy
  int32_t k;  // top-k; <= 0 or >= V: off
  float p;    // top-p; not < 1: off
};

__device__ __forceinline__ Setting setting_of(const sg_sampling& s, int b) {
  Setting r;
  r.t = s.temperature ? s.temperature[b] : s.temperature_all;
  r.k = s.top_k ? s.top_k[b] : s.top_k_all;
  r.p = s.top_p ? s.top_p[b] : s.top_p_all;
  return r;
}

// Host-side checks of a row set; batch and positions may be 0.
inline int check_rows(const sg_rows* r, bool probs) {
  if (!r || r->batch < 0 || r->positions < 0) return SG_ERR_INVALID;
  if (r->vocab < 1 || r->vocab >= (int64_t{1} << 31) - 1024)
    return SG_ERR_INVALID;
  if (r->dtype < SG_F32 || r->dtype > SG_F16) return SG_ERR_INVALID;
  if (probs && r->dtype != SG_F32) return SG_ERR_UNSUPPORTED;
  if (r->batch == 0 || r->positions == 0) return SG_OK;
  if (r->row_start != nullptr) {
    if (r->n_rows < 0 || r->stride_b < 0) return SG_ERR_INVALID;
    if (r->n_rows > 0 && !r->data) return SG_ERR_INVALID;
    return SG_OK;
  }
  if (!r->data || r->stride_b < 0 || r->stride_j < 0) return SG_ERR_INVALID;
  return SG_OK;
}

}  // namespace sg
