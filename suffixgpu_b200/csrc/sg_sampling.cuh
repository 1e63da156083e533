// Shared pieces of the draft-verification kernels (verify.cu,
// target_probs.cu): where a row of logits or probabilities lies, how its
// values are read and ordered, and a token's weight under a temperature.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <cmath>

#include "sg_common.cuh"

namespace sg {

// What a verification with top-k or top-p knows of a row.
struct RowStat {
  int32_t token;   // what follows if the row's draft is not accepted, -1: none
  int32_t accept;  // 1: it is
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

// Exact weights: exp((l - m) / T) in 64 bits without branches, so that the
// eight of a vector overlap (with a called exp() and its branches a block's
// warps took 300 clocks each for a weight a lane). 2^y = 2^n * 2^(i / 16) *
// 2^f with y = n + i / 16 + f, |f| <= 1 / 32: 2^(i / 16) from a table in
// shared memory (16 doubles lie in the 32 banks without conflicts), 2^f by
// its Taylor series to f^6 (the next term is below 2^-50). Weights below
// 2^-1022 count as 0, and so do NaN and -inf. m is not +inf.
constexpr int kExpTable = 16;

__device__ __forceinline__ void fill_exp_table(double* tab) {
  if (threadIdx.x < kExpTable) tab[threadIdx.x] = exp2(threadIdx.x / 16.0);
}

__device__ __forceinline__ double scale64_of(float t) {
  return 1.4426950408889634074 / static_cast<double>(t);
}

__device__ __forceinline__ double weight64(float l, double m, double scale,
                                           const double* tab) {
  constexpr double c1 = 0.69314718055994530942;  // ln2^k / k!
  constexpr double c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4,
                   c5 = c4 * c1 / 5, c6 = c5 * c1 / 6;
  const double y = (static_cast<double>(l) - m) * scale;
  // 1.5 * 2^48: its unit is 1 / 16, so the sum's low word is 16 * y rounded
  const double magic = 422212465065984.0;
  const double t = y + magic;
  const int i = __double2loint(t);
  const double f = y - (t - magic);
  double r = fma(f, c6, c5);
  r = fma(f, r, c4);
  r = fma(f, r, c3);
  r = fma(f, r, c2);
  r = fma(f, r, c1);
  r = fma(f, r, 1.0);
  r *= tab[i & (kExpTable - 1)];
  r = __hiloint2double(__double2hiint(r) + ((i >> 4) << 20),
                       __double2loint(r));
  // y below -1022, infinite or NaN (-inf under an infinite temperature)
  return (__double2hiint(y) & 0x7fffffff) > 0x408ff000 ? 0.0 : r;
}

// Probabilities read from memory: NaN, infinities and negative values
// count as 0.
__device__ __forceinline__ float clean_prob(float p) {
  return (p > 0.0f && p < CUDART_INF_F) ? p : 0.0f;
}

// Largest value over the warp (-inf at least).
__device__ __forceinline__ float warp_max(float m) {
  return key_value(__reduce_max_sync(SG_FULL_MASK, order_key(m)));
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
  if (r.t > 0.0f) r.t = fmaxf(r.t, 1.17549435e-38f);  // 1 / T stays finite
  r.k = s.top_k ? s.top_k[b] : s.top_k_all;
  r.p = s.top_p ? s.top_p[b] : s.top_p_all;
  return r;
}

inline bool has_filter(const sg_sampling& s) {
  return s.top_k || s.top_p || s.top_k_all > 0 || s.top_p_all < 1.0f;
}

// Statistics of the rows that a verification with top-k or top-p reads
// (target_probs.cu). rejected [B] and *taken are zero at the start.
int launch_row_stats(const sg_rows& rows, const sg_sampling& set,
                     const int32_t* draft, const int32_t* num_valid,
                     const float* uniforms, RowStat* stats, int32_t* rejected,
                     int32_t* taken, cudaStream_t st);

// A launch that may become resident while the previous kernel on the stream
// finishes (it waits for that kernel before it reads anything).
template <class Args>
inline int launch_after(void (*kernel)(Args), unsigned grid, int threads,
                        int cluster, const Args& a, cudaStream_t st,
                        size_t smem = 0) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    cudaGetLastError();
    return SG_ERR_CUDA;
  }
  return check_launch();
}

// Host-side checks of a row set; batch and positions may be 0.
inline int check_rows(const sg_rows* r, bool probs) {
  if (!r || r->batch < 0 || r->positions < 0) return SG_ERR_INVALID;
  if (r->vocab < 1 || r->vocab >= (int64_t{1} << 31) - 1024)
    return SG_ERR_INVALID;
  if (r->dtype < SG_F32 || r->dtype > SG_F16) return SG_ERR_INVALID;
  if (probs && r->dtype != SG_F32) return SG_ERR_UNSUPPORTED;
  if (r->batch == 0 || r->positions == 0) return SG_OK;
  const uintptr_t size = r->dtype == SG_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(r->data) % size) return SG_ERR_INVALID;
  if (r->row_start != nullptr) {
    if (r->n_rows < 0 || r->stride_b < 0) return SG_ERR_INVALID;
    if (r->n_rows > 0 && !r->data) return SG_ERR_INVALID;
    return SG_OK;
  }
  if (!r->data || r->stride_b < 0 || r->stride_j < 0) return SG_ERR_INVALID;
  return SG_OK;
}

// ---------------------------------------------------------------------------
// A row as 16-byte vectors
// ---------------------------------------------------------------------------
// Rows start anywhere (odd vocabularies, slices), so a row is read on the
// 16-byte grid of its addresses: vector v holds elements v * E - head + e,
// e < E; the first and the last may stick out of the row, and are then read
// element by element. Elements outside the row read as -inf.
template <class T>
struct RowVecs {
  static constexpr int E = 16 / sizeof(T);
  const T* row;
  int64_t v;     // elements
  int head;      // elements of the first vector that lie before the row
  int nv;        // vectors
  int in0, in1;  // vectors [in0, in1) lie wholly inside

  __device__ __forceinline__ RowVecs(const T* r, int64_t vocab) : row(r) {
    v = r ? vocab : 0;
    head = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    nv = v ? static_cast<int>((head + v + E - 1) / E) : 0;
    in0 = head ? 1 : 0;
    in1 = static_cast<int>((head + v) / E);
  }
  // Row index of a vector's first element.
  __device__ __forceinline__ int64_t first(int vec) const {
    return static_cast<int64_t>(vec) * E - head;
  }
  __device__ __forceinline__ bool inner(int vec) const {
    return vec >= in0 && vec < in1;
  }
};

template <class T>
struct Raw;  // 16 bytes of a row
template <>
struct Raw<float> {
  static constexpr uint32_t kMasked = 0xff800000u;  // -inf
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    x[0] = __uint_as_float(r.x);
    x[1] = __uint_as_float(r.y);
    x[2] = __uint_as_float(r.z);
    x[3] = __uint_as_float(r.w);
  }
  // Largest of the vectors' values, NaN ignored (NaN only if all are).
  template <int U>
  static __device__ __forceinline__ float vec_max(const uint4 (&r)[U]) {
    float m = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < U; ++u)
      m = fmaxf(fmaxf(fmaxf(__uint_as_float(r[u].x), __uint_as_float(r[u].y)),
                      fmaxf(__uint_as_float(r[u].z), __uint_as_float(r[u].w))),
                m);
    return m;
  }
};

// The same for two 16-bit values a word, compared in pairs.
template <class T2, int U>
__device__ __forceinline__ T2 packed_max(const uint4 (&r)[U]) {
  auto as = [](const uint32_t& w) { return *reinterpret_cast<const T2*>(&w); };
  T2 m = __hmax2(__hmax2(as(r[0].x), as(r[0].y)),
                 __hmax2(as(r[0].z), as(r[0].w)));
#pragma unroll
  for (int u = 1; u < U; ++u)
    m = __hmax2(m, __hmax2(__hmax2(as(r[u].x), as(r[u].y)),
                           __hmax2(as(r[u].z), as(r[u].w))));
  return m;
}
template <>
struct Raw<__nv_bfloat16> {
  static constexpr uint32_t kMasked = 0xff80ff80u;
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  template <int U>
  static __device__ __forceinline__ float vec_max(const uint4 (&r)[U]) {
    const __nv_bfloat162 m = packed_max<__nv_bfloat162>(r);
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <>
struct Raw<__half> {
  static constexpr uint32_t kMasked = 0xfc00fc00u;
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  template <int U>
  static __device__ __forceinline__ float vec_max(const uint4 (&r)[U]) {
    const __half2 m = packed_max<__half2>(r);
    return fmaxf(__low2float(m), __high2float(m));
  }
};

__device__ __forceinline__ uint4 load_16(const void* p) {
  return __ldg(static_cast<const uint4*>(p));
}

// A vector at the edge of the row, element by element.
template <class T>
__device__ __forceinline__ uint4 edge_vec(const RowVecs<T>& rv, int vec) {
  constexpr int E = RowVecs<T>::E;
  uint4 r;
  r.x = r.y = r.z = r.w = Raw<T>::kMasked;
  T* t = reinterpret_cast<T*>(&r);
  const int64_t i0 = rv.first(vec);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (i0 + e >= 0 && i0 + e < rv.v) t[e] = rv.row[i0 + e];
  return r;
}

// Vector `vec` of the row, or -inf past `end`.
template <class T>
__device__ __forceinline__ uint4 load_vec(const RowVecs<T>& rv, int vec,
                                          int end) {
  uint4 r;
  r.x = r.y = r.z = r.w = Raw<T>::kMasked;
  if (vec < end) {
    if (rv.inner(vec))
      r = load_16(rv.row + rv.first(vec));
    else
      r = edge_vec(rv, vec);
  }
  return r;
}

// 2^x, 2 ulp (ex2.approx: 2^-22 relative, results below 2^-126 flushed).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)),
        "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)),
        "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}

// log2(e) / T for 2^((l - m) * scale); finite (see setting_of).
__device__ __forceinline__ float scale_of(float t) {
  return static_cast<float>(1.4426950408889634074 / static_cast<double>(t));
}

// exp((l - m) / T) in fp32. Relative error: half a step each for l - m, the
// product and the scale act on the exponent, 3 * 2^-24 * ln2 * |z|, z = the
// exponent of 2; plus 2^-22 of ex2. Next to m = +inf nothing else has weight,
// at an infinite temperature (scale 0) either. Where l - m passes fp32's
// range, halves of both do not (and twice the scale is finite).
__device__ __forceinline__ float weight32(float l, float m, float scale) {
  if (l == m) return 1.0f;
  if (!(l > -CUDART_INF_F) || m == CUDART_INF_F) return 0.0f;
  const float d = l - m;
  return exp2_fast(d > -CUDART_INF_F ? d * scale
                                     : (0.5f * l - 0.5f * m) * (2.0f * scale));
}

// Scales below this one (temperatures above 2^100) leave weight where l - m
// passes fp32's range, and have no second part: they are left to weight32.
constexpr float kFlatScale = 1.138e-30f;

// The scale in two parts, so that its rounding, which would act on all
// weights alike and shift a row's probabilities by 2^-24 times their mean
// depth, does not count: z = d * (hi + lo) is rounded once, by itself. hi is
// rounded down and lo above 0 (by the smallest number there is, next to
// nothing beside any scale above kFlatScale), so that -inf keeps its sign.
struct FineScale {
  float hi, lo;
};
__device__ __forceinline__ FineScale fine_scale_of(float t) {
  FineScale f;
  const double s = 1.4426950408889634074 / static_cast<double>(t);
  f.hi = s < kFlatScale ? static_cast<float>(s) : __double2float_rd(s);
  f.lo = fmaxf(static_cast<float>(s - static_cast<double>(f.hi)), 1.4e-45f);
  return f;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)),
        "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}
// Weights of two values; NaN for NaN, and for m = +inf.
__device__ __forceinline__ float2 fine_weight2(float2 l, float m,
                                               const FineScale& f) {
  const float2 d = add2(l, make_float2(-m, -m));
  const float2 z = fma2(d, make_float2(f.hi, f.hi),
                        mul2(d, make_float2(f.lo, f.lo)));
  return make_float2(exp2_fast(z.x), exp2_fast(z.y));
}

// ---------------------------------------------------------------------------
// One pass over values: largest and sum of weights
// ---------------------------------------------------------------------------
// What a lane knows of its warp's span so far.
struct LaneStat {
  float m;      // the warp's largest value
  double s;     // this lane's sum, relative to m
  int32_t arg;  // lowest index of the largest value
};

// Takes U vectors a lane into `st`; index(u) is the row index of vector u's
// first element. kArg: the lowest index of the largest value, looked for
// where the vectors reach the block's largest so far (s_top); kSum: the
// weights' sum, from fp32 weights or finer ones.
enum SumKind : int { kNoSum, kFastSum, kFineSum };

template <class T, bool kArg, SumKind kSum, int U, class Index>
__device__ __forceinline__ void take_vecs(const uint4 (&raw)[U], Index index,
                                          const FineScale& f,
                                          uint32_t* s_top, LaneStat& st) {
  const float scale = f.hi;
  constexpr int E = RowVecs<T>::E;
  const float tm = warp_max(canon(Raw<T>::vec_max(raw)));
  bool up = kArg ? tm >= st.m && tm > -CUDART_INF_F : tm > st.m;
  if (kArg && up) {
    uint32_t old = 0;
    if (lane_id() == 0) old = atomicMax(s_top, order_key(tm));
    up = order_key(tm) >= __shfl_sync(SG_FULL_MASK, old, 0);
  }
  if (up) {
    if (kSum != kNoSum && st.s != 0.0) st.s *= weight32(st.m, tm, scale);
    if (kArg) {
      int32_t at = tm == st.m ? st.arg : INT32_MAX;
#pragma unroll
      for (int u = U - 1; u >= 0; --u) {
        float x[E];
        Raw<T>::unpack(raw[u], x);
        const int32_t i0 = static_cast<int32_t>(index(u));
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
          if (x[e] == tm) at = min(at, i0 + e);
      }
      st.arg = __reduce_min_sync(SG_FULL_MASK, at);
    }
    st.m = tm;
  }
  if (kSum != kNoSum && st.m > -CUDART_INF_F) {
    const float2 nm = make_float2(-st.m, -st.m);
    const float2 sc = make_float2(scale, scale);
    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[E];
      Raw<T>::unpack(raw[u], x);
      float2 p[E / 2];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        p[e] = make_float2(x[2 * e], x[2 * e + 1]);
        if (kSum == kFineSum) {
          p[e] = fine_weight2(p[e], st.m, f);
        } else {
          p[e] = mul2(add2(p[e], nm), sc);
          p[e] = make_float2(exp2_fast(p[e].x), exp2_fast(p[e].y));
        }
      }
#pragma unroll
      for (int w = E / 4; w > 0; w /= 2)
#pragma unroll
        for (int e = 0; e < w; ++e) p[e] = add2(p[e], p[e + w]);
      acc = add2(acc, p[0]);
    }
    float ts = acc.x + acc.y;
    // NaN: masked NaN logits, or +inf; such vectors, and all at the largest
    // temperatures, are summed again with each case told apart
    if (ts != ts || scale < kFlatScale) {
      ts = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[E];
        Raw<T>::unpack(raw[u], x);
        float us = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
          us += weight32(canon(x[e]), st.m, scale);
        ts += us;
      }
    }
    st.s += ts;
  }
}

// Sums over parts of a row, relative to the parts' largest values.
struct SpanSum {
  double s;
  float m;
  int32_t arg;
};

// The row's from those of its n <= 32 parts, in every lane of the warp; with
// factors in 64 bits (t > 0; else only m and arg count).
__device__ __forceinline__ SpanSum join_sums(const SpanSum* parts, int n,
                                             float t) {
  SpanSum p{0.0, -CUDART_INF_F, INT32_MAX};
  if (lane_id() < n) p = parts[lane_id()];
  const float m = warp_max(p.m);
  p.arg = __reduce_min_sync(SG_FULL_MASK, p.m == m ? p.arg : INT32_MAX);
  double s = 0.0;
  if (p.s != 0.0 && t > 0.0f && (p.m == m || m < CUDART_INF_F))
    s = p.m == m ? p.s
                 : p.s * exp((static_cast<double>(p.m) -
                              static_cast<double>(m)) /
                             static_cast<double>(t));
  p.s = warp_sum64(s);
  p.m = m;
  return p;
}

// A weight's relative error is 3 * 2^-24 * ln2 = 1.24e-7 times its depth z
// (its exponent of 2) plus 2^-22: at most kDeepGuard for one weight, whose
// depth ends at 126. In a row's sum it counts by weight, and the weights'
// mean depth is at most log2(V): it is their entropy less log2 of their sum,
// and the largest weight is 1. Further errors: 2^-22 for each time the
// largest value grew (at most once a tile) or spans were joined (2), and
// 2^-24 for each of the at most 20 fp32 operations on a weight's way.
constexpr double kDeepGuard = 1.7e-5;
// `tile`: values of a row taken in at a time.
inline double guard_of(int64_t vocab, int64_t tile) {
  const int64_t tiles = ceil_div(vocab, tile) + 1;
  return 1.25e-7 * std::log2(static_cast<double>(vocab) + 1.0) +
         2.4e-7 * static_cast<double>(2 + tiles) + 1.2e-6;
}

// ---------------------------------------------------------------------------
// Drawing a token over a cluster, in 64 bits
// ---------------------------------------------------------------------------
constexpr int kCWarps = 8;  // of a block that draws
constexpr int kCThreads = kCWarps * 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxSpans = 128;  // contiguous spans a row is cut into

// The vectors [v0, v1) of a row in span `w` of `n`.
struct Span {
  int v0, v1;
};
__device__ __forceinline__ Span nth_span(int nv, int w, int per) {
  Span s;
  s.v0 = min(nv, w * per);
  s.v1 = min(nv, s.v0 + per);
  return s;
}
__device__ __forceinline__ Span span_of(int nv, int w, int n) {
  return nth_span(nv, w, (nv + n - 1) / n);
}

// The span that holds u times the total of `spans` sums, sum_of(i) giving
// them (called for lane * per + i): the first whose running sum exceeds the
// target, else the last with mass, -1 without any; `ahead` is the sum in
// front of it. The same in every lane of the warp.
struct Pick {
  int span;
  double ahead;
  double target;
  double total;
};
template <class SumOf>
__device__ __forceinline__ Pick pick_span(int spans, double u, SumOf sum_of) {
  constexpr int kPer = kMaxSpans / 32;
  const int per = (spans + 31) / 32;
  double v[kPer];
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = lane_id() * per + i;
    v[i] = i < per && at < spans ? sum_of(at) : 0.0;
    sum += v[i];
  }
  double incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(SG_FULL_MASK, incl, o);
    if (lane_id() >= o) incl += t;
  }
  Pick r;
  r.total = __shfl_sync(SG_FULL_MASK, incl, 31);
  r.target = u * r.total;
  const unsigned over = __ballot_sync(SG_FULL_MASK, incl > r.target);
  const unsigned has = __ballot_sync(SG_FULL_MASK, sum > 0.0);
  r.span = -1;
  r.ahead = 0.0;
  if (has == 0) return r;
  const int src = over ? __ffs(over) - 1 : 31 - __clz(has);
  // within the lane: the first span that passes, else its last with mass
  double run = incl - sum;
  int at = -1;
  double ahead = run;
  bool done = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (!done && v[i] > 0.0) {
      at = lane_id() * per + i;
      ahead = run;
      run += v[i];
      done = run > r.target;
    }
  }
  r.span = __shfl_sync(SG_FULL_MASK, at, src);
  r.ahead = __shfl_sync(SG_FULL_MASK, ahead, src);
  return r;
}

// The lowest index whose running sum of the source's weights exceeds u
// times their total; the last one with a weight when rounding leaves none;
// -1 without mass. Warps own contiguous spans over the cluster; the block
// that owns the span with the target scans it. Called by every thread of
// the cluster, same result in all.
//   Src::E              weights of a vector
//   src.first(v)        index of a vector's first weight
//   src.span(w, n)      vectors of span w of n = 8 a block, in order
//   src.sum(v, end, st) sum of the weights of vectors v, v + st, ... < end
//   src.vec(v, end, w)  weights of vector v
struct DrawShared {
  double seg[kMaxCluster * kCWarps];
  double red[32];
  int32_t tok, first, last;
};
template <class Src>
__device__ int32_t cluster_draw(const cooperative_groups::cluster_group& cl,
                                const Src& src, double u, DrawShared& sh) {
  constexpr int E = Src::E;
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int spans = cs * kCWarps;
  const int mine = rank * kCWarps + warp_id();
  const Span sp = src.span(mine, spans);
  const double s = warp_sum64(src.sum(sp.v0 + lane_id(), sp.v1, 32));
  cl.sync();  // sh is free
  if (lane_id() < cs) *cl.map_shared_rank(&sh.seg[mine], lane_id()) = s;
  cl.sync();
  const Pick pick = pick_span(spans, u, [&](int i) { return sh.seg[i]; });
  if (pick.span < 0) return -1;
  if (pick.span / kCWarps == rank) {
    // a contiguous run of vectors a thread
    const Span seg = src.span(pick.span, spans);
    const int per = (seg.v1 - seg.v0 + kCThreads - 1) / kCThreads;
    const int v0 = min(seg.v1, seg.v0 + static_cast<int>(threadIdx.x) * per);
    const int v1 = min(seg.v1, v0 + per);
    const double mass = src.sum(v0, v1, 1);
    double incl = mass;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(SG_FULL_MASK, incl, o);
      if (lane_id() >= o) incl += t;
    }
    if (lane_id() == 31) sh.red[warp_id()] = incl;
    if (threadIdx.x == 0) {
      sh.first = INT32_MAX;
      sh.last = -1;
    }
    __syncthreads();
    double lo = pick.ahead;
    for (int i = 0; i < warp_id(); ++i) lo += sh.red[i];
    lo += incl - mass;
    if (mass > 0.0 && !(lo > pick.target)) {  // or u is NaN
      double run = lo;
      int32_t at = -1;
      bool over = false;
      double w[E];
      for (int v = v0; v < v1 && !over; ++v) {
        src.vec(v, v1, w);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (!over && w[e] > 0.0) {
            at = static_cast<int32_t>(src.first(v) + e);
            run += w[e];
            over = run > pick.target;
          }
        }
      }
      if (over)
        atomicMin(&sh.first, at);
      else
        atomicMax(&sh.last, at);
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < cs)
      *cl.map_shared_rank(&sh.tok, static_cast<int>(threadIdx.x)) =
          sh.first != INT32_MAX ? sh.first : sh.last;
  }
  cl.sync();
  return sh.tok;
}

}  // namespace sg
