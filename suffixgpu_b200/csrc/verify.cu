// Draft verification: from the target's logits (greedy or by given random
// numbers) and from probabilities. Definitions in include/suffixgpu.h.
#include <cuda_runtime.h>

#include "sg_sampling.cuh"

namespace sg {

constexpr int kVThreads = 512;

// ---------------------------------------------------------------------------
// statistics: one block a row
// ---------------------------------------------------------------------------
struct StatArgs {
  sg_rows rows;
  sg_sampling set;
  const int32_t* draft;      // [B, K] or NULL (statistics only)
  const int32_t* num_valid;  // [B] or NULL
  const float* uniforms;     // [B, K + 1] or NULL (greedy)
  RowStat* stats;            // [B * positions]
};

template <class T>
__device__ __forceinline__ float value_at(const T* row, int64_t i) {
  return canon(to_f32(row[i]));
}

// Largest value and its lowest index, in every thread.
template <class T>
__device__ void block_argmax(const T* row, int64_t v, float* m_out,
                             int32_t* arg_out) {
  __shared__ float s_m[32];
  __shared__ int32_t s_i[32];
  float m = -CUDART_INF_F;
  int32_t arg = INT32_MAX;
  for (int64_t i = threadIdx.x; i < v; i += blockDim.x) {
    const float x = value_at(row, i);
    if (x > m) {
      m = x;
      arg = static_cast<int32_t>(i);
    }
  }
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) {
      __syncthreads();
      if (lane_id() == 0) {
        s_m[warp_id()] = m;
        s_i[warp_id()] = arg;
      }
      __syncthreads();
      const bool in = lane_id() < static_cast<int>(blockDim.x >> 5);
      m = in ? s_m[lane_id()] : -CUDART_INF_F;
      arg = in ? s_i[lane_id()] : INT32_MAX;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(SG_FULL_MASK, m, o);
      const int32_t oi = __shfl_xor_sync(SG_FULL_MASK, arg, o);
      if (om > m || (om == m && oi < arg)) {
        m = om;
        arg = oi;
      }
    }
  }
  *m_out = m;
  *arg_out = m > -CUDART_INF_F ? arg : -1;
}

template <class T, bool kGreedy>
__global__ void __launch_bounds__(kVThreads) row_stats_kernel(StatArgs a) {
  __shared__ double red[32];
  const int b = blockIdx.x % a.rows.batch;
  const int j = blockIdx.x / a.rows.batch;
  const int k = a.rows.positions - 1;
  int n = k;
  if (a.draft != nullptr || k == 0) {
    n = valid_drafts(a.num_valid, b, k);
    if (j > n) return;
  }
  RowStat* out = a.stats + static_cast<int64_t>(b) * a.rows.positions + j;
  const T* row = row_ptr<T>(a.rows, b, j);
  const int64_t v = a.rows.vocab;
  RowStat st;
  st.z = 0.0;
  st.m = -CUDART_INF_F;
  st.arg = -1;
  st.tkey = 0;
  st.accept = 0;
  if (row != nullptr) block_argmax(row, v, &st.m, &st.arg);
  Setting set{0.0f, 0, 1.0f};
  if (!kGreedy) set = setting_of(a.set, b);
  const bool greedy = kGreedy || !(set.t > 0.0f);
  if (!greedy && st.arg >= 0) {
    const double inv_t = 1.0 / static_cast<double>(set.t);
    // top-k: the largest key held by at least k tokens from it on
    uint32_t low = 0;
    if (set.k > 0 && set.k < v) {
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t cand = low | (1u << bit);
        int c = 0;
        for (int64_t i = threadIdx.x; i < v; i += blockDim.x)
          c += order_key(value_at(row, i)) >= cand;
        if (block_sum64(c, red) >= set.k) low = cand;
      }
    }
    auto mass = [&](uint32_t from) {
      double s = 0.0;
      for (int64_t i = threadIdx.x; i < v; i += blockDim.x) {
        const float x = value_at(row, i);
        if (order_key(x) >= from) s += weight64(x, st.m, inv_t);
      }
      return block_sum64(s, red);
    };
    if (set.p < 1.0f) {
      if (set.p > 0.0f) {
        const double need = static_cast<double>(set.p) * mass(low);
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t cand = t | (1u << bit);
          if (mass(max(cand, low)) >= need) t = cand;
        }
        low = max(low, t);
      } else {
        low = order_key(st.m);
      }
    }
    st.tkey = low;
    st.z = mass(low);
  }
  if (threadIdx.x == 0) {
    if (a.draft != nullptr && j < n) {
      const int32_t x = a.draft[static_cast<int64_t>(b) * k + j];
      if (x >= 0 && x < v && st.arg >= 0) {
        const double u = a.uniforms
            ? static_cast<double>(
                  a.uniforms[static_cast<int64_t>(b) * (k + 1) + j])
            : 0.0;
        if (greedy) {
          st.accept = x == st.arg && u < 1.0;
        } else {
          const float l = value_at(row, x);
          const double w = order_key(l) >= st.tkey
              ? weight64(l, st.m, 1.0 / static_cast<double>(set.t)) : 0.0;
          st.accept = u < w / st.z;
        }
      }
    }
    *out = st;
  }
}

// ---------------------------------------------------------------------------
// drawing one token from a row of weights
// ---------------------------------------------------------------------------
// The lowest i < v whose running sum of weight(i) exceeds u times the sum;
// the last i with a weight when rounding leaves none; -1 without mass. A
// warp owns a contiguous segment of the row. Same result in every thread.
template <class W>
__device__ int32_t block_draw(int64_t v, double u, W weight, double* seg) {
  __shared__ int32_t s_tok;
  const int warps = blockDim.x >> 5;
  const int64_t len = ceil_div(ceil_div(v, warps), 32) * 32;
  const int64_t lo = min(v, warp_id() * len);
  const int64_t hi = min(v, lo + len);
  double s = 0.0;
  for (int64_t i = lo + lane_id(); i < hi; i += 32) s += weight(i);
  s = warp_sum64(s);
  __syncthreads();
  if (threadIdx.x == 0) s_tok = -1;
  if (lane_id() == 0) seg[warp_id()] = s;
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < warps; ++w) total += seg[w];
  const double target = u * total;
  double before = 0.0;
  int pick = -1;
  for (int w = 0; w < warps; ++w) {
    if (seg[w] > 0.0) pick = w;
    if (before + seg[w] > target) break;
    before += seg[w];
  }
  if (pick == warp_id()) {
    // `before` covers the segments ahead of the one that passes the target;
    // when none passes (rounding), the last segment with mass is scanned
    double run = 0.0;
    for (int w = 0; w < pick; ++w) run += seg[w];
    int32_t tok = -1;
    for (int64_t i0 = lo; i0 < hi; i0 += 32) {
      const int64_t i = i0 + lane_id();
      const double w = i < hi ? weight(i) : 0.0;
      double incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(SG_FULL_MASK, incl, o);
        if (lane_id() >= o) incl += t;
      }
      const unsigned has = __ballot_sync(SG_FULL_MASK, w > 0.0);
      const unsigned over =
          __ballot_sync(SG_FULL_MASK, w > 0.0 && run + incl > target);
      if (has) tok = static_cast<int32_t>(i0 + 31 - __clz(has));
      if (over) {
        tok = static_cast<int32_t>(i0 + __ffs(over) - 1);
        break;
      }
      run += __shfl_sync(SG_FULL_MASK, incl, 31);
    }
    if (lane_id() == 0) s_tok = tok;
  }
  __syncthreads();
  return s_tok;
}

// Writes a request's ids and count: the first s drafts and the token after
// them (-1: none).
__device__ __forceinline__ void emit(const int32_t* drow, int s, int32_t tok,
                                     int k, int32_t* out, int32_t* count) {
  for (int j = threadIdx.x; j <= k; j += blockDim.x)
    out[j] = j < s ? drow[j] : (j == s ? tok : -1);
  if (threadIdx.x == 0) *count = s + (tok >= 0 ? 1 : 0);
}

// ---------------------------------------------------------------------------
// picking from logits: one block a request
// ---------------------------------------------------------------------------
struct PickArgs {
  sg_rows rows;
  sg_sampling set;
  const RowStat* stats;
  const int32_t* draft;
  const int32_t* num_valid;
  const float* uniforms;  // NULL: greedy
  int32_t* sampled;
  int32_t* count;
};

template <class T>
__global__ void __launch_bounds__(kVThreads) pick_kernel(PickArgs a) {
  __shared__ double seg[32];
  const int b = blockIdx.x;
  const int k = a.rows.positions - 1;
  const int n = valid_drafts(a.num_valid, b, k);
  const int32_t* drow = a.draft + static_cast<int64_t>(b) * k;
  int32_t* out = a.sampled + static_cast<int64_t>(b) * (k + 1);
  if (n < 0) {
    emit(drow, 0, -1, k, out, a.count + b);
    return;
  }
  const RowStat* stats = a.stats + static_cast<int64_t>(b) * (k + 1);
  int s = 0;
  while (s < n && stats[s].accept) ++s;
  const RowStat st = stats[s];
  int32_t tok = st.arg;
  if (a.uniforms != nullptr && st.arg >= 0) {
    const Setting set = setting_of(a.set, b);
    if (set.t > 0.0f) {
      const T* row = row_ptr<T>(a.rows, b, s);
      const double inv_t = 1.0 / static_cast<double>(set.t);
      const double u = a.uniforms[static_cast<int64_t>(b) * (k + 1) + k];
      const int64_t out_tok = s < n ? drow[s] : -1;
      auto weight = [&](int64_t i) {
        const float x = value_at(row, i);
        return order_key(x) >= st.tkey ? weight64(x, st.m, inv_t) : 0.0;
      };
      tok = block_draw(
          a.rows.vocab, u,
          [&](int64_t i) { return i == out_tok ? 0.0 : weight(i); }, seg);
      if (tok < 0) tok = block_draw(a.rows.vocab, u, weight, seg);
    }
  }
  emit(drow, s, tok, k, out, a.count + b);
}

// ---------------------------------------------------------------------------
// verification from probabilities: one block a request
// ---------------------------------------------------------------------------
struct ProbArgs {
  sg_rows p;
  sg_rows q;
  int32_t has_q;
  const int32_t* draft;
  const int32_t* num_valid;
  const float* uniforms;
  int32_t* sampled;
  int32_t* count;
};

__global__ void __launch_bounds__(kVThreads) probs_kernel(ProbArgs a) {
  __shared__ double seg[32];
  __shared__ int s_stop;
  const int b = blockIdx.x;
  const int k = a.p.positions - 1;
  const int64_t v = a.p.vocab;
  const int n = valid_drafts(a.num_valid, b, k);
  const int32_t* drow = a.draft + static_cast<int64_t>(b) * k;
  const float* u = a.uniforms + static_cast<int64_t>(b) * (k + 1);
  int32_t* out = a.sampled + static_cast<int64_t>(b) * (k + 1);
  if (n < 0) {
    emit(drow, 0, -1, k, out, a.count + b);
    return;
  }
  if (threadIdx.x == 0) s_stop = n;
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int32_t x = drow[j];
    const float* prow = row_ptr<float>(a.p, b, j);
    bool ok = false;
    if (x >= 0 && x < v && prow != nullptr) {
      const double q =
          a.has_q ? clean_prob(row_ptr<float>(a.q, b, j)[x]) : 1.0f;
      ok = static_cast<double>(u[j]) * q < clean_prob(prow[x]);
    }
    if (!ok) atomicMin(&s_stop, j);
  }
  __syncthreads();
  const int s = s_stop;
  const float* prow = row_ptr<float>(a.p, b, s);
  int32_t tok = -1;
  if (prow != nullptr) {
    auto p_of = [&](int64_t i) {
      return static_cast<double>(clean_prob(prow[i]));
    };
    if (s < n && a.has_q) {
      const float* qrow = row_ptr<float>(a.q, b, s);
      tok = block_draw(
          v, u[k],
          [&](int64_t i) {
            return fmax(p_of(i) - static_cast<double>(clean_prob(qrow[i])),
                        0.0);
          },
          seg);
    } else if (s < n) {
      const int64_t x = drow[s];
      tok = block_draw(
          v, u[k], [&](int64_t i) { return i == x ? 0.0 : p_of(i); }, seg);
    }
    if (tok < 0) tok = block_draw(v, u[k], p_of, seg);
  }
  emit(drow, s, tok, k, out, a.count + b);
}

// ---------------------------------------------------------------------------
// probabilities of every row
// ---------------------------------------------------------------------------
template <class T>
__global__ void __launch_bounds__(kVThreads)
    write_probs_kernel(sg_rows rows, sg_sampling sampling,
                       const RowStat* stats, float* out) {
  const int b = blockIdx.x % rows.batch;
  const int j = blockIdx.x / rows.batch;
  const int64_t at = static_cast<int64_t>(b) * rows.positions + j;
  const RowStat st = stats[at];
  const T* row = row_ptr<T>(rows, b, j);
  const Setting set = setting_of(sampling, b);
  const double inv_t = 1.0 / static_cast<double>(set.t);
  float* orow = out + at * rows.vocab;
  for (int64_t i = threadIdx.x; i < rows.vocab; i += blockDim.x) {
    float p = 0.0f;
    if (st.arg >= 0) {
      if (!(set.t > 0.0f)) {
        p = i == st.arg ? 1.0f : 0.0f;
      } else {
        const float x = value_at(row, i);
        if (order_key(x) >= st.tkey)
          p = static_cast<float>(weight64(x, st.m, inv_t) / st.z);
      }
    }
    orow[i] = p;
  }
}

static int check_workspace(const sg_rows* r, const void* ws, size_t bytes) {
  const size_t need = sg_verify_workspace_size(r->batch, r->positions);
  if (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15))
    return SG_ERR_WORKSPACE;
  return SG_OK;
}

template <bool kGreedy>
static int launch_stats(const StatArgs& a, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.rows.batch) * a.rows.positions;
  if (rows > INT32_MAX) return SG_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(rows);
  switch (a.rows.dtype) {
    case SG_F32:
      row_stats_kernel<float, kGreedy><<<grid, kVThreads, 0, st>>>(a);
      break;
    case SG_BF16:
      row_stats_kernel<__nv_bfloat16, kGreedy><<<grid, kVThreads, 0, st>>>(a);
      break;
    default:
      row_stats_kernel<__half, kGreedy><<<grid, kVThreads, 0, st>>>(a);
  }
  return check_launch();
}

static int launch_pick(const PickArgs& a, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(a.rows.batch);
  switch (a.rows.dtype) {
    case SG_F32:
      pick_kernel<float><<<grid, kVThreads, 0, st>>>(a);
      break;
    case SG_BF16:
      pick_kernel<__nv_bfloat16><<<grid, kVThreads, 0, st>>>(a);
      break;
    default:
      pick_kernel<__half><<<grid, kVThreads, 0, st>>>(a);
  }
  return check_launch();
}

static int verify(const sg_rows* logits, const sg_sampling* sampling,
                  const int32_t* draft, const int32_t* num_valid,
                  const float* uniforms, int32_t* sampled, int32_t* count,
                  void* workspace, size_t workspace_bytes,
                  cudaStream_t st) {
  int rc = check_rows(logits, false);
  if (rc != SG_OK) return rc;
  if (logits->positions < 1) return SG_ERR_INVALID;
  if (logits->batch == 0) return SG_OK;
  if (!sampled || !count || (logits->positions > 1 && !draft))
    return SG_ERR_INVALID;
  rc = check_workspace(logits, workspace, workspace_bytes);
  if (rc != SG_OK) return rc;
  StatArgs sa{};
  sa.rows = *logits;
  if (sampling) sa.set = *sampling;
  sa.draft = draft;
  sa.num_valid = num_valid;
  sa.uniforms = uniforms;
  sa.stats = static_cast<RowStat*>(workspace);
  rc = sampling ? launch_stats<false>(sa, st) : launch_stats<true>(sa, st);
  if (rc != SG_OK) return rc;
  return launch_pick(PickArgs{*logits, sa.set, sa.stats, draft, num_valid,
                              uniforms, sampled, count},
                     st);
}

}  // namespace sg

using namespace sg;

extern "C" size_t sg_verify_workspace_size(int32_t batch, int32_t positions) {
  if (batch < 0 || positions < 0) return 0;
  return static_cast<size_t>(batch) * static_cast<size_t>(positions) *
         sizeof(RowStat);
}

extern "C" int sg_verify_greedy(const sg_rows* logits, const int32_t* draft,
                                const int32_t* num_valid, int32_t* sampled,
                                int32_t* count, void* workspace,
                                size_t workspace_bytes, sg_stream_t stream) {
  NvtxScope nvtx("sg_verify_greedy");
  return verify(logits, nullptr, draft, num_valid, nullptr, sampled, count,
                workspace, workspace_bytes,
                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int sg_verify_sampled(const sg_rows* logits,
                                 const sg_sampling* sampling,
                                 const int32_t* draft,
                                 const int32_t* num_valid,
                                 const float* uniforms, int32_t* sampled,
                                 int32_t* count, void* workspace,
                                 size_t workspace_bytes, sg_stream_t stream) {
  NvtxScope nvtx("sg_verify_sampled");
  if (!sampling || (!uniforms && logits && logits->batch > 0))
    return SG_ERR_INVALID;
  return verify(logits, sampling, draft, num_valid, uniforms, sampled, count,
                workspace, workspace_bytes,
                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int sg_verify_probs(const sg_rows* probs,
                               const sg_rows* draft_probs,
                               const int32_t* draft, const int32_t* num_valid,
                               const float* uniforms, int32_t* sampled,
                               int32_t* count, sg_stream_t stream) {
  NvtxScope nvtx("sg_verify_probs");
  int rc = check_rows(probs, true);
  if (rc != SG_OK) return rc;
  if (probs->positions < 1) return SG_ERR_INVALID;
  if (draft_probs) {
    rc = check_rows(draft_probs, true);
    if (rc != SG_OK) return rc;
    if (draft_probs->batch != probs->batch ||
        draft_probs->positions != probs->positions - 1 ||
        draft_probs->vocab != probs->vocab || draft_probs->row_start)
      return SG_ERR_INVALID;
  }
  if (probs->batch == 0) return SG_OK;
  if (!sampled || !count || !uniforms || (probs->positions > 1 && !draft))
    return SG_ERR_INVALID;
  ProbArgs a{};
  a.p = *probs;
  if (draft_probs) a.q = *draft_probs;
  a.has_q = draft_probs != nullptr;
  a.draft = draft;
  a.num_valid = num_valid;
  a.uniforms = uniforms;
  a.sampled = sampled;
  a.count = count;
  probs_kernel<<<static_cast<unsigned>(probs->batch), kVThreads, 0,
                 reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return check_launch();
}

extern "C" int sg_target_probs(const sg_rows* logits,
                               const sg_sampling* sampling, float* out,
                               void* workspace, size_t workspace_bytes,
                               sg_stream_t stream) {
  NvtxScope nvtx("sg_target_probs");
  int rc = check_rows(logits, false);
  if (rc != SG_OK) return rc;
  if (!sampling || logits->row_start) return SG_ERR_INVALID;
  if (logits->batch == 0 || logits->positions == 0) return SG_OK;
  if (!out) return SG_ERR_INVALID;
  rc = check_workspace(logits, workspace, workspace_bytes);
  if (rc != SG_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  StatArgs sa{};
  sa.rows = *logits;
  sa.set = *sampling;
  sa.stats = static_cast<RowStat*>(workspace);
  rc = launch_stats<false>(sa, st);
  if (rc != SG_OK) return rc;
  const unsigned grid = static_cast<unsigned>(
      static_cast<int64_t>(logits->batch) * logits->positions);
  switch (logits->dtype) {
    case SG_F32:
      write_probs_kernel<float><<<grid, kVThreads, 0, st>>>(
          *logits, *sampling, sa.stats, out);
      break;
    case SG_BF16:
      write_probs_kernel<__nv_bfloat16><<<grid, kVThreads, 0, st>>>(
          *logits, *sampling, sa.stats, out);
      break;
    default:
      write_probs_kernel<__half><<<grid, kVThreads, 0, st>>>(
          *logits, *sampling, sa.stats, out);
  }
  return check_launch();
}
