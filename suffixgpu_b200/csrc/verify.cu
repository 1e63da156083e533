// Draft verification: from the target's logits (greedy or by given random
// numbers) and from probabilities. Definitions in include/suffixgpu.h.
#include <cuda_runtime.h>

#include <algorithm>

#include "sg_sampling.cuh"

namespace sg {

// Writes a request's ids and count: the first s drafts and the token after
// them (-1: none).
__device__ __forceinline__ void emit(const int32_t* drow, int s, int32_t tok,
                                     int k, int32_t* out, int32_t* count) {
  for (int j = threadIdx.x; j <= k; j += blockDim.x)
    out[j] = j < s ? drow[j] : (j == s ? tok : -1);
  if (threadIdx.x == 0) *count = s + (tok >= 0 ? 1 : 0);
}

// ---------------------------------------------------------------------------
// verification from logits without filters
// ---------------------------------------------------------------------------
// Two launches. The first reads every row once, in spans (one a warp, `split`
// blocks a row), and stores each span's largest value and the sum of its
// weights relative to it. The second decides, a cluster a request, from the
// spans' sums; it reads again only the span that holds the drawn token.
//
// Whether u < P(x) is decided from fp32 weights where u * Z and the weight
// of x are further apart than their error can be (guard_of); otherwise the
// row is summed again in 64 bits. The drawn token is found the same way:
// in fp32 while the target lies clear of both borders of the token found,
// else in 64 bits.
constexpr int kSWarps = 8;  // warps of a block that reads rows
constexpr int kSThreads = kSWarps * 32;
constexpr int kMaxSplit = kMaxSpans / kSWarps;  // blocks that share a row
constexpr int kSBlocks = 3;  // such blocks on an SM
constexpr int kUnroll = 8;  // 16-byte loads in flight per thread

struct Part {  // a span of a row
  float s;     // sum of 2^((l - m) * scale)
  float m;
  int32_t arg;
};

struct VerifyArgs {
  sg_rows rows;
  sg_sampling set;
  const int32_t* draft;
  const int32_t* num_valid;
  const float* uniforms;  // NULL: greedy
  int32_t* sampled;
  int32_t* count;
  int32_t split;       // blocks that share a row
  int32_t warp_spans;  // spans of each of their warps
  double guard;   // relative error of sums of fp32 weights
  Part* parts;    // [B * positions][split * kSWarps * warp_spans]
  // many rows only (else NULL); zero at the start
  int32_t* rejected;  // [B] positions - the lowest position known rejected
  int32_t* arrived;   // [B * positions] blocks of the row that are done
  int32_t* marks;     // requests to be decided by sums in 64 bits,
  int32_t* marked;    // and which
};

// One warp's span of a row. The row's partial vectors at its two ends are
// loaded first and taken last, so that they cost no latency of their own.
template <class T, bool kArg, bool kSum>
__device__ __forceinline__ Part warp_stats(const RowVecs<T>& rv, Span sp,
                                           float scale, uint32_t* s_top) {
  uint4 edge[1];
  edge[0].x = edge[0].y = edge[0].z = edge[0].w = Raw<T>::kMasked;
  const int ev = lane_id() == 0 ? sp.v0 : sp.v1 - 1;
  const bool edges =
      sp.v0 < sp.v1 && (!rv.inner(sp.v0) || !rv.inner(sp.v1 - 1));
  if (edges && lane_id() < 2 && !rv.inner(ev) &&
      (lane_id() == 0 || sp.v1 - 1 != sp.v0))
    edge[0] = edge_vec(rv, ev);
  LaneStat st{-CUDART_INF_F, 0.0, INT32_MAX};
  for (int t0 = sp.v0; t0 < sp.v1; t0 += kUnroll * 32) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      raw[u].x = raw[u].y = raw[u].z = raw[u].w = Raw<T>::kMasked;
      const int v = t0 + u * 32 + lane_id();
      if (v < sp.v1 && rv.inner(v)) raw[u] = load_16(rv.row + rv.first(v));
    }
    take_vecs<T, kArg, kSum ? kFastSum : kNoSum>(
        raw, [&](int u) { return rv.first(t0 + u * 32 + lane_id()); },
        FineScale{scale, 0.0f}, s_top, st);
  }
  if (edges)
    take_vecs<T, kArg, kSum ? kFastSum : kNoSum>(
        edge, [&](int) { return rv.first(ev); },
        FineScale{scale, 0.0f}, s_top, st);
  float s = 0.0f;
  if (kSum) {
    s = static_cast<float>(st.s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(SG_FULL_MASK, s, o);
  }
  return Part{s, st.m, st.arg};
}

// A row from the Parts of its `n` spans, in every lane of the warp. kFresh:
// past the L1 cache, since other blocks of the same launch wrote them.
struct RowSum {
  double s;
  float m;
  int32_t arg;
};
template <bool kArg, bool kSum, bool kFresh = false>
__device__ __forceinline__ RowSum join_parts(const Part* parts, int n,
                                             float scale) {
  constexpr int kPer = kMaxSpans / 32;
  Part p[kPer];
  float m = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    p[i] = Part{0.0f, -CUDART_INF_F, INT32_MAX};
    if (i * 32 + lane_id() < n) {
      const Part* q = parts + i * 32 + lane_id();
      p[i] = kFresh ? Part{__ldcg(&q->s), __ldcg(&q->m), __ldcg(&q->arg)} : *q;
    }
    m = fmaxf(m, p[i].m);
  }
  RowSum r{0.0, warp_max(m), INT32_MAX};
  int32_t arg = INT32_MAX;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (kSum && p[i].s != 0.0f)
      r.s += static_cast<double>(p[i].s * weight32(p[i].m, r.m, scale));
    if (kArg && p[i].m == r.m) arg = min(arg, p[i].arg);
  }
  if (kSum) r.s = warp_sum64(r.s);
  if (kArg) r.arg = __reduce_min_sync(SG_FULL_MASK, arg);
  return r;
}

// Spans of a warp, so that a span is one or two tiles.
static int warp_spans_of(int64_t vocab, int elems, int split) {
  const int64_t tile = static_cast<int64_t>(kUnroll) * 32 * elems;
  const int64_t want = ceil_div(vocab, 2 * tile * split * kSWarps);
  return static_cast<int>(
      std::min<int64_t>(want, kMaxSpans / (split * kSWarps)));
}

// Whether a draft is accepted, where fp32 weights can tell: not within their
// errors, nor where both sides are as small as a weight that is flushed to 0.
enum Verdict : int { kReject = 0, kAccept = 1, kUnsure = 2 };

__device__ __forceinline__ Verdict verdict(const RowSum& row, float l, double u,
                                           float scale, double guard) {
  const double w = weight32(l, row.m, scale);
  const double uz = u * row.s;
  if (!(fabs(uz - w) > guard * uz + kDeepGuard * w + 1.2e-38)) return kUnsure;
  return uz < w ? kAccept : kReject;
}

// One block's spans of row (b, j): block c's warps own a.warp_spans each.
template <class T, bool kSampled>
__device__ __forceinline__ void block_spans(const VerifyArgs& a, int b, int j,
                                            int c, bool greedy, float scale,
                                            uint32_t* s_top) {
  const RowVecs<T> rv(row_ptr<T>(a.rows, b, j), a.rows.vocab);
  const int spans = a.split * kSWarps * a.warp_spans;
  Part* out = a.parts +
              (static_cast<int64_t>(b) * a.rows.positions + j) * spans;
  const int per = (rv.nv + spans - 1) / spans;
#pragma unroll 1
  for (int i = 0; i < a.warp_spans; ++i) {
    const int w = (c * kSWarps + warp_id()) * a.warp_spans + i;
    const Span sp = nth_span(rv.nv, w, per);
    const Part p = greedy ? warp_stats<T, true, false>(rv, sp, scale, s_top)
                          : warp_stats<T, false, true>(rv, sp, scale, s_top);
    if (lane_id() == 0) out[w] = p;
  }
}

// Greedy rows take 64 registers a thread, four blocks on an SM: those of 16
// bits by themselves, of 32 bits when told to (37 packed requests of up to 8
// rows of 50021: 15.3 us against 17.3; told the same, 16-bit rows spill and
// lose 5%).
template <class T, bool kSampled>
constexpr int blocks_on_sm() {
  return !kSampled && sizeof(T) == 4 ? kSBlocks + 1 : kSBlocks;
}

// a.split blocks a row, the rows of low positions first. With many rows
// (a.rejected), the last block of a row to arrive tells whether its draft is
// surely rejected, and rows behind such a position are left out. What is
// left out depends on timing; the rows that the decision reads do not.
template <class T, bool kSampled>
__global__ void __launch_bounds__(kSThreads, blocks_on_sm<T, kSampled>())
    spans_kernel(VerifyArgs a) {
  __shared__ uint32_t s_top;
  __shared__ int32_t s_skip;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int k = a.rows.positions - 1;
  const int c = static_cast<int>(blockIdx.x % a.split);
  const int item = static_cast<int>(blockIdx.x / a.split);
  const int b = item % a.rows.batch;
  const int j = item / a.rows.batch;
  if (threadIdx.x == 0) {
    // read by one thread for the block: other blocks change it meanwhile
    const int r = a.rejected
        ? *static_cast<volatile int32_t*>(a.rejected + b) : 0;
    s_skip = j > min(valid_drafts(a.num_valid, b, k), k + 1 - r);
    s_top = 0;
  }
  __syncthreads();
  if (s_skip) return;
  Setting set{0.0f, 0, 1.0f};
  if (kSampled) set = setting_of(a.set, b);
  const bool greedy = !kSampled || !(set.t > 0.0f);
  const float scale = greedy ? 0.0f : scale_of(set.t);
  block_spans<T, kSampled>(a, b, j, c, greedy, scale, &s_top);
  if (a.rejected == nullptr || j >= k) return;
  if (lane_id() == 0) __threadfence();  // the warp's Parts, before the count
  __syncthreads();
  if (warp_id() != 0) return;
  const int64_t at = static_cast<int64_t>(b) * (k + 1) + j;
  int last = 0;
  if (lane_id() == 0) last = atomicAdd(a.arrived + at, 1) == a.split - 1;
  if (!__shfl_sync(SG_FULL_MASK, last, 0)) return;
  __threadfence();
  __syncwarp();
  const int spans = a.split * kSWarps * a.warp_spans;
  const Part* row_parts = a.parts + at * spans;
  const RowSum r =
      greedy ? join_parts<true, false, true>(row_parts, spans, scale)
             : join_parts<false, true, true>(row_parts, spans, scale);
  if (lane_id() != 0) return;
  const int32_t x = a.draft[static_cast<int64_t>(b) * k + j];
  bool reject = x < 0 || x >= a.rows.vocab || !(r.m > -CUDART_INF_F);
  if (!reject) {
    if (greedy) {
      reject = x != r.arg;
    } else {
      const double u = a.uniforms[static_cast<int64_t>(b) * (k + 1) + j];
      const float l = canon(to_f32(row_ptr<T>(a.rows, b, j)[x]));
      reject = verdict(r, l, u, scale, a.guard) == kReject;
    }
  }
  if (reject) atomicMax(a.rejected + b, k + 1 - j);
}

// A row's weights; `skip` (an index, or -1) has none.
template <class T>
struct RowWeights : RowVecs<T> {
  using RowVecs<T>::E;
  float m;
  float scale;
  double scale64;
  int64_t skip;
  const double* tab;

  __device__ __forceinline__ RowWeights(const T* row, int64_t vocab, float m_,
                                        float scale_, double scale64_,
                                        int64_t skip_, const double* tab_)
      : RowVecs<T>(row, vocab), m(m_), scale(scale_), scale64(scale64_),
        skip(skip_), tab(tab_) {}

  // fp32 weights of vector v; their sum.
  __device__ __forceinline__ float fast_vec(int v, int end, float* w) const {
    float x[E];
    Raw<T>::unpack(load_vec(*this, v, end), x);
    const int64_t i0 = this->first(v);
#pragma unroll
    for (int e = 0; e < E; ++e)
      w[e] = i0 + e == skip ? 0.0f : weight32(canon(x[e]), m, scale);
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = w[e];
#pragma unroll
    for (int h = E / 2; h > 0; h /= 2)
#pragma unroll
      for (int e = 0; e < h; ++e) s[e] += s[e + h];
    return s[0];
  }

  __device__ __forceinline__ void exact(const uint4& raw, int v,
                                        double* w) const {
    float x[E];
    Raw<T>::unpack(raw, x);
    if (m == CUDART_INF_F) {
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = x[e] == m ? 1.0 : 0.0;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = weight64(x[e], m, scale64, tab);
    }
    const int64_t at = skip - this->first(v);
    if (at >= 0 && at < E) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e == at) w[e] = 0.0;
    }
  }
  // Exact weights (cluster_draw's source).
  __device__ __forceinline__ Span span(int w, int n) const {
    return span_of(this->nv, w, n);
  }
  __device__ __forceinline__ void vec(int v, int end, double* w) const {
    exact(load_vec(*this, v, end), v, w);
  }
  __device__ __forceinline__ double sum(int v, int end, int step) const {
    double s = 0.0;
    if (v >= end) return s;
    uint4 next = load_vec(*this, v, end);
    for (; v < end; v += step) {
      const uint4 raw = next;
      next = load_vec(*this, v + step, end);  // in flight meanwhile
      double w[E];
      exact(raw, v, w);
#pragma unroll
      for (int h = E / 2; h > 0; h /= 2)
#pragma unroll
        for (int e = 0; e < h; ++e) w[e] += w[e + h];
      s += w[0];
    }
    return s;
  }
};

// Sum of a row's exact weights over the cluster, the same in every thread.
template <class T>
__device__ double cluster_sum64(const cooperative_groups::cluster_group& cl,
                                const RowWeights<T>& weights,
                                DrawShared& sh) {
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const Span sp = span_of(weights.nv, rank * kCWarps + warp_id(),
                          cs * kCWarps);
  const double s = block_sum64(
      weights.sum(sp.v0 + lane_id(), sp.v1, 32), sh.red);
  cl.sync();  // sh.seg is free
  if (static_cast<int>(threadIdx.x) < cs)
    *cl.map_shared_rank(&sh.seg[rank], static_cast<int>(threadIdx.x)) = s;
  cl.sync();
  double z = 0.0;
  for (int c = 0; c < cs; ++c) z += sh.seg[c];
  cl.sync();  // and free again
  return z;
}

// The token that cluster_draw gives, looked for in one span by the whole
// block from fp32 weights: the span's running sums start `ahead` of the
// row's; -2 when the target is nearer to a border of the token found than
// `guard`.
template <class W>
__device__ int32_t span_draw(const W& weights, Span sp, double ahead,
                             double target, double guard, float* red,
                             int32_t* s_found) {
  constexpr int E = W::E;
  // a contiguous run of vectors a thread; exclusive sums over the block
  const int per = (sp.v1 - sp.v0 + kCThreads - 1) / kCThreads;
  const int v0 = min(sp.v1, sp.v0 + static_cast<int>(threadIdx.x) * per);
  const int v1 = min(sp.v1, v0 + per);
  float w[E];
  double sum = 0.0;
  for (int v = v0; v < v1; ++v) sum += weights.fast_vec(v, v1, w);
  const float s = static_cast<float>(sum);
  float incl = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float t = __shfl_up_sync(SG_FULL_MASK, incl, o);
    if (lane_id() >= o) incl += t;
  }
  __syncthreads();
  if (threadIdx.x == 0) *s_found = -2;
  if (lane_id() == 31) red[warp_id()] = incl;
  __syncthreads();
  float before = 0.0f;
#pragma unroll
  for (int i = 0; i < kCWarps; ++i) before += i < warp_id() ? red[i] : 0.0f;
  // at most one token is clear of both of its borders
  const double need = target - ahead;
  double lo = before + (incl - s);
  if (need - lo > guard && lo + sum - need > guard) {
    for (int v = v0; v < v1; ++v) {
      weights.fast_vec(v, v1, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (need - lo > guard && lo + w[e] - need > guard)
          *s_found = static_cast<int32_t>(weights.first(v) + e);
        lo += w[e];
      }
    }
  }
  __syncthreads();
  return *s_found;
}

// Every CTA of a request's cluster decides alike from the same numbers; the
// cluster is needed where a row has to be summed in 64 bits. With many
// requests that is left to a second launch: the first, a block a request,
// only marks those that need it.
enum Stage : int { kWhole, kMark, kMarked };

struct DecideShared {
  RowSum row[kCWarps];
  int32_t x[kCWarps];
  float l[kCWarps];
  int32_t verdict[kCWarps];
  DrawShared draw;
  double tab[kExpTable];
  float red[kCWarps];
  int32_t found;
};

template <class T, bool kSampled, Stage kStage>
__device__ void decide(const VerifyArgs& a,
                       const cooperative_groups::cluster_group& cl, int b,
                       bool leader, DecideShared& sh) {
  const int k = a.rows.positions - 1;
  const int64_t vocab = a.rows.vocab;
  const int spans = a.split * kSWarps * a.warp_spans;
  const int n = valid_drafts(a.num_valid, b, k);
  const int32_t* drow = a.draft + static_cast<int64_t>(b) * k;
  const float* urow = kSampled
      ? a.uniforms + static_cast<int64_t>(b) * (k + 1) : nullptr;
  int32_t* out = a.sampled + static_cast<int64_t>(b) * (k + 1);
  if (n < 0) {
    if (leader) emit(drow, 0, -1, k, out, a.count + b);
    return;
  }
  const Setting set = kSampled ? setting_of(a.set, b)
                               : Setting{0.0f, 0, 1.0f};
  const bool greedy = !kSampled || !(set.t > 0.0f);
  const float scale = greedy ? 0.0f : scale_of(set.t);
  const double scale64 = greedy ? 0.0 : scale64_of(set.t);
  const Part* parts = a.parts + static_cast<int64_t>(b) * (k + 1) * spans;

  const auto mark = [&] {
    if (threadIdx.x == 0) a.marked[atomicAdd(a.marks, 1)] = b;
  };

  // a warp a position, until one is not accepted; position n never is
  int s = -1;
  int32_t skip = -1;
  float skip_l = 0.0f;
  RowSum stop{};
  for (int j0 = 0; s < 0; j0 += kCWarps) {
    const int j = j0 + warp_id();
    if (j <= n) {
      int32_t x = -1;
      float l = 0.0f;
      double u = 0.0;
      if (j < n) {
        x = drow[j];
        const T* r = row_ptr<T>(a.rows, b, j);
        if (x < 0 || x >= vocab || r == nullptr) x = -1;
        if (kSampled) u = urow[j];
        if (!greedy && x >= 0) l = canon(to_f32(r[x]));
      }
      const Part* rp = parts + static_cast<int64_t>(j) * spans;
      const RowSum row = greedy ? join_parts<true, false>(rp, spans, scale)
                              : join_parts<false, true>(rp, spans, scale);
      Verdict v = kReject;
      if (x >= 0 && row.m > -CUDART_INF_F)
        v = greedy ? (x == row.arg && u < 1.0 ? kAccept : kReject)
                   : verdict(row, l, u, scale, a.guard);
      if (lane_id() == 0) {
        sh.row[warp_id()] = row;
        sh.x[warp_id()] = x;
        sh.l[warp_id()] = l;
        sh.verdict[warp_id()] = v;
      }
    }
    __syncthreads();
    for (int g = 0; g < kCWarps && s < 0; ++g) {
      int v = sh.verdict[g];
      if (v == kUnsure) {
        if (kStage == kMark) {
          mark();
          return;
        }
        const float m = sh.row[g].m;
        const RowWeights<T> weights(row_ptr<T>(a.rows, b, j0 + g), vocab, m,
                                    scale, scale64, -1, sh.tab);
        const double z = cluster_sum64(cl, weights, sh.draw);
        const double u = urow[j0 + g];
        const double w = m == CUDART_INF_F
            ? (sh.l[g] == m ? 1.0 : 0.0)
            : weight64(sh.l[g], m, scale64, sh.tab);
        v = u < w / z ? kAccept : kReject;
      }
      if (v == kReject) {
        s = j0 + g;
        stop = sh.row[g];
        skip = s < n ? sh.x[g] : -1;
        skip_l = sh.l[g];
      }
    }
    __syncthreads();
  }
  int32_t tok = stop.m > -CUDART_INF_F ? stop.arg : -1;
  if (!greedy && stop.m > -CUDART_INF_F) {
    RowWeights<T> weights(row_ptr<T>(a.rows, b, s), vocab, stop.m, scale,
                          scale64, skip, sh.tab);
    const double u = urow[k];
    // The span that holds the target, from the spans' sums; every warp
    // finds it for itself. The rejected token's weight leaves its span.
    const Part* rp = parts + static_cast<int64_t>(s) * spans;
    const int skip_span =
        skip < 0 ? -1
                 : static_cast<int>((static_cast<int64_t>(skip) +
                                     weights.head) / RowVecs<T>::E) /
                       ((weights.nv + spans - 1) / spans);
    const Pick pick = pick_span(spans, u, [&](int i) {
      const Part p = rp[i];
      double v = p.s == 0.0f ? 0.0f : p.s * weight32(p.m, stop.m, scale);
      if (i == skip_span)
        v = fmax(v - weight32(skip_l, stop.m, scale), 0.0);
      return v;
    });
    tok = -2;
    if (pick.span >= 0)
      tok = span_draw(weights, span_of(weights.nv, pick.span, spans),
                      pick.ahead, pick.target, stop.s * a.guard, sh.red,
                      &sh.found);
    if (kStage == kMark && tok == -2) {
      mark();
      return;
    }
    if (tok == -2) tok = cluster_draw(cl, weights, u, sh.draw);
    if (tok < 0) {  // nothing but the rejected token
      weights.skip = -1;
      tok = cluster_draw(cl, weights, u, sh.draw);
    }
  }
  if (leader) emit(drow, s, tok, k, out, a.count + b);
}

template <class T, bool kSampled, Stage kStage>
__global__ void __launch_bounds__(kCThreads) decide_kernel(VerifyArgs a) {
  const auto cl = cooperative_groups::this_cluster();
  __shared__ DecideShared sh;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (kSampled) fill_exp_table(sh.tab);
  __syncthreads();
  const int cs = static_cast<int>(cl.num_blocks());
  const bool leader = cl.block_rank() == 0;
  const int first = static_cast<int>(blockIdx.x) / cs;
  if (kStage != kMarked) {
    decide<T, kSampled, kStage>(a, cl, first, leader, sh);
    return;
  }
  // clusters take the marked requests in turns
  const int marks = *a.marks;
  for (int i = first; i < marks; i += static_cast<int>(gridDim.x) / cs) {
    decide<T, kSampled, kStage>(a, cl, a.marked[i], leader, sh);
    __syncthreads();
  }
}

template <class T, bool kSampled>
static int launch_verify_t(const VerifyArgs& a, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(a.rows.batch) *
                        static_cast<unsigned>(a.rows.positions) *
                        static_cast<unsigned>(a.split);
  int rc = launch_after(spans_kernel<T, kSampled>, grid, kSThreads, 1,
                              a, st);
  if (rc != SG_OK) return rc;
  const unsigned requests = static_cast<unsigned>(a.rows.batch);
  if constexpr (!kSampled) {
    return launch_after(decide_kernel<T, false, kWhole>, requests, kCThreads,
                        1, a, st);
  } else {
    if (a.marks == nullptr)
      return launch_after(decide_kernel<T, true, kWhole>, requests * kMaxCluster,
                          kCThreads, kMaxCluster, a, st);
    rc = launch_after(decide_kernel<T, true, kMark>, requests, kCThreads, 1,
                      a, st);
    if (rc != SG_OK) return rc;
    return launch_after(decide_kernel<T, true, kMarked>,
                        std::min(requests, 74u) * kMaxCluster, kCThreads,
                        kMaxCluster, a, st);
  }
}

template <bool kSampled>
static int launch_verify(const VerifyArgs& a, cudaStream_t st) {
  switch (a.rows.dtype) {
    case SG_F32:
      return launch_verify_t<float, kSampled>(a, st);
    case SG_BF16:
      return launch_verify_t<__nv_bfloat16, kSampled>(a, st);
    default:
      return launch_verify_t<__half, kSampled>(a, st);
  }
}

// With many rows (more than resident blocks) two blocks share a row: rows
// read in vain before a rejection is known get fewer than with one (256 x 17
// rows of 128256 bf16: 78 us against 87; with four the blocks that find
// nothing to do outweigh that, 80 us).
constexpr int kManySplit = 2;

// Up to this batch one launch with a cluster a request decides everything
// (64 requests without drafts: 24 us against 35 with the second launch;
// 256 requests: 65 against 50).
constexpr int kWholeBatch = 128;

// Blocks that share a row: enough to fill the machine's resident blocks.
static int split_of(int64_t rows) {
  const int64_t s = rows > 0 ? (kSBlocks * 148 + rows / 2) / rows : 1;
  return static_cast<int>(std::min<int64_t>(kMaxSplit,
                                            std::max<int64_t>(1, s)));
}

// ---------------------------------------------------------------------------
// verification from logits with top-k or top-p
// ---------------------------------------------------------------------------
// The rows' kernel (target_probs.cu) has left the verdict on each draft and
// the token that follows a rejection; a warp a request puts them together.
struct GatherArgs {
  const RowStat* stats;
  const int32_t* draft;
  const int32_t* num_valid;
  int32_t* sampled;
  int32_t* count;
  int32_t batch;
  int32_t k;
};

__global__ void __launch_bounds__(kCThreads) gather_kernel(GatherArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = static_cast<int>(blockIdx.x) * kCWarps + warp_id();
  if (b >= a.batch) return;
  const int n = valid_drafts(a.num_valid, b, a.k);
  const RowStat* stats = a.stats + static_cast<int64_t>(b) * (a.k + 1);
  const int32_t* drow = a.draft + static_cast<int64_t>(b) * a.k;
  int32_t* out = a.sampled + static_cast<int64_t>(b) * (a.k + 1);
  int s = n;  // -1: inactive
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane_id();
    const unsigned no =
        __ballot_sync(SG_FULL_MASK, j >= n || !stats[j].accept);
    if (no) {
      s = j0 + __ffs(no) - 1;
      break;
    }
  }
  const int32_t tok = s >= 0 ? stats[s].token : -1;
  for (int j = lane_id(); j <= a.k; j += 32)
    out[j] = j < s ? drow[j] : (j == s ? tok : -1);
  if (lane_id() == 0) a.count[b] = max(s, 0) + (tok >= 0 ? 1 : 0);
}

// ---------------------------------------------------------------------------
// verification from probabilities: one cluster a request
// ---------------------------------------------------------------------------
// The acceptance tests are K gathers, which every block of the cluster makes
// for itself; then the one row the token is drawn from (and the drafter's)
// is read once, split over the cluster. Its sums are fp32 over a few
// vectors and 64 bits beyond; where the target is not clear of the borders
// of the token found, the row is summed again with every weight in 64 bits
// (differences of fp32 probabilities are exact there). Converting every
// value to 64 bits in the first place took twice the time of its bytes.
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

// max(p - q, 0) (q NULL: p), without token `skip`: cluster_draw's source.
struct ProbWeights : RowVecs<float> {
  const float* q;
  bool q_vecs;  // q's rows lie on the same 16-byte grid as p's
  int64_t skip;

  __device__ __forceinline__ ProbWeights(const float* p, const float* q_,
                                         int64_t vocab, int64_t skip_)
      : RowVecs<float>(p, vocab), q(q_), skip(skip_) {
    q_vecs = ((reinterpret_cast<uintptr_t>(p) ^
               reinterpret_cast<uintptr_t>(q_)) & 15) == 0;
  }
  __device__ __forceinline__ uint4 load(const float* row, int vec,
                                        bool vecs) const {
    uint4 r;
    r.x = r.y = r.z = r.w = 0;
    const int64_t i0 = first(vec);
    if (vecs && inner(vec)) return load_16(row + i0);
    if (i0 >= 0 && i0 < v) r.x = __float_as_uint(row[i0]);
    if (i0 + 1 >= 0 && i0 + 1 < v) r.y = __float_as_uint(row[i0 + 1]);
    if (i0 + 2 >= 0 && i0 + 2 < v) r.z = __float_as_uint(row[i0 + 2]);
    if (i0 + 3 >= 0 && i0 + 3 < v) r.w = __float_as_uint(row[i0 + 3]);
    return r;
  }
  __device__ __forceinline__ double weight(uint32_t a, uint32_t b) const {
    const double d =
        static_cast<double>(clean_prob(__uint_as_float(a))) -
        static_cast<double>(clean_prob(__uint_as_float(b)));
    return d > 0.0 ? d : 0.0;
  }
  __device__ __forceinline__ void weights(const uint4& a, const uint4& b,
                                          int vec, double* w) const {
    w[0] = weight(a.x, b.x);
    w[1] = weight(a.y, b.y);
    w[2] = weight(a.z, b.z);
    w[3] = weight(a.w, b.w);
    const int64_t at = skip - first(vec);
    if (at >= 0 && at < E) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e == at) w[e] = 0.0;
    }
  }
  __device__ __forceinline__ Span span(int w, int n) const {
    return span_of(nv, w, n);
  }
  __device__ __forceinline__ void vec(int at, int end, double* w) const {
    uint4 a, b;
    a.x = a.y = a.z = a.w = 0;
    b = a;
    if (at < end) {
      a = load(row, at, true);
      if (q) b = load(q, at, q_vecs);
    }
    weights(a, b, at, w);
  }
  // fp32 weights of a vector; their sum. A weight is off by 2^-24 of it; an
  // infinite p gives an infinite sum, which no token is clear of.
  __device__ __forceinline__ float fast(const uint4& a, const uint4& b,
                                        int vec, float* w) const {
    const uint32_t pa[E] = {a.x, a.y, a.z, a.w};
    const uint32_t qa[E] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = fmaxf(__uint_as_float(pa[e]), 0.0f);
      if (q) w[e] = fmaxf(w[e] - clean_prob(__uint_as_float(qa[e])), 0.0f);
    }
    const int64_t at = skip - first(vec);
    if (at >= 0 && at < E) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e == at) w[e] = 0.0f;
    }
    return (w[0] + w[1]) + (w[2] + w[3]);
  }
  __device__ __forceinline__ float fast_vec(int at, int end, float* w) const {
    uint4 a, b;
    a.x = a.y = a.z = a.w = 0;
    b = a;
    if (at < end) {
      a = load(row, at, true);
      if (q) b = load(q, at, q_vecs);
    }
    return fast(a, b, at, w);
  }
  __device__ __forceinline__ double fast_sum(int at, int end, int step) const {
    constexpr int U = 4;  // loads in flight
    double s = 0.0;
    for (; at < end; at += U * step) {
      uint4 a[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u].x = a[u].y = a[u].z = a[u].w = 0;
        b[u] = a[u];
        const int i = at + u * step;
        if (i < end) {
          a[u] = load(row, i, true);
          if (q) b[u] = load(q, i, q_vecs);
        }
      }
      float t[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float w[E];
        t[u] = fast(a[u], b[u], at + u * step, w);
      }
#pragma unroll
      for (int h = U / 2; h > 0; h /= 2)
#pragma unroll
        for (int u = 0; u < h; ++u) t[u] += t[u + h];
      s += t[0];
    }
    return s;
  }
  __device__ __forceinline__ double sum(int at, int end, int step) const {
    constexpr int U = 4;  // loads of each row in flight
    double s = 0.0;
    for (; at < end; at += U * step) {
      uint4 a[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u].x = a[u].y = a[u].z = a[u].w = 0;
        b[u] = a[u];
        const int i = at + u * step;
        if (i < end) {
          a[u] = load(row, i, true);
          if (q) b[u] = load(q, i, q_vecs);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        double w[E];
        weights(a[u], b[u], at + u * step, w);
        s += (w[0] + w[1]) + (w[2] + w[3]);
      }
    }
    return s;
  }
};

// The fp32 additions on a weight's way (at most 17) and its own rounding.
constexpr double kProbGuard = 1.2e-6;

// cluster_draw from fp32 sums; -2 where they cannot tell.
__device__ int32_t cluster_try_draw(
    const cooperative_groups::cluster_group& cl, const ProbWeights& weights,
    double u, DrawShared& sh, float* red, int32_t* s_found) {
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int spans = cs * kCWarps;
  const int mine = rank * kCWarps + warp_id();
  const Span sp = span_of(weights.nv, mine, spans);
  const double s = warp_sum64(weights.fast_sum(sp.v0 + lane_id(), sp.v1, 32));
  cl.sync();  // every block runs before any writes into another
  if (lane_id() < cs) *cl.map_shared_rank(&sh.seg[mine], lane_id()) = s;
  cl.sync();
  const Pick pick = pick_span(spans, u, [&](int i) { return sh.seg[i]; });
  if (pick.span < 0) return -1;
  if (pick.span / kCWarps == rank) {
    const int32_t tok =
        span_draw(weights, span_of(weights.nv, pick.span, spans), pick.ahead,
                  pick.target, pick.total * kProbGuard, red, s_found);
    if (static_cast<int>(threadIdx.x) < cs)
      *cl.map_shared_rank(&sh.tok, static_cast<int>(threadIdx.x)) = tok;
  }
  cl.sync();
  return sh.tok;
}

__global__ void __launch_bounds__(kCThreads, 5) probs_kernel(ProbArgs a) {
  const auto cl = cooperative_groups::this_cluster();
  __shared__ DrawShared sh;
  __shared__ float s_red[kCWarps];
  __shared__ int32_t s_found;
  __shared__ int s_stop;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cs = static_cast<int>(cl.num_blocks());
  const int b = static_cast<int>(blockIdx.x) / cs;
  const bool leader = cl.block_rank() == 0;
  const int k = a.p.positions - 1;
  const int64_t v = a.p.vocab;
  const int n = valid_drafts(a.num_valid, b, k);
  const int32_t* drow = a.draft + static_cast<int64_t>(b) * k;
  const float* u = a.uniforms + static_cast<int64_t>(b) * (k + 1);
  int32_t* out = a.sampled + static_cast<int64_t>(b) * (k + 1);
  if (n < 0) {  // the whole cluster leaves: no barrier is waited for
    if (leader) emit(drow, 0, -1, k, out, a.count + b);
    return;
  }
  if (threadIdx.x == 0) s_stop = n;
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += kCThreads) {
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
    const float* qrow =
        s < n && a.has_q ? row_ptr<float>(a.q, b, s) : nullptr;
    const int64_t skip = s < n && !a.has_q ? drow[s] : -1;
    const ProbWeights weights(prow, qrow, v, skip);
    tok = cluster_try_draw(cl, weights, u[k], sh, s_red, &s_found);
    if (tok == -2) tok = cluster_draw(cl, weights, u[k], sh);
    if (tok < 0 && s < n)  // nothing left: the row itself
      tok = cluster_draw(cl, ProbWeights(prow, nullptr, v, -1), u[k], sh);
  }
  if (leader) emit(drow, s, tok, k, out, a.count + b);
}

// 64-bit indices as the nearest 32-bit ones, a thread each. The launch bounds
// it: 8 x 5 x 32000 greedy with 64-bit drafts takes 12.3 us a call, 8.9 with
// 32-bit ones (19.3 with a library's clamp and conversion).
struct ClampArgs {
  const int64_t* src;
  int64_t n, cols, stride_row, stride_col;
  int32_t* out;
};
constexpr int kClampThreads = 256;
constexpr int64_t kClampBlocks = 148 * 8;

__global__ void __launch_bounds__(kClampThreads) clamp_kernel(ClampArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t step = static_cast<int64_t>(gridDim.x) * kClampThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kClampThreads +
                   threadIdx.x;
       i < a.n; i += step) {
    const int64_t x =
        a.src[i / a.cols * a.stride_row + i % a.cols * a.stride_col];
    a.out[i] = static_cast<int32_t>(
        max(static_cast<int64_t>(INT32_MIN),
            min(static_cast<int64_t>(INT32_MAX), x)));
  }
}

static int check_workspace(const sg_rows* r, const void* ws, size_t bytes) {
  const size_t need = sg_verify_workspace_size(r->batch, r->positions);
  if (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15))
    return SG_ERR_WORKSPACE;
  return SG_OK;
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
  if (static_cast<int64_t>(logits->batch) * logits->positions >
      INT32_MAX / kMaxSplit)
    return SG_ERR_UNSUPPORTED;
  if (!sampling || !has_filter(*sampling)) {
    VerifyArgs va{};
    va.rows = *logits;
    if (sampling) va.set = *sampling;
    va.draft = draft;
    va.num_valid = num_valid;
    va.uniforms = uniforms;
    va.sampled = sampled;
    va.count = count;
    const int64_t rows =
        static_cast<int64_t>(logits->batch) * logits->positions;
    va.split = split_of(rows);
    const bool many = rows > kSBlocks * 148 && logits->positions > 1;
    if (many) va.split = kManySplit;
    va.parts = static_cast<Part*>(workspace);
    const int elems = logits->dtype == SG_F32 ? 4 : 8;
    va.warp_spans = warp_spans_of(logits->vocab, elems, va.split);
    const int spans = va.split * kSWarps * va.warp_spans;
    va.guard = guard_of(logits->vocab, kUnroll * 32 * elems * spans);
    int32_t* ctl = reinterpret_cast<int32_t*>(va.parts + rows * spans);
    size_t zero = 0;
    if (sampling && logits->batch > kWholeBatch) {
      va.marks = ctl;
      va.marked = ctl + 1 + logits->batch + rows;
      zero = 1;
    }
    if (many) {
      va.rejected = ctl + 1;
      va.arrived = va.rejected + logits->batch;
      zero = 1 + logits->batch + rows;
    }
    if (zero) {
      const cudaError_t err = cudaMemsetAsync(ctl, 0, zero * sizeof(int32_t), st);
      if (err != cudaSuccess) {
        set_cuda_error(err);
        return SG_ERR_CUDA;
      }
    }
    return sampling ? launch_verify<true>(va, st)
                    : launch_verify<false>(va, st);
  }
  // rows' statistics, then [B] rejected positions and the rows handed out
  RowStat* stats = static_cast<RowStat*>(workspace);
  const int64_t rows = static_cast<int64_t>(logits->batch) * logits->positions;
  int32_t* rejected = reinterpret_cast<int32_t*>(stats + rows);
  const cudaError_t err = cudaMemsetAsync(
      rejected, 0, (static_cast<size_t>(logits->batch) + 1) * sizeof(int32_t),
      st);
  if (err != cudaSuccess) {
    set_cuda_error(err);
    return SG_ERR_CUDA;
  }
  rc = launch_row_stats(*logits, *sampling, draft, num_valid, uniforms, stats,
                        rejected, rejected + logits->batch, st);
  if (rc != SG_OK) return rc;
  const GatherArgs ga{stats, draft,         num_valid,
                      sampled, count, logits->batch, logits->positions - 1};
  return launch_after(
      gather_kernel,
      static_cast<unsigned>(ceil_div(logits->batch, kCWarps)), kCThreads, 1,
      ga, st);
}

}  // namespace sg

using namespace sg;

extern "C" int sg_clamp_i32(const int64_t* src, int64_t rows, int64_t cols,
                            int64_t stride_row, int64_t stride_col,
                            int32_t* out, sg_stream_t stream) {
  NvtxScope nvtx("sg_clamp_i32");
  if (rows < 0 || cols < 0 || stride_row < 0 || stride_col < 0)
    return SG_ERR_INVALID;
  if (rows == 0 || cols == 0) return SG_OK;
  if (!src || !out) return SG_ERR_INVALID;
  if (rows > INT64_MAX / cols) return SG_ERR_UNSUPPORTED;
  const ClampArgs a{src, rows * cols, cols, stride_row, stride_col, out};
  const int64_t blocks = std::min(kClampBlocks, ceil_div(a.n, kClampThreads));
  return launch_after(clamp_kernel, static_cast<unsigned>(blocks),
                      kClampThreads, 1, a,
                      reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t sg_verify_workspace_size(int32_t batch, int32_t positions) {
  if (batch <= 0 || positions <= 0) return 0;
  const size_t rows = static_cast<size_t>(batch) * positions;
  const size_t spans = rows * kMaxSpans * sizeof(Part) +
      (1 + 2 * static_cast<size_t>(batch) + rows) * sizeof(int32_t);
  const size_t stats = rows * sizeof(RowStat) +
                       (static_cast<size_t>(batch) + 1) * sizeof(int32_t);
  return std::max(spans, stats);
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
  if (probs->batch > INT32_MAX / kMaxCluster) return SG_ERR_UNSUPPORTED;
  return launch_after(probs_kernel,
                      static_cast<unsigned>(probs->batch) * kMaxCluster,
                      kCThreads, kMaxCluster, a,
                      reinterpret_cast<cudaStream_t>(stream));
}
