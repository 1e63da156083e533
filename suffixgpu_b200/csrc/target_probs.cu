// The target's probabilities under temperature, top-k and top-p: written out
// (sg_target_probs), or as statistics per row for the verification that
// draws from logits (verify.cu). Definitions in include/suffixgpu.h.
//
// One cluster a row; each block keeps its share of the row in shared memory,
// so that the row is read from HBM once whatever the number of passes.
#include <cuda_runtime.h>

#include <algorithm>

#include "sg_sampling.cuh"

namespace sg {

constexpr int kFThreads = 256;
constexpr int kFWarps = kFThreads / 32;
constexpr int kSoftBlocks = 5;  // blocks on an SM, plain softmax
constexpr int kKeptBlocks = 3;  // with filters
constexpr int kStatBlocks = 2;  // with filters, nothing written
constexpr int kBins = 1024;      // of a window; the last takes the rest
constexpr float kPlaces = 64.0f;  // places told apart in a bin
constexpr int kWindows = 4;      // looked at before bisect_row
constexpr int kList = 1024;      // candidates the first block can hold
constexpr int kOwn = kList / kFThreads;
constexpr int kFixBits = 46;     // of a candidate's weight in fixed point

// What a cluster finds for a row.
struct Kept {
  double z;   // sum of the kept weights
  float m;    // largest value
  float low;  // smallest kept value
  int32_t arg;
};

struct RowShared {
  SpanSum part[kFWarps];
  SpanSum slot[kMaxCluster];  // the cluster's blocks write into each other
  double s[kMaxCluster];
  uint32_t top;
  int32_t next;
  float redf[kFWarps];
  int32_t redi[kFWarps];
  uint32_t redu[kFWarps];
  double red[32];
  double tab[kExpTable];
};

// How the first block goes on after a window's counts.
struct Plan {
  int32_t off;    // >= 0: count the window of bins from here on
  int32_t give;   // 1: bisect_row
  int32_t bk;     // bin of the k-th value
  int32_t above;  // values in bins before it
  int32_t p0, p1; // bins in which top-p's border is looked for
};

struct FilterShared {
  uint32_t hist[kBins];  // this block's counts
  uint32_t offs[kBins];  // and their places in the bins, summed
  uint32_t list[kList];  // this block's candidates (order keys)
  int32_t listed;
  int32_t n[kMaxCluster];
  uint32_t nall[kMaxCluster];
  double a[kMaxCluster];
  uint64_t redl[2][kFWarps];
  Plan plan;
  // first block, over the windows so far
  int32_t seen;          // values in earlier windows
  float mass;            // and their weights, about
  int32_t k_found, pick, pick_most;
  float need, need_most;  // top-p's share, with fewest and most values kept
  // the result; done 0: bisect_row, 2: sum the row exactly and come again
  double z;
  float low;
  int32_t done;
};

__device__ __forceinline__ int32_t block_sum_i32(int32_t v, int32_t* red) {
  v = __reduce_add_sync(SG_FULL_MASK, v);
  __syncthreads();
  if (lane_id() == 0) red[warp_id()] = v;
  __syncthreads();
  v = lane_id() < kFWarps ? red[lane_id()] : 0;
  return __reduce_add_sync(SG_FULL_MASK, v);
}
__device__ __forceinline__ uint32_t block_or(uint32_t v, uint32_t* red) {
  v = __reduce_or_sync(SG_FULL_MASK, v);
  __syncthreads();
  if (lane_id() == 0) red[warp_id()] = v;
  __syncthreads();
  v = lane_id() < kFWarps ? red[lane_id()] : 0u;
  return __reduce_or_sync(SG_FULL_MASK, v);
}
__device__ __forceinline__ uint32_t block_max_u32(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(SG_FULL_MASK, v);
  __syncthreads();
  if (lane_id() == 0) red[warp_id()] = v;
  __syncthreads();
  v = lane_id() < kFWarps ? red[lane_id()] : 0u;
  return __reduce_max_sync(SG_FULL_MASK, v);
}
// The first block's sums over its candidates: one barrier each, `turn`
// alternating between two sets of slots.
__device__ __forceinline__ int32_t turn_sum_i32(int32_t v, int& turn,
                                                uint64_t (*red)[kFWarps]) {
  v = __reduce_add_sync(SG_FULL_MASK, v);
  turn ^= 1;
  if (lane_id() == 0) red[turn][warp_id()] = static_cast<uint32_t>(v);
  __syncthreads();
  uint32_t s = 0;
#pragma unroll
  for (int i = 0; i < kFWarps; ++i) s += static_cast<uint32_t>(red[turn][i]);
  return static_cast<int32_t>(s);
}
// v < 2^49: two parts, whose warp sums fit 32 bits.
__device__ __forceinline__ uint64_t turn_sum_u64(uint64_t v, int& turn,
                                                 uint64_t (*red)[kFWarps]) {
  const uint32_t lo = __reduce_add_sync(
      SG_FULL_MASK, static_cast<uint32_t>(v) & 0xffffffu);
  const uint32_t hi =
      __reduce_add_sync(SG_FULL_MASK, static_cast<uint32_t>(v >> 24));
  turn ^= 1;
  if (lane_id() == 0)
    red[turn][warp_id()] = (static_cast<uint64_t>(hi) << 24) + lo;
  __syncthreads();
  uint64_t s = 0;
#pragma unroll
  for (int i = 0; i < kFWarps; ++i) s += red[turn][i];
  return s;
}

// One row's share of a block, and what the passes over it need.
template <class T>
struct Share : RowVecs<T> {
  using RowVecs<T>::E;
  const uint4* buf;  // vectors [v0, v0 + n) of the row
  int v0, n;
  float m, scale;
  double m64, scale64;
  const double* tab;
  float bin_scale;  // bins per unit of m - l

  __device__ __forceinline__ Share(const T* row, int64_t vocab)
      : RowVecs<T>(row, vocab) {}

  // Bins of equal width down from the largest value, rounded to nearest;
  // NaN and -inf come last. Monotone in x.
  __device__ __forceinline__ int bin(float x) const {
    const float t = fminf((m - x) * bin_scale, 4194303.0f);
    return __float_as_uint(t + 8388608.0f) & 0x7fffff;
  }
  // Where in its bin a value lies, from 0 to kPlaces.
  __device__ __forceinline__ uint32_t place(float x, int b) const {
    const float t = (m - x) * bin_scale - (static_cast<float>(b) - 0.5f);
    return static_cast<uint32_t>(fmaxf(t, 0.0f) * kPlaces + 0.5f);
  }
  __device__ __forceinline__ double weight(float x) const {
    return weight64(x, m64, scale64, tab);
  }
  // f(value, row index) for this thread's values; the vectors' order is the
  // same in every pass. Values outside the row are left out. With kTop,
  // vectors without a value >= from are passed over.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    each_from<false>(0.0f, f);
  }
  template <bool kTop, class F>
  __device__ __forceinline__ void each_from(float from, F f) const {
    for (int i = threadIdx.x; i < n; i += kFThreads) {
      const uint4 raw[1] = {buf[i]};
      if (kTop && !(Raw<T>::vec_max(raw) >= from)) continue;
      float x[E];
      Raw<T>::unpack(raw[0], x);
      const int64_t at = this->first(v0 + i);
      if (this->inner(v0 + i)) {
#pragma unroll
        for (int e = 0; e < E; ++e) f(x[e], at + e);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at + e >= 0 && at + e < this->v) f(x[e], at + e);
      }
    }
  }
};

// The row's values >= some k-th, >= some top-p border: by bisection of the
// order keys over the whole cluster. Takes the rows whose candidates do not
// fit the first block's list (many values close to one another).
template <class T>
__device__ void bisect_row(const cooperative_groups::cluster_group& cl,
                           const Share<T>& sh, int32_t k, float p,
                           RowShared& rs, FilterShared& fs) {
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  auto total_count = [&](uint32_t from) {
    int32_t c = 0;
    sh.each([&](float x, int64_t) { c += order_key(canon(x)) >= from; });
    c = block_sum_i32(c, rs.redi);
    if (static_cast<int>(threadIdx.x) < cs)
      *cl.map_shared_rank(&fs.n[rank], static_cast<int>(threadIdx.x)) = c;
    cl.sync();
    int32_t s = 0;
    for (int i = 0; i < cs; ++i) s += fs.n[i];
    cl.sync();
    return s;
  };
  auto total_mass = [&](uint32_t from) {
    double s = 0.0;
    sh.each([&](float x, int64_t) {
      if (order_key(canon(x)) >= from) s += sh.weight(x);
    });
    s = block_sum64(s, rs.red);
    if (static_cast<int>(threadIdx.x) < cs)
      *cl.map_shared_rank(&fs.a[rank], static_cast<int>(threadIdx.x)) = s;
    cl.sync();
    double t = 0.0;
    for (int i = 0; i < cs; ++i) t += fs.a[i];
    cl.sync();
    return t;
  };
  // bits in which the row's keys differ: only those are looked at
  uint32_t any = 0, not_all = 0;
  sh.each([&](float x, int64_t) {
    any |= order_key(canon(x));
    not_all |= ~order_key(canon(x));
  });
  any = block_or(any, rs.redu);
  not_all = block_or(not_all, rs.redu);
  if (static_cast<int>(threadIdx.x) < cs) {
    *cl.map_shared_rank(&fs.n[rank], static_cast<int>(threadIdx.x)) =
        static_cast<int32_t>(any);
    *cl.map_shared_rank(&fs.nall[rank], static_cast<int>(threadIdx.x)) =
        not_all;
  }
  cl.sync();
  any = not_all = 0;
  for (int i = 0; i < cs; ++i) {
    any |= static_cast<uint32_t>(fs.n[i]);
    not_all |= fs.nall[i];
  }
  cl.sync();
  const uint32_t differ = any & not_all;
  const uint32_t common = any & ~not_all;
  uint32_t low = common;
  if (k > 0) {
    for (uint32_t bits = differ; bits;) {
      const uint32_t bit = 0x80000000u >> __clz(bits);
      bits &= ~bit;
      if (total_count(low | bit) >= k) low |= bit;
    }
  }
  double z = total_mass(low);
  if (p < 1.0f) {
    const double need = static_cast<double>(p) * z;
    uint32_t t = common;
    for (uint32_t bits = differ; bits;) {
      const uint32_t bit = 0x80000000u >> __clz(bits);
      bits &= ~bit;
      if (total_mass(max(t | bit, low)) >= need) t |= bit;
    }
    if (t > low) {
      low = t;
      z = total_mass(low);
    }
  }
  if (threadIdx.x == 0) {
    fs.low = low == common ? -CUDART_INF_F : key_value(low);
    fs.z = z;
  }
  __syncthreads();
}

// First block: reads the plan off a window's counts (all its threads).
__device__ __forceinline__ void plan_window(
    const cooperative_groups::cluster_group& cl, int32_t off, int32_t k,
    float p, float octaves, float row_sum, RowShared& rs, FilterShared& fs,
    Plan& plan) {
  constexpr int kPer = kBins / kFThreads;
  static_assert(kPer == 4, "a thread reads its bins as one vector");
  const int cs = static_cast<int>(cl.num_blocks());
  const int tid = static_cast<int>(threadIdx.x);
  int32_t c[kPer] = {0, 0, 0, 0};
  float o[kPer] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int r = 0; r < kMaxCluster; ++r) {
    if (r >= cs) break;
    const FilterShared* from = cl.map_shared_rank(&fs, r);
    const uint4 h = reinterpret_cast<const uint4*>(from->hist)[tid];
    const uint4 f = reinterpret_cast<const uint4*>(from->offs)[tid];
    c[0] += h.x;
    c[1] += h.y;
    c[2] += h.z;
    c[3] += h.w;
    o[0] += f.x;
    o[1] += f.y;
    o[2] += f.z;
    o[3] += f.w;
  }
  float w[kPer];  // the weight at the mean place of a bin's values
  int32_t cnt = 0;
  float mass = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float at = static_cast<float>(off + tid * kPer + i) - 0.5f +
                     o[i] / (kPlaces * fmaxf(1.0f, static_cast<float>(c[i])));
    w[i] = exp2_fast(-at * octaves);
    cnt += c[i];
    mass += static_cast<float>(c[i]) * w[i];
  }
  const int32_t ci = warp_incl_scan(cnt);
  float mi = mass;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float t = __shfl_up_sync(SG_FULL_MASK, mi, o);
    if (lane_id() >= o) mi += t;
  }
  if (lane_id() == 31) {
    rs.redi[warp_id()] = ci;
    rs.redf[warp_id()] = mi;
  }
  if (tid == 0) {
    fs.pick = fs.pick_most = INT32_MAX;
    if (off == 0 && !fs.k_found) {
      fs.seen = 0;
      fs.mass = 0.0f;
    }
  }
  __syncthreads();
  const int32_t seen = fs.seen;
  const float mass_seen = fs.mass;
  int32_t run = seen + ci - cnt;
  float mr = mass_seen + (mi - mass);
  int32_t all_c = seen;
  float all_m = mass_seen;
#pragma unroll
  for (int i = 0; i < kFWarps; ++i) {
    if (i < warp_id()) {
      run += rs.redi[i];
      mr += rs.redf[i];
    }
    all_c += rs.redi[i];
    all_m += rs.redf[i];
  }
  if (k > 0 && !fs.k_found) {
    int32_t r = run;
    float q = mr;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (r < k && k <= r + c[i]) {
        plan.bk = off + tid * kPer + i;
        plan.above = r;
        fs.pick = plan.bk;
        // values equal to the k-th are kept too: up to the whole bin
        fs.need = p * (q + static_cast<float>(k - r) * w[i]);
        fs.need_most = p * (q + static_cast<float>(c[i]) * w[i]);
      }
      r += c[i];
      q += static_cast<float>(c[i]) * w[i];
    }
  }
  if (k <= 0 && tid == 0) fs.need = fs.need_most = p * row_sum;
  __syncthreads();
  bool k_now = false;
  if (k > 0 && !fs.k_found) {
    k_now = fs.pick != INT32_MAX;
    __syncthreads();
    if (tid == 0) {
      fs.pick = INT32_MAX;
      if (k_now) fs.k_found = 1;
    }
    __syncthreads();
  }
  // the border of top-p, once the kept mass is known
  int32_t next = -1;
  if (p < 1.0f && (k <= 0 || fs.k_found)) {
    if (k_now && off > 0) {
      next = 0;  // it may lie in an earlier window
    } else {
      float q = mr;
      int32_t at = INT32_MAX, most = INT32_MAX;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        q += static_cast<float>(c[i]) * w[i];
        if (tid * kPer + i < kBins - 1) {
          if (q >= fs.need) at = min(at, off + tid * kPer + i);
          if (q >= fs.need_most) most = min(most, off + tid * kPer + i);
        }
      }
      if (at != INT32_MAX) atomicMin(&fs.pick, at);
      if (most != INT32_MAX) atomicMin(&fs.pick_most, most);
      __syncthreads();
      at = fs.pick;
      most = fs.pick_most;
      // the border does not lie beyond the k-th value
      if (k > 0 && plan.bk < off + kBins - 1) {
        at = min(at, plan.bk);
        most = min(most, plan.bk);
      }
      if (most == INT32_MAX) {
        next = off + kBins - 1;
        if (at != INT32_MAX) next = kWindows * kBins;  // split: bisect_row
      } else if (tid == 0) {
        plan.p0 = max(at - 1, 0);
        plan.p1 = k > 0 ? min(most + 1, plan.bk) : most + 1;
      }
    }
  } else if (k > 0 && !fs.k_found) {
    next = off + kBins - 1;
  }
  __syncthreads();
  if (tid == 0) {
    plan.off = next;
    plan.give = next >= kWindows * (kBins - 1);
    fs.seen = next == 0 ? 0 : all_c;
    fs.mass = next == 0 ? 0.0f : all_m;
  }
  __syncthreads();
}

// The smallest kept value and the kept mass of a row with top-k (k > 0) or
// top-p (0 < p < 1) or both; left in fs.low and fs.z of every block.
//
// One pass counts the values in bins from the largest down, a window of bins
// at a time (one or two mostly: a window is 10.7 logits at T = 1, and the
// border at p = 0.95 to 0.99 lies 10.5 to 13 down in rows of a normal bulk
// and a few likely tokens); the first block finds the bin of the
// k-th value from the counts, and from counts and mean places in the bins
// (off by about 1e-5) the bin top-p's border should lie in. A second pass
// sums the weights ahead of those bins in 64 bits and lists the values inside
// them, from which the first block takes both borders: top-k by counting,
// top-p by 64-bit sums, whose order does not matter (fixed point). Their unit
// follows the bins: 2^-46 of the weight the first of them begins with, so
// that a sum over the whole list is off by about 2^-36 of one candidate's
// weight, however deep it lies (with a unit for all rows, 2^-44 of the
// largest weight, borders of top-p next to 1 missed by a token). Whether the
// border lies in the bins looked at shows in the sums; if not, or if the list
// is too short, or the border lies beyond the windows (k-th values of -inf
// among them), bisect_row finds it. Without top-k, top-p's share is taken of
// the row's fp32 sum where the border is clear of that sum's error, else of
// its 64-bit sum.
template <class T>
__device__ void filter_row(const cooperative_groups::cluster_group& cl,
                           Share<T>& sh, int32_t k, float p, double row_sum,
                           double guard, RowShared& rs, FilterShared& fs) {
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int tid = static_cast<int>(threadIdx.x);
  const bool with_p = p < 1.0f;
  // 16 bins an octave of weight, 96 a unit of logits at least
  sh.bin_scale = fminf(fmaxf(16.0f * sh.scale, 96.0f), 1e30f);
  if (tid == 0) {
    fs.listed = 0;
    fs.k_found = 0;
    fs.plan.bk = -1;
  }
  // fs.hist is zero (cleared by the caller before its barrier)
  for (int32_t off = 0;;) {
    const float from = sh.m - (off + kBins) / sh.bin_scale;
    sh.template each_from<true>(from, [&](float x, int64_t) {
      const int b = sh.bin(x) - off;
      if (b >= 0 && b < kBins - 1) {
        atomicAdd(&fs.hist[b], 1u);
        if (with_p) atomicAdd(&fs.offs[b], sh.place(x, b + off));
      }
    });
    cl.sync();
    if (rank == 0) {
      plan_window(cl, off, k, p, sh.scale / sh.bin_scale,
                  static_cast<float>(row_sum), rs, fs, fs.plan);
      const Plan plan = fs.plan;
      __syncthreads();
      if (tid > 0 && tid < cs) cl.map_shared_rank(&fs, tid)->plan = plan;
    }
    cl.sync();
    off = fs.plan.off;
    if (off < 0 || fs.plan.give) break;
    for (int i = tid; i < kBins; i += kFThreads) fs.hist[i] = fs.offs[i] = 0;
    __syncthreads();
  }
  if (fs.plan.give) {
    bisect_row(cl, sh, k, p, rs, fs);
    return;
  }

  // exact sums ahead of the bins looked at, and the values inside them
  const int bk = k > 0 ? fs.plan.bk : -1;
  const int p0 = with_p ? fs.plan.p0 : INT32_MAX;
  const int p1 = with_p ? fs.plan.p1 : -1;
  double s = 0.0, a = 0.0;
  sh.template each_from<true>(
      sh.m - (max(bk, p1) + 1) / sh.bin_scale, [&](float x, int64_t) {
        const int b = sh.bin(x);
        if (b < bk || (with_p && b < p0)) {
          const double w = sh.weight(x);
          if (b < bk) s += w;
          if (b < p0) a += w;
        }
        if (b == bk || (b >= p0 && b <= p1)) {
          const int at = atomicAdd(&fs.listed, 1);
          if (at < kList) fs.list[at] = order_key(canon(x));
        }
      });
  if (k > 0) s = block_sum64(s, rs.red);
  if (with_p) a = block_sum64(a, rs.red);
  __syncthreads();
  if (tid == 0) {
    *cl.map_shared_rank(&rs.s[rank], 0) = s;
    *cl.map_shared_rank(&fs.a[rank], 0) = a;
    *cl.map_shared_rank(&fs.n[rank], 0) = fs.listed;
  }
  cl.sync();
  for (bool exact = k > 0;; exact = true) {
    if (rank == 0) {
      int n = 0;
      bool fits = true;
      double kept = 0.0;  // values before bin bk, or the row's sum
      a = 0.0;
      for (int r = 0; r < cs; ++r) {
        n += fs.n[r];
        fits = fits && fs.n[r] <= kList;
        kept += rs.s[r];
        a += fs.a[r];
      }
      if (!exact) kept = row_sum;
      int done = fits && n <= kList;
      int turn = 0;
      float low = -CUDART_INF_F;
      if (done) {
        // 2^kFixBits over a power of two that no candidate's weight exceeds:
        // values of bin b lie more than b - 1 bins below the largest
        const int top = min(p0, k > 0 ? bk : INT32_MAX);
        const int down = static_cast<int>(
            fminf(static_cast<float>(max(top - 1, 0)) *
                      (sh.scale / sh.bin_scale), 512.0f));
        const double fix = __hiloint2double((1023 + kFixBits + down) << 20, 0);
        const double unit = __hiloint2double((1023 - kFixBits - down) << 20, 0);
        // this thread's candidates: their keys, bins and fixed-point weights
        uint32_t key[kOwn];
        uint64_t w[kOwn];
        bool in_k[kOwn], in_p[kOwn];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          int at = tid + i * kFThreads;
          key[i] = 0;
          w[i] = 0;
          in_k[i] = in_p[i] = false;
          if (at < n) {
            int r = 0;
            while (at >= fs.n[r]) at -= fs.n[r++];
            key[i] = cl.map_shared_rank(fs.list, r)[at];
            const float x = key_value(key[i]);
            const int b = sh.bin(x);
            in_k[i] = b == bk;
            in_p[i] = b >= p0 && b <= p1;
            w[i] = static_cast<uint64_t>(
                __double2ll_rn(sh.weight(x) * fix));
          }
        }
        // The greatest key of a set that `enough` accepts (its smallest, if
        // none but that): bit by bit over the bits in which its keys differ.
        auto border = [&](const bool (&in)[kOwn], auto enough) {
          uint32_t any = 0, not_all = 0, least = 0xffffffffu;
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            if (in[i]) {
              any |= key[i];
              not_all |= ~key[i];
              least = min(least, key[i]);
            }
          }
          any = block_or(any, rs.redu);
          not_all = block_or(not_all, rs.redu);
          least = ~block_max_u32(~least, rs.redu);
          uint32_t t = any & ~not_all;
          for (uint32_t bits = any & not_all; bits;) {
            const uint32_t bit = 0x80000000u >> __clz(bits);
            bits &= ~bit;
            if (enough(t | bit)) t |= bit;
          }
          return max(t, least);
        };
        if (k > 0) {
          const int32_t want = k - fs.plan.above;
          const uint32_t tk = border(in_k, [&](uint32_t from) {
            int32_t c = 0;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) c += in_k[i] && key[i] >= from;
            return turn_sum_i32(c, turn, fs.redl) >= want;
          });
          uint64_t f = 0;
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            f += in_k[i] && key[i] >= tk ? w[i] : 0;
            in_p[i] = in_p[i] && key[i] >= tk;
          }
          kept += static_cast<double>(turn_sum_u64(f, turn, fs.redl)) * unit;
          low = key_value(tk);
        }
        if (with_p) {
          const double need = static_cast<double>(p) * kept;
          const double slack = exact ? 0.0 : need * guard;
          auto mass = [&](uint32_t from) {
            uint64_t f = 0;
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
              f += in_p[i] && key[i] >= from ? w[i] : 0;
            return a +
                   static_cast<double>(turn_sum_u64(f, turn, fs.redl)) * unit;
          };
          if (!(a < need - slack && mass(0) >= need + slack)) {
            done = exact ? 0 : 2;
          } else {
            const uint32_t t = border(
                in_p, [&](uint32_t from) { return mass(from) >= need; });
            low = key_value(t);
            kept = mass(t);
            if (!exact &&
                !(kept >= need + slack && mass(t + 1) < need - slack))
              done = 2;
          }
        }
      }
      if (tid < cs) {
        FilterShared* o = cl.map_shared_rank(&fs, tid);
        o->low = low;
        o->z = kept;
        o->done = done;
      }
    }
    cl.sync();
    if (fs.done != 2) break;
    double all = 0.0;
    sh.each([&](float x, int64_t) { all += sh.weight(x); });
    all = block_sum64(all, rs.red);
    if (tid == 0) *cl.map_shared_rank(&rs.s[rank], 0) = all;
    cl.sync();
  }
  if (!fs.done) bisect_row(cl, sh, k, p, rs, fs);
}

// Loads a row's shares into shared memory and gives its largest value, the
// lowest index of that (t not > 0) or the fp32 sum of its weights (with_sum):
// a running maximum a warp, one exchange over the cluster. rs.top is 0.
template <int U, class T>
__device__ __forceinline__ SpanSum
load_row(const cooperative_groups::cluster_group& cl, Share<T>& sh, uint4* buf,
         float t, bool with_sum, RowShared& rs) {
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int tid = static_cast<int>(threadIdx.x);
  const Span sp = span_of(sh.nv, rank, cs);
  sh.buf = buf;
  sh.v0 = sp.v0;
  sh.n = sp.v1 - sp.v0;
  const bool greedy = !(t > 0.0f);
  const FineScale f = greedy ? FineScale{0.0f, 0.0f} : fine_scale_of(t);
  LaneStat st{-CUDART_INF_F, 0.0, INT32_MAX};
  for (int i0 = 0; i0 < sh.n; i0 += U * kFThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = load_vec(sh, sp.v0 + i0 + u * kFThreads + tid, sp.v1);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * kFThreads + tid < sh.n)
        buf[i0 + u * kFThreads + tid] = raw[u];
    auto index = [&](int u) {
      return sh.first(sp.v0 + i0 + u * kFThreads + tid);
    };
    if (greedy)
      take_vecs<T, true, kNoSum>(raw, index, f, &rs.top, st);
    else if (with_sum)
      take_vecs<T, false, kFineSum>(raw, index, f, &rs.top, st);
    else
      take_vecs<T, false, kNoSum>(raw, index, f, &rs.top, st);
  }
  if (with_sum) st.s = warp_sum64(st.s);
  if (lane_id() == 0) rs.part[warp_id()] = SpanSum{st.s, st.m, st.arg};
  __syncthreads();
  if (warp_id() == 0) {
    const SpanSum p = join_sums(rs.part, kFWarps, t);
    if (lane_id() < cs) *cl.map_shared_rank(&rs.slot[rank], lane_id()) = p;
    if (lane_id() == 0) rs.top = 0;
  }
  cl.sync();
  return join_sums(rs.slot, cs, t);
}

// ---------------------------------------------------------------------------
// a row's statistics
// ---------------------------------------------------------------------------
template <class T>
__device__ Kept keep_row(const cooperative_groups::cluster_group& cl,
                         Share<T>& sh, uint4* buf, const Setting& set,
                         double guard, RowShared& rs, FilterShared& fs) {
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int tid = static_cast<int>(threadIdx.x);
  for (int i = tid; i < kBins; i += kFThreads) fs.hist[i] = fs.offs[i] = 0;
  const int32_t k = set.k > 0 && set.k < sh.v ? set.k : 0;
  const float p = set.p < 1.0f ? set.p : 1.0f;
  // the row's sum is what top-p without top-k takes its share of
  const SpanSum row =
      load_row<8>(cl, sh, buf, set.t, set.t > 0.0f && k == 0 && p < 1.0f, rs);
  Kept kept{0.0, row.m, -CUDART_INF_F, -1};
  if (!(row.m > -CUDART_INF_F)) return kept;  // no mass
  kept.arg = 0;
  if (!(set.t > 0.0f)) {  // greedy: the first largest value
    kept.arg = row.arg;
    kept.z = 1.0;
    return kept;
  }
  sh.m = row.m;
  sh.m64 = static_cast<double>(row.m);
  sh.scale = scale_of(set.t);
  sh.scale64 = scale64_of(set.t);
  sh.tab = rs.tab;
  double s = 0.0;
  if (row.m == CUDART_INF_F || !(p > 0.0f)) {
    // only the largest value has mass, or is kept
    sh.each([&](float x, int64_t) { s += x == row.m ? 1.0 : 0.0; });
    kept.low = row.m;
  } else if (k > 0 || p < 1.0f) {
    filter_row(cl, sh, k, p, row.s, guard, rs, fs);
    kept.low = fs.low;
    kept.z = fs.z;
    return kept;
  } else {
    sh.each([&](float x, int64_t) { s += sh.weight(x); });
  }
  s = block_sum64(s, rs.red);
  if (tid < cs) *cl.map_shared_rank(&rs.s[rank], tid) = s;
  cl.sync();
  for (int i = 0; i < cs; ++i) kept.z += rs.s[i];
  return kept;
}

// ---------------------------------------------------------------------------
// kernels
// ---------------------------------------------------------------------------
struct RowArgs {
  sg_rows rows;
  sg_sampling set;
  double guard;  // relative error of a row's fp32 sum
  float* out;    // [B, positions, V]
  // statistics for the verification
  const int32_t* draft;
  const int32_t* num_valid;
  const float* uniforms;
  RowStat* stats;     // [B, positions]
  int32_t* rejected;  // [B] positions - the lowest position known rejected
  int32_t* taken;     // rows handed out
};

extern __shared__ uint4 row_smem[];

// Eight (or, at odd places, single) probabilities.
__device__ __forceinline__ void store_8(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p),
               "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]),
               "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

// Writes a block's share of a row, f(pair of values) giving the
// probabilities: vectors whole where the output lies on the vectors' grid,
// else value by value (neighbouring threads on neighbouring values).
template <class T, class F>
__device__ __forceinline__ void write_share(const Share<T>& sh, float* orow,
                                            F f) {
  constexpr int E = Share<T>::E;
  const int64_t base = sh.first(sh.v0);
  if (sh.n > 0 && sh.inner(sh.v0) && sh.inner(sh.v0 + sh.n - 1) &&
      (reinterpret_cast<uintptr_t>(orow + base) & (4 * E - 1)) == 0) {
    for (int i = threadIdx.x; i < sh.n; i += kFThreads) {
      float x[E];
      Raw<T>::unpack(sh.buf[i], x);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 p = f(make_float2(x[e], x[e + 1]));
        x[e] = p.x;
        x[e + 1] = p.y;
      }
      float* o = orow + base + static_cast<int64_t>(i) * E;
      if constexpr (E == 8)
        store_8(o, x);
      else
        *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
    }
    return;
  }
  const int64_t i0 = max(int64_t{0}, base);
  const int64_t i1 = min(sh.v, sh.first(sh.v0 + sh.n));
  const T* share = reinterpret_cast<const T*>(sh.buf) - base;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kFThreads) {
    const float x = to_f32(share[i]);
    orow[i] = f(make_float2(x, x)).x;
  }
}

// One-hot and empty rows.
template <class T>
__device__ __forceinline__ void write_one_hot(const Share<T>& sh, float* orow,
                                              int64_t arg) {
  const int64_t i0 = max(int64_t{0}, sh.first(sh.v0));
  const int64_t i1 = min(sh.v, sh.first(sh.v0 + sh.n));
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kFThreads)
    orow[i] = i == arg ? 1.0f : 0.0f;
}

// Kept values' probabilities (kAll: every value is kept).
template <class T, bool kAll>
__device__ __forceinline__ void write_kept(const Share<T>& sh, float* orow,
                                           float m, float low, double z,
                                           float t) {
  const float inv_z = static_cast<float>(1.0 / z);
  const FineScale f = fine_scale_of(t);
  if (m == CUDART_INF_F || f.hi < kFlatScale) {
    write_share(sh, orow, [&](float2 x) {
      return make_float2(x.x >= low ? weight32(x.x, m, f.hi) * inv_z : 0.0f,
                         x.y >= low ? weight32(x.y, m, f.hi) * inv_z : 0.0f);
    });
    return;
  }
  write_share(sh, orow, [&](float2 x) {
    float2 p = mul2(fine_weight2(x, m, f), make_float2(inv_z, inv_z));
    if (kAll) return make_float2(fmaxf(p.x, 0.0f), fmaxf(p.y, 0.0f));  // NaN
    return make_float2(x.x >= low ? p.x : 0.0f, x.y >= low ? p.y : 0.0f);
  });
}

// Probabilities with top-k or top-p for some rows at least.
template <class T>
__global__ void __launch_bounds__(kFThreads, kKeptBlocks) kept_rows_kernel(RowArgs a) {
  const auto cl = cooperative_groups::this_cluster();
  __shared__ RowShared rs;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  FilterShared* fs = reinterpret_cast<FilterShared*>(row_smem);
  uint4* buf = row_smem + (sizeof(FilterShared) + 15) / 16;
  fill_exp_table(rs.tab);
  if (threadIdx.x == 0) rs.top = 0;
  cl.sync();  // every block runs before any writes into another
  const int64_t r = blockIdx.x / cl.num_blocks();
  const int b = static_cast<int>(r / a.rows.positions);
  const int j = static_cast<int>(r % a.rows.positions);
  const Setting set = setting_of(a.set, b);
  Share<T> sh(row_ptr<T>(a.rows, b, j), a.rows.vocab);
  const Kept kept = keep_row(cl, sh, buf, set, a.guard, rs, *fs);
  float* orow = a.out + r * a.rows.vocab;
  if (kept.arg < 0 || !(set.t > 0.0f))
    write_one_hot(sh, orow, kept.arg);
  else
    write_kept<T, false>(sh, orow, kept.m, kept.low, kept.z, set.t);
  cl.sync();  // no block leaves while another may still write into it
}

// Plain softmax rows: the largest value and the sum in the pass that loads
// the row into shared memory (a running maximum a warp), one exchange over
// the cluster, and the pass that writes. Memory bounds it.
template <class T>
__global__ void __launch_bounds__(kFThreads, kSoftBlocks)
    soft_rows_kernel(RowArgs a) {
  const auto cl = cooperative_groups::this_cluster();
  __shared__ RowShared rs;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) rs.top = 0;
  cl.sync();  // every block runs before any writes into another
  const int64_t r = blockIdx.x / cl.num_blocks();
  const int b = static_cast<int>(r / a.rows.positions);
  const int j = static_cast<int>(r % a.rows.positions);
  const float t = setting_of(a.set, b).t;
  Share<T> sh(row_ptr<T>(a.rows, b, j), a.rows.vocab);
  const SpanSum row = load_row<4>(cl, sh, row_smem, t, t > 0.0f, rs);
  float* orow = a.out + r * a.rows.vocab;
  if (!(row.m > -CUDART_INF_F))
    write_one_hot(sh, orow, -1);
  else if (!(t > 0.0f))
    write_one_hot(sh, orow, row.arg);
  else
    write_kept<T, true>(sh, orow, row.m, -CUDART_INF_F, row.s, t);
}

// The next row that may be needed, found by the first block's first warp:
// rows are handed out in order of position, as many at a time as it takes
// to find one (their requests' known rejections are looked up together).
struct RowQueue {
  int64_t base;
  uint32_t open;  // rows base + lane still to be looked at
  int step;
};
__device__ __forceinline__ int64_t next_row(const RowArgs& a, RowQueue& q) {
  const int64_t rows = static_cast<int64_t>(a.rows.batch) * a.rows.positions;
  const int k = a.rows.positions - 1;
  auto live = [&](int64_t r) {
    if (r >= rows) return false;
    const int b = static_cast<int>(r % a.rows.batch);
    const int j = static_cast<int>(r / a.rows.batch);
    const int rej = *static_cast<volatile int32_t*>(a.rejected + b);
    return j <= min(valid_drafts(a.num_valid, b, k), k + 1 - rej);
  };
  for (;;) {
    if (q.open) {
      // what was live when the rows were taken may be known rejected now
      q.open &= __ballot_sync(SG_FULL_MASK, live(q.base + lane_id()));
      if (q.open) {
        const int i = __ffs(q.open) - 1;
        q.open &= q.open - 1;
        return q.base + i;
      }
    }
    int at = 0;
    if (lane_id() == 0) at = atomicAdd(a.taken, q.step);
    q.base = __shfl_sync(SG_FULL_MASK, at, 0);
    if (q.base >= rows) return -1;
    q.open = __ballot_sync(SG_FULL_MASK,
                           lane_id() < q.step && live(q.base + lane_id()));
    const int n = __popc(q.open);
    if (n == 0) q.step = min(32, 2 * q.step);
    if (n > 1) q.step = max(1, q.step / 2);
  }
}

// Exact weights of a row's kept values, without token `skip`, from the blocks'
// shares: cluster_draw's source. Weights are formed only where a vector holds
// such a value.
template <class T>
struct KeptShare {
  static constexpr int E = Share<T>::E;
  const Share<T>& sh;
  float low;
  int64_t skip;

  __device__ __forceinline__ int64_t first(int v) const { return sh.first(v); }
  __device__ __forceinline__ Span span(int w, int n) const {
    const Span block = span_of(sh.nv, w / kCWarps, n / kCWarps);
    Span s = span_of(block.v1 - block.v0, w % kCWarps, kCWarps);
    s.v0 += block.v0;
    s.v1 += block.v0;
    return s;
  }
  __device__ __forceinline__ double value_weight(float x) const {
    if (!(x >= low)) return 0.0;
    return x == sh.m ? 1.0 : sh.weight(x);
  }
  __device__ __forceinline__ void vec(int v, int, double* w) const {
    const uint4 raw[1] = {sh.buf[v - sh.v0]};
    float x[E];
    Raw<T>::unpack(raw[0], x);
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = 0.0;
    if (!(Raw<T>::vec_max(raw) >= low)) return;
    const int64_t at = first(v);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (at + e != skip) w[e] = value_weight(x[e]);
  }
  __device__ __forceinline__ double sum(int v, int end, int step) const {
    double s = 0.0;
    for (; v < end; v += step) {
      const uint4 raw[1] = {sh.buf[v - sh.v0]};
      if (!(Raw<T>::vec_max(raw) >= low)) continue;
      double w[E];
      vec(v, end, w);
#pragma unroll
      for (int e = 0; e < E; ++e) s += w[e];
    }
    return s;
  }
};

template <class T>
__global__ void __launch_bounds__(kFThreads, kStatBlocks)
    stat_rows_kernel(RowArgs a) {
  static_assert(kFThreads == kCThreads, "cluster_draw's blocks");
  const auto cl = cooperative_groups::this_cluster();
  __shared__ RowShared rs;
  __shared__ DrawShared ds;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  FilterShared* fs = reinterpret_cast<FilterShared*>(row_smem);
  uint4* buf = row_smem + (sizeof(FilterShared) + 15) / 16;
  fill_exp_table(rs.tab);
  if (threadIdx.x == 0) rs.top = 0;
  const int cs = static_cast<int>(cl.num_blocks());
  const bool leader = cl.block_rank() == 0;
  const int k = a.rows.positions - 1;
  RowQueue queue{0, 0u, 1};
  cl.sync();  // every block runs before any writes into another
  for (;;) {
    if (leader && warp_id() == 0) {
      const int64_t r = next_row(a, queue);
      if (lane_id() < cs)
        *cl.map_shared_rank(&rs.next, lane_id()) = static_cast<int32_t>(r);
    }
    cl.sync();
    const int32_t r = rs.next;
    if (r < 0) return;  // every block of the cluster leaves here
    const int b = r % a.rows.batch;
    const int j = r / a.rows.batch;
    const Setting set = setting_of(a.set, b);
    const T* row = row_ptr<T>(a.rows, b, j);
    Share<T> sh(row, a.rows.vocab);
    const Kept kept = keep_row(cl, sh, buf, set, a.guard, rs, *fs);
    // Every block comes to the same verdict. The token that follows if the
    // draft is not accepted is drawn while the row is at hand.
    const int n = valid_drafts(a.num_valid, b, k);
    const float* urow = a.uniforms + static_cast<int64_t>(b) * (k + 1);
    const int32_t x = j < n ? a.draft[static_cast<int64_t>(b) * k + j] : -1;
    RowStat st{kept.arg, 0};
    if (kept.arg >= 0) {
      const bool greedy = !(set.t > 0.0f);
      const bool inside = x >= 0 && x < a.rows.vocab;
      const double u = inside ? urow[j] : 0.0f;
      if (greedy) {
        st.accept = inside && x == kept.arg && u < 1.0;
      } else {
        KeptShare<T> src{sh, kept.low, x};
        if (inside)
          st.accept =
              u < src.value_weight(canon(to_f32(row[x]))) / kept.z;
        if (!st.accept) {
          st.token = cluster_draw(cl, src, urow[k], ds);
          if (st.token < 0) {  // nothing but the rejected token
            src.skip = -1;
            st.token = cluster_draw(cl, src, urow[k], ds);
          }
        }
      }
    }
    if (leader && threadIdx.x == 0) {
      a.stats[static_cast<int64_t>(b) * (k + 1) + j] = st;
      if (!st.accept && j < k) atomicMax(a.rejected + b, k + 1 - j);
    }
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Blocks a row is split over: shares of at most `share` bytes, but enough
// blocks to fill the machine where rows are few. 32 KiB where rows are
// written; 64 KiB for the statistics, whose passes cost every block much the
// same whatever its share (128 x 33 rows of 128256 bf16, top-k and top-p:
// 371 us against 504, and 566 with 128 KiB; not measured with few rows).
static int row_cluster(const sg_rows& r, int64_t share) {
  const int64_t rows = static_cast<int64_t>(r.batch) * r.positions;
  const int64_t bytes = r.vocab * (r.dtype == SG_F32 ? 4 : 2);
  int cs = 1;
  while (cs < kMaxCluster &&
         (bytes > cs * share || (rows * cs < 148 && bytes > cs * 4096)))
    cs *= 2;
  return cs;
}

template <class Kernel>
static int launch_rows(Kernel* kernel, RowArgs& a, bool filter, int64_t share,
                       int64_t most, int* cache, cudaStream_t st) {
  const int cs = row_cluster(a.rows, share);
  const int elems = a.rows.dtype == SG_F32 ? 4 : 8;
  a.guard = guard_of(a.rows.vocab, 4 * kFThreads * cs * elems);
  const int64_t vecs = ceil_div(ceil_div(a.rows.vocab + elems - 1, elems), cs);
  const int64_t bytes =
      16 * vecs + (filter ? (sizeof(FilterShared) + 15) / 16 * 16 : 0);
  if (bytes > 200 * 1024) return SG_ERR_UNSUPPORTED;
  // 2 KiB more: the static shared memory counts towards the same limit
  static_assert(sizeof(RowShared) + sizeof(DrawShared) <= 2048, "");
  const int rc =
      ensure_dyn_smem(kernel, static_cast<size_t>(bytes) + 2048, cache);
  if (rc != SG_OK) return rc;
  const int64_t rows = static_cast<int64_t>(a.rows.batch) * a.rows.positions;
  if (rows > INT32_MAX / kMaxCluster) return SG_ERR_UNSUPPORTED;
  const int64_t clusters = std::min(rows, most / cs);
  return launch_after(kernel, static_cast<unsigned>(clusters * cs), kFThreads,
                      cs, a, st, static_cast<size_t>(bytes));
}

template <class T>
static int write_rows(RowArgs& a, bool filter, cudaStream_t st) {
  static int cache[2][64];
  return filter ? launch_rows(kept_rows_kernel<T>, a, true, 32768,
                              INT32_MAX, cache[1], st)
                : launch_rows(soft_rows_kernel<T>, a, false, 32768,
                              INT32_MAX, cache[0], st);
}

template <class T>
static int stat_rows(RowArgs& a, cudaStream_t st) {
  static int cache[64];
  return launch_rows(stat_rows_kernel<T>, a, true, 65536,
                     kStatBlocks * 148, cache, st);
}

int launch_row_stats(const sg_rows& rows, const sg_sampling& set,
                     const int32_t* draft, const int32_t* num_valid,
                     const float* uniforms, RowStat* stats, int32_t* rejected,
                     int32_t* taken, cudaStream_t st) {
  RowArgs a{};
  a.rows = rows;
  a.set = set;
  a.draft = draft;
  a.num_valid = num_valid;
  a.uniforms = uniforms;
  a.stats = stats;
  a.rejected = rejected;
  a.taken = taken;
  switch (rows.dtype) {
    case SG_F32: return stat_rows<float>(a, st);
    case SG_BF16: return stat_rows<__nv_bfloat16>(a, st);
    default: return stat_rows<__half>(a, st);
  }
}

}  // namespace sg

using namespace sg;

extern "C" int sg_target_probs(const sg_rows* logits,
                               const sg_sampling* sampling, float* out,
                               sg_stream_t stream) {
  NvtxScope nvtx("sg_target_probs");
  const int rc = check_rows(logits, false);
  if (rc != SG_OK) return rc;
  if (!sampling || logits->row_start) return SG_ERR_INVALID;
  if (logits->batch == 0 || logits->positions == 0) return SG_OK;
  if (!out) return SG_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  RowArgs a{};
  a.rows = *logits;
  a.set = *sampling;
  a.out = out;
  const bool filter = has_filter(*sampling);
  switch (logits->dtype) {
    case SG_F32: return write_rows<float>(a, filter, st);
    case SG_BF16: return write_rows<__nv_bfloat16>(a, filter, st);
    default: return write_rows<__half>(a, filter, st);
  }
}
