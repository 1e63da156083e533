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
constexpr int kKeptBlocks = 3;  // and with filters
constexpr int kBins = 2048;
constexpr int kList = 2048;      // candidates the first block can hold
constexpr int kOwn = kList / kFThreads;
constexpr double kFix = 17592186044416.0;  // 2^44: unit of candidates' sums

// What a cluster finds for a row.
struct Kept {
  double z;   // sum of the kept weights
  float m;    // largest value
  float low;  // smallest kept value
  int32_t arg;
};

struct RowShared {
  float m[kMaxCluster];  // slots the cluster's blocks write into each other
  int32_t arg[kMaxCluster];
  double s[kMaxCluster];
  int32_t next;
  float redf[kFWarps];
  int32_t redi[kFWarps];
  uint32_t redu[kFWarps];
  double red[32];
  double tab[kExpTable];
};

struct FilterShared {
  uint32_t hist[kBins];  // this block's counts
  uint32_t tot[kBins];   // first block: the row's
  uint32_t list[kList];  // this block's candidates (order keys)
  int32_t listed;
  int32_t n[kMaxCluster];
  double a[kMaxCluster];
  uint64_t redl[kFWarps];
  // the plan: the bin of the k-th value, the values in bins before it, and
  // the bins [p0, p1] in which top-p's border is looked for
  int32_t bk, above, p0, p1;
  // the result
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
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(SG_FULL_MASK, v, o);
  __syncthreads();
  if (lane_id() == 0) red[warp_id()] = v;
  __syncthreads();
  uint64_t s = 0;
#pragma unroll
  for (int i = 0; i < kFWarps; ++i) s += red[i];
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
  // the last takes everything beyond, NaN and -inf too. Monotone in x.
  __device__ __forceinline__ int bin(float x) const {
    const float t = fminf((m - x) * bin_scale, kBins - 1.0f);
    return __float_as_uint(t + 8388608.0f) & (kBins - 1);
  }
  __device__ __forceinline__ double weight(float x) const {
    return weight64(x, m64, scale64, tab);
  }
  // f(value, row index) for this thread's values; the vectors' order is the
  // same in every pass. Values outside the row are left out.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x; i < n; i += kFThreads) {
      float x[E];
      Raw<T>::unpack(buf[i], x);
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
    *cl.map_shared_rank(&rs.arg[rank], static_cast<int>(threadIdx.x)) =
        static_cast<int32_t>(not_all);
  }
  cl.sync();
  any = not_all = 0;
  for (int i = 0; i < cs; ++i) {
    any |= static_cast<uint32_t>(fs.n[i]);
    not_all |= static_cast<uint32_t>(rs.arg[i]);
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

// The smallest kept value and the kept mass of a row with top-k (k > 0) or
// top-p (0 < p < 1) or both; left in fs.low and fs.z of every block.
//
// One pass counts the values in bins; the first block finds the bin of the
// k-th value from the counts, and from counts times the bins' middle weights
// the bin top-p's border should lie in. A second pass sums the weights
// ahead of those bins in 64 bits and lists the values inside them, from
// which the first block takes both borders exactly: top-k by counting,
// top-p by 64-bit sums, whose order does not matter (fixed point). Whether
// the border lies in the bins looked at shows in the exact sums; if not, or
// if the list is too short, bisect_row finds it.
template <class T>
__device__ void filter_row(const cooperative_groups::cluster_group& cl,
                           Share<T>& sh, int32_t k, float p, RowShared& rs,
                           FilterShared& fs) {
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int tid = static_cast<int>(threadIdx.x);
  const bool with_p = p < 1.0f;
  // 32 octaves of weight or 32 units of logits, whichever is shorter
  const float range = fminf(32.0f / sh.scale, 32.0f);
  sh.bin_scale = fminf((kBins - 1.0f) / range, 1e30f);

  // fs.hist is zero (cleared by the caller before its barrier)
  sh.each([&](float x, int64_t) {
    const int b = sh.bin(x);
    if (b < kBins - 1) atomicAdd(&fs.hist[b], 1u);
  });
  if (tid == 0) fs.listed = 0;
  cl.sync();
  {  // the row's counts, a slice of bins a block, into the first block
    const int slice = kBins / cs;
    uint32_t* tot = cl.map_shared_rank(fs.tot, 0);
    for (int i = rank * slice + tid; i < (rank + 1) * slice; i += kFThreads) {
      uint32_t c = 0;
      for (int r = 0; r < cs; ++r) c += cl.map_shared_rank(fs.hist, r)[i];
      tot[i] = c;
    }
  }
  cl.sync();
  if (rank == 0) {
    constexpr int kPer = kBins / kFThreads;
    const float octaves = sh.scale / sh.bin_scale;  // a bin's
    int32_t c[kPer];
    float w[kPer];
    int32_t cnt = 0;
    float mass = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = tid * kPer + i;
      c[i] = static_cast<int32_t>(fs.tot[b]);
      w[i] = exp2_fast(-static_cast<float>(b) * octaves);
      cnt += c[i];
      mass += static_cast<float>(c[i]) * w[i];
    }
    int32_t ci = warp_incl_scan(cnt);
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
      fs.bk = kBins;  // top-k off: every bin lies ahead of it
      fs.above = 0;
      fs.p0 = kBins;
      rs.red[0] = 0.0;
    }
    __syncthreads();
    int32_t c0 = ci - cnt;
    float m0 = mi - mass;
    float all = 0.0f;
    for (int i = 0; i < kFWarps; ++i) {
      if (i < warp_id()) {
        c0 += rs.redi[i];
        m0 += rs.redf[i];
      }
      all += rs.redf[i];
    }
    if (k > 0) {
      int32_t run = c0;
      float mr = m0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int b = tid * kPer + i;
        const bool last = b == kBins - 1;
        if (run < k && (k <= run + c[i] || last)) {
          fs.bk = b;
          fs.above = run;
          rs.red[0] = mr + static_cast<float>(k - run) * w[i];
        }
        run += c[i];
        mr += static_cast<float>(c[i]) * w[i];
      }
      __syncthreads();
      all = static_cast<float>(rs.red[0]);
    }
    if (with_p) {
      const float need = p * all;
      float incl = m0;
      int at = kBins;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        incl += static_cast<float>(c[i]) * w[i];
        if (incl >= need) at = min(at, tid * kPer + i);
      }
      if (at < kBins) atomicMin(&fs.p0, at);
      __syncthreads();
    }
    const int bk = fs.bk;
    const int mid = min(min(fs.p0, kBins - 1), bk);
    const int above = fs.above;
    __syncthreads();
    if (tid < cs) {
      FilterShared* o = cl.map_shared_rank(&fs, tid);
      o->bk = bk;
      o->above = above;
      o->p0 = with_p ? max(mid - 1, 0) : kBins;
      o->p1 = with_p ? min(mid + 1, min(bk, kBins - 1)) : -1;
    }
  }
  cl.sync();

  // exact sums ahead of the bins looked at, and the values inside them
  const int bk = fs.bk, p0 = fs.p0, p1 = fs.p1;
  double s = 0.0, a = 0.0;
  sh.each([&](float x, int64_t) {
    const int b = sh.bin(x);
    if (b < bk) {
      const double w = sh.weight(x);
      s += w;
      if (b < p0) a += w;
    }
    if (b == bk || (b >= p0 && b <= p1)) {
      const int at = atomicAdd(&fs.listed, 1);
      if (at < kList) fs.list[at] = order_key(canon(x));
    }
  });
  s = block_sum64(s, rs.red);
  if (with_p) a = block_sum64(a, rs.red);
  __syncthreads();
  if (tid == 0) {
    *cl.map_shared_rank(&rs.s[rank], 0) = s;
    *cl.map_shared_rank(&fs.a[rank], 0) = a;
    *cl.map_shared_rank(&fs.n[rank], 0) = fs.listed;
  }
  cl.sync();
  if (rank == 0) {
    int n = 0;
    bool fits = true;
    s = a = 0.0;
    for (int r = 0; r < cs; ++r) {
      n += fs.n[r];
      fits = fits && fs.n[r] <= kList;
      s += rs.s[r];
      a += fs.a[r];
    }
    bool done = fits && n <= kList;
    float low = -CUDART_INF_F;
    double z = s;
    if (done) {
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
              __double2ll_rn(sh.weight(x) * kFix));
        }
      }
      // keys' differing bits among a set; the greatest key that `enough`
      // accepts, and the set's smallest key where none but it does
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
      uint32_t tk = 0;
      if (k > 0) {
        const int32_t want = k - fs.above;
        tk = border(in_k, [&](uint32_t from) {
          int32_t c = 0;
#pragma unroll
          for (int i = 0; i < kOwn; ++i) c += in_k[i] && key[i] >= from;
          return block_sum_i32(c, rs.redi) >= want;
        });
        uint64_t f = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          f += in_k[i] && key[i] >= tk ? w[i] : 0;
          in_p[i] = in_p[i] && key[i] >= tk;
        }
        z += static_cast<double>(block_sum_u64(f, fs.redl)) / kFix;
        low = key_value(tk);
      }
      if (with_p) {
        const double need = static_cast<double>(p) * z;
        auto mass = [&](uint32_t from) {
          uint64_t f = 0;
#pragma unroll
          for (int i = 0; i < kOwn; ++i)
            f += in_p[i] && key[i] >= from ? w[i] : 0;
          return a + static_cast<double>(block_sum_u64(f, fs.redl)) / kFix;
        };
        done = a < need && mass(0) >= need;
        if (done) {
          const uint32_t t =
              border(in_p, [&](uint32_t from) { return mass(from) >= need; });
          low = key_value(t);
          z = mass(t);
        }
      }
    }
    if (tid < cs) {
      FilterShared* o = cl.map_shared_rank(&fs, tid);
      o->low = low;
      o->z = z;
      o->done = done;
    }
  }
  cl.sync();
  if (!fs.done) bisect_row(cl, sh, k, p, rs, fs);
}

// ---------------------------------------------------------------------------
// a row's statistics
// ---------------------------------------------------------------------------
template <class T>
__device__ Kept keep_row(const cooperative_groups::cluster_group& cl,
                         Share<T>& sh, uint4* buf, const Setting& set,
                         RowShared& rs, FilterShared& fs) {
  constexpr int U = 8;
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int tid = static_cast<int>(threadIdx.x);
  const Span sp = span_of(sh.nv, rank, cs);
  sh.buf = buf;
  sh.v0 = sp.v0;
  sh.n = sp.v1 - sp.v0;
  sh.tab = rs.tab;
  for (int i = tid; i < kBins; i += kFThreads) fs.hist[i] = 0;
  float m = -CUDART_INF_F;
  for (int i0 = tid; i0 < sh.n; i0 += U * kFThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = load_vec(sh, sp.v0 + i0 + u * kFThreads, sp.v1);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * kFThreads < sh.n) buf[i0 + u * kFThreads] = raw[u];
    m = fmaxf(m, Raw<T>::vec_max(raw));
  }
  m = warp_max(canon(m));
  if (lane_id() == 0) rs.redf[warp_id()] = m;
  __syncthreads();
  for (int i = 0; i < kFWarps; ++i) m = fmaxf(m, rs.redf[i]);
  if (tid < cs) *cl.map_shared_rank(&rs.m[rank], tid) = m;
  cl.sync();
  Kept kept{0.0, -CUDART_INF_F, -CUDART_INF_F, -1};
  for (int i = 0; i < cs; ++i) kept.m = fmaxf(kept.m, rs.m[i]);
  if (!(kept.m > -CUDART_INF_F)) return kept;  // no mass
  sh.m = kept.m;
  sh.m64 = static_cast<double>(kept.m);
  kept.arg = 0;
  if (!(set.t > 0.0f)) {  // greedy: the first largest value
    int32_t at = INT32_MAX;
    sh.each([&](float x, int64_t i) {
      if (x == kept.m) at = min(at, static_cast<int32_t>(i));
    });
    at = __reduce_min_sync(SG_FULL_MASK, at);
    if (lane_id() == 0) rs.redi[warp_id()] = at;
    __syncthreads();
    for (int i = 0; i < kFWarps; ++i) at = min(at, rs.redi[i]);
    if (tid < cs) *cl.map_shared_rank(&rs.arg[rank], tid) = at;
    cl.sync();
    for (int i = 0; i < cs; ++i) at = min(at, rs.arg[i]);
    kept.arg = at;
    kept.z = 1.0;
    return kept;
  }
  sh.scale = scale_of(set.t);
  sh.scale64 = scale64_of(set.t);
  const int32_t k = set.k > 0 && set.k < sh.v ? set.k : 0;
  const float p = set.p < 1.0f ? set.p : 1.0f;
  if (kept.m == CUDART_INF_F || !(p > 0.0f)) {
    // only the largest value has mass, or is kept
    int32_t c = 0;
    sh.each([&](float x, int64_t) { c += x == kept.m; });
    c = block_sum_i32(c, rs.redi);
    if (tid < cs) *cl.map_shared_rank(&rs.arg[rank], tid) = c;
    cl.sync();
    for (int i = 0; i < cs; ++i) kept.z += rs.arg[i];
    kept.low = kept.m;
    return kept;
  }
  if (k > 0 || p < 1.0f) {
    filter_row(cl, sh, k, p, rs, fs);
    kept.low = fs.low;
    kept.z = fs.z;
    return kept;
  }
  double s = 0.0;
  sh.each([&](float x, int64_t) { s += sh.weight(x); });
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
  float* out;  // [B, positions, V]
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
  if (m == CUDART_INF_F || t == CUDART_INF_F) {
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
  __syncthreads();
  cl.sync();  // every block runs before any writes into another
  const int64_t r = blockIdx.x / cl.num_blocks();
  const int b = static_cast<int>(r / a.rows.positions);
  const int j = static_cast<int>(r % a.rows.positions);
  const Setting set = setting_of(a.set, b);
  Share<T> sh(row_ptr<T>(a.rows, b, j), a.rows.vocab);
  const Kept kept = keep_row(cl, sh, buf, set, rs, *fs);
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
struct SoftShared {
  SpanSum part[kFWarps];
  uint32_t top;
  SpanSum slot[kMaxCluster];  // the cluster's blocks
};

template <class T>
__global__ void __launch_bounds__(kFThreads, kSoftBlocks)
    soft_rows_kernel(RowArgs a) {
  constexpr int U = 4;
  const auto cl = cooperative_groups::this_cluster();
  __shared__ SoftShared ss;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cs = static_cast<int>(cl.num_blocks());
  const int rank = static_cast<int>(cl.block_rank());
  const int tid = static_cast<int>(threadIdx.x);
  if (tid == 0) ss.top = 0;
  cl.sync();  // every block runs before any writes into another
  const int64_t r = blockIdx.x / cs;
  const int b = static_cast<int>(r / a.rows.positions);
  const int j = static_cast<int>(r % a.rows.positions);
  const float t = setting_of(a.set, b).t;
  const bool greedy = !(t > 0.0f);
  Share<T> sh(row_ptr<T>(a.rows, b, j), a.rows.vocab);
  const Span sp = span_of(sh.nv, rank, cs);
  sh.buf = row_smem;
  sh.v0 = sp.v0;
  sh.n = sp.v1 - sp.v0;
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
        row_smem[i0 + u * kFThreads + tid] = raw[u];
    auto index = [&](int u) {
      return sh.first(sp.v0 + i0 + u * kFThreads + tid);
    };
    if (greedy)
      take_vecs<T, true, kNoSum>(raw, index, f, &ss.top, st);
    else
      take_vecs<T, false, kFineSum>(raw, index, f, &ss.top, st);
  }
  st.s = warp_sum64(st.s);
  if (lane_id() == 0) ss.part[warp_id()] = SpanSum{st.s, st.m, st.arg};
  __syncthreads();
  if (warp_id() == 0) {
    const SpanSum p = join_sums(ss.part, kFWarps, t);
    if (lane_id() < cs) *cl.map_shared_rank(&ss.slot[rank], lane_id()) = p;
  }
  cl.sync();
  const SpanSum row = join_sums(ss.slot, cs, t);
  float* orow = a.out + r * a.rows.vocab;
  if (greedy || !(row.m > -CUDART_INF_F))
    write_one_hot(sh, orow, row.m > -CUDART_INF_F ? row.arg : -1);
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

template <class T>
__global__ void __launch_bounds__(kFThreads, kKeptBlocks) stat_rows_kernel(RowArgs a) {
  const auto cl = cooperative_groups::this_cluster();
  __shared__ RowShared rs;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  FilterShared* fs = reinterpret_cast<FilterShared*>(row_smem);
  uint4* buf = row_smem + (sizeof(FilterShared) + 15) / 16;
  fill_exp_table(rs.tab);
  __syncthreads();
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
    const Kept kept = keep_row(cl, sh, buf, set, rs, *fs);
    if (leader && threadIdx.x == 0) {
      RowStat st;
      st.z = kept.z;
      st.m = kept.m;
      st.arg = kept.arg;
      st.low = kept.low;
      st.accept = 0;
      const int32_t x =
          j < k ? a.draft[static_cast<int64_t>(b) * k + j] : -1;
      if (x >= 0 && x < a.rows.vocab && kept.arg >= 0) {
        const double u = a.uniforms[static_cast<int64_t>(b) * (k + 1) + j];
        if (!(set.t > 0.0f)) {
          st.accept = x == kept.arg && u < 1.0;
        } else {
          const float l = canon(to_f32(row[x]));
          double w = 0.0;
          if (l >= kept.low)
            w = l == kept.m ? 1.0
                            : weight64(l, static_cast<double>(kept.m),
                                       scale64_of(set.t), rs.tab);
          st.accept = u < w / kept.z;
        }
      }
      a.stats[static_cast<int64_t>(b) * (k + 1) + j] = st;
      if (!st.accept && j < k) atomicMax(a.rejected + b, k + 1 - j);
    }
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Blocks a row is split over: shares of at most 32 KiB (more blocks on an
// SM), but enough blocks to fill the machine where rows are few.
static int row_cluster(const sg_rows& r) {
  const int64_t rows = static_cast<int64_t>(r.batch) * r.positions;
  const int64_t bytes = r.vocab * (r.dtype == SG_F32 ? 4 : 2);
  int cs = 1;
  while (cs < kMaxCluster &&
         (bytes > cs * 32768 || (rows * cs < 148 && bytes > cs * 4096)))
    cs *= 2;
  return cs;
}

template <class Kernel>
static int launch_rows(Kernel* kernel, const RowArgs& a, bool filter,
                       int64_t most, int* cache, cudaStream_t st) {
  const int cs = row_cluster(a.rows);
  const int elems = a.rows.dtype == SG_F32 ? 4 : 8;
  const int64_t vecs = ceil_div(ceil_div(a.rows.vocab + elems - 1, elems), cs);
  const int64_t bytes =
      16 * vecs + (filter ? (sizeof(FilterShared) + 15) / 16 * 16 : 0);
  if (bytes > 200 * 1024) return SG_ERR_UNSUPPORTED;
  // 1 KiB more: the static shared memory counts towards the same limit
  const int rc =
      ensure_dyn_smem(kernel, static_cast<size_t>(bytes) + 1024, cache);
  if (rc != SG_OK) return rc;
  const int64_t rows = static_cast<int64_t>(a.rows.batch) * a.rows.positions;
  if (rows > INT32_MAX / kMaxCluster) return SG_ERR_UNSUPPORTED;
  const int64_t clusters = std::min(rows, most / cs);
  return launch_after(kernel, static_cast<unsigned>(clusters * cs), kFThreads,
                      cs, a, st, static_cast<size_t>(bytes));
}

template <class T>
static int write_rows(const RowArgs& a, bool filter, cudaStream_t st) {
  static int cache[2][64];
  return filter ? launch_rows(kept_rows_kernel<T>, a, true, INT32_MAX,
                              cache[1], st)
                : launch_rows(soft_rows_kernel<T>, a, false, INT32_MAX,
                              cache[0], st);
}

template <class T>
static int stat_rows(const RowArgs& a, cudaStream_t st) {
  static int cache[64];
  return launch_rows(stat_rows_kernel<T>, a, true, kKeptBlocks * 148, cache,
                     st);
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
