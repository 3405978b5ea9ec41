// One token per row of logits: temperature, top-k, top-p, min-p, given
// uniforms.  The reference decodes greedily (argmax in PipelineRuntime.generate,
// helm/runtime/pipeline_runtime.py:300-338); sampling has no counterpart.
//
// Definition.  Candidates are ordered by (logit descending, index ascending);
// w_i = exp((l_i - l_max) / T).
//   top-k: the first k.   top-p: of those, the shortest prefix whose weights
//   reach top_p of their sum.   min-p: w_i >= min_p.
//   token = the smallest index i whose running sum, in index order over what is
//   left, exceeds u times the sum of what is left.   T = 0: the first candidate.
// NaN logits count as -inf; a row without a finite (or +inf) logit gives -1.
//
// A token is right or wrong, so every comparison is made in integers that no
// order of summation changes: w is computed in fp64 (relative error < 1e-13,
// 64-entry table of 2^(j/64) and a quartic) and rounded to a multiple of 2^-44;
// sums of up to 2^18 of those fit 64 bits exactly.  Two runs, grids or cluster
// sizes give the same token.
//
// With few rows a row is held by one cluster, its logits in the CTAs' shared
// memory.  With at least as many rows as SMs one CTA does a row, reading it from
// L2 once per pass: no cluster barriers, and two rows share an SM, one computing
// while the other waits (256 x 151936 bf16, every filter mixed: 184 -> 118 us).
// Bound by instructions: some 30 per logit for its weight, 10 for a bin; a long bf16
// row looks its weights up in a table of its possible values instead.  A call also
// waits for its heaviest rows, each one CTA from start to end: 256 rows of top-p
// alone take 137 us, of top-k alone 78, without a filter 80.
//
// A filter needs its last kept candidate.  A histogram of counts over 2048 equal
// steps of the logit (equal steps spread a bell-shaped row over the bins; digits
// of its bit pattern would not) says in which bin it falls: exactly for top-k, and
// for top-p by an estimate from counts times the weight at the bins' centres, good
// to a bin or two among many candidates (a window of 8 bins is kept around it, a
// margin of 64 candidates where they are few).  Then
//   few: when at most 1024 candidates lie in that bin (window) or above, they are
//        sorted in one CTA, which finishes the row; the others are done;
//   many: one pass in fp64 sums the weights above the window, per warp, and each
//        bin's of the window; only the candidates of the bin that the sums point
//        to are sorted.  The sums serve the draw as well.
// For a small k the histogram need not see every logit: the threads' own largest
// ones bound the k-th from below (k of them at or above a bin are k candidates),
// and the candidates from that bin up are few.
// A long bf16 row counts its logits by value instead (by_value), which says exactly
// where the filters cut.
// Whatever these cannot decide (more than 1024 equal logits at the cut, say) is
// bisected over the order of candidates, pass by pass.
#include <cooperative_groups.h>

#include <cstddef>
#include <type_traits>

#include "common.cuh"

namespace helm {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampThreads = 512;
constexpr int kSampWarps = kSampThreads / 32;
constexpr int kSampBins = 2048;
constexpr int kSampWindow = 8;               // bins around the estimate of top-p's cut
constexpr int kSampMargin = 64;              // candidates beyond it that few-candidate rows sort too
constexpr int kSampList = 1024;              // candidates sorted in one CTA
constexpr int kSampMaxVocab = 1 << 18;       // 2^18 weights of 2^44 stay below 2^63
constexpr int kSampSliceBytes = 160 * 1024;  // most logits a CTA can hold
constexpr int kSampSliceGoal = 80 * 1024;    // two CTAs an SM: one loads while the other computes
constexpr int kSampMaxCluster = 8;
// Table of weights (bf16): sixteen binades of magnitudes of either sign, and an
// entry for what lies beyond.
constexpr int kSampLutSide = 2048 + 1;
constexpr int kSampLutBytes = 2 * kSampLutSide * (8 + 4);  // weights and counts
constexpr int kSampLutLogits = 65536;  // of a row that has the table (launch_sample says why)
typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* ids;
  float* logprobs;
  int vocab, slice;  // logits of a row and of a CTA's slice
  int tabled;        // room was given for the table of weights
};

// 2^(j/64), j = 0 .. 63, rounded to nearest
__device__ const double kExp2Table[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0,
    0x1.0874518759bc8p+0, 0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0,
    0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0, 0x1.172b83c7d517bp+0,
    0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0,
    0x1.2d285a6e4030bp+0, 0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0,
    0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0, 0x1.3dea64c123422p+0,
    0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0,
    0x1.56f4736b527dap+0, 0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0,
    0x1.6247eb03a5585p+0, 0x1.6623882552225p+0, 0x1.6a09e667f3bcdp+0,
    0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0,
    0x1.868d99b4492edp+0, 0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0,
    0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0, 0x1.9c49182a3f090p+0,
    0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0,
    0x1.bcc1e904bc1d2p+0, 0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0,
    0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0, 0x1.d5818dcfba487p+0,
    0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0,
    0x1.fa7c1819e90d8p+0,
};

// w = exp(x) in units of 2^-44 for -31.4 < x <= 0, given y = x * 64 / ln 2, by Tang's
// table-driven method (ACM Trans. Math. Softw. 15, 1989) with a Taylor tail:
// 2^(j/64) from the table, e^r = 2^(y/64 - k/64) by its series to the fourth
// power (|r| <= ln2/128, next term < 4e-14), rounded to nearest by adding 2^52.
// No branches: the caller's loop interleaves several of these chains, which is
// what fp64's latency needs.
__device__ __forceinline__ u64 weight_fixed(double y, const double* table) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the integer
  constexpr double kStep = 0.0108304246962491454596;  // ln2 / 64
  const double k = y + kMagic;
  const int n = static_cast<int>(__double_as_longlong(k));
  const double r = y - (k - kMagic);
  double p = fma(r, kStep * kStep * kStep * kStep / 24.0, kStep * kStep * kStep / 6.0);
  p = fma(p, r, kStep * kStep / 2.0);
  p = fma(p, r, kStep);
  p = fma(p, r, 1.0);
  p *= table[n & 63];
  p = __longlong_as_double(__double_as_longlong(p) +
                           (static_cast<long long>(44 + (n >> 6)) << 52));
  return static_cast<u64>(__double_as_longlong(p + 4503599627370496.0)) & 0xfffffffffffffull;
}

// Order-preserving bits of a float (NaN was replaced; -0 counts as +0), and back.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Larger = earlier in the order of candidates.
__device__ __forceinline__ u64 order_of(float f, int index) {
  return (static_cast<u64>(order_key(f)) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}

template <typename V, typename Op>
__device__ __forceinline__ V warp_reduce(V v, Op op) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
struct AddOp {
  template <typename V>
  __device__ __forceinline__ V operator()(V a, V b) const {
    return a + b;
  }
};

struct __align__(16) SampleShared {
  double table[64];
  float warp_max[kSampWarps], warp_min[kSampWarps];
  u64 warp_a[kSampWarps], warp_b[kSampWarps];
  double warp_d[kSampWarps];
  // published to the cluster
  float pub_max, pub_min;
  u64 pub_a, pub_b;
  uint32_t pub_n;
  // results, the same for every CTA of the cluster
  int bin_k, bin_p;               // bins of the filters' last candidates (bin_p: estimate)
  uint32_t upto_k, in_k;          // candidates up to and in bin_k
  uint32_t upto_p, upto_w, upto_f;  // up to bin_p, up to the window's end, up to bin_f
  int bin_f;                      // bin with kSampMargin candidates beyond bin_p
  uint32_t win_lo[kSampWindow], win_hi[kSampWindow];  // weights of the window's bins
  int win_bin;                    // the window's bin that the weights point to
  u64 win_over;                   // weight above it
  uint32_t list_n;        // rank 0: candidates in its list
  u64 last, last_mass;    // rank 0: last kept candidate, weight up to it
  __align__(16) uint32_t hist[kSampBins];  // read four at a time
  u64 list[kSampList], weight[kSampList];
};

static_assert(offsetof(SampleShared, hist) % 16 == 0, "");

template <typename T, bool kResident>
struct Sampler {
  static constexpr int kVec = 16 / sizeof(T);
  const SampleArgs& a;
  SampleShared& s;
  const T* slice;    // in shared memory, or the row itself
  cg::cluster_group cluster;
  int base, n;       // first index and number of logits of this CTA
  int vecs;          // 16-byte groups of its slice (padded with -inf)
  int ranks, rank, lane, warp;
  float top;         // largest logit of the row
  double top_finite;
  double inv_temp, scale;  // z = (l - l_max) inv_temp, y = (l - l_max) scale
  float bin_scale;
  float least_logit;  // below it weights round to 0
  u64* lut;           // weights by bf16 code, once `tabled`
  int lut_base;       // magnitude code of its first entry
  bool tabled = false;

  __device__ Sampler(const SampleArgs& a_, SampleShared& s_, const T* sl)
      : a(a_), s(s_), slice(sl), cluster(cg::this_cluster()) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    ranks = static_cast<int>(cluster.num_blocks());
    rank = static_cast<int>(cluster.block_rank());
  }

  // (+inf stands for the largest finite float here: infinities share the weight)
  __device__ __forceinline__ u64 weight(float f) const {
    const double d = static_cast<double>(fminf(f, 3.402823466e38f)) - top_finite;
    const u64 w = weight_fixed(d * scale, s.table);
    return f >= least_logit ? w : 0;  // -inf is below it
  }
  // weight() of a logit, from the table where there is one: a row has a few
  // thousand bf16 values at most, and looking one up takes a third of the
  // instructions.  Magnitudes below the table's are computed; those above are of
  // logits too small to weigh, or +inf.
  __device__ __forceinline__ u64 weight_of(float f) const {
    if (!kResident && std::is_same<T, __nv_bfloat16>::value && tabled) {
      const int at = lut_entry(f);
      if (at >= 0) return lut[at];
    }
    return weight(f);
  }
  __device__ __forceinline__ int lut_entry(float f) const {  // -1: below the table
    const uint32_t u = __float_as_uint(f);
    const int d = min(static_cast<int>((u & 0x7fffffffu) >> 16) - lut_base, kSampLutSide - 1);
    return d < 0 ? -1 : d + (u >> 31 ? kSampLutSide : 0);
  }
  // smallest: the row's smallest finite logit
  __device__ void build_table(float smallest) {
    auto mag = [](float f) { return static_cast<int>((__float_as_uint(f) & 0x7fffffffu) >> 16); };
    const int most = max(mag(static_cast<float>(top_finite)), mag(fmaxf(least_logit, smallest)));
    lut_base = max(0, most + 2 - kSampLutSide);
    for (int i = threadIdx.x; i < 2 * kSampLutSide; i += kSampThreads) {
      const bool neg = i >= kSampLutSide;
      const int d = neg ? i - kSampLutSide : i;
      const float f = d < kSampLutSide - 1 ? __uint_as_float(static_cast<uint32_t>(lut_base + d) << 16)
                                           : INFINITY;
      lut[i] = weight(neg ? -f : f);
    }
    tabled = true;
    __syncthreads();
  }
  // Place on the bins' scale, 0 .. inf; bin b holds the places from b to b + 1, the
  // last bin all beyond.  (inf - inf and 0 * inf, of the largest logits: place 0.)
  __device__ __forceinline__ float place(float f) const {
    return fmaxf((top - f) * bin_scale, 0.f);
  }
  __device__ __forceinline__ static bool between(float x, int b0, int b1) {  // bins b0 .. b1
    return x >= static_cast<float>(b0) && (x < static_cast<float>(b1 + 1) || b1 == kSampBins - 1);
  }
  __device__ __forceinline__ int bin(float f) const {
    return min(kSampBins - 1, static_cast<int>(place(f)));
  }
  __device__ __forceinline__ uint4 raw(int vec) const {
    const uint4* p = reinterpret_cast<const uint4*>(slice) + vec;
    return kResident ? *p : __ldg(p);
  }
  // fn(value, index within the slice) for every logit of vectors v0, v0 + step ..
  template <typename Fn>
  __device__ __forceinline__ void each(int v0, int v1, int step, Fn fn) const {
    if (v0 >= v1) return;
    uint4 next = raw(v0);
    for (int v = v0; v < v1; v += step) {
      const uint4 now = next;
      if (v + step < v1) next = raw(v + step);
      const T* e = reinterpret_cast<const T*>(&now);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float f = to_float<T>(e[i]);
        fn(kResident || f == f ? f : -INFINITY, v * kVec + i);
      }
    }
  }
  // A warp owns a contiguous run of vectors, its lanes take turns.
  __device__ __forceinline__ int seg_vecs() const { return (vecs + kSampWarps - 1) / kSampWarps; }
  __device__ __forceinline__ int seg_begin(int w) const { return min(vecs, w * seg_vecs()); }

  // Exclusive running sums over the block, thread by thread; total to all.
  template <typename V>
  __device__ __forceinline__ V block_scan(V v, V* warp_sums, V& total) {
    V inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const V x = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += x;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    V w = lane < kSampWarps ? warp_sums[lane] : V(0), winc = w;
#pragma unroll
    for (int off = 1; off < kSampWarps; off <<= 1) {
      const V x = __shfl_up_sync(0xffffffffu, winc, off);
      if (lane >= off) winc += x;
    }
    total = __shfl_sync(0xffffffffu, winc, kSampWarps - 1);
    const V before = __shfl_sync(0xffffffffu, winc - w, warp);
    __syncthreads();
    return before + inc - v;
  }

  // Sums of a and b over the cluster.
  __device__ void cluster_sum(u64& x, u64& y) {
    x = warp_reduce(x, AddOp());
    y = warp_reduce(y, AddOp());
    if (lane == 0) {
      s.warp_a[warp] = x;
      s.warp_b[warp] = y;
    }
    __syncthreads();
    if (warp == 0) {
      x = warp_reduce(lane < kSampWarps ? s.warp_a[lane] : u64(0), AddOp());
      y = warp_reduce(lane < kSampWarps ? s.warp_b[lane] : u64(0), AddOp());
      if (lane == 0) {
        s.pub_a = x;
        s.pub_b = y;
      }
    }
    cluster.sync();
    x = y = 0;
    for (int r = 0; r < ranks; ++r) {
      const SampleShared* o = cluster.map_shared_rank(&s, r);
      x += o->pub_a;
      y += o->pub_b;
    }
    cluster.sync();  // everyone has read before the words are used again
  }

  // Descending bitonic sort of list[0 .. size), a power of two, by this CTA.
  __device__ void sort(int size) {
    const int t = threadIdx.x;
    for (int k = 2; k <= size; k <<= 1) {
      for (int j = k >> 1; j > 0; j >>= 1) {
        if (t < size / 2) {
          const int i = 2 * t - (t & (j - 1));
          const u64 x = s.list[i], y = s.list[i + j];
          if ((x < y) == ((i & k) == 0)) {
            s.list[i] = y;
            s.list[i + j] = x;
          }
        }
        // pairs less than 64 apart stay within a warp's 64 entries
        if (j > 32 || (j == 1 && k >= 64))
          __syncthreads();
        else
          __syncwarp();
      }
    }
    __syncthreads();
  }

  // Adds a candidate to rank 0's list (counted beyond its end as well).
  __device__ __forceinline__ void push(SampleShared* home, float f, int i) const {
    const uint32_t at = atomicAdd(&home->list_n, 1u);
    if (at < kSampList) home->list[at] = order_of(f, base + i);
  }

  // Rank 0: sorts its list, weighs it and leaves exclusive running sums in
  // registers: entries 2t and 2t + 1 are this thread's.
  __device__ void order_list(int count, u64 (&w)[2], u64 (&ex)[2], u64& total) {
    int size = 64;
    while (size < count) size <<= 1;
    for (int i = count + threadIdx.x; i < size; i += kSampThreads) s.list[i] = 0;
    __syncthreads();
    sort(size);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 2 * threadIdx.x + i;
      w[i] = at < count ? weight(key_value(static_cast<uint32_t>(s.list[at] >> 32))) : 0;
    }
    ex[0] = block_scan(w[0] + w[1], s.warp_a, total);
    ex[1] = ex[0] + w[0];
  }

  // The slow and general way: the order of the last candidate kept by a filter
  // that keeps candidates until their count (or weight) reaches `target`, by
  // bisection over the order itself.  `mass`: weight up to and including it.
  __device__ u64 bisect(bool by_mass, u64 target, u64& mass) {
    u64 lo = 0, hi = ~u64(0), at_lo = 0;  // the set from lo on reaches the target, from hi on not
    bool have = false;
    while (hi - lo > 1) {
      const u64 mid = lo + (hi - lo) / 2;
      u64 c = 0, m = 0;
      each(threadIdx.x, vecs, kSampThreads, [&](float f, int i) {
        if (f > -INFINITY && order_of(f, base + i) >= mid) {
          ++c;
          m += weight_of(f);
        }
      });
      cluster_sum(c, m);
      if ((by_mass ? m : c) >= target) {
        lo = mid;
        at_lo = m;
        have = true;
      } else {
        hi = mid;
      }
    }
    if (!have) {  // nothing reaches it: everything is kept
      u64 c = 0, m = 0;
      each(threadIdx.x, vecs, kSampThreads, [&](float f, int) { m += weight_of(f); });
      cluster_sum(c, m);
      at_lo = m;
    }
    mass = at_lo;
    return lo;
  }

  // Cluster-wide histogram of the candidates' logits, and the bins in which the
  // filters' last candidates fall (the last bin where a filter keeps everything).
  static constexpr int kPer = kSampBins / kSampThreads;
  static_assert(kPer == 4, "");
  // This thread's kPer bins over the whole cluster.
  __device__ __forceinline__ void cluster_bins(uint32_t (&c)[kPer]) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) c[i] = 0;
#pragma unroll
    for (int r = 0; r < kSampMaxCluster; ++r) {
      if (r < ranks) {
        const uint4 x = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&s, r)->hist +
                                                        threadIdx.x * kPer);
        c[0] += x.x;
        c[1] += x.y;
        c[2] += x.z;
        c[3] += x.w;
      }
    }
  }

  // From the threads' largest logits: a bin at or above which k candidates lie,
  // the last bin if there is none.
  __device__ int bound_k(float largest, int k) {
    if (largest > -INFINITY) atomicAdd(&s.hist[bin(largest)], 1u);
    if (threadIdx.x == 0) s.bin_k = kSampBins - 1;
    cluster.sync();
    uint32_t c[kPer], total;
    cluster_bins(c);
    const uint32_t uk = static_cast<uint32_t>(k);
    uint32_t before = block_scan(c[0] + c[1] + c[2] + c[3],
                                 reinterpret_cast<uint32_t*>(s.warp_a), total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (before < uk && before + c[i] >= uk) s.bin_k = threadIdx.x * kPer + i;
      before += c[i];
    }
    __syncthreads();
    return s.bin_k;
  }

  __device__ void histogram(int k, bool use_k, float p, bool use_p) {
    each(threadIdx.x, vecs, kSampThreads, [&](float f, int) {
      if (f > -INFINITY) atomicAdd(&s.hist[bin(f)], 1u);
    });
    cluster.sync();
    const int b0 = threadIdx.x * kPer;
    uint32_t c[kPer];
    cluster_bins(c);
    if (threadIdx.x == 0) {
      s.bin_k = s.bin_p = kSampBins - 1;
      s.in_k = s.upto_k = 0xffffffffu;
    }
    const uint32_t uk = static_cast<uint32_t>(k);
    uint32_t total;
    const uint32_t ex = block_scan(c[0] + c[1] + c[2] + c[3],
                                   reinterpret_cast<uint32_t*>(s.warp_a), total);
    uint32_t before = ex;
    if (use_k) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (before < uk && before + c[i] >= uk) {
          s.bin_k = b0 + i;
          s.in_k = c[i];
          s.upto_k = before + c[i];
        }
        before += c[i];
      }
    }
    if (use_p) {
      // weights at the bins' centres (an estimate); with top-k the first k.  In whole
      // numbers, steps of 2^-40 and one at least: the threads' shares then tile the
      // sum exactly, so one thread of the CTA holds the bin, and the same bin in
      // every CTA of the cluster (fp32 running sums overlap by their rounding).
      const float step = bin_scale > 0.f ? static_cast<float>(inv_temp) / bin_scale : 0.f;
      u64 m[kPer], sum = 0, all;
      before = ex;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t count = use_k ? min(c[i], before < uk ? uk - before : 0u) : c[i];
        const float e = fmaxf(__expf(-(b0 + i + 0.5f) * step), 0.f);  // (NaN: 0)
        m[i] = count * (static_cast<u64>(e * 0x1p40f) + 1);
        sum += m[i];
        before += c[i];
      }
      u64 at = block_scan(sum, s.warp_a, all);
      const u64 want = top_p_target(p, all);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (at < want && at + m[i] >= want) s.bin_p = b0 + i;
        at += m[i];
      }
    }
    __syncthreads();
    if (!use_p) return;
    // Where candidates are few and heavy the estimate may be off by the empty bins
    // between two of them: the margin for sorting goes by candidates.
    const int end = window_begin() + kSampWindow - 1, at_p = s.bin_p;
    if (threadIdx.x == 0) {
      s.bin_f = kSampBins - 1;
      s.upto_f = total;
    }
    before = ex;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      before += c[i];
      if (b0 + i == end) s.upto_w = before;
      if (b0 + i == at_p) s.upto_p = before;
    }
    __syncthreads();
    const uint32_t goal = s.upto_p + kSampMargin;
    before = ex;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (before < goal && before + c[i] >= goal) {
        s.bin_f = b0 + i;
        s.upto_f = before + c[i];
      }
      before += c[i];
    }
    __syncthreads();
  }
  __device__ __forceinline__ int window_begin() const {
    return max(0, min(s.bin_p - kSampWindow / 2, kSampBins - kSampWindow));
  }

  // Weights of the whole row, per lane: its sum (total), what lies above bin lo
  // (above) and of that what min-p keeps (kept); the weights of the bins lo ..
  // lo + kSampWindow - 1 are added up in shared memory, the candidates of bin
  // `which` sent to rank 0's (empty) list.
  __device__ __forceinline__ void weigh(int lo, int which, u64 least, u64& total, u64& above, u64& kept) {
    if (threadIdx.x < kSampWindow) s.win_lo[threadIdx.x] = s.win_hi[threadIdx.x] = 0;
    __syncthreads();
    const int s1 = seg_begin(warp + 1);
    SampleShared* home = cluster.map_shared_rank(&s, 0);
    each(seg_begin(warp) + lane, s1, 32, [&](float f, int i) {
      const u64 w = weight_of(f);
      const float at_f = place(f);
      const bool over = at_f < static_cast<float>(lo);
      total += w;
      above += over ? w : 0;
      kept += over && w >= least ? w : 0;
      if (between(at_f, lo, lo + kSampWindow - 1) && f > -INFINITY) {
        const int at = bin(f) - lo;
        if (at + lo == which) push(home, f, i);
        const uint32_t x = static_cast<uint32_t>(w);
        const uint32_t old = atomicAdd(&s.win_lo[at], x);
        const uint32_t hi = static_cast<uint32_t>(w >> 32) + (old + x < old ? 1u : 0u);
        if (hi) atomicAdd(&s.win_hi[at], hi);
      }
    });
  }

  // The filters of a row whose values have a table (one CTA): the logits are counted
  // by value, and counts times weights, taken in the order of the values, say
  // exactly in which value each filter ends and how many of its candidates, in
  // index order, are kept.  One more pass sums what is kept and finds the last of
  // those.  (256 x 151936, top-p: 212 us without it, 137 with.)  False where a filter
  // ends among the values below the table, which are counted as one.
  static constexpr int kLutPos = 2 * kSampLutSide + 1;  // positive, below the table, negative
  static constexpr int kLutPer = (kLutPos + kSampThreads - 1) / kSampThreads;
  __device__ bool by_value(int k, bool use_k, float p, bool use_p, u64 least, u64& total, u64& last,
                           u64& warp_kept, bool& known) {
    uint32_t* counts = reinterpret_cast<uint32_t*>(lut + 2 * kSampLutSide);
    for (int i = threadIdx.x; i < 2 * kSampLutSide; i += kSampThreads) counts[i] = 0;
    if (threadIdx.x == 0) {
      s.bin_k = s.bin_p = -1;
      s.in_k = 0;      // candidates below the table
      s.win_over = 0;  // and their weight
    }
    __syncthreads();
    uint32_t tiny_n = 0;
    u64 tiny_w = 0;
    each(threadIdx.x, vecs, kSampThreads, [&](float f, int) {
      if (!(f > -INFINITY)) return;
      const int at = lut_entry(f + 0.f);  // -0 with +0
      if (at >= 0) {
        atomicAdd(counts + at, 1u);
      } else {
        ++tiny_n;
        tiny_w += weight(f);
      }
    });
    if (__any_sync(0xffffffffu, tiny_n != 0)) {
      tiny_n = warp_reduce(tiny_n, AddOp());
      tiny_w = warp_reduce(tiny_w, AddOp());
      if (lane == 0) {
        atomicAdd(&s.in_k, tiny_n);
        atomicAdd(&s.win_over, tiny_w);
      }
    }
    __syncthreads();
    // places in descending order of value; this thread's are first .. first + kLutPer - 1
    const int first = threadIdx.x * kLutPer;
    auto at_place = [&](int pos, uint32_t& c, u64& w) {  // candidates and weight of each; its mass
      c = 0;
      w = 0;
      if (pos >= kLutPos) return u64(0);
      if (pos == kSampLutSide) {
        c = s.in_k;
        return s.win_over;
      }
      const int at = lut_of(pos);
      c = counts[at];
      w = lut[at];
      return c * w;
    };
    uint32_t c, n = 0, all_n;
    u64 w, m = 0;
    for (int i = 0; i < kLutPer; ++i) {
      m += at_place(first + i, c, w);
      n += c;
    }
    const uint32_t n0 = block_scan(n, reinterpret_cast<uint32_t*>(s.warp_a), all_n);
    const u64 m0 = block_scan(m, s.warp_a, total);
    const uint32_t uk = static_cast<uint32_t>(k);
    if (use_k && n0 < uk && n0 + n >= uk) {
      u64 mass = m0;
      for (int i = 0, before = n0; i < kLutPer; ++i) {
        const u64 here = at_place(first + i, c, w);
        if (before < k && before + static_cast<int>(c) >= k) {
          s.bin_k = first + i;
          s.upto_k = uk - before;
          s.last_mass = mass + s.upto_k * w;
        }
        before += c;
        mass += here;
      }
    }
    __syncthreads();
    int cut = -1;
    uint32_t need = 0;
    u64 of = total;
    if (use_k && s.bin_k >= 0) {
      cut = s.bin_k;
      need = s.upto_k;
      of = s.last_mass;
      if (cut == kSampLutSide) return false;
    }
    if (use_p) {
      const u64 target = top_p_target(p, of);
      if (m0 < target && m0 + m >= target) {
        u64 mass = m0;
        for (int i = 0; i < kLutPer; ++i) {
          const u64 here = at_place(first + i, c, w);
          if (mass < target && mass + here >= target) {
            s.bin_p = first + i;
            s.upto_p = w != 0 ? static_cast<uint32_t>((target - mass + w - 1) / w) : 0;
          }
          mass += here;
        }
      }
      __syncthreads();
      cut = s.bin_p;
      need = s.upto_p;
      if (cut < 0 || cut == kSampLutSide) return false;
    }
    last = 0;
    known = false;
    const int at = cut < 0 ? 0 : lut_of(cut);
    const u64 w_cut = cut < 0 ? 0 : lut[at];
    if (w_cut == 0) return true;  // whatever has a weight is kept
    const bool neg = at >= kSampLutSide;
    const int d = neg ? at - kSampLutSide : at;
    const float mag = d == kSampLutSide - 1
                          ? INFINITY
                          : __uint_as_float(static_cast<uint32_t>(lut_base + d) << 16);
    const float v = neg ? -mag : mag;
    uint32_t equal = 0;
    u64 above = 0;
    each(seg_begin(warp) + lane, seg_begin(warp + 1), 32, [&](float f, int) {
      if (f > v) {
        const u64 x = weight_of(f);
        above += x >= least ? x : 0;
      }
      equal += f == v ? 1 : 0;
    });
    above = warp_reduce(above, AddOp());
    equal = warp_reduce(equal, AddOp());
    if (lane == 0) s.warp_b[warp] = equal;
    __syncthreads();
    const uint32_t mine = lane < kSampWarps ? static_cast<uint32_t>(s.warp_b[lane]) : 0;
    uint32_t inc = mine;
#pragma unroll
    for (int off = 1; off < kSampWarps; off <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += x;
    }
    const uint32_t ex = inc - mine, ahead = __shfl_sync(0xffffffffu, ex, warp);
    const uint32_t kept = min(equal, need > ahead ? need - ahead : 0u);
    warp_kept = above + (w_cut >= least ? kept * w_cut : 0);
    known = true;
    if (need >= counts[at]) {
      last = static_cast<u64>(order_key(v)) << 32;
      return true;
    }
    // the need-th candidate of this value: the warp's run that holds it, again
    const unsigned hit = __ballot_sync(0xffffffffu, lane < kSampWarps && ex < need && inc >= need);
    const int run = max(0, __ffs(hit) - 1);
    const uint32_t rest = need - __shfl_sync(0xffffffffu, ex, run);
    const int v0 = seg_begin(run), v1 = seg_begin(run + 1);
    const int per = (v1 - v0 + kSampThreads - 1) / kSampThreads;
    const int t0 = min(v1, v0 + static_cast<int>(threadIdx.x) * per), t1 = min(v1, t0 + per);
    uint32_t here = 0, sum;
    each(t0, t1, 1, [&](float f, int) { here += f == v ? 1 : 0; });
    uint32_t seen = block_scan(here, reinterpret_cast<uint32_t*>(s.warp_a), sum);
    if (seen < rest && seen + here >= rest) {
      each(t0, t1, 1, [&](float f, int i) {
        if (f == v && ++seen == rest) s.last = order_of(f, base + i);
      });
    }
    __syncthreads();
    last = s.last;
    return true;
  }
  __device__ __forceinline__ static int lut_of(int pos) {  // table entry of a place
    return pos < kSampLutSide ? kSampLutSide - 1 - pos : pos - 1;
  }

  // After weigh() and a cluster barrier: the bin of the window in which the
  // weight from the top reaches target, -1 if none; over: the weight above it.
  __device__ int window_find(int lo, u64 above, u64 target, u64& over) {
    if (threadIdx.x == 0) s.win_bin = -1;
    __syncthreads();
    if (warp == 0) {
      u64 m = 0;
      for (int r = 0; r < ranks && lane < kSampWindow; ++r) {
        const SampleShared* o = cluster.map_shared_rank(&s, r);
        m += (static_cast<u64>(o->win_hi[lane]) << 32) + o->win_lo[lane];
      }
      u64 inc = m;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += x;
      }
      const u64 ex = above + inc - m;
      if (ex < target && ex + m >= target) {
        s.win_bin = lo + lane;
        s.win_over = ex;
      }
    }
    static_assert(kSampWindow <= 32, "");
    __syncthreads();
    over = s.win_over;
    return s.win_bin;
  }

  // target of top-p in units of weight: kept while the weight before is below it
  __device__ __forceinline__ static u64 top_p_target(float p, u64 of) {
    const u64 t = static_cast<u64>(ceil(static_cast<double>(p) * static_cast<double>(of)));
    return max(u64(1), min(of, t));
  }
  __device__ __forceinline__ static u64 draw_goal(float u, u64 whole) {
    const u64 g = static_cast<u64>(fmax(static_cast<double>(u), 0.0) * static_cast<double>(whole));
    return g >= whole ? whole - 1 : g;
  }

  // The general way for one CTA alone, over the row in global memory: sums of
  // weights, bisected for top-p's last candidate and then for the drawn index.
  template <typename Pred>
  __device__ u64 row_sum(const T* src, Pred pred) {
    u64 x = 0, sum;
    for (int i = threadIdx.x; i < a.vocab; i += kSampThreads) {
      const float f = to_float<T>(src[i]);
      if (f == f && pred(f, i)) x += weight(f);
    }
    block_scan(x, s.warp_a, sum);
    return sum;
  }
  __device__ void alone(int row, float p, u64 least, float u, u64 row_total) {
    const T* src = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.row_stride;
    const u64 target = top_p_target(p, row_total);
    u64 lo = 0, hi = ~u64(0);
    while (hi - lo > 1) {
      const u64 mid = lo + (hi - lo) / 2;
      const u64 m = row_sum(src, [&](float f, int i) { return order_of(f, i) >= mid; });
      (m >= target ? lo : hi) = mid;
    }
    auto keep = [&](float f, int i) {
      return order_of(f, i) >= lo && weight(f) >= least;
    };
    const u64 goal = draw_goal(u, row_sum(src, keep));
    int first = -1, end = a.vocab - 1;  // the sum up to `end` exceeds the goal, up to `first` not
    while (end - first > 1) {
      const int mid = first + (end - first) / 2;
      const u64 m = row_sum(src, [&](float f, int i) { return i <= mid && keep(f, i); });
      (m > goal ? end : first) = mid;
    }
    if (threadIdx.x == 0) finish(row, end, to_float<T>(src[end]), row_total);
  }

  // The token is found: by the thread that holds it.
  __device__ __forceinline__ void finish(int row, int index, float f, u64 total) {
    a.ids[row] = index;
    if (a.logprobs != nullptr) {
      const double z =
          f == top ? 0.0 : (static_cast<double>(f) - static_cast<double>(top)) * inv_temp;
      a.logprobs[row] = static_cast<float>(z - log(static_cast<double>(total) * 0x1p-44));
    }
  }

  __device__ void run(int row, float mx, float mn) {
    const float own_max = mx;  // this thread's largest logit
    const float temp = a.temperature != nullptr ? a.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    const int k = greedy || a.top_k == nullptr ? 0 : a.top_k[row];
    const float p = greedy || a.top_p == nullptr ? 1.f : a.top_p[row];
    const float mp = greedy || a.min_p == nullptr ? 0.f : a.min_p[row];
    const float u32 = a.uniforms[row];
    const bool use_k = k > 0 && k < a.vocab, use_p = p < 1.f;
    if (threadIdx.x < 64) s.table[threadIdx.x] = kExp2Table[threadIdx.x];
    for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) s.hist[i] = 0;
    if (threadIdx.x == 0) s.list_n = 0;

    // ---- the row's largest and smallest finite logit -------------------------
    auto fmax_op = [](float x, float y) { return fmaxf(x, y); };
    auto fmin_op = [](float x, float y) { return fminf(x, y); };
    mx = warp_reduce(mx, fmax_op);
    mn = warp_reduce(mn, fmin_op);
    if (lane == 0) {
      s.warp_max[warp] = mx;
      s.warp_min[warp] = mn;
    }
    __syncthreads();
    if (warp == 0) {
      mx = warp_reduce(lane < kSampWarps ? s.warp_max[lane] : -INFINITY, fmax_op);
      mn = warp_reduce(lane < kSampWarps ? s.warp_min[lane] : INFINITY, fmin_op);
      if (lane == 0) {
        s.pub_max = mx;
        s.pub_min = mn;
      }
    }
    cluster.sync();
    top = -INFINITY;
    mn = INFINITY;
    for (int r = 0; r < ranks; ++r) {
      const SampleShared* o = cluster.map_shared_rank(&s, r);
      top = fmaxf(top, o->pub_max);
      mn = fminf(mn, o->pub_min);
    }
    if (top == -INFINITY) {  // nothing to draw from (the same for every CTA)
      if (rank == 0 && threadIdx.x == 0) {
        a.ids[row] = -1;
        if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
      }
      cluster.sync();
      return;
    }
    top_finite = static_cast<double>(fminf(top, 3.402823466e38f));
    inv_temp = greedy ? 1.0 : 1.0 / static_cast<double>(temp);
    scale = 92.332482616893656877 * inv_temp;  // 64 / ln 2
    // bins span the finite logits, at most 64 T (weights below e^-64 vanish)
    least_logit = fmaxf(top - 31.3f * (greedy ? 1.f : temp), -3.402823466e38f);
    const float span = fminf(top - mn, fmaxf(64.f * temp, 32.f));
    bin_scale = span > 0.f && span < INFINITY ? (kSampBins - 1) / span : 0.f;
    // min_p in units of 2^-44; the largest candidates (weight 2^44) always stay
    const u64 least =
        mp > 0.f ? min(u64(1) << 44, static_cast<u64>(ceil(static_cast<double>(mp) * 17592186044416.0)))
                 : 0;

    const bool small_k = use_k && k <= ranks * (kSampThreads / 4);
    // (greedy rows and those of a small k seldom weigh all logits)
    if (!kResident && std::is_same<T, __nv_bfloat16>::value && a.tabled &&
        (a.logprobs != nullptr || !(greedy || small_k)))
      build_table(mn);

    // ---- where the filters cut -------------------------------------------------
    const int s0 = seg_begin(warp), s1 = seg_begin(warp + 1);
    u64 row_total = 0, above = 0;
    SampleShared* home = cluster.map_shared_rank(&s, 0);
    // Sends the candidates of bins 0 .. upto to rank 0, which finishes the row if
    // they fit its list; sums the row where rank 0 needs that: for top-p without
    // top-k and for log probabilities.
    auto try_few = [&](int upto) {
      // every logit of those bins (and, by rounding, perhaps a few more)
      const float low = bin_scale > 0.f ? top - (upto + 1) / bin_scale * 1.00001f : -INFINITY;
      const float from = upto < kSampBins - 1 && low > -3.402823466e38f ? low : -3.402823466e38f;
      if (a.logprobs != nullptr || !use_k) {
        each(s0 + lane, s1, 32, [&](float f, int i) {
          row_total += weight_of(f);
          if (f >= from) push(home, f, i);
        });
      } else {
        each(s0 + lane, s1, 32, [&](float f, int i) {
          if (f >= from) push(home, f, i);
        });
      }
      cluster_sum(row_total, above);
      if (home->list_n > kSampList) {  // (seen by all alike)
        row_total = above = 0;
        cluster.sync();
        if (threadIdx.x == 0) s.list_n = 0;
        cluster.sync();
        return false;
      }
      cluster.sync();  // all have seen the count: rank 0 may use its list, the others leave
      if (rank == 0) finish_few(row, k, use_k, p, use_p, least, u32, row_total);
      return true;  // rank 0 touches no other CTA's memory from here on
    };
    if (small_k) {
      if (try_few(bound_k(own_max, k))) return;
      // more than the list holds: start over with all logits
      for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) s.hist[i] = 0;
      __syncthreads();
    }
    u64 last = 0;        // every candidate from this order on is kept
    u64 warp_kept = 0;   // of this warp's run of vectors
    bool known = true;   // warp_kept is right
    bool counted = false;
    if (!kResident && std::is_same<T, __nv_bfloat16>::value && tabled && (use_k || use_p)) {
      counted = by_value(k, use_k, p, use_p, least, row_total, last, warp_kept, known);
      if (!counted) row_total = 0;
    }
    if (!counted && (use_k || use_p)) {
      histogram(k, use_k, p, use_p);
      // (top-p alone: the window and the margin, whichever reaches further)
      if ((use_k ? s.upto_k : max(s.upto_w, s.upto_f)) <= kSampList &&
          try_few(use_k ? s.bin_k : max(s.bin_f, window_begin() + kSampWindow - 1)))
        return;
    }

    // ---- many candidates, or no filter ------------------------------------------
    if (counted) {
      // (by_value has what the draw needs)
    } else if (greedy) {
      if (a.logprobs != nullptr)
        each(s0 + lane, s1, 32, [&](float f, int) { row_total += weight_of(f); });
      each(s0 + lane, s1, 32, [&](float f, int) { warp_kept += f == top ? 1 : 0; });
      warp_kept = warp_reduce(warp_kept, AddOp());
      if (a.logprobs != nullptr) cluster_sum(row_total, above);
    } else if (!use_k && !use_p) {
      each(s0 + lane, s1, 32, [&](float f, int) {
        const u64 w = weight_of(f);
        row_total += w;
        warp_kept += w >= least ? w : 0;
      });
      warp_kept = warp_reduce(warp_kept, AddOp());
      cluster_sum(row_total, above);
    } else {
      // Many candidates.  top-k first: its bin is exact.
      u64 mass = 0;
      int lo = use_k ? min(s.bin_k, kSampBins - kSampWindow) : window_begin();
      weigh(lo, use_k ? s.bin_k : s.bin_p, least, row_total, above, warp_kept);
      warp_kept = warp_reduce(warp_kept, AddOp());
      cluster_sum(row_total, above);
      mass = row_total;
      int cut = -1;  // bin of the last kept candidate
      if (use_k && s.in_k != 0xffffffffu) {
        if (s.in_k <= kSampList) {
          u64 over = above;
          for (int b = lo; b < s.bin_k; ++b)  // (the window may begin before bin_k)
            for (int r = 0; r < ranks; ++r) {
              const SampleShared* o = cluster.map_shared_rank(&s, r);
              over += (static_cast<u64>(o->win_hi[b - lo]) << 32) + o->win_lo[b - lo];
            }
          last = bin_last(s.bin_k, true, false, static_cast<u64>(k) - (s.upto_k - s.in_k), over, mass);
          cut = s.bin_k;
        } else {
          last = bisect(false, static_cast<u64>(k), mass);
          known = false;
        }
      }
      if (use_p) {
        if (use_k) {  // the sums were taken at top-k's bin: again at top-p's
          if (threadIdx.x == 0) s.list_n = 0;
          cluster.sync();
          lo = window_begin();
          u64 again = 0;
          above = warp_kept = 0;
          weigh(lo, s.bin_p, least, again, above, warp_kept);
          warp_kept = warp_reduce(warp_kept, AddOp());
          cluster_sum(again, above);
          known = true;
        }
        const u64 target = top_p_target(p, mass);
        u64 over = 0, m = 0, by_p = 0;
        const int found = window_find(lo, above, target, over);
        uint32_t in_bin = 0;
        if (found >= 0)
          for (int r = 0; r < ranks; ++r) in_bin += cluster.map_shared_rank(&s, r)->hist[found];
        if (found >= 0 && in_bin <= kSampList) {
          by_p = bin_last(found, found == s.bin_p, true, target - over, over, m);
          cut = found;
        }
        if (by_p == 0) {
          by_p = bisect(true, target, m);
          known = false;
        }
        if (by_p < last) known = false;  // equal weights at the border: top-k is the stricter one
        last = max(last, by_p);
      }
      if (known && last != 0) {
        // what is kept of the bins lo .. cut joins the sums
        u64 more = 0;
        each(s0 + lane, s1, 32, [&](float f, int i) {
          if (between(place(f), lo, cut) && f > -INFINITY && order_of(f, base + i) >= last) {
            const u64 w = weight(f);
            more += w >= least ? w : 0;
          }
        });
        warp_kept += warp_reduce(more, AddOp());
      } else {
        known = false;
      }
    }

    // ---- the draw: running sums in index order ---------------------------------
    auto keep = [&](float f, int i) -> u64 {
      if (greedy) return f == top ? 1 : 0;
      if (last != 0 && order_of(f, base + i) < last) return 0;
      const u64 w = weight_of(f);
      return w >= least ? w : 0;
    };
    if (!known) {
      u64 x = 0;
      each(s0 + lane, s1, 32, [&](float f, int i) { x += keep(f, i); });
      warp_kept = warp_reduce(x, AddOp());
    }
    __syncthreads();
    if (lane == 0) s.warp_b[warp] = warp_kept;
    __syncthreads();
    u64 mine = lane < kSampWarps ? s.warp_b[lane] : 0, inc = mine;  // every warp: the CTA's warps
#pragma unroll
    for (int off = 1; off < kSampWarps; off <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += x;
    }
    const u64 cta = __shfl_sync(0xffffffffu, inc, kSampWarps - 1);
    if (threadIdx.x == 0) s.pub_a = cta;
    cluster.sync();
    u64 before = 0, whole = 0;
    for (int r = 0; r < ranks; ++r) {
      const u64 m = cluster.map_shared_rank(&s, r)->pub_a;
      if (r < rank) before += m;
      whole += m;
    }
    // the token is the first whose running sum exceeds u * whole
    const u64 goal = greedy ? 0 : draw_goal(u32, whole);
    if (before <= goal && before + cta > goal) {  // in this CTA: which warp's run of vectors?
      const u64 ex = before + inc - mine;
      const unsigned hit = __ballot_sync(0xffffffffu, lane < kSampWarps && ex <= goal && ex + mine > goal);
      const int w = max(0, __ffs(hit) - 1);
      u64 at = __shfl_sync(0xffffffffu, ex, w);
      // that run again, spread over the whole CTA in index order
      const int v0 = seg_begin(w), v1 = seg_begin(w + 1);
      const int per = (v1 - v0 + kSampThreads - 1) / kSampThreads;
      const int t0 = min(v1, v0 + static_cast<int>(threadIdx.x) * per), t1 = min(v1, t0 + per);
      u64 x = 0;
      each(t0, t1, 1, [&](float f, int i) { x += keep(f, i); });
      u64 sum;
      at += block_scan(x, s.warp_a, sum);
      if (at <= goal && at + x > goal) {
        bool found = false;
        each(t0, t1, 1, [&](float f, int i) {
          if (found) return;
          at += keep(f, i);
          if (at > goal) {
            found = true;
            finish(row, base + i, f, row_total);
          }
        });
      }
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
  }

  // Rank 0, its list holding every candidate that may be kept: the row's token.
  __device__ void finish_few(int row, int k, bool use_k, float p, bool use_p, u64 least, float u,
                             u64 row_total) {
    const int count = static_cast<int>(min(s.list_n, static_cast<uint32_t>(kSampList)));
    u64 w[2], ex[2], sum;
    order_list(count, w, ex, sum);
    // top-p's share is of the first k, or of the row where there is no top-k
    u64 of = row_total;
    if (use_k) {
      if (threadIdx.x == 0) s.last_mass = sum;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (2 * static_cast<int>(threadIdx.x) + i == k) s.last_mass = ex[i];
      __syncthreads();
      of = s.last_mass;
    }
    const u64 target = use_p ? top_p_target(p, of) : ~u64(0);
    if (!use_k && sum < target) {  // the estimate fell short by more than the window
      alone(row, p, least, u, row_total);
      return;
    }
    // what is kept, in index order: (index complemented, place in the list)
    u64 key[2] = {0, 0};
    float value[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 2 * threadIdx.x + i;
      const bool keep = at < count && (!use_k || at < k) && ex[i] < target &&
                        w[i] >= least;
      const u64 entry = at < count ? s.list[at] : 0;
      value[i] = key_value(static_cast<uint32_t>(entry >> 32));
      if (keep) key[i] = (entry << 32) | static_cast<u64>(at) | 0x80000000ull;
      s.weight[at] = keep ? w[i] : 0;
    }
    const int kept_n = __syncthreads_count(key[0] != 0) + __syncthreads_count(key[1] != 0);
    if (threadIdx.x == 0) s.pub_n = 0;
    int size = 64;
    while (size < kept_n) size <<= 1;
    for (int i = threadIdx.x; i < size; i += kSampThreads) s.list[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (key[i] != 0) s.list[atomicAdd(&s.pub_n, 1u)] = key[i];
    __syncthreads();
    sort(size);  // larger = smaller index
    u64 iw[2], iex[2], whole;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 2 * threadIdx.x + i;
      iw[i] = at < kept_n ? s.weight[s.list[at] & 0x7fffffffu] : 0;
    }
    iex[0] = block_scan(iw[0] + iw[1], s.warp_a, whole);
    iex[1] = iex[0] + iw[0];
    const u64 goal = draw_goal(u, whole);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (iex[i] <= goal && iex[i] + iw[i] > goal) {
        const u64 entry = s.list[2 * threadIdx.x + i];
        s.bin_k = static_cast<int>(entry & 0x7fffffffu);  // its place in the first order
        s.bin_p = static_cast<int>(0xffffffffu - static_cast<uint32_t>(entry >> 32));
      }
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) == s.bin_k / 2)
      finish(row, s.bin_p, s.bin_k & 1 ? value[1] : value[0], row_total);
  }

  // The order of the last kept candidate within a bin of at most kSampList
  // candidates, where `need` more (counted or weighed) are to be kept; mass =
  // above + the bin's weight up to it.  0 when the bin does not hold enough.
  // listed: rank 0's list holds the bin's candidates already.
  __device__ u64 bin_last(int which, bool listed, bool by_mass, u64 need, u64 above, u64& mass) {
    if (!listed) {
      cluster.sync();
      if (threadIdx.x == 0) s.list_n = 0;
      cluster.sync();
      SampleShared* home = cluster.map_shared_rank(&s, 0);
      each(threadIdx.x, vecs, kSampThreads, [&](float f, int i) {
        if (between(place(f), which, which) && f > -INFINITY) push(home, f, i);
      });
      cluster.sync();
    }
    if (rank == 0) {
      const int count = static_cast<int>(min(s.list_n, static_cast<uint32_t>(kSampList)));
      u64 w[2], ex[2], sum;
      order_list(count, w, ex, sum);
      if (threadIdx.x == 0) s.last = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u64 at = 2 * threadIdx.x + i;
        const bool here = by_mass ? ex[i] < need && ex[i] + w[i] >= need : at + 1 == need;
        if (here && at < static_cast<u64>(count)) {
          s.last = s.list[at];
          s.last_mass = above + ex[i] + w[i];
        }
      }
    }
    cluster.sync();
    const SampleShared* o = cluster.map_shared_rank(&s, 0);
    const u64 last = o->last;
    mass = o->last_mass;
    cluster.sync();
    return last;
  }
};

template <typename T, bool kResident>
__global__ void __launch_bounds__(kSampThreads, 2) sample_tokens_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(s_raw);
  T* slice = reinterpret_cast<T*>(s_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  Sampler<T, kResident> job(a, s, slice);
  job.lut = reinterpret_cast<u64*>(slice);  // where the row is not resident
  constexpr int kVec = 16 / sizeof(T);
  const int row = blockIdx.x / job.ranks;
  job.base = min(a.vocab, job.rank * a.slice);
  job.n = min(a.slice, a.vocab - job.base);
  job.vecs = (job.n + kVec - 1) / kVec;
  const T* src = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.row_stride + job.base;
  float mx = -INFINITY, mn = INFINITY;
  if (kResident) {
    // into shared memory, NaN as -inf and the last vector padded with it
    const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
#pragma unroll 4
    for (int v = threadIdx.x; v < job.vecs; v += kSampThreads) {
      uint4 raw;
      T* e = reinterpret_cast<T*>(&raw);
      if (aligned && (v + 1) * kVec <= job.n) {
        raw = __ldg(reinterpret_cast<const uint4*>(src) + v);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          e[i] = v * kVec + i < job.n ? src[v * kVec + i] : from_float<T>(-INFINITY);
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float f = to_float<T>(e[i]);
        if (f != f) e[i] = from_float<T>(-INFINITY);
        mx = fmaxf(mx, f);  // NaN loses
        if (f > -INFINITY) mn = fminf(mn, f);
      }
      reinterpret_cast<uint4*>(slice)[v] = raw;
    }
  } else {
    job.slice = src;  // 16-byte aligned, a whole number of vectors
#pragma unroll 4
    for (int v = threadIdx.x; v < job.vecs; v += kSampThreads) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src) + v);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float f = to_float<T>(e[i]);
        mx = fmaxf(mx, f);
        if (f > -INFINITY) mn = fminf(mn, f);
      }
    }
  }
  job.run(row, mx, mn);
}

template <typename T, bool kResident>
cudaError_t launch_sample(SampleArgs a, int batch, int ctas, cudaStream_t stream) {
  static unsigned long long configured = 0;  // one bit per device
  constexpr int kFixed = (sizeof(SampleShared) + 15) / 16 * 16;
  static_assert(kFixed + kSampSliceBytes <= 227 * 1024, "");
  static_assert(2 * (kFixed + kSampLutBytes) <= 226 * 1024, "two CTAs an SM");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(configured & (1ull << dev))) {
    e = cudaFuncSetAttribute(sample_tokens_kernel<T, kResident>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kFixed + (kResident ? kSampSliceBytes : kSampLutBytes));
    if (e != cudaSuccess) return e;
    if (dev < 64) configured |= 1ull << dev;
  }
  a.slice = ((a.vocab + ctas - 1) / ctas + 15) / 16 * 16;
  // The table of weights costs 4098 of them: slower with the slices of a cluster
  // (64 x 151936 in slices of 19k: 66.8 -> 69.8 us), faster with whole rows (256 x
  // 151936, no filter: 104 -> 80, top-k 103 -> 78, top-p with by_value 234 -> 137; at
  // 65536 logits 46 -> 38, mixed filters 86 -> 58).  Shorter whole rows would gain as
  // well (16384 logits: no filter 19.9 -> 18.8, mixed 40 -> 28); they share the path of
  // fp16 and fp32 rows.
  a.tabled = !kResident && std::is_same<T, __nv_bfloat16>::value && a.vocab >= kSampLutLogits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * ctas));
  cfg.blockDim = dim3(kSampThreads);
  cfg.dynamicSmemBytes = kFixed + (kResident ? static_cast<size_t>(a.slice) * sizeof(T) : 0) +
                         (a.tabled ? kSampLutBytes : 0);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T, kResident>, a);
}

template <typename T>
cudaError_t dispatch_sample(const SampleArgs& a, int batch, cudaStream_t stream) {
  const int sms = num_sms_current_device();
  constexpr int kVec = 16 / sizeof(T);
  // Whole rows from L2 or clusters, mixed filters, us: 151936 bf16 at 74 rows 92 / 71,
  // 120: 94 / 100, 148: 97 / 121, 256: 118 / 184; fp32 at 120: 143 / 130, 148: 145 / 161,
  // 256: 182 / 261; fp16 (no table) at 148: 139 / 122, 200: 170 / 147, 256: 170 / 182.
  // 32000 bf16 and fp16: within a tenth from 120 rows on; fp32 at 148: 43 / 38, 200: 49
  // / 56.
  if (batch >= sms && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 &&
      a.row_stride % kVec == 0 && a.vocab % kVec == 0)
    return launch_sample<T, false>(a, batch, 1, stream);
  // CTAs of a row: as many as hold its logits two to an SM (one to an SM where a
  // cluster of eight leaves more); more while SMs would be idle and every CTA
  // keeps a few thousand logits
  int ctas = 1;
  auto bytes = [&](int c) { return (static_cast<int64_t>(a.vocab) + c - 1) / c * static_cast<int64_t>(sizeof(T)); };
  while (ctas < kSampMaxCluster && bytes(ctas) > kSampSliceGoal) ctas *= 2;
  while (ctas < kSampMaxCluster && batch * ctas * 2 <= sms &&
         bytes(ctas) > 8192 * static_cast<int64_t>(sizeof(T)))
    ctas *= 2;
  return launch_sample<T, true>(a, batch, ctas, stream);
}

}  // namespace
}  // namespace helm

extern "C" int helm_sample_tokens(const void* logits, int64_t row_stride, int dtype,
                                  const float* uniforms, const float* temperature,
                                  const int32_t* top_k, const float* top_p, const float* min_p,
                                  int64_t* ids, float* logprobs, int batch, int vocab,
                                  void* stream) {
  using namespace helm;
  if (logits == nullptr || uniforms == nullptr || ids == nullptr || batch < 0 || vocab <= 0)
    return HELM_ERR_INVALID_ARGUMENT;
  if (batch == 0) return HELM_OK;
  if (vocab > kSampMaxVocab || batch > (1 << 24)) return HELM_ERR_UNSUPPORTED;
  const SampleArgs a = {logits, row_stride, uniforms, temperature, top_k, top_p,
                        min_p,  ids,        logprobs, vocab,       0,           0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (dtype) {
    case HELM_DTYPE_BF16:
      e = dispatch_sample<__nv_bfloat16>(a, batch, s);
      break;
    case HELM_DTYPE_FP16:
      e = dispatch_sample<__half>(a, batch, s);
      break;
    case HELM_DTYPE_FP32:
      e = dispatch_sample<float>(a, batch, s);
      break;
    default:
      return HELM_ERR_UNSUPPORTED;
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}
