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
// A row is held by one cluster, its logits in the CTAs' shared memory: HBM is
// read once.  Each filter's last kept candidate is found by a histogram over
// 2048 equal steps of the logit (counts and weights; steps equal in the logit
// spread the atomics of a bell-shaped row, digits of its bit pattern would not),
// then by ranking the candidates of the one bin that it falls in.  A bin of more
// than 1024 candidates (all logits equal, huge outliers) is bisected instead.
#include <cooperative_groups.h>

#include "common.cuh"

namespace helm {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampThreads = 1024;
constexpr int kSampWarps = kSampThreads / 32;
constexpr int kSampBins = 2048;
constexpr int kSampCand = 1024;              // candidates ranked against each other
constexpr int kSampMaxVocab = 1 << 18;       // 2^18 weights of 2^44 stay below 2^63
constexpr int kSampSliceBytes = 160 * 1024;  // logits held by a CTA
constexpr int kSampMaxCluster = 8;
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

// exp(x) in units of 2^-44, for x <= 0, rounded to nearest.  x = (64 m + j)
// ln2/64 + r with |r| <= ln2/128, e^r by its series to r^4 (next term < 4e-14).
__device__ __forceinline__ u64 weight_fixed(double x, const double* table) {
  if (!(x > -31.0)) return 0;  // below half a unit (2^-45 = e^-31.2)
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the integer
  const double k = fma(x, 0x1.71547652b82fep+6, kMagic);
  const int n = static_cast<int>(__double_as_longlong(k));
  const double kd = k - kMagic;
  double r = fma(kd, -0x1.62e42fcp-7, x);
  r = fma(kd, -0x1.7d1cf79abc9e4p-34, r);
  double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  p *= table[n & 63];
  // times 2^(44 + floor(n / 64)), then rounded to an integer by adding 2^52
  p = __longlong_as_double(__double_as_longlong(p) +
                           (static_cast<long long>(44 + (n >> 6)) << 52));
  const double y = p + 4503599627370496.0;
  return static_cast<u64>(__double_as_longlong(y)) & 0xfffffffffffffull;
}

// Order-preserving bits of a float (NaN was replaced; -0 counts as +0).
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Larger = earlier in the order of candidates.
__device__ __forceinline__ u64 order_of(float f, int index) {
  return (static_cast<u64>(order_key(f)) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}

__device__ __forceinline__ u64 shfl_up64(u64 v, int off) { return __shfl_up_sync(0xffffffffu, v, off); }

template <typename V, typename Op>
__device__ __forceinline__ V warp_reduce(V v, Op op) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

struct SampleShared {
  double table[64];
  u64 warp_u64[kSampWarps];
  uint32_t warp_u32[kSampWarps];
  float warp_f32[2][kSampWarps];
  // published to the cluster
  float pub_max, pub_min;
  u64 pub_mass;
  uint32_t pub_count;
  int pub_index;
  uint32_t pub_cand;
  // results of block-wide searches
  int found_bin;
  u64 found_above, found_order, found_mass;
  uint32_t found_count;
  int result;
  uint32_t hist_count[kSampBins], hist_lo[kSampBins], hist_hi[kSampBins];
  u64 cand_order[kSampCand], cand_weight[kSampCand];      // this CTA's
  u64 all_order[kSampCand], all_weight[kSampCand];        // the cluster's
};

template <typename T>
struct Sampler {
  const SampleArgs& a;
  SampleShared& s;
  const T* slice;
  cg::cluster_group cluster;
  int base, n;       // first index and number of logits of this CTA
  float top;         // largest logit of the row
  double inv_temp;
  float bin_scale;

  __device__ Sampler(const SampleArgs& a_, SampleShared& s_, const T* sl)
      : a(a_), s(s_), slice(sl), cluster(cg::this_cluster()) {}

  __device__ __forceinline__ float logit(int i) const {
    const float f = to_float<T>(slice[i]);
    return f == f ? f : -INFINITY;
  }
  __device__ __forceinline__ u64 weight(float f) const {
    if (f == top) return u64(1) << 44;
    return weight_fixed((static_cast<double>(f) - static_cast<double>(top)) * inv_temp, s.table);
  }
  __device__ __forceinline__ int bin(float f) const {
    return max(0, min(kSampBins - 1, static_cast<int>((top - f) * bin_scale)));
  }

  // Block-wide then cluster-wide sums of (count, mass).
  __device__ void cluster_sum(uint32_t& count, u64& mass) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto add32 = [](uint32_t x, uint32_t y) { return x + y; };
    auto add64 = [](u64 x, u64 y) { return x + y; };
    count = warp_reduce(count, add32);
    mass = warp_reduce(mass, add64);
    if (lane == 0) {
      s.warp_u32[warp] = count;
      s.warp_u64[warp] = mass;
    }
    __syncthreads();
    if (warp == 0) {
      count = warp_reduce(s.warp_u32[lane], add32);
      mass = warp_reduce(s.warp_u64[lane], add64);
      if (lane == 0) {
        s.pub_count = count;
        s.pub_mass = mass;
      }
    }
    cluster.sync();
    count = 0;
    mass = 0;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
      count += *cluster.map_shared_rank(&s.pub_count, r);
      mass += *cluster.map_shared_rank(&s.pub_mass, r);
    }
    cluster.sync();  // everyone has read before the words are used again
  }

  // Candidates (by count) or weight (by mass) before and in each bin: the first
  // bin whose inclusive sum reaches the target.  Needs the complete histogram.
  __device__ void find_bin(bool by_mass, u64 target) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kPer = kSampBins / kSampThreads;
    uint32_t c[kPer];
    u64 m[kPer], sum_c = 0, sum_m = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int bn = threadIdx.x * kPer + i;
      c[i] = 0;
      m[i] = 0;
      for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
        const SampleShared* o = cluster.map_shared_rank(&s, r);
        c[i] += o->hist_count[bn];
        m[i] += (static_cast<u64>(o->hist_hi[bn]) << 32) + o->hist_lo[bn];
      }
      sum_c += c[i];
      sum_m += m[i];
    }
    const u64 mine = by_mass ? sum_m : sum_c, mine_m = sum_m;
    u64 inc = mine, inc_m = mine_m;
    for (int off = 1; off < 32; off <<= 1) {
      const u64 x = shfl_up64(inc, off), y = shfl_up64(inc_m, off);
      if (lane >= off) {
        inc += x;
        inc_m += y;
      }
    }
    if (lane == 31) {
      s.warp_u64[warp] = inc;
      s.all_weight[warp] = inc_m;
    }
    if (threadIdx.x == 0) s.found_bin = -1;
    __syncthreads();
    u64 before = 0, before_m = 0;
    for (int w = 0; w < warp; ++w) {
      before += s.warp_u64[w];
      before_m += s.all_weight[w];
    }
    u64 ex = before + inc - mine, ex_m = before_m + inc_m - mine_m;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const u64 q = by_mass ? m[i] : c[i];
      if (ex < target && ex + q >= target) {
        s.found_bin = threadIdx.x * kPer + i;
        s.found_above = ex;        // in the target's unit
        s.found_mass = ex_m;       // weight above the bin
        s.found_count = c[i];
      }
      ex += q;
      ex_m += m[i];
    }
    __syncthreads();
  }

  // The order of the last candidate kept by a filter that keeps candidates
  // until their count (or weight) reaches `target`; `mass` gets the weight of
  // all candidates up to and including it.
  __device__ u64 last_kept(bool by_mass, u64 target, u64& mass) {
    find_bin(by_mass, target);
    const int fb = s.found_bin;
    const u64 above = s.found_above, above_m = s.found_mass;
    const uint32_t in_bin = s.found_count;
    if (fb >= 0 && in_bin <= kSampCand) {
      if (threadIdx.x == 0) s.pub_cand = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kSampThreads) {
        const float f = logit(i);
        if (bin(f) == fb) {
          const uint32_t at = atomicAdd(&s.pub_cand, 1u);
          s.cand_order[at] = order_of(f, base + i);
          s.cand_weight[at] = weight(f);
        }
      }
      cluster.sync();
      uint32_t at = 0;
      for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
        const SampleShared* o = cluster.map_shared_rank(&s, r);
        const uint32_t m = o->pub_cand;
        for (uint32_t i = threadIdx.x; i < m; i += kSampThreads) {
          s.all_order[at + i] = o->cand_order[i];
          s.all_weight[at + i] = o->cand_weight[i];
        }
        at += m;
      }
      cluster.sync();  // copied: the lists may be used again
      if (threadIdx.x < at) {
        const u64 me = s.all_order[threadIdx.x], w = s.all_weight[threadIdx.x];
        u64 before = 0, before_m = 0;
        for (uint32_t j = 0; j < at; ++j) {
          const bool earlier = s.all_order[j] > me;
          before += earlier ? 1 : 0;
          before_m += earlier ? s.all_weight[j] : 0;
        }
        const u64 ex = above + (by_mass ? before_m : before);
        const u64 q = by_mass ? w : 1;
        if (ex < target && ex + q >= target) {
          s.found_order = me;
          s.found_above = above_m + before_m + w;
        }
      }
      __syncthreads();
      mass = s.found_above;
      const u64 r = s.found_order;
      __syncthreads();
      return r;
    }
    // bisection over the order itself: the largest order whose candidates (it
    // and all earlier ones) reach the target
    u64 lo = 0, hi = ~u64(0);  // reach(lo) holds, reach(hi) does not
    u64 at_lo = 0;
    bool have = false;
    while (hi - lo > 1) {
      const u64 mid = lo + (hi - lo) / 2;
      uint32_t c = 0;
      u64 m = 0;
      for (int i = threadIdx.x; i < n; i += kSampThreads) {
        const float f = logit(i);
        if (order_of(f, base + i) >= mid) {
          ++c;
          m += weight(f);
        }
      }
      cluster_sum(c, m);
      if ((by_mass ? m : static_cast<u64>(c)) >= target) {
        lo = mid;
        at_lo = m;
        have = true;
      } else {
        hi = mid;
      }
    }
    if (!have) {  // nothing reaches it: everything is kept
      uint32_t c = 0;
      u64 m = 0;
      for (int i = threadIdx.x; i < n; i += kSampThreads) m += weight(logit(i));
      cluster_sum(c, m);
      at_lo = m;
    }
    mass = at_lo;
    return lo;
  }

  __device__ void run(int row) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ranks = static_cast<int>(cluster.num_blocks());
    const int rank = static_cast<int>(cluster.block_rank());
    if (threadIdx.x < 64) s.table[threadIdx.x] = kExp2Table[threadIdx.x];
    const float temp = a.temperature != nullptr ? a.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    inv_temp = greedy ? 1.0 : 1.0 / static_cast<double>(temp);
    const int k = greedy || a.top_k == nullptr ? 0 : a.top_k[row];
    const float p = greedy || a.top_p == nullptr ? 1.f : a.top_p[row];
    const float mp = greedy || a.min_p == nullptr ? 0.f : a.min_p[row];
    const bool use_k = k > 0 && k < a.vocab, use_p = p < 1.f;

    // ---- the row's largest and smallest finite logit -------------------------
    float mx = -INFINITY, mn = INFINITY;
    for (int i = threadIdx.x; i < n; i += kSampThreads) {
      const float f = logit(i);
      mx = fmaxf(mx, f);
      if (f > -INFINITY) mn = fminf(mn, f);
    }
    mx = warp_reduce(mx, [](float x, float y) { return fmaxf(x, y); });
    mn = warp_reduce(mn, [](float x, float y) { return fminf(x, y); });
    if (lane == 0) {
      s.warp_f32[0][warp] = mx;
      s.warp_f32[1][warp] = mn;
    }
    for (int i = threadIdx.x; i < kSampBins; i += kSampThreads)
      s.hist_count[i] = s.hist_lo[i] = s.hist_hi[i] = 0;
    __syncthreads();
    if (warp == 0) {
      mx = warp_reduce(s.warp_f32[0][lane], [](float x, float y) { return fmaxf(x, y); });
      mn = warp_reduce(s.warp_f32[1][lane], [](float x, float y) { return fminf(x, y); });
      if (lane == 0) {
        s.pub_max = mx;
        s.pub_min = mn;
      }
    }
    cluster.sync();
    top = -INFINITY;
    mn = INFINITY;
    for (int r = 0; r < ranks; ++r) {
      top = fmaxf(top, *cluster.map_shared_rank(&s.pub_max, r));
      mn = fminf(mn, *cluster.map_shared_rank(&s.pub_min, r));
    }
    if (top == -INFINITY) {  // nothing to draw from (the same for every CTA)
      if (rank == 0 && threadIdx.x == 0) {
        a.ids[row] = -1;
        if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
      }
      cluster.sync();
      return;
    }
    // bins span the finite logits, at most 64 T (weights below e^-64 vanish)
    const float span = fminf(top - mn, fmaxf(64.f * temp, 32.f));
    bin_scale = span > 0.f && span < INFINITY ? (kSampBins - 1) / span : 0.f;

    // ---- weights of all candidates, and the histogram --------------------------
    u64 total = 0;
    const bool want_hist = use_k || use_p;
    const bool want_total = a.logprobs != nullptr || use_p || (!use_k && !greedy);
    if (want_hist || want_total) {
      for (int i = threadIdx.x; i < n; i += kSampThreads) {
        const float f = logit(i);
        const u64 w = weight(f);
        total += w;
        if (want_hist) {
          const int bn = bin(f);
          atomicAdd(&s.hist_count[bn], 1u);
          if (w != 0) {
            const uint32_t lo = static_cast<uint32_t>(w);
            const uint32_t old = atomicAdd(&s.hist_lo[bn], lo);
            const uint32_t hi = static_cast<uint32_t>(w >> 32) + (old + lo < old ? 1u : 0u);
            if (hi) atomicAdd(&s.hist_hi[bn], hi);
          }
        }
      }
      uint32_t none = 0;
      cluster_sum(none, total);  // its barriers also complete the histogram
    }
    u64 last = 0, mass = total;  // everything is kept
    if (use_k) last = last_kept(false, static_cast<u64>(k), mass);
    if (use_p) {
      // kept while the weight before a candidate is below p * mass
      const double want = static_cast<double>(p) * static_cast<double>(mass);
      const u64 target = max(u64(1), min(mass, static_cast<u64>(ceil(want))));
      u64 unused;
      last = max(last, last_kept(true, target, unused));
    }
    const double least = static_cast<double>(mp) * 17592186044416.0;  // min_p in units of 2^-44

    // ---- the draw: running sums in index order ---------------------------------
    const int seg = (n + kSampThreads - 1) / kSampThreads * 32;  // of a warp, within the slice
    const int s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
    auto kept = [&](int i) -> u64 {
      const float f = logit(i);
      if (greedy) return f == top ? 1 : 0;
      if (last != 0 && order_of(f, base + i) < last) return 0;
      const u64 w = weight(f);
      return static_cast<double>(w) >= least || f == top ? w : 0;
    };
    u64 sum = 0;
    for (int i = s0 + lane; i < s1; i += 32) sum += kept(i);
    sum = warp_reduce(sum, [](u64 x, u64 y) { return x + y; });
    if (lane == 0) s.warp_u64[warp] = sum;
    __syncthreads();
    u64 before = 0, mine = 0;  // before this warp, within the CTA
    for (int w = 0; w < kSampWarps; ++w) {
      if (w < warp) before += s.warp_u64[w];
      mine += s.warp_u64[w];
    }
    if (threadIdx.x == 0) s.pub_mass = mine;
    cluster.sync();
    u64 whole = 0;
    for (int r = 0; r < ranks; ++r) {
      const u64 m = *cluster.map_shared_rank(&s.pub_mass, r);
      if (r < rank) before += m;
      whole += m;
    }
    // the token is the first whose running sum exceeds u * whole
    const double u = greedy ? 0.0 : static_cast<double>(a.uniforms[row]);
    u64 target = static_cast<u64>(fmax(u, 0.0) * static_cast<double>(whole));
    if (target >= whole) target = whole - 1;
    if (before <= target && before + sum > target) {  // in this warp's segment
      u64 run_sum = before;
      for (int i0 = s0; i0 < s1; i0 += 32) {
        const int i = i0 + lane;
        const u64 w = i < s1 ? kept(i) : 0;
        u64 inc = w;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const u64 x = shfl_up64(inc, off);
          if (lane >= off) inc += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, run_sum + inc > target);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            a.ids[row] = base + i;
            if (a.logprobs != nullptr) {
              const float f = logit(i);
              const double z = f == top ? 0.0
                                        : (static_cast<double>(f) - static_cast<double>(top)) * inv_temp;
              a.logprobs[row] =
                  static_cast<float>(z - log(static_cast<double>(total) * 0x1p-44));
            }
          }
          break;
        }
        run_sum += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
  }
};

template <typename T>
__global__ void __launch_bounds__(kSampThreads, 1) sample_tokens_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(s_raw);
  T* slice = reinterpret_cast<T*>(s_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  Sampler<T> job(a, s, slice);
  const int rank = static_cast<int>(job.cluster.block_rank());
  const int row = blockIdx.x / job.cluster.num_blocks();
  job.base = min(a.vocab, rank * a.slice);
  job.n = min(a.slice, a.vocab - job.base);
  const T* src = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.row_stride + job.base;
  constexpr int kVec = 16 / sizeof(T);
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int nv = job.n / kVec;
    for (int i = threadIdx.x; i < nv; i += kSampThreads)
      reinterpret_cast<uint4*>(slice)[i] = reinterpret_cast<const uint4*>(src)[i];
    for (int i = nv * kVec + threadIdx.x; i < job.n; i += kSampThreads) slice[i] = src[i];
  } else {
    for (int i = threadIdx.x; i < job.n; i += kSampThreads) slice[i] = src[i];
  }
  __syncthreads();
  job.run(row);
}

template <typename T>
cudaError_t launch_sample(SampleArgs a, int batch, cudaStream_t stream) {
  static unsigned long long configured = 0;  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  constexpr int kFixed = (sizeof(SampleShared) + 15) / 16 * 16;
  if (dev >= 64 || !(configured & (1ull << dev))) {
    e = cudaFuncSetAttribute(sample_tokens_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kFixed + kSampSliceBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) configured |= 1ull << dev;
  }
  // CTAs of a row: as many as hold its logits; more while SMs would be idle
  // and every CTA keeps a few thousand logits
  int ctas = 1;
  auto slice_of = [&](int c) { return ((a.vocab + c - 1) / c + 15) / 16 * 16; };
  while (ctas < kSampMaxCluster && static_cast<int64_t>(slice_of(ctas)) * sizeof(T) > kSampSliceBytes)
    ctas *= 2;
  while (ctas < kSampMaxCluster && batch * ctas * 2 <= num_sms_current_device() &&
         slice_of(ctas) > 8192)
    ctas *= 2;
  a.slice = slice_of(ctas);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * ctas));
  cfg.blockDim = dim3(kSampThreads);
  cfg.dynamicSmemBytes = kFixed + static_cast<size_t>(a.slice) * sizeof(T);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T>, a);
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
                        min_p,  ids,        logprobs, vocab,       0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (dtype) {
    case HELM_DTYPE_BF16:
      e = launch_sample<__nv_bfloat16>(a, batch, s);
      break;
    case HELM_DTYPE_FP16:
      e = launch_sample<__half>(a, batch, s);
      break;
    case HELM_DTYPE_FP32:
      e = launch_sample<float>(a, batch, s);
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
