// Decode attention over the 4-bit page pool (layout and format: fp4.cuh).
//
// The single-token attention of paged_attention.cu for a cache that holds 4.5
// bits a value: 18 * D bytes bring 16 tokens of K and V, 3.56x fewer than the
// 16-bit pool.  HELM has no counterpart (its cache is in the model's dtype,
// helm/runtime/kv_cache.py:405-662).
//
// The bound is HBM, but not by much: at the measured copy rate a tile of D =
// 128 (2304 bytes) arrives on an SM about every 100 cycles, i.e. every 400
// issue slots of its four schedulers, and has 4096 values to widen.  So the
// kernel is built around few instructions per value:
//   * cvt.rn.f16x2.e2m1x2 widens two values, one HMUL2 applies their scale
//     (exact: see fp4.cuh); both matrix products run as fp16 mma.sync m16n8k16
//     with fp32 accumulation.  tcgen05's fp16 kind would need the widened tile
//     written back to shared memory for its operand, more work than the product
//     itself; its block-scaled FP4 kind takes K as it lies, but wants q as a sum of
//     FP4 numbers, and has no place for V, whose blocks run along the other axis.
//   * The reduction index of a product may be taken in any order, so a lane
//     reads 16 contiguous bytes of a K row (32 dims) as its A fragments of all
//     eight k-steps, and a V chunk's dims as its rows of all m-tiles; the
//     tile's layout makes those reads conflict-free.
//   * V fragments pair two tokens of one dim.  Nibbles of two token words are
//     interleaved before widening (four logic ops per 16 values).
//   * P is taken against a reference that lies 2^11 below the running maximum and
//     moves only when a P would exceed 2^15, fp16's last binade: a unit normally
//     costs one vote instead of a max reduction and a rescale of O, and weights
//     down to 2^-25 of the largest keep all of fp16's bits.
//   * Work goes by UNITS of two tiles (32 tokens): their chains of LDS, cvt,
//     mma and exp2 are independent, and waits, votes and bookkeeping are paid
//     once for both.
// q is scaled per head by a power of two into fp16's range.  P is rounded to
// fp16 where O is bf16 (half a step 2^-8): it is off by 2^-11 of itself, or by 2^-36
// of the largest where that is more; where O is fp16 itself it is carried as the sum
// of two fp16 numbers (2^-22, the same floor), the second in a product's idle
// columns where there are enough.  The sum l and all state are fp32.
//
// All units of all (sequence, KV head) pairs lie in one flattened order, cut into
// equal contiguous ranges, one per warp (paged_attention.cu's split).  A warp's
// ring of bulk copies is its own (its next copy is issued by the warp itself
// once the stage is read), so no producer warp and no empty barriers are
// needed.  Pairs split across warps are merged by a programmatic-dependent
// kernel.
#include "common.cuh"
#include "fp4.cuh"

namespace helm {
namespace {

struct DecodeFp4Args {
  const void* q;
  int64_t q_sb, q_sh;
  const uint8_t* pool;
  int64_t pool_pages;
  const int32_t* page_table;
  int64_t pt_sb;
  int most;  // tokens that a row of the table, and of the mask, can describe
  const int32_t* kv_lens;
  const void* mask;
  int mask_dtype;
  int64_t mask_sb;
  void* out;
  int64_t out_sb, out_sh;
  float* lse;
  float* part_o;   // warp partials [num_workers + pairs][G][D]
  float* part_ml;  // warp partials [num_workers + pairs][G][2]
  int batch, hq, hkv, group, page_size, tiles_per_page;
  uint32_t tpp_magic;  // x / tiles_per_page = (x * tpp_magic) >> 32, 0: shift
  int tpp_shift;
  int warps;         // workers of a CTA
  int num_workers;
  int early;         // decode overlap: the lengths and tables may be read before the wait
  float score_scale; // softmax scale x K cache scale
  float softcap, softcap_inv;
  float v_scale;
  // A state's reference m is in log2 units in the plain form (no mask, no softcap,
  // scale > 0), in natural units of the score otherwise (a mask of the type's
  // lowest value must not overflow):
  float unit_log2;   // exp2 factor of a difference of references: 1 or log2(e)
  float unit_ln;     // natural units of m: ln 2 or 1
};

constexpr float kLowest = -3.402823466e38f;
// log2 of the largest P, and of P at the maximum when the reference has just moved:
// the maximum may rise by the difference before it moves again.
constexpr float kMostP = 15.f, kTopP = 11.f;
constexpr int kUnitTokens = 2 * kFp4TileTokens;
constexpr int kFp4MaxWarps = 16;  // of a CTA (sizes the workspace)

// Shape of a CTA: warps (= workers) and ring stages (of one unit) per warp.
template <int D, int NT>
struct Fp4Shape {
  static constexpr int NCW = (D <= 128 && NT == 1) ? 16 : 8;
  static constexpr int NS = D == 64 ? 4 : (NCW == 16 ? 2 : (D == 128 ? 4 : 2));
  static constexpr int kThreads = NCW * 32;
  static constexpr int kTile = Fp4Tile<D>::kBytes;
  static constexpr int kUnit = 2 * kTile;
  static constexpr int kData = NCW * NS * kUnit;
  static constexpr size_t smem_bytes(int batch) {
    return 128 + kData + NCW * NS * sizeof(uint64_t) + (2 * batch + 1) * sizeof(int);
  }
  static_assert(NCW <= kFp4MaxWarps, "");
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh without a branch: its Taylor series to x^11 below 1/4 (next term 2e-10), else
// the identity 1 - 2 / (e^2x + 1) (3e-7 absolute).
__device__ __forceinline__ float tanh_fast(float x) {
  const float z = x * x;
  float p = fmaf(z, -1382.f / 155925.f, 62.f / 2835.f);
  p = fmaf(p, z, -17.f / 315.f);
  p = fmaf(p, z, 2.f / 15.f);
  p = fmaf(p, z, -1.f / 3.f);
  const float small = fmaf(p * z, x, x);
  const float e = exp2_fast(fabsf(x) * (2.f * kLog2e));  // inf: 1
  const float large = copysignf(1.f - __fdividef(2.f, e + 1.f), x);
  return z < 0.0625f ? small : (e == INFINITY ? copysignf(1.f, x) : large);  // NaN stays NaN
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[N]) {
  static_assert(N == 1 || N == 2 || N == 4, "");
  if (N == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[N > 1 ? 1 : 0]), "=r"(w[N > 2 ? 2 : 0]),
                   "=r"(w[N > 3 ? 3 : 0])
                 : "r"(addr));
  else if (N == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                 : "=r"(w[0]), "=r"(w[N > 1 ? 1 : 0])
                 : "r"(addr));
  else
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ uint32_t bcast_lo(uint32_t h2) { return __byte_perm(h2, h2, 0x1010); }
__device__ __forceinline__ uint32_t bcast_hi(uint32_t h2) { return __byte_perm(h2, h2, 0x3232); }

// d = a . b (no accumulator to clear first)
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32"
      " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Tokens of sequence b (a length beyond its row of the table, or of the mask, is
// cut and reported).
__device__ __forceinline__ int fp4_len(const DecodeFp4Args& a, int b) {
  const int len = a.kv_lens[b];
  if (len > a.most) {
    report_status(HELM_DEV_BAD_PAGE);
    return a.most;
  }
  return max(len, 0);
}

// s_cum[b]: units of one KV head before sequence b, s_len[b]: its tokens (one
// warp fills both).
__device__ void fp4_build_prefix(const DecodeFp4Args& a, int* s_cum, int* s_len, int lane) {
  int carry = 0;
  if (lane == 0) s_cum[0] = 0;
  for (int base = 0; base < a.batch; base += 32) {
    const int b = base + lane;
    const int len = b < a.batch ? fp4_len(a, b) : 0;
    if (s_len != nullptr && b < a.batch) s_len[b] = len;
    int v = div_up(len, kUnitTokens);
    for (int off = 1; off < 32; off <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v += n;
    }
    if (b < a.batch) s_cum[b + 1] = carry + v;
    carry += __shfl_sync(0xffffffffu, v, 31);
  }
}

__device__ __forceinline__ float fp4_mask(const DecodeFp4Args& a, int b, int tok) {
  const int64_t off = static_cast<int64_t>(b) * a.mask_sb + tok;
  if (a.mask_dtype == HELM_DTYPE_FP32) return static_cast<const float*>(a.mask)[off];
  if (a.mask_dtype == HELM_DTYPE_BF16)
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.mask)[off]);
  return __half2float(static_cast<const __half*>(a.mask)[off]);
}

template <typename T>
__device__ __forceinline__ T* fp4_out_row(const DecodeFp4Args& a, int b, int qh) {
  return static_cast<T*>(a.out) + static_cast<int64_t>(b) * a.out_sb +
         static_cast<int64_t>(qh) * a.out_sh;
}

__device__ __forceinline__ float fp4_lse(const DecodeFp4Args& a, float m, float l) {
  return l > 0.f ? m * a.unit_ln + logf(l) : (l == l ? -INFINITY : l);
}

// O of a state is kept in the order in which lanes hold it: place i is this dim.
template <int D>
__device__ __forceinline__ int fp4_state_dim(int i) {
  return (D / 8) * ((i >> 1) & 7) + 2 * (i >> 4) + (i & 1);
}

// x / y for x < 2^30 and a quotient below 2^20: the float product is at most one
// off.  The kernel divides a handful of times per warp, at its start and end,
// where nothing else runs: a general division there is microseconds in all.
__device__ __forceinline__ int fp4_div(int x, int y) {
  int q = static_cast<int>(__fdividef(static_cast<float>(x), static_cast<float>(y)));
  const int r = x - q * y;
  q += r >= y ? 1 : 0;
  q -= r < 0 ? 1 : 0;
  return q;
}

// locate() of the flattened unit order with that division.
__device__ __forceinline__ TilePos fp4_locate(const int* s_cum, int batch, int hkv, int x) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {  // largest b with s_cum[b] * hkv <= x
    const int mid = (lo + hi + 1) >> 1;
    if (s_cum[mid] * hkv <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int tb = s_cum[lo + 1] - s_cum[lo];
  const int r = x - s_cum[lo] * hkv;
  TilePos p;
  p.b = lo;
  p.h = fp4_div(r, tb);
  p.t = r - p.h * tb;
  return p;
}

// The workers vf .. vl whose ranges hold units of KV head h of sequence b.
struct Fp4Span {
  int vf, vl;
};

__device__ __forceinline__ Fp4Span fp4_span(const DecodeFp4Args& a, const int* s_cum, int W, int b,
                                            int h) {
  const int units = s_cum[b + 1] - s_cum[b], st = s_cum[b] * a.hkv + h * units;
  Fp4Span ps;
  ps.vf = fp4_div(st, W);
  ps.vl = fp4_div(st + units - 1, W);
  return ps;
}

// kFold (fp16, at most four heads a KV head): heads 0 .. 3 stand again in columns
// 4 .. 7 of the products, whose P is the low half; so the second product of a
// split P costs nothing.
template <typename T, int D, int NT, bool kPlain, bool kFold>
struct Fp4Worker {
  static constexpr int KS = D / 16;
  static constexpr bool kSplitP = std::is_same<T, __half>::value && !kFold;
  static_assert(!kFold || (NT == 1 && std::is_same<T, __half>::value), "");
  using L = Fp4Tile<D>;
  float m[NT][2];       // what P is taken against (units: see DecodeFp4Args)
  float l[NT][2];
  float o[NT][KS][4];
  uint32_t qf[NT][KS][2];
  float cx[NT][2];      // plain: dot product to log2 units; else to the natural score
  int cur_b = -1, cur_h = -1;
  // byte offsets in a tile of what this lane reads (kept: they cost more to redo)
  uint32_t kA, kB, kS, v0, v1, v2, v3, vS;

  // A lane's K rows: row i of S^T (i < 8: r, else r + 8) is token 4 (r >> 1) +
  // (r & 1) [+ 2]; its V tokens: 4c .. 4c + 3.
  __device__ __forceinline__ void lane_offsets(int lane) {
    const int r = lane >> 2, c = lane & 3;
    const int tA = 4 * (r >> 1) + (r & 1);
    const int at = D == 64 ? c * 8 : (D == 128 ? c * 16 : (c ^ (4 * (r & 1))) * 16);
    kA = L::row_of(tA) * L::kRow + at;
    kB = L::row_of(tA + 2) * L::kRow + at;
    kS = L::kKScale + lane * (D / 32);
    const int chunk = L::kV + (r ^ L::v_turn(4 * c)) * (D / 16);
    v0 = chunk + L::row_of(4 * c) * L::kRow;
    v1 = chunk + L::row_of(4 * c + 1) * L::kRow;
    v2 = chunk + L::row_of(4 * c + 2) * L::kRow;
    v3 = chunk + L::row_of(4 * c + 3) * L::kRow;
    vS = L::kVScale + (D == 64 ? r >> 1 : (D == 128 ? r : 2 * r)) * 16 + 4 * c;
    // opaque to the compiler, which would rather compute them again at every use
    asm volatile("" : "+r"(kA), "+r"(kB), "+r"(kS), "+r"(vS));
    asm volatile("" : "+r"(v0), "+r"(v1), "+r"(v2), "+r"(v3));
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[nt][j] = kLowest;
        l[nt][j] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < KS; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
    }
  }

  // First dim of k-step kk on lane column c: a lane's A fragments cover 16
  // (D = 64) or 32 contiguous dims of a K row, four per k-step.
  __device__ __forceinline__ static int q_dim(int kk, int c) {
    if (D == 64) return 16 * c + 4 * kk;
    return 128 * (kk >> 3) + 32 * c + 4 * (kk & 7);
  }

  __device__ __forceinline__ void load_q(const DecodeFp4Args& a, int b, int h, int lane) {
    const int r = lane >> 2, c = lane & 3;
    const T* qb = static_cast<const T*>(a.q) + static_cast<int64_t>(b) * a.q_sb;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int hg = kFold ? r & 3 : nt * 8 + r;
      const bool ok = hg < a.group;
      const T* qh = qb + static_cast<int64_t>(h * a.group + (ok ? hg : 0)) * a.q_sh;
      float amax = 0.f;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        const T* p = qh + q_dim(kk, c);
        qf[nt][kk][0] = ok ? *reinterpret_cast<const uint32_t*>(p) : 0u;
        qf[nt][kk][1] = ok ? *reinterpret_cast<const uint32_t*>(p + 2) : 0u;
      }
      float back = 1.f;
      if (!std::is_same<T, __half>::value) {
        // bf16 -> fp16 after a power-of-two scaling that puts the head's largest
        // |q| into [2^14, 2^15): exact down to 2^-29 of it
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float lo = __uint_as_float(qf[nt][kk][e] << 16);
            const float hi = __uint_as_float(qf[nt][kk][e] & 0xffff0000u);
            amax = fmaxf(amax, fmaxf(fabsf(lo), fabsf(hi)));
          }
        amax = warp_max_xor(amax, 1, 2);
        int up = 0;
        if (amax > 0.f && amax < INFINITY) {
          up = 14 - (static_cast<int>(__float_as_uint(amax) >> 23) - 127);
          up = min(up, 100);
        }
        const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
        back = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float lo = __uint_as_float(qf[nt][kk][e] << 16) * f;
            const float hi = __uint_as_float(qf[nt][kk][e] & 0xffff0000u) * f;
            qf[nt][kk][e] = MmaOp<__half>::pack(lo, hi);
          }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float bk = __shfl_sync(0xffffffffu, back, (2 * c + j) * 4);
        cx[nt][j] = a.score_scale * bk * (kPlain ? kLog2e : 1.f);
      }
    }
  }

  // Ends the current pair: the final output when this warp covered the whole
  // pair, else its partial state at slot worker + pair.
  __device__ __forceinline__ void flush(const DecodeFp4Args& a, bool alone, int v, int lane) {
    const int r = lane >> 2, c = lane & 3;
    const int p = cur_b * a.hkv + cur_h;
    if (kFold) {  // columns 4 .. 7 (lanes c + 2) join 0 .. 3
#pragma unroll
      for (int mt = 0; mt < KS; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][mt][e] += __shfl_xor_sync(0xffffffffu, o[0][mt][e], 2);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float lt = warp_sum_xor(l[nt][j], 4, 16);
        const int hg = nt * 8 + 2 * c + j;
        if (hg >= a.group) continue;
        if (alone) {
          const int qh = cur_h * a.group + hg;
          const float inv = lt != 0.f ? a.v_scale / lt : 0.f;
          T* po = fp4_out_row<T>(a, cur_b, qh) + r * (D / 8);
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
            po[2 * mt] = from_float<T>(o[nt][mt][j] * inv);
            po[2 * mt + 1] = from_float<T>(o[nt][mt][2 + j] * inv);
          }
          if (r == 0 && a.lse != nullptr)
            a.lse[static_cast<int64_t>(cur_b) * a.hq + qh] = fp4_lse(a, m[nt][j], lt);
        } else {
          const int64_t slot = static_cast<int64_t>(v + p) * a.group + hg;
          float* po = a.part_o + slot * D + 2 * r;
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
            *reinterpret_cast<float2*>(po + 16 * mt) = make_float2(o[nt][mt][j], o[nt][mt][2 + j]);
          if (r == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(m[nt][j], lt);
        }
      }
    }
  }

  // S^T = K . Q^T of the tile at shared address `base`.
  __device__ __forceinline__ void scores(uint32_t base, float (&s)[NT][4]) {
    constexpr int kHalves = D == 256 ? 2 : 1;  // 32-dim chunks of a lane
    constexpr int kWords = D == 64 ? 2 : 4;    // code words per chunk
    float s2[NT][4];
    uint32_t scA[2], scB[2];  // f16x2 scale pairs per chunk
    if (D == 64) {
      const uint32_t two = e4m3x2_to_half2(lds_u16(base + kS));
      scA[0] = bcast_lo(two);
      scB[0] = bcast_hi(two);
    } else if (D == 128) {
      uint32_t w[1];
      lds_words<1>(base + kS, w);
      scA[0] = e4m3x2_to_half2(w[0]);
      scB[0] = e4m3x2_to_half2(w[0] >> 16);
    } else {
      uint32_t w[2];
      lds_words<2>(base + kS, w);
      scA[0] = e4m3x2_to_half2(w[0]);
      scA[1] = e4m3x2_to_half2(w[0] >> 16);
      scB[0] = e4m3x2_to_half2(w[1]);
      scB[1] = e4m3x2_to_half2(w[1] >> 16);
    }
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
      uint32_t wa[kWords], wb[kWords];
      // the second chunk of D = 256 is 64 bytes on, modulo the row's turn
      lds_words<kWords>(base + (kA ^ (64 * hf)), wa);
      lds_words<kWords>(base + (kB ^ (64 * hf)), wb);
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint32_t ha[4], hb[4];
        fp4x8_to_half(wa[w], ha);
        fp4x8_to_half(wb[w], hb);
        const uint32_t sa = D == 64 ? scA[0] : (w < 2 ? bcast_lo(scA[hf]) : bcast_hi(scA[hf]));
        const uint32_t sb = D == 64 ? scB[0] : (w < 2 ? bcast_lo(scB[hf]) : bcast_hi(scB[hf]));
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // two k-steps per code word
          const int kk = hf * 8 + 2 * w + e;
          uint32_t af[4] = {hmul2(ha[2 * e], sa), hmul2(hb[2 * e], sb), hmul2(ha[2 * e + 1], sa),
                            hmul2(hb[2 * e + 1], sb)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (kk < 2)
              mma_f16_zero(e ? s2[nt] : s[nt], af, qf[nt][kk][0], qf[nt][kk][1]);
            else
              MmaOp<__half>::run(e ? s2[nt] : s[nt], af, qf[nt][kk][0], qf[nt][kk][1]);
          }
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
  }

  // O^T += V^T . P^T of the tile at `base`; pb: P fragments (and their low
  // halves), keep: lanes' tokens 4c .. 4c+3 that count, as f16x2 masks.  Row r
  // (r + 8) of m-tile mt is dim D/8 r + 2 mt (+ 1).
  __device__ __forceinline__ void values(uint32_t base, const uint32_t (&pb)[NT][2],
                                         const uint32_t (&pl)[NT][2], uint32_t keep01,
                                         uint32_t keep23) {
    constexpr int kWords = D / 64 < 1 ? 1 : D / 64;  // code words of a lane per token
    uint32_t w[4][kWords];
    lds_words<kWords>(base + v0, w[0]);
    lds_words<kWords>(base + v1, w[1]);
    lds_words<kWords>(base + v2, w[2]);
    lds_words<kWords>(base + v3, w[3]);
    uint32_t sc01[2], sc23[2];
    constexpr int kGroups = D == 256 ? 2 : 1;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      uint32_t sw[1];
      lds_words<1>(base + vS + g * 16, sw);
      sc01[g] = e4m3x2_to_half2(sw[0]) & keep01;
      sc23[g] = e4m3x2_to_half2(sw[0] >> 16) & keep23;
    }
#pragma unroll
    for (int q = 0; q < kWords; ++q) {
      constexpr uint32_t kLo = 0x0f0f0f0fu, kHi = 0xf0f0f0f0u;
      uint32_t e01[4], d01[4], e23[4], d23[4];
      fp4x8_to_half((w[0][q] & kLo) | ((w[1][q] << 4) & kHi), e01);  // even dims of tokens 0, 1
      fp4x8_to_half(((w[0][q] >> 4) & kLo) | (w[1][q] & kHi), d01);  // odd dims
      fp4x8_to_half((w[2][q] & kLo) | ((w[3][q] << 4) & kHi), e23);
      fp4x8_to_half(((w[2][q] >> 4) & kLo) | (w[3][q] & kHi), d23);
      const int g = D == 256 ? q >> 1 : 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t af[4] = {hmul2(e01[b], sc01[g]), hmul2(d01[b], sc01[g]), hmul2(e23[b], sc23[g]),
                          hmul2(d23[b], sc23[g])};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          MmaOp<__half>::run(o[nt][4 * q + b], af, pb[nt][0], pb[nt][1]);
          if (kSplitP) MmaOp<__half>::run(o[nt][4 * q + b], af, pl[nt][0], pl[nt][1]);
        }
      }
    }
  }

  // One unit at shared address `base`.  kFull: all of its 32 tokens exist and
  // no mask is given; else its first token is tok0 and `valid` (1 .. 32) exist.
  template <bool kFull>
  __device__ __forceinline__ void unit(const DecodeFp4Args& a, uint32_t base, int valid, int tok0,
                                       int lane) {
    // mask values of this lane's tokens (rows A and B of both tiles): asked for
    // before the products, used after them
    float mask[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    const bool masked = !kFull && !kPlain && a.mask != nullptr;
    if (masked) {
      const int r = lane >> 2, first = 4 * (r >> 1) + (r & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = (i >> 1) * kFp4TileTokens + first + 2 * (i & 1);
        mask[i >> 1][i & 1] = t < valid ? fp4_mask(a, cur_b, tok0 + t) : -INFINITY;
      }
    }
    float s[2][NT][4];
    scores(base, s[0]);
    scores(base + L::kBytes, s[1]);
    uint32_t keep01[2] = {0xffffffffu, 0xffffffffu}, keep23[2] = {0xffffffffu, 0xffffffffu};
    if (!kPlain) {
#pragma unroll
      for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = s[ti][nt][e] * cx[nt][e & 1];
            if (a.softcap > 0.f) x = a.softcap * tanh_fast(x * a.softcap_inv);
            s[ti][nt][e] = x;
          }
    }
    if (!kFull) {
      const int r = lane >> 2, c = lane & 3;
      const int tA = 4 * (r >> 1) + (r & 1), tB = tA + 2;
#pragma unroll
      for (int ti = 0; ti < 2; ++ti) {
        const int v = valid - ti * kFp4TileTokens;
        bool seeA = tA < v, seeB = tB < v;
        if (masked) {
          const float mA = mask[ti][0], mB = mask[ti][1];
          seeA = mA != -INFINITY;
          seeB = mB != -INFINITY;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              s[ti][nt][j] += mA;
              s[ti][nt][2 + j] += mB;
            }
        }
        // an excluded key contributes nothing, whatever its page holds: its score
        // is -inf and its V scales are cleared (codes are finite, scales may be NaN)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (!seeA) s[ti][nt][j] = -INFINITY;
            if (!seeB) s[ti][nt][2 + j] = -INFINITY;
          }
        // token 4c + i is row r' = 2c + (i & 1) of A (i < 2) or B: lane 4 r'
        const unsigned eA = __ballot_sync(0xffffffffu, seeA);
        const unsigned eB = __ballot_sync(0xffffffffu, seeB);
        keep01[ti] =
            ((eA >> (8 * c)) & 1 ? 0x0000ffffu : 0u) | ((eA >> (8 * c + 4)) & 1 ? 0xffff0000u : 0u);
        keep23[ti] =
            ((eB >> (8 * c)) & 1 ? 0x0000ffffu : 0u) | ((eB >> (8 * c + 4)) & 1 ? 0xffff0000u : 0u);
      }
    }
    // exponents against the reference; it moves when one exceeds kMostP
    float t[2][NT][4];
    auto exponents = [&]() {
      float hi = -1.f;
#pragma unroll
      for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[ti][nt][e];
            t[ti][nt][e] = kPlain ? fmaf(x, cx[nt][e & 1], -m[nt][e & 1])
                                  : (x - m[nt][e & 1]) * kLog2e;
            hi = fmaxf(hi, t[ti][nt][e]);
          }
      return hi;
    };
    if (__any_sync(0xffffffffu, exponents() > kMostP)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(fmaxf(s[0][nt][j], s[0][nt][2 + j]), fmaxf(s[1][nt][j], s[1][nt][2 + j]));
          mx = warp_max_xor(mx, 4, 16);
          if (kPlain) mx *= cx[nt][j];
          const float m_new = fmaxf(m[nt][j], mx - (kPlain ? kTopP : kTopP * kLn2));
          const float alpha = exp2_fast((m[nt][j] - m_new) * (kPlain ? 1.f : kLog2e));
          m[nt][j] = m_new;
          l[nt][j] *= alpha;
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
            o[nt][mt][j] *= alpha;
            o[nt][mt][2 + j] *= alpha;
          }
        }
      exponents();
    }
    uint32_t pb[2][NT][2], pl[2][NT][2];
#pragma unroll
    for (int ti = 0; ti < 2; ++ti)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = exp2_fast(t[ti][nt][e]);
        l[nt][0] += p[0] + p[2];
        l[nt][1] += p[1] + p[3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t hi = MmaOp<__half>::pack(p[2 * i], p[2 * i + 1]);
          uint32_t lo = 0;
          if (kSplitP || kFold) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            lo = MmaOp<__half>::pack(p[2 * i] - f.x, p[2 * i + 1] - f.y);
          }
          pb[ti][nt][i] = movmatrix_trans(kFold && (lane & 2) ? lo : hi);
          pl[ti][nt][i] = kSplitP ? movmatrix_trans(lo) : 0;
        }
      }
    values(base, pb[0], pl[0], keep01[0], keep23[0]);
    values(base + L::kBytes, pb[1], pl[1], keep01[1], keep23[1]);
  }
};

template <typename T, int D, int NT, bool kPlain, bool kFold>
__global__ void __launch_bounds__(Fp4Shape<D, NT>::kThreads, 1)
    paged_decode_fp4_kernel(const DecodeFp4Args a) {
  using S = Fp4Shape<D, NT>;
  constexpr int NCW = S::NCW, NS = S::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128 - (smem_addr(smem_raw) & 127)) & 127);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kData);
  int* s_cum = reinterpret_cast<int*>(bars + NCW * NS);
  int* s_len = s_cum + a.batch + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = bars + warp * NS;
  // Always a programmatic dependent: the CTA is placed while the kernel before
  // it ends.  Without decode overlap it reads nothing before that one is done.
  if (!a.early) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 0) fp4_build_prefix(a, s_cum, s_len, lane);
  if (lane < NS) mbar_init(&full[lane], 1);
  fence_barrier_init();
  __syncthreads();
  // the merge kernel may be placed now; it waits for this grid to complete
  asm volatile("griddepcontrol.launch_dependents;");

  // As in paged_decode_kernel: with decode overlap this grid may run before the
  // kernel before it has finished; up to the wait it reads lengths, the page
  // table and tiles outside each sequence's last page only.
  const int total = s_cum[a.batch] * a.hkv;
  const int W = total > 0 ? div_up(total, a.num_workers) : 0;
  const int v = blockIdx.x * a.warps + warp;
  const int64_t first64 = static_cast<int64_t>(v) * W;
  const int first = first64 < total ? static_cast<int>(first64) : total;
  const int my_len = min(W, total - first);
  const uint32_t ring = smem_addr(smem) + warp * NS * S::kUnit;

  // Lane 2i + j of a window of 16 units holds the source of tile j of unit i
  // (nullptr where there is none), one window ahead of the copies.
  auto page_of = [&](int tile) {
    return a.tpp_magic == 0 ? tile >> a.tpp_shift
                            : static_cast<int>(__umulhi(static_cast<uint32_t>(tile), a.tpp_magic));
  };
  auto tile_src = [&](int s, const uint8_t*& src, bool& tail) {
    src = nullptr;
    tail = false;
    if (s >= my_len) return;
    const TilePos p = fp4_locate(s_cum, a.batch, a.hkv, first + s);
    const int tile = 2 * p.t + (lane & 1);
    const int last = div_up(s_len[p.b], kFp4TileTokens) - 1;
    if (tile > last) return;
    const int page = page_of(tile);
    tail = page == page_of(last);
    int64_t slot = a.page_table[static_cast<int64_t>(p.b) * a.pt_sb + page];
    if (slot < 0 || slot >= a.pool_pages) {
      report_status(HELM_DEV_BAD_PAGE);
      slot = 0;
    }
    src = a.pool +
          ((slot * a.hkv + p.h) * a.tiles_per_page + (tile - page * a.tiles_per_page)) * S::kTile;
  };
  const uint8_t *src_cur, *src_nxt;
  bool tail_cur, tail_nxt;
  tile_src(lane >> 1, src_cur, tail_cur);
  // the first NS units (2 NS <= 32 lanes), then the last-page tiles among them
  unsigned have = __ballot_sync(0xffffffffu, src_cur != nullptr);
  const int two = __popc(have >> (lane & 30) & 3u);
  const bool opens = lane < 2 * NS && src_cur != nullptr;
  const uint32_t open_dst = ring + (lane >> 1) * S::kUnit + (lane & 1) * S::kTile;
  if (opens && (lane & 1) == 0) mbar_arrive_expect_tx(&full[lane >> 1], two * S::kTile);
  __syncwarp();
  if (opens && !tail_cur) bulk_load(open_dst, src_cur, S::kTile, &full[lane >> 1]);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (opens && tail_cur) bulk_load(open_dst, src_cur, S::kTile, &full[lane >> 1]);
  tile_src(16 + (lane >> 1), src_nxt, tail_nxt);

  // Pairs without tokens: zero output, LSE = -inf.
  for (int p = blockIdx.x; p < a.batch * a.hkv; p += gridDim.x) {
    const int b = p / a.hkv, h = p - b * a.hkv;
    if (s_cum[b + 1] != s_cum[b]) continue;
    for (int e = threadIdx.x; e < a.group * D; e += blockDim.x)
      fp4_out_row<T>(a, b, h * a.group + e / D)[e % D] = from_float<T>(0.f);
    if (a.lse != nullptr && threadIdx.x < a.group)
      a.lse[static_cast<int64_t>(b) * a.hq + h * a.group + threadIdx.x] = -INFINITY;
  }
  Fp4Worker<T, D, NT, kPlain, kFold> st;
  st.lane_offsets(lane);
  bool ok = true;
  int stage = 0, parity = 0;
  for (int s = 0; s < my_len;) {
    // the part of this warp's range that lies in one pair
    const TilePos pos = fp4_locate(s_cum, a.batch, a.hkv, first + s);
    st.cur_b = pos.b;
    st.cur_h = pos.h;
    st.reset();
    st.load_q(a, pos.b, pos.h, lane);
    const int units = s_cum[pos.b + 1] - s_cum[pos.b];
    const int end = min(my_len, s + units - pos.t);
    const int len = s_len[pos.b];
    // units before `whole` need no checks: all of their tokens exist and count
    const int whole = (kPlain || a.mask == nullptr) ? s + (len / kUnitTokens - pos.t) : s;
    for (int tok0 = pos.t * kUnitTokens; s < end; ++s, tok0 += kUnitTokens) {
      if (!__all_sync(0xffffffffu, mbar_try_wait(&full[stage], parity))) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], parity));
        if (!ok) break;
      }
      const uint32_t at = ring + stage * S::kUnit;
      if (s < whole)
        st.template unit<true>(a, at, kUnitTokens, tok0, lane);
      else
        st.template unit<false>(a, at, min(kUnitTokens, len - tok0), tok0, lane);
      __syncwarp();
      const int nx = s + NS;  // the stage is read: its next unit
      if ((nx & 15) == 0) {
        src_cur = src_nxt;
        have = __ballot_sync(0xffffffffu, src_cur != nullptr);
        tile_src(nx + 16 + (lane >> 1), src_nxt, tail_nxt);
      }
      if (nx < my_len) {
        if (lane == 0)
          mbar_arrive_expect_tx(&full[stage], (have >> (2 * (nx & 15)) & 2u) ? S::kUnit : S::kTile);
        __syncwarp();
        if ((lane >> 1) == (nx & 15) && src_cur != nullptr)
          bulk_load(at + (lane & 1) * S::kTile, src_cur, S::kTile, &full[stage]);
      }
      if (++stage == NS) {
        stage = 0;
        parity ^= 1;
      }
    }
    if (!ok) break;
    const Fp4Span ps = fp4_span(a, s_cum, W, st.cur_b, st.cur_h);
    st.flush(a, ps.vf == ps.vl, v, lane);
  }
  // A wait that gave up leaves copies in flight into this CTA's shared memory:
  // wait (bounded) for those of this warp before it ends.
  if (!ok) {
    for (int i = 0; i < NS; ++i) {
      if (!mbar_wait(&full[stage], parity)) break;
      if (++stage == NS) {
        stage = 0;
        parity ^= 1;
      }
    }
  }
}

// Merges the pairs whose units were split across warps.  A CTA owns 32 places of
// the row of one query head of one pair: eight threads cover them, the 32 groups
// of eight take disjoint subsets of the sources, all loads in flight at once,
// each against its own maximum, and meet in shared memory.  (Combining the warps
// of a CTA in shared memory first was slower: that put 2.2 us behind the last
// unit, the larger merge here costs less.)
constexpr int kFp4MergeThreads = 256;
constexpr int kFp4MergeCols = 8;  // float4 places of a CTA

template <typename T, int D>
__global__ void __launch_bounds__(kFp4MergeThreads) merge_fp4_kernel(const DecodeFp4Args a) {
  constexpr int kGroups = kFp4MergeThreads / kFp4MergeCols, kBatch = 5;
  constexpr int kParts = 8;  // threads that add up the groups of one float4
  extern __shared__ int s_cum_m[];
  __shared__ float4 s_acc[kGroups][kFp4MergeCols];
  __shared__ float2 s_ml[kGroups];
  asm volatile("griddepcontrol.launch_dependents;");
  const int p = blockIdx.x, hg = blockIdx.y, col0 = blockIdx.z * kFp4MergeCols;
  const int b = p / a.hkv, h = p - b * a.hkv, G = a.group;
  // the lengths were there before the decode kernel's wait, hence before this
  // kernel could be placed
  if (threadIdx.x < 32) fp4_build_prefix(a, s_cum_m, nullptr, threadIdx.x);
  __syncthreads();
  const int total = s_cum_m[a.batch] * a.hkv;
  const int W = total > 0 ? div_up(total, a.num_workers) : 1;
  const Fp4Span ps = fp4_span(a, s_cum_m, W, b, h);
  const int K = s_cum_m[b + 1] == s_cum_m[b] || ps.vf == ps.vl ? 0 : ps.vl - ps.vf + 1;
  // every thread waits, also those with nothing to merge: this grid must not
  // complete before the decode kernel
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (K == 0) return;
  const int64_t slot0 = static_cast<int64_t>(ps.vf + p) * G + hg;  // source k: k * G further
  const int el = threadIdx.x % kFp4MergeCols, grp = threadIdx.x / kFp4MergeCols;
  const float2* src_ml = reinterpret_cast<const float2*>(a.part_ml) + slot0;
  const float4* src_o = reinterpret_cast<const float4*>(a.part_o) + slot0 * (D / 4) + col0 + el;
  float top = kLowest, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = grp; k0 < K; k0 += kGroups * kBatch) {
    float2 ml[kBatch];
    float4 o[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int k = k0 + i * kGroups;
      ml[i] = make_float2(kLowest, 0.f);
      o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < K) {
        const int64_t at = static_cast<int64_t>(k) * G;
        ml[i] = __ldcg(src_ml + at);
        o[i] = __ldcg(src_o + at * (D / 4));
      }
    }
    float t = top;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) t = fmaxf(t, ml[i].x);
    const float f = exp2_fast((top - t) * a.unit_log2);
    top = t;
    sum *= f;
    acc.x *= f;
    acc.y *= f;
    acc.z *= f;
    acc.w *= f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float w = exp2_fast((ml[i].x - top) * a.unit_log2);
      sum = fmaf(w, ml[i].y, sum);
      acc.x = fmaf(w, o[i].x, acc.x);
      acc.y = fmaf(w, o[i].y, acc.y);
      acc.z = fmaf(w, o[i].z, acc.z);
      acc.w = fmaf(w, o[i].w, acc.w);
    }
  }
  s_acc[grp][el] = acc;
  if (el == 0) s_ml[grp] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x >= kFp4MergeCols * kParts) return;  // whole warps
  const int e2 = threadIdx.x / kParts, part = threadIdx.x % kParts;
  float2 ml[kGroups / kParts];
  top = kLowest;
#pragma unroll
  for (int i = 0; i < kGroups / kParts; ++i) {
    ml[i] = s_ml[part + i * kParts];
    top = fmaxf(top, ml[i].x);
  }
  top = warp_max_xor(top, 1, kParts / 2);
  sum = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kGroups / kParts; ++i) {
    const float w = exp2_fast((ml[i].x - top) * a.unit_log2);
    const float4 x = s_acc[part + i * kParts][e2];
    sum = fmaf(w, ml[i].y, sum);
    acc.x = fmaf(w, x.x, acc.x);
    acc.y = fmaf(w, x.y, acc.y);
    acc.z = fmaf(w, x.z, acc.z);
    acc.w = fmaf(w, x.w, acc.w);
  }
  sum = warp_sum_xor(sum, 1, kParts / 2);
  acc.x = warp_sum_xor(acc.x, 1, kParts / 2);
  acc.y = warp_sum_xor(acc.y, 1, kParts / 2);
  acc.z = warp_sum_xor(acc.z, 1, kParts / 2);
  acc.w = warp_sum_xor(acc.w, 1, kParts / 2);
  if (part != 0) return;
  const int qh = h * G + hg, place = (col0 + e2) * 4;
  const float inv = sum != 0.f ? a.v_scale / sum : 0.f;
  T* out = fp4_out_row<T>(a, b, qh);
  T* lo = out + fp4_state_dim<D>(place);
  T* hi = out + fp4_state_dim<D>(place + 2);
  lo[0] = from_float<T>(acc.x * inv);
  lo[1] = from_float<T>(acc.y * inv);
  hi[0] = from_float<T>(acc.z * inv);
  hi[1] = from_float<T>(acc.w * inv);
  if (place == 0 && a.lse != nullptr)
    a.lse[static_cast<int64_t>(b) * a.hq + qh] = fp4_lse(a, top, sum);
}

// ----------------------------------------------------------------- host side --
template <typename T, int D, int NT, bool kPlain, bool kFold = false>
cudaError_t launch_decode_fp4(DecodeFp4Args a, int64_t max_units, cudaStream_t stream) {
  using S = Fp4Shape<D, NT>;
  static unsigned long long configured = 0;  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(configured & (1ull << dev))) {
    e = cudaFuncSetAttribute(paged_decode_fp4_kernel<T, D, NT, kPlain, kFold>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(S::smem_bytes(kMaxBatch)));
    if (e != cudaSuccess) return e;
    if (dev < 64) configured |= 1ull << dev;
  }
  // one unit per warp where there are few: first over SMs, then over warps
  const int sms = num_sms_current_device();
  a.warps = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(S::NCW, max_units / sms)));
  const int grid = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(sms, (max_units + a.warps - 1) / a.warps)));
  a.num_workers = grid * a.warps;
  a.early = decode_overlap_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = stream;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(a.warps * 32);
  cfg.dynamicSmemBytes = S::smem_bytes(a.batch);
  e = cudaLaunchKernelEx(&cfg, paged_decode_fp4_kernel<T, D, NT, kPlain, kFold>, a);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch * a.hkv), static_cast<unsigned>(a.group),
                     D / 4 / kFp4MergeCols);
  cfg.blockDim = dim3(kFp4MergeThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(a.batch + 1) * sizeof(int);
  return cudaLaunchKernelEx(&cfg, merge_fp4_kernel<T, D>, a);
}

template <typename T, int D>
cudaError_t dispatch_decode_fp4_nt(const DecodeFp4Args& a, bool plain, int64_t units,
                                   cudaStream_t s) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  if (kHalf && a.group <= 4)  // 16 x 2k tokens, one head a KV head: 50.2 us, two products 53.9
    return plain ? launch_decode_fp4<T, D, 1, true, kHalf>(a, units, s)
                 : launch_decode_fp4<T, D, 1, false, kHalf>(a, units, s);
  if (a.group <= 8)
    return plain ? launch_decode_fp4<T, D, 1, true>(a, units, s)
                 : launch_decode_fp4<T, D, 1, false>(a, units, s);
  return plain ? launch_decode_fp4<T, D, 2, true>(a, units, s)
               : launch_decode_fp4<T, D, 2, false>(a, units, s);
}

template <typename T>
cudaError_t dispatch_decode_fp4(int head_dim, const DecodeFp4Args& a, bool plain, int64_t units,
                                cudaStream_t s) {
  switch (head_dim) {
    case 64:
      return dispatch_decode_fp4_nt<T, 64>(a, plain, units, s);
    case 128:
      return dispatch_decode_fp4_nt<T, 128>(a, plain, units, s);
    default:
      return dispatch_decode_fp4_nt<T, 256>(a, plain, units, s);
  }
}

// Workspace: warp partials, O then (m, l), 256-byte aligned regions.
struct Fp4Workspace {
  int64_t o, ml;
  Fp4Workspace(int batch, int hq, int hkv, int d) {
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t slots = static_cast<int64_t>(num_sms_current_device()) * kFp4MaxWarps +
                          static_cast<int64_t>(batch) * hkv;
    o = up(slots * (hq / hkv) * d * 4);
    ml = up(slots * (hq / hkv) * 8);
  }
  int64_t total() const { return o + ml; }
};

}  // namespace
}  // namespace helm

extern "C" int64_t helm_paged_decode_fp4_workspace_bytes(int batch, int num_q_heads,
                                                         int num_kv_heads, int head_dim) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0) return 0;
  return helm::Fp4Workspace(batch, num_q_heads, num_kv_heads, head_dim).total();
}

extern "C" int helm_paged_decode_attention_fp4(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* kv_pool, int64_t pool_pages,
    const int32_t* page_table, int64_t pt_stride_b, int max_pages, const int32_t* kv_lens,
    const void* mask, int mask_dtype, int64_t mask_stride_b, int64_t mask_len, void* out,
    int64_t out_stride_b, int64_t out_stride_h, float* lse, void* workspace, int64_t workspace_bytes, int batch,
    int num_q_heads, int num_kv_heads, int head_dim, int page_size, int dtype, float scale,
    float softcap, float k_scale, float v_scale, int max_kv_len_hint, void* stream) {
  using namespace helm;
  if (q == nullptr || kv_pool == nullptr || page_table == nullptr || kv_lens == nullptr ||
      out == nullptr || workspace == nullptr)
    return HELM_ERR_INVALID_ARGUMENT;
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || page_size <= 0 || max_pages < 0 ||
      pool_pages <= 0 || num_q_heads % num_kv_heads != 0)
    return HELM_ERR_INVALID_ARGUMENT;
  if (!fp4_scale_ok(k_scale) || !fp4_scale_ok(v_scale)) return HELM_ERR_INVALID_ARGUMENT;
  if (mask != nullptr && mask_len < 0) return HELM_ERR_INVALID_ARGUMENT;
  if (mask != nullptr && mask_dtype != HELM_DTYPE_FP32 && mask_dtype != HELM_DTYPE_BF16 &&
      mask_dtype != HELM_DTYPE_FP16)
    return HELM_ERR_INVALID_ARGUMENT;
  const int group = num_q_heads / num_kv_heads;
  if (group > 16 || batch > kMaxBatch) return HELM_ERR_UNSUPPORTED;
  if (dtype != HELM_DTYPE_BF16 && dtype != HELM_DTYPE_FP16) return HELM_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return HELM_ERR_UNSUPPORTED;
  if (page_size % kFp4TileTokens != 0) return HELM_ERR_UNSUPPORTED;
  const int64_t tpp = page_size / kFp4TileTokens;
  const int64_t table_tiles = static_cast<int64_t>(batch) * max_pages * tpp * num_kv_heads;
  // tile and token positions are 32-bit
  if (table_tiles >= (int64_t(1) << 30) ||
      static_cast<int64_t>(max_pages) * page_size >= (int64_t(1) << 31))
    return HELM_ERR_UNSUPPORTED;
  // The page of tile x is (x * magic) >> 32 with magic = ceil(2^32 / tpp): the product
  // exceeds x / tpp * 2^32 by x * over / tpp, which must stay below the 1 / tpp * 2^32
  // that the tile before a page's end leaves.
  const uint64_t magic = ((uint64_t(1) << 32) + tpp - 1) / tpp;
  const uint64_t over = magic * tpp - (uint64_t(1) << 32);
  if (static_cast<uint64_t>(max_pages) * tpp * over > (uint64_t(1) << 32))
    return HELM_ERR_UNSUPPORTED;
  // q is read as 32-bit words, the pool with bulk copies (16-byte rule)
  if ((reinterpret_cast<uintptr_t>(q) & 3) || (q_stride_b & 1) || (q_stride_h & 1) ||
      (reinterpret_cast<uintptr_t>(kv_pool) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return HELM_ERR_ALIGNMENT;
  if (workspace_bytes <
      helm_paged_decode_fp4_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim))
    return HELM_ERR_WORKSPACE;
  const Fp4Workspace ws(batch, num_q_heads, num_kv_heads, head_dim);
  DecodeFp4Args a;
  a.q = q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.pool = static_cast<const uint8_t*>(kv_pool);
  a.pool_pages = pool_pages;
  a.page_table = page_table;
  a.pt_sb = pt_stride_b;
  int64_t tokens = static_cast<int64_t>(max_pages) * page_size;
  if (mask != nullptr) tokens = std::min(tokens, mask_len);
  a.most = static_cast<int>(tokens);
  a.kv_lens = kv_lens;
  a.mask = mask;
  a.mask_dtype = mask_dtype;
  a.mask_sb = mask_stride_b;
  a.out = out;
  a.out_sb = out_stride_b;
  a.out_sh = out_stride_h;
  a.lse = lse;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(w);
  a.part_ml = reinterpret_cast<float*>(w + ws.o);
  a.batch = batch;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = group;
  a.page_size = page_size;
  a.tiles_per_page = static_cast<int>(tpp);
  a.tpp_magic = 0;
  a.tpp_shift = 0;
  if ((tpp & (tpp - 1)) == 0)
    while ((int64_t(1) << a.tpp_shift) < tpp) ++a.tpp_shift;
  else
    a.tpp_magic = static_cast<uint32_t>(magic);
  const bool plain = mask == nullptr && !(softcap > 0.f) && scale > 0.f;
  a.score_scale = scale * k_scale;
  a.softcap = softcap;
  a.softcap_inv = softcap > 0.f ? 1.f / softcap : 0.f;
  a.v_scale = v_scale;
  a.unit_log2 = plain ? 1.f : kLog2e;
  a.unit_ln = plain ? kLn2 : 1.f;
  // bound on the units of the call: it sizes the grid
  if (max_kv_len_hint > 0) tokens = std::min<int64_t>(tokens, max_kv_len_hint);
  const int64_t units = (tokens + kUnitTokens - 1) / kUnitTokens * batch * num_kv_heads;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == HELM_DTYPE_BF16
                            ? dispatch_decode_fp4<__nv_bfloat16>(head_dim, a, plain, units, s)
                            : dispatch_decode_fp4<__half>(head_dim, a, plain, units, s);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}
