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
//     with fp32 accumulation.  tcgen05 would need the widened tile written
//     back to shared memory for its operand, more work than the product itself.
//   * The reduction index of a product may be taken in any order, so a lane
//     reads 16 contiguous bytes of a K row (32 dims) as its A fragments of all
//     eight k-steps, and a V chunk's dims as its rows of all m-tiles; the
//     tile's layout makes those reads conflict-free.
//   * V fragments pair two tokens of one dim.  Nibbles of two token words are
//     interleaved before widening (four logic ops per 16 values).
//   * The running maximum moves only when a score exceeds it by 8 in log2
//     units (then P <= 2^8, far inside fp16), so a tile normally costs one
//     vote instead of a max reduction and a rescale of O.
//   * q is scaled per head by a power of two into fp16's range; P is rounded
//     to fp16 (2^-12 relative); the sum l and all state stay fp32.
//
// Work split and merge follow paged_attention.cu: all tiles of all (sequence,
// KV head) pairs in one flattened order, cut into equal contiguous ranges, one
// per warp; a warp's ring of bulk copies is its own (its next copy is issued
// by the warp itself once the stage is read), so no producer warp and no empty
// barriers are needed.  States of warps that end in the same pair are combined
// in the CTA; pairs split across CTAs by a programmatic-dependent merge kernel.
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
  int max_pages;
  const int32_t* kv_lens;
  const void* mask;
  int mask_dtype;
  int64_t mask_sb;
  void* out;
  int64_t out_sb, out_sh;
  float* lse;
  float* part_o;   // warp partials [num_workers + pairs][G][D]
  float* part_ml;  // warp partials [num_workers + pairs][G][2]
  float* cta_o;    // CTA partials [grid + pairs][G][D]
  float* cta_ml;
  int batch, hq, hkv, group, page_size, tiles_per_page;
  int num_workers;
  int plain;         // no mask, no softcap, scale > 0: scores stay unscaled
  float score_scale; // softmax scale x K cache scale
  float softcap;
  float v_scale;
  // A state's maximum m is in log2 units when `plain`, in natural units of the
  // score otherwise (a mask of the type's lowest value must not overflow):
  float unit_log2;   // exp2 factor of a difference of maxima: 1 or log2(e)
  float unit_ln;     // natural units of m: ln 2 or 1
};

constexpr float kLowest = -3.402823466e38f;

// Shape of a CTA: consumer warps and ring stages per warp.
template <int D, int NT>
struct Fp4Shape {
  static constexpr int NCW = (D <= 128 && NT == 1) ? 16 : 8;
  static constexpr int NS = D == 64 ? 8 : (D == 128 && NT == 2 ? 8 : 5);
  static constexpr int kThreads = NCW * 32;
  static constexpr int kTile = Fp4Tile<D>::kBytes;
  static constexpr int kHeads = 8 * NT;
  static constexpr int kRec = 2 * kHeads + kHeads * D;  // floats of a warp's end state
  static constexpr int kRing = NCW * NS * kTile;
  static constexpr int kState = NCW * kRec * 4;
  static constexpr int kData = ((kRing > kState ? kRing : kState) + 127) / 128 * 128;
  static constexpr size_t smem_bytes(int batch) {
    return 128 + kData + NCW * NS * sizeof(uint64_t) + (batch + 1) * sizeof(int);
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

__device__ __forceinline__ int fp4_tiles_of_seq(const DecodeFp4Args& a, int b) {
  const int len = a.kv_lens[b];
  if (len <= 0) return 0;
  if (static_cast<int64_t>(len) > static_cast<int64_t>(a.max_pages) * a.page_size) {
    report_status(HELM_DEV_BAD_PAGE);
    return a.max_pages * a.tiles_per_page;
  }
  return div_up(len, kFp4TileTokens);
}

__device__ void fp4_build_prefix(const DecodeFp4Args& a, int* s_cum, int lane) {
  int carry = 0;
  if (lane == 0) s_cum[0] = 0;
  for (int base = 0; base < a.batch; base += 32) {
    const int b = base + lane;
    int v = b < a.batch ? fp4_tiles_of_seq(a, b) : 0;
    for (int off = 1; off < 32; off <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v += n;
    }
    if (b < a.batch) s_cum[b + 1] = carry + v;
    carry += __shfl_sync(0xffffffffu, v, 31);
  }
}

// Mask value of a token (0 without a mask).
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

// Where a pair's tiles lie in the flattened order (as PairSpan there).
struct Fp4Span {
  int tiles, vf, vl;
  bool last_continues;
};

__device__ __forceinline__ Fp4Span fp4_span(const int* s_cum, int hkv, int W, int total, int b,
                                            int h) {
  Fp4Span ps;
  ps.tiles = s_cum[b + 1] - s_cum[b];
  ps.vf = ps.vl = 0;
  ps.last_continues = false;
  if (ps.tiles > 0) {
    const int st = s_cum[b] * hkv + h * ps.tiles, en = st + ps.tiles;
    ps.vf = st / W;
    ps.vl = (en - 1) / W;
    ps.last_continues = static_cast<int64_t>(ps.vl + 1) * W > en && en < total;
  }
  return ps;
}

template <typename T, int D, int NT>
struct Fp4Worker {
  static constexpr int KS = D / 16;
  using L = Fp4Tile<D>;
  float m[NT][2];       // scores' units: unscaled dot products (plain) or natural
  float l[NT][2];
  float o[NT][KS][4];
  uint32_t qf[NT][KS][2];
  float xs[NT][2];      // natural score = dot * xs
  float cx[NT][2];      // exp2 factor of a difference of scores
  int cur_b = -1, cur_h = -1, cur_len = 0;

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
      const int hg = nt * 8 + r;
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
        xs[nt][j] = a.score_scale * bk;
        cx[nt][j] = a.plain ? xs[nt][j] * kLog2e : kLog2e;
      }
    }
  }

  __device__ __forceinline__ float m_unit(const DecodeFp4Args& a, int nt, int j) const {
    return a.plain ? fmaxf(m[nt][j] * cx[nt][j], kLowest) : m[nt][j];
  }

  // Ends the current pair: the final output when this warp covered the whole
  // pair, else its partial state at slot worker + pair.
  __device__ __forceinline__ void flush(const DecodeFp4Args& a, bool alone, int v, int lane) {
    const int r = lane >> 2, c = lane & 3;
    const int p = cur_b * a.hkv + cur_h;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float lt = warp_sum_xor(l[nt][j], 4, 16);
        const float mu = m_unit(a, nt, j);
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
            a.lse[static_cast<int64_t>(cur_b) * a.hq + qh] = fp4_lse(a, mu, lt);
        } else {
          const int64_t slot = static_cast<int64_t>(v + p) * a.group + hg;
          float* po = a.part_o + slot * D + r * (D / 8);
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
            *reinterpret_cast<float2*>(po + 2 * mt) = make_float2(o[nt][mt][j], o[nt][mt][2 + j]);
          if (r == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(mu, lt);
        }
      }
    }
  }

  // End state into a shared-memory record m[kHeads] | l[kHeads] | O[kHeads][D].
  __device__ __forceinline__ void save(const DecodeFp4Args& a, float* rec, int lane) {
    constexpr int kHeads = 8 * NT;
    const int r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float lt = warp_sum_xor(l[nt][j], 4, 16);
        const float mu = m_unit(a, nt, j);
        const int hg = nt * 8 + 2 * c + j;
        if (hg >= a.group) continue;
        float* po = rec + 2 * kHeads + hg * D + r * (D / 8);
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
          *reinterpret_cast<float2*>(po + 2 * mt) = make_float2(o[nt][mt][j], o[nt][mt][2 + j]);
        if (r == 0) {
          rec[hg] = mu;
          rec[kHeads + hg] = lt;
        }
      }
    }
  }

  // One tile at shared address `base`; its first token is tok0, the first
  // `valid` of its 16 tokens exist.
  __device__ __forceinline__ void tile(const DecodeFp4Args& a, uint32_t base, int valid, int tok0,
                                       int lane) {
    const int r = lane >> 2, c = lane & 3;
    // ---- S^T = K . Q^T.  Row i of the product (i < 8: r, else r + 8) is token
    // 4 (r >> 1) + (r & 1) [+ 2]: then the transposed P has the token order in
    // which a lane reads V (tokens 4c .. 4c + 3).
    const int tA = 4 * (r >> 1) + (r & 1), tB = tA + 2;
    const int turn = ((r & 2)) | (r >> 2);  // row_of(t) ^ t of both tokens
    float s[NT][4];
    {
      float s2[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
      constexpr int kHalves = D == 256 ? 2 : 1;         // 32-dim chunks of a lane
      constexpr int kWords = D == 64 ? 2 : 4;           // code words per chunk
      uint32_t scA[2], scB[2];                          // f16x2 scale pairs per chunk
      if (D == 64) {
        const uint32_t two = e4m3x2_to_half2(lds_u16(base + L::kKScale + lane * 2));
        scA[0] = bcast_lo(two);
        scB[0] = bcast_hi(two);
      } else if (D == 128) {
        uint32_t w[1];
        lds_words<1>(base + L::kKScale + lane * 4, w);
        scA[0] = e4m3x2_to_half2(w[0]);
        scB[0] = e4m3x2_to_half2(w[0] >> 16);
      } else {
        uint32_t w[2];
        lds_words<2>(base + L::kKScale + lane * 8, w);
        scA[0] = e4m3x2_to_half2(w[0]);
        scA[1] = e4m3x2_to_half2(w[0] >> 16);
        scB[0] = e4m3x2_to_half2(w[1]);
        scB[1] = e4m3x2_to_half2(w[1] >> 16);
      }
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        uint32_t wa[kWords], wb[kWords];
        const uint32_t at = D == 64 ? c * 8 : (D == 128 ? c * 16 : ((c + 4 * hf) ^ (4 * (r & 1))) * 16);
        lds_words<kWords>(base + (tA ^ turn) * L::kRow + at, wa);
        lds_words<kWords>(base + (tB ^ turn) * L::kRow + at, wb);
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
            for (int nt = 0; nt < NT; ++nt)
              MmaOp<__half>::run(e ? s2[nt] : s[nt], af, qf[nt][kk][0], qf[nt][kk][1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
    }
    // ---- scores -> probabilities ---------------------------------------------
    uint32_t keep01 = 0xffffffffu, keep23 = 0xffffffffu;  // V tokens 4c..4c+3 that count
    if (!a.plain) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[nt][e] * xs[nt][e & 1];
          if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
          s[nt][e] = x;
        }
    }
    bool seeA = true, seeB = true;
    if (valid < kFp4TileTokens) {
      seeA = tA < valid;
      seeB = tB < valid;
    }
    if (a.mask != nullptr) {
      const float mA = seeA ? fp4_mask(a, cur_b, tok0 + tA) : -INFINITY;
      const float mB = seeB ? fp4_mask(a, cur_b, tok0 + tB) : -INFINITY;
      seeA = mA != -INFINITY;
      seeB = mB != -INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[nt][j] += mA;
          s[nt][2 + j] += mB;
        }
    }
    if (__any_sync(0xffffffffu, !(seeA && seeB))) {
      // an excluded key contributes nothing, whatever its page holds: its score
      // is -inf and its V scales are cleared (codes are finite, scales may be NaN)
      const unsigned eA = __ballot_sync(0xffffffffu, seeA), eB = __ballot_sync(0xffffffffu, seeB);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!seeA) s[nt][j] = -INFINITY;
          if (!seeB) s[nt][2 + j] = -INFINITY;
        }
      // token 4c + i is row r' = 2c + (i & 1) of A (i < 2) or B: lane 4 r'
      keep01 = ((eA >> (8 * c)) & 1 ? 0x0000ffffu : 0u) | ((eA >> (8 * c + 4)) & 1 ? 0xffff0000u : 0u);
      keep23 = ((eB >> (8 * c)) & 1 ? 0x0000ffffu : 0u) | ((eB >> (8 * c + 4)) & 1 ? 0xffff0000u : 0u);
    }
    float t[NT][4];
    bool high = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        t[nt][e] = (s[nt][e] - m[nt][e & 1]) * cx[nt][e & 1];
        high |= t[nt][e] > 8.f;
      }
    if (__any_sync(0xffffffffu, high)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float mx = warp_max_xor(fmaxf(s[nt][j], s[nt][2 + j]), 4, 16);
          const float m_new = fmaxf(m[nt][j], mx);
          const float alpha = exp2_fast((m[nt][j] - m_new) * cx[nt][j]);
          m[nt][j] = m_new;
          l[nt][j] *= alpha;
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
            o[nt][mt][j] *= alpha;
            o[nt][mt][2 + j] *= alpha;
          }
          t[nt][j] = (s[nt][j] - m_new) * cx[nt][j];
          t[nt][2 + j] = (s[nt][2 + j] - m_new) * cx[nt][j];
        }
    }
    uint32_t pb0[NT], pb1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = exp2_fast(t[nt][e]);
      l[nt][0] += p[0] + p[2];
      l[nt][1] += p[1] + p[3];
      pb0[nt] = movmatrix_trans(MmaOp<__half>::pack(p[0], p[1]));
      pb1[nt] = movmatrix_trans(MmaOp<__half>::pack(p[2], p[3]));
    }
    // ---- O^T += V^T . P^T: row r (r + 8) of m-tile mt is dim D/8 r + 2 mt (+ 1)
    {
      constexpr int kWords = D / 64 < 1 ? 1 : D / 64;  // code words of a lane per token
      const int vturn = D == 128 ? 4 * (c & 1) : (D == 256 ? 2 * c : 0);
      const int x = ((c & 1) << 1) | (c >> 1);         // row_of(t) ^ t of tokens 4c + i
      const uint32_t vb = base + L::kV + 4 * c * L::kRow + (r ^ vturn) * (D / 16);
      uint32_t w[4][kWords];
#pragma unroll
      for (int i = 0; i < 4; ++i) lds_words<kWords>(vb + (i ^ x) * L::kRow, w[i]);
      uint32_t sc01[2], sc23[2];
      constexpr int kGroups = D == 256 ? 2 : 1;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        uint32_t sw[1];
        const int grp = D == 64 ? r >> 1 : (D == 128 ? r : 2 * r + g);
        lds_words<1>(base + L::kVScale + grp * 16 + 4 * c, sw);
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
          for (int nt = 0; nt < NT; ++nt) MmaOp<__half>::run(o[nt][4 * q + b], af, pb0[nt], pb1[nt]);
        }
      }
    }
  }
};

// Combines `n` states read through `get(k, m, l, o4)` for one float4 of O.
struct Fp4Sum {
  float m, l;
  float4 o;
};

__device__ __forceinline__ void fp4_fold(Fp4Sum& acc, float m, float l, float4 o, float unit) {
  const float top = fmaxf(acc.m, m);
  const float a = exp2_fast((acc.m - top) * unit), b = exp2_fast((m - top) * unit);
  acc.l = acc.l * a + l * b;
  acc.o.x = acc.o.x * a + o.x * b;
  acc.o.y = acc.o.y * a + o.y * b;
  acc.o.z = acc.o.z * a + o.z * b;
  acc.o.w = acc.o.w * a + o.w * b;
  acc.m = top;
}

template <typename T>
__device__ __forceinline__ void fp4_write(const DecodeFp4Args& a, int b, int qh, int d4,
                                          const Fp4Sum& s) {
  const float inv = s.l != 0.f ? a.v_scale / s.l : 0.f;
  T* p = fp4_out_row<T>(a, b, qh) + d4 * 4;
  p[0] = from_float<T>(s.o.x * inv);
  p[1] = from_float<T>(s.o.y * inv);
  p[2] = from_float<T>(s.o.z * inv);
  p[3] = from_float<T>(s.o.w * inv);
  if (d4 == 0 && a.lse != nullptr)
    a.lse[static_cast<int64_t>(b) * a.hq + qh] = fp4_lse(a, s.m, s.l);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Fp4Shape<D, NT>::kThreads, 1)
    paged_decode_fp4_kernel(const DecodeFp4Args a) {
  using S = Fp4Shape<D, NT>;
  constexpr int NCW = S::NCW, NS = S::NS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_endpair[NCW];
  __shared__ int s_abort;
  uint8_t* smem = smem_raw + ((128 - (smem_addr(smem_raw) & 127)) & 127);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kData);
  int* s_cum = reinterpret_cast<int*>(bars + NCW * NS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = bars + warp * NS;
  if (warp == 0) fp4_build_prefix(a, s_cum, lane);
  if (lane < NS) mbar_init(&full[lane], 1);
  fence_barrier_init();
  if (threadIdx.x == 0) s_abort = 0;
  __syncthreads();
  // the merge kernel may be placed now; it waits for this grid to complete
  asm volatile("griddepcontrol.launch_dependents;");

  // As in paged_decode_kernel: with decode overlap this grid may run before the
  // kernel before it has finished; up to the wait it reads lengths, the page
  // table and tiles outside each sequence's last page only.
  const int total = s_cum[a.batch] * a.hkv;
  const int W = total > 0 ? div_up(total, a.num_workers) : 0;
  const int v = blockIdx.x * NCW + warp;
  const int64_t first64 = static_cast<int64_t>(v) * W;
  const int first = first64 < total ? static_cast<int>(first64) : total;
  const int my_len = min(W, total - first);
  const uint32_t ring = smem_addr(smem) + warp * NS * S::kTile;

  auto tile_src = [&](int s, const uint8_t*& src, bool& tail) {
    src = a.pool;
    tail = false;
    if (s >= my_len) return;
    const TilePos p = locate(s_cum, a.batch, a.hkv, first + s);
    const int page = p.t / a.tiles_per_page;
    tail = page == (s_cum[p.b + 1] - s_cum[p.b] - 1) / a.tiles_per_page;
    int64_t slot = a.page_table[static_cast<int64_t>(p.b) * a.pt_sb + page];
    if (slot < 0 || slot >= a.pool_pages) {
      report_status(HELM_DEV_BAD_PAGE);
      slot = 0;
    }
    src = a.pool + ((slot * a.hkv + p.h) * a.tiles_per_page + (p.t - page * a.tiles_per_page)) *
                       S::kTile;
  };
  // lane i holds the source of tile 32 * window + i, one window ahead
  const uint8_t *src_cur, *src_nxt;
  bool tail_cur, tail_nxt;
  tile_src(lane, src_cur, tail_cur);
  const bool opens = lane < NS && lane < my_len;
  if (opens) {
    mbar_arrive_expect_tx(&full[lane], S::kTile);
    if (!tail_cur) bulk_load(ring + lane * S::kTile, src_cur, S::kTile, &full[lane]);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (opens && tail_cur) bulk_load(ring + lane * S::kTile, src_cur, S::kTile, &full[lane]);
  tile_src(32 + lane, src_nxt, tail_nxt);

  // Pairs without tokens: zero output, LSE = -inf.
  for (int p = blockIdx.x; p < a.batch * a.hkv; p += gridDim.x) {
    const int b = p / a.hkv, h = p - b * a.hkv;
    if (s_cum[b + 1] != s_cum[b]) continue;
    for (int e = threadIdx.x; e < a.group * D; e += blockDim.x)
      fp4_out_row<T>(a, b, h * a.group + e / D)[e % D] = from_float<T>(0.f);
    if (a.lse != nullptr && threadIdx.x < a.group)
      a.lse[static_cast<int64_t>(b) * a.hq + h * a.group + threadIdx.x] = -INFINITY;
  }
  if (blockIdx.x * static_cast<int64_t>(NCW) * W >= total) return;  // whole CTA without work

  Fp4Worker<T, D, NT> st;
  TilePos pos;
  if (my_len > 0) pos = locate(s_cum, a.batch, a.hkv, first);
  bool ok = true;
  int stage = 0, parity = 0;
  for (int s = 0; s < my_len; ++s) {
    if (pos.b != st.cur_b || pos.h != st.cur_h) {
      if (st.cur_b >= 0) {
        const Fp4Span ps = fp4_span(s_cum, a.hkv, W, total, st.cur_b, st.cur_h);
        st.flush(a, ps.vf == ps.vl, v, lane);
      }
      st.cur_b = pos.b;
      st.cur_h = pos.h;
      st.cur_len = min(a.kv_lens[pos.b], (s_cum[pos.b + 1] - s_cum[pos.b]) * kFp4TileTokens);
      st.reset();
      st.load_q(a, pos.b, pos.h, lane);
    }
    if (!mbar_wait(&full[stage], parity)) ok = false;
    if (__any_sync(0xffffffffu, !ok)) {
      ok = false;
      break;
    }
    const int tok0 = pos.t * kFp4TileTokens;
    st.tile(a, ring + stage * S::kTile, min(kFp4TileTokens, st.cur_len - tok0), tok0, lane);
    __syncwarp();
    const int nx = s + NS;  // the stage is read: its next tile
    if ((nx & 31) == 0) {
      src_cur = src_nxt;
      tile_src(nx + 32 + lane, src_nxt, tail_nxt);
    }
    if (nx < my_len && lane == (nx & 31)) {
      mbar_arrive_expect_tx(&full[stage], S::kTile);
      bulk_load(ring + stage * S::kTile, src_cur, S::kTile, &full[stage]);
    }
    advance(pos, s_cum, a.batch, a.hkv);
    if (++stage == NS) {
      stage = 0;
      parity ^= 1;
    }
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
    if (lane == 0) s_abort = 1;
  }
  __syncthreads();
  if (s_abort) return;
  // ============ merge: as paged_decode_kernel, records over the idle ring =====
  float* s_states = reinterpret_cast<float*>(smem);
  int end_pair = -1;
  if (st.cur_b >= 0) {
    end_pair = st.cur_b * a.hkv + st.cur_h;
    const Fp4Span ps = fp4_span(s_cum, a.hkv, W, total, st.cur_b, st.cur_h);
    if (ps.vf == ps.vl) {
      st.flush(a, true, v, lane);
      end_pair = -1;
    } else {
      st.save(a, s_states + warp * S::kRec, lane);
    }
  }
  if (lane == 0) s_endpair[warp] = end_pair;
  __syncthreads();
  constexpr int D4 = D / 4;
  for (int w0 = 0; w0 < NCW;) {
    const int p = s_endpair[w0];
    int w1 = w0 + 1;
    while (w1 < NCW && s_endpair[w1] == p) ++w1;
    if (p >= 0) {
      const int b = p / a.hkv, h = p - b * a.hkv;
      const Fp4Span ps = fp4_span(s_cum, a.hkv, W, total, b, h);
      const bool whole = ps.vf / NCW == ps.vl / NCW;  // the pair lies in this CTA
      for (int e = threadIdx.x; e < a.group * D4; e += S::kThreads) {
        const int hg = e / D4, d4 = e - hg * D4;
        Fp4Sum acc = {kLowest, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
        for (int w = w0; w < w1; ++w) {
          const float* rec = s_states + w * S::kRec;
          fp4_fold(acc, rec[hg], rec[S::kHeads + hg],
                   *reinterpret_cast<const float4*>(rec + 2 * S::kHeads + hg * D + d4 * 4),
                   a.unit_log2);
        }
        if (whole && ps.last_continues) {
          // the pair's last warp went on past it: its state for the pair is in
          // the warp partials (written before the barrier above)
          const int64_t slot = static_cast<int64_t>(ps.vl + p) * a.group + hg;
          const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml + slot * 2));
          fp4_fold(acc, ml.x, ml.y,
                   __ldcg(reinterpret_cast<const float4*>(a.part_o + slot * D + d4 * 4)),
                   a.unit_log2);
        }
        if (whole) {
          fp4_write<T>(a, b, h * a.group + hg, d4, acc);
        } else {
          const int64_t slot = static_cast<int64_t>(blockIdx.x + p) * a.group + hg;
          *reinterpret_cast<float4*>(a.cta_o + slot * D + d4 * 4) = acc.o;
          if (d4 == 0)
            *reinterpret_cast<float2*>(a.cta_ml + slot * 2) = make_float2(acc.m, acc.l);
        }
      }
    }
    w0 = w1;
  }
}

// Merges the pairs whose tiles were split across CTAs.  CTA (pair, chunk) owns
// kMergeElems float4 elements; its half-warps take disjoint subsets of the
// sources and meet in shared memory (see merge_split_pairs_kernel).
template <typename T, int D, int NCW>
__global__ void __launch_bounds__(kMergeThreads, 4) merge_fp4_kernel(const DecodeFp4Args a) {
  extern __shared__ int s_cum_m[];
  __shared__ float s_st[kMergeGroups][6][kMergeElems];
  asm volatile("griddepcontrol.launch_dependents;");
  const int p = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) fp4_build_prefix(a, s_cum_m, lane);
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int total = s_cum_m[a.batch] * a.hkv;
  if (total == 0) return;
  const int W = div_up(total, a.num_workers);
  const int b = p / a.hkv, h = p - b * a.hkv;
  const Fp4Span ps = fp4_span(s_cum_m, a.hkv, W, total, b, h);
  if (ps.tiles == 0 || ps.vf / NCW == ps.vl / NCW) return;  // not split across CTAs
  const int vl_end = ps.last_continues ? ps.vl - 1 : ps.vl;
  const int c0 = ps.vf / NCW, n_cta = vl_end / NCW - c0 + 1;
  const int K = n_cta + (ps.last_continues ? 1 : 0);
  const int G = a.group;
  constexpr int D4 = D / 4;
  const int el = lane & (kMergeElems - 1);
  const int grp = warp * 2 + (lane >> 4);
  const int e = blockIdx.y * kMergeElems + el;
  const bool active = e < G * D4;
  const int hg = active ? e / D4 : 0, d4 = active ? e - hg * D4 : 0;
  Fp4Sum acc = {kLowest, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int k0 = grp; active && k0 < K; k0 += kMergeGroups * 2) {
    float2 ml[2];
    float4 o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = k0 + i * kMergeGroups;
      ml[i] = make_float2(kLowest, 0.f);
      o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < K) {
        const bool cta_src = k < n_cta;
        const int64_t slot = static_cast<int64_t>((cta_src ? c0 + k : ps.vl) + p) * G + hg;
        ml[i] = __ldcg(reinterpret_cast<const float2*>((cta_src ? a.cta_ml : a.part_ml) + slot * 2));
        o[i] = __ldcg(
            reinterpret_cast<const float4*>((cta_src ? a.cta_o : a.part_o) + slot * D + d4 * 4));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) fp4_fold(acc, ml[i].x, ml[i].y, o[i], a.unit_log2);
  }
  s_st[grp][0][el] = acc.m;
  s_st[grp][1][el] = acc.l;
  s_st[grp][2][el] = acc.o.x;
  s_st[grp][3][el] = acc.o.y;
  s_st[grp][4][el] = acc.o.z;
  s_st[grp][5][el] = acc.o.w;
  __syncthreads();
  if (threadIdx.x >= kMergeElems || !active) return;
  Fp4Sum sum = {kLowest, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
  for (int g = 0; g < kMergeGroups; ++g)
    fp4_fold(sum, s_st[g][0][el], s_st[g][1][el],
             make_float4(s_st[g][2][el], s_st[g][3][el], s_st[g][4][el], s_st[g][5][el]),
             a.unit_log2);
  fp4_write<T>(a, b, h * G + hg, d4, sum);
}

// ----------------------------------------------------------------- host side --
template <typename T, int D, int NT>
cudaError_t launch_decode_fp4(DecodeFp4Args a, int64_t max_tiles, cudaStream_t stream) {
  using S = Fp4Shape<D, NT>;
  static unsigned long long configured = 0;  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(configured & (1ull << dev))) {
    e = cudaFuncSetAttribute(paged_decode_fp4_kernel<T, D, NT>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(S::smem_bytes(kMaxBatch)));
    if (e != cudaSuccess) return e;
    if (dev < 64) configured |= 1ull << dev;
  }
  const int64_t want = (max_tiles + S::NCW - 1) / S::NCW;
  const int grid = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(num_sms_current_device(), want)));
  a.num_workers = grid * S::NCW;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.stream = stream;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::smem_bytes(a.batch);
  cfg.numAttrs = decode_overlap_enabled() ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, paged_decode_fp4_kernel<T, D, NT>, a);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch * a.hkv),
                     static_cast<unsigned>((a.group * (D / 4) + kMergeElems - 1) / kMergeElems));
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(a.batch + 1) * sizeof(int);
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, merge_fp4_kernel<T, D, S::NCW>, a);
}

template <typename T>
cudaError_t dispatch_decode_fp4(int head_dim, const DecodeFp4Args& a, int64_t tiles,
                                cudaStream_t s) {
  const bool one = a.group <= 8;
  switch (head_dim) {
    case 64:
      return one ? launch_decode_fp4<T, 64, 1>(a, tiles, s) : launch_decode_fp4<T, 64, 2>(a, tiles, s);
    case 128:
      return one ? launch_decode_fp4<T, 128, 1>(a, tiles, s)
                 : launch_decode_fp4<T, 128, 2>(a, tiles, s);
    default:
      return one ? launch_decode_fp4<T, 256, 1>(a, tiles, s)
                 : launch_decode_fp4<T, 256, 2>(a, tiles, s);
  }
}

// Workspace: warp partials and CTA partials, O then (m, l) of each, 256-byte
// aligned regions.
struct Fp4Workspace {
  int64_t o, ml, cta_o, cta_ml;
  Fp4Workspace(int batch, int hq, int hkv, int d) {
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t group = hq / hkv, pairs = static_cast<int64_t>(batch) * hkv;
    const int64_t sms = num_sms_current_device();
    const int64_t warps = (sms * 16 + pairs) * group, ctas = (sms + pairs) * group;
    o = up(warps * d * 4);
    ml = up(warps * 8);
    cta_o = up(ctas * d * 4);
    cta_ml = up(ctas * 8);
  }
  int64_t total() const { return o + ml + cta_o + cta_ml; }
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
    const void* mask, int mask_dtype, int64_t mask_stride_b, void* out, int64_t out_stride_b,
    int64_t out_stride_h, float* lse, void* workspace, int64_t workspace_bytes, int batch,
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
  a.max_pages = max_pages;
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
  a.cta_o = reinterpret_cast<float*>(w + ws.o + ws.ml);
  a.cta_ml = reinterpret_cast<float*>(w + ws.o + ws.ml + ws.cta_o);
  a.batch = batch;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = group;
  a.page_size = page_size;
  a.tiles_per_page = static_cast<int>(tpp);
  a.plain = mask == nullptr && !(softcap > 0.f) && scale > 0.f ? 1 : 0;
  a.score_scale = scale * k_scale;
  a.softcap = softcap;
  a.v_scale = v_scale;
  a.unit_log2 = a.plain ? 1.f : kLog2e;
  a.unit_ln = a.plain ? kLn2 : 1.f;
  // bound on the tiles of the call: it sizes the grid
  int64_t tiles = table_tiles;
  if (max_kv_len_hint > 0)
    tiles = std::min<int64_t>(tiles, (static_cast<int64_t>(max_kv_len_hint) + 15) / 16 * batch *
                                         num_kv_heads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == HELM_DTYPE_BF16
                            ? dispatch_decode_fp4<__nv_bfloat16>(head_dim, a, tiles, s)
                            : dispatch_decode_fp4<__half>(head_dim, a, tiles, s);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}
