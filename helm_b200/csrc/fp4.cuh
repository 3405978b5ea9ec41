// The 4-bit K/V format: e2m1 values in blocks of 16 along the head dim, one
// e4m3 scale per block, and the byte layout of a tile of 16 tokens.
//
//   s     = e4m3(max|x| / 6)             (round to nearest even, saturating)
//   code  = nearest of 0 .5 1 1.5 2 3 4 6 (and negatives) to x / s, ties to even
//   value = code * s
// Both factors are short (2 and 4 significant bits), so every value is exact in
// fp16 and in bf16 and the dequantising multiply rounds nothing.
//
// Tile of 16 tokens of one KV head, 18 * D bytes (4.5 bits a value):
//   [0, 8D)    K codes   [8D, 16D)  V codes    16 rows of D/2 bytes each
//   [16D, 17D) K scales  [17D, 18D) V scales
// Code byte i of a row holds dims 2i (low four bits) and 2i + 1.  The order of
// rows and chunks is chosen so that the decode kernel's shared-memory reads are
// free of bank conflicts with no padding (a bulk copy lands the tile as it is):
//   * token t's row is row t ^ x, x = (bit 2 of t) << 1 | (bit 3 of t);
//   * K, D = 256: 16-byte chunk j is at j ^ 4 * (t & 1);
//   * V: chunk u of D/16 bytes is at u ^ 4 * (bit 2 of t) for D = 128 and at
//     u ^ 2 * ((t >> 2) & 3) for D = 256;
//   * K scales are grouped by the lane that reads them (its dims, tokens t and
//     t + 2 together); V scales are [block][token].
#pragma once

#include "common.cuh"

namespace helm {

constexpr int kFp4TileTokens = 16;
constexpr int kFp4Block = 16;  // values that share a scale

template <int D>
struct Fp4Tile {
  static constexpr int kBytes = 18 * D;
  static constexpr int kRow = D / 2;       // code bytes of a token
  static constexpr int kV = 8 * D;         // V codes
  static constexpr int kKScale = 16 * D;
  static constexpr int kVScale = 17 * D;

  __device__ __forceinline__ static int row_of(int t) {
    return t ^ (((t >> 1) & 2) | ((t >> 3) & 1));
  }
  // byte offset of K code byte i of token t
  __device__ __forceinline__ static int k_code(int t, int i) {
    return row_of(t) * kRow + (D == 256 ? i ^ (64 * (t & 1)) : i);
  }
  // XOR applied to a V chunk index of token t
  __device__ __forceinline__ static int v_turn(int t) {
    return D == 128 ? 4 * ((t >> 2) & 1) : (D == 256 ? 2 * ((t >> 2) & 3) : 0);
  }
  __device__ __forceinline__ static int v_code(int t, int i) {
    constexpr int kChunk = D / 16;
    return kV + row_of(t) * kRow + ((i / kChunk) ^ v_turn(t)) * kChunk + i % kChunk;
  }
  __device__ __forceinline__ static int k_scale(int t, int g) {
    const int c = D == 64 ? g : (D == 128 ? g >> 1 : (g & 7) >> 1);
    const int k = D == 64 ? 0 : (D == 128 ? g & 1 : ((g & 1) | ((g >> 3) << 1)));
    const int pair = ((t >> 2) << 1) | (t & 1);
    return kKScale + (pair * 4 + c) * (D / 32) + ((t >> 1) & 1) * (D / 64) + k;
  }
  __device__ __forceinline__ static int v_scale(int t, int g) { return kVScale + g * 16 + t; }
};

// Eight values of a register (four bytes of codes) as four f16x2 registers.
__device__ __forceinline__ void fp4x8_to_half(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

// Eight fp32 values rounded to e2m1 (nearest, ties to even, saturating at 6).
__device__ __forceinline__ uint32_t float8_to_fp4(const float (&x)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return w;
}

// Two e4m3 scales (low 16 bits) as f16x2.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
      : "=r"(h)
      : "r"(two));
  return h;
}

__device__ __forceinline__ uint32_t float_to_e4m3(float x) {
  uint32_t r;
  asm("{\n\t.reg .b16 p;\n\tcvt.rn.satfinite.e4m3x2.f32 p, %2, %1;\n\tcvt.u32.u16 %0, p;\n\t}"
      : "=r"(r)
      : "f"(x), "f"(0.f));
  return r & 0xffu;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a),
                            *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// A scale of the whole cache must be a power of two: then dividing by it on the
// way in and multiplying by it on the way out round nothing.
inline bool fp4_scale_ok(float s) {
  int e;
  return s > 0.f && s <= 0x1p60f && s >= 0x1p-60f && frexpf(s, &e) == 0.5f;
}

}  // namespace helm
