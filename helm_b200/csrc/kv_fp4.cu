// Append to, and read back from, the 4-bit page pool (layout: fp4.cuh).
//
// helm_kv_append_fp4 is helm_kv_append's form for 4-bit pages: RMSNorm of q and
// k, rotary embedding, page write.  HELM keeps its cache in the model's dtype
// (helm/runtime/kv_cache.py:113-171); the 4-bit form has no counterpart there.
// Everything up to the last step is fp32: q_out rounds once to its dtype, k and
// v once to 4 bits (kv_append rounds where HF's eager modules do, because its
// rows are compared with theirs bit for bit; a 4-bit row cannot be).
#include "common.cuh"
#include "fp4.cuh"

namespace helm {
namespace {

struct AppendFp4Args {
  const void* src[3];     // q, k, v: indexed by a row's kind
  int64_t st[3], sh[3];   // their token and head strides
  const void* weight[3];  // norm weights of q and k
  float eps;
  const void* cos;
  const void* sin;
  int64_t rope_st;
  void* q_out;
  int64_t qo_st, qo_sh;
  uint8_t* pool;
  int64_t pool_rows;  // pool_pages * page_size
  const int64_t* slot_rows;
  int hq, hkv, page_size;
  int page_shift;  // page_size = 1 << page_shift, or -1
  float inv[3];    // 1 / cache scale (a power of two) of k and v
};

template <typename T>
__device__ __forceinline__ void widen8(const uint4& r, float (&x)[8]) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(MmaOp<T>::pack(x[0], x[1]), MmaOp<T>::pack(x[2], x[3]),
                 MmaOp<T>::pack(x[4], x[5]), MmaOp<T>::pack(x[6], x[7]));
}

// Slot and row inside the page of a pool row (a shift or a 32-bit division where
// that does).
__device__ __forceinline__ void split_row(int64_t row, int page_size, int page_shift, int64_t& slot,
                                          int& r_in) {
  if (page_shift >= 0) {
    slot = row >> page_shift;
    r_in = static_cast<int>(row) & (page_size - 1);
  } else if (row < (int64_t(1) << 32)) {
    const uint32_t u = static_cast<uint32_t>(row), s = u / static_cast<uint32_t>(page_size);
    slot = s;
    r_in = static_cast<int>(u - s * page_size);
  } else {
    slot = row / page_size;
    r_in = static_cast<int>(row - slot * page_size);
  }
}

// log2 of a power of two, else -1.
inline int shift_of(int x) {
  int s = -1;
  if ((x & (x - 1)) == 0)
    while ((1 << ++s) < x) {
    }
  return s;
}

// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// First byte of the tile that holds pool row (slot, r_in) of KV head h.
template <int D>
__device__ __forceinline__ int64_t tile_base(int64_t slot, int r_in, int h, int hkv,
                                             int page_size) {
  return ((slot * hkv + h) * (page_size / kFp4TileTokens) + r_in / kFp4TileTokens) *
         Fp4Tile<D>::kBytes;
}

// One head row of D values on D / 8 lanes, eight values a lane (16-byte loads);
// the rows of a warp are neighbouring head rows of one token, so the row's place
// in the pool is found once per warp and needs no division by the head count.  A
// quantisation block is two neighbouring lanes.  Rows of different kinds (q, k,
// v) may share a warp, so the shuffles run for every lane and the results are
// selected; a warp of q rows alone ends before the quantising half.  Bytes per
// token: 2 (2 Hq + 2 Hkv) D + 1.125 Hkv D, but at D = 128 the instructions weigh
// more: 4096 tokens with 32/8 heads, norm and rotation take 29.5 us (3.1 TB/s; 81 %
// of the issue slots busy), about 40 with a division per row and quantised q rows.
constexpr int kFp4RowWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kFp4RowWarps * 32) kv_append_fp4_kernel(const AppendFp4Args a) {
  // programmatic dependent launch both ways, as kv_append_kernel
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tok = blockIdx.x;
  const int part = lane % kLanes;  // dims [8 part, 8 part + 8)
  const int want = (blockIdx.y * kFp4RowWarps + warp) * kRows + lane / kLanes;
  const int rows = a.hq + 2 * a.hkv;
  if ((blockIdx.y * kFp4RowWarps + warp) * kRows >= rows) return;  // the whole warp
  const bool live = want < rows;
  const int hr = live ? want : rows - 1;
  const int kind = hr < a.hq ? 0 : (hr < a.hq + a.hkv ? 1 : 2);
  const bool is_q = kind == 0, is_v = kind == 2;
  const int h = hr - (is_q ? 0 : (is_v ? a.hq + a.hkv : a.hq));
  // everything the row needs is loaded at once
  const T* w = static_cast<const T*>(a.weight[kind]);
  const bool turn = a.cos != nullptr && !is_v;
  uint4 raw_w = {}, raw_c = {}, raw_s = {};
  const uint4 raw_x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.src[kind]) +
                                                      tok * a.st[kind] + h * a.sh[kind] + part * 8);
  if (w != nullptr) raw_w = *reinterpret_cast<const uint4*>(w + part * 8);
  if (turn) {
    raw_c = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.cos) + tok * a.rope_st + part * 8);
    raw_s = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.sin) + tok * a.rope_st + part * 8);
  }
  const int64_t row = is_q ? -1 : a.slot_rows[tok];
  float x[8];
  widen8<T>(raw_x, x);
  if (__any_sync(0xffffffffu, w != nullptr)) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
    ss = warp_sum_xor(ss, 1, kLanes / 2);
    if (w != nullptr) {
      const float r = rsqrtf(fmaf(ss, 1.f / static_cast<float>(D), a.eps));
      float wv[8];
      widen8<T>(raw_w, wv);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wv[i];
    }
  }
  if (__any_sync(0xffffffffu, turn)) {
    float other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl_xor_sync(0xffffffffu, x[i], kLanes / 2);
    if (turn) {
      float c[8], s[8];
      widen8<T>(raw_c, c);
      // rotate_half negates the partner of the lower half: the sine's sign does
      const uint32_t flip = part < kLanes / 2 ? 0x80008000u : 0u;
      raw_s.x ^= flip;
      raw_s.y ^= flip;
      raw_s.z ^= flip;
      raw_s.w ^= flip;
      widen8<T>(raw_s, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(other[i], s[i], x[i] * c[i]);
    }
  }
  if (is_q && live) store8<T>(static_cast<T*>(a.q_out) + tok * a.qo_st + h * a.qo_sh + part * 8, x);
  if (__all_sync(0xffffffffu, is_q)) return;
  // ---- quantise (q rows take part in the shuffle only) -----------------------
  const float inv_cache = a.inv[kind];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] *= inv_cache;
    amax = max_nan(amax, fabsf(x[i]));
  }
  amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));  // NaN marks the whole block
  if (!live || row < 0) return;
  if (row >= a.pool_rows) {
    if (part == 0) report_status(HELM_DEV_BAD_PAGE);
    return;
  }
  // Quotients by the residual: the product with a rounded reciprocal, corrected by
  // the remainder that an fma gives exactly (Markstein, "Computation of elementary
  // functions on the IBM RISC System/6000 processor", IBM J. Res. Dev. 34, 1990); the
  // reciprocal itself is an approximation with one Newton-Raphson step.
  // max / 6:
  const float sixth = amax * (1.f / 6.f);
  const float most = amax < INFINITY ? fmaf(fmaf(-6.f, sixth, amax), 1.f / 6.f, sixth) : amax;
  const uint32_t s8 = amax != amax ? 0x7fu : float_to_e4m3(most);
  const uint32_t sh = e4m3x2_to_half2(s8);
  const float s = __low2float(*reinterpret_cast<const __half2*>(&sh));
  // x / s.  s has four significant bits and the borders between
  // codes three, so a border is met exactly, and the value next to it is at least
  // 1.06 half steps of the quotient away: it stays on its side.
  const float r0 = rcp_fast(s);
  const float inv = s > 0.f ? fmaf(fmaf(-s, r0, 1.f), r0, r0) : 0.f;
  if (!(amax < INFINITY)) {  // infinities saturate
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -3.0e38f), 3.0e38f);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q0 = x[i] * inv;
    x[i] = fmaf(-fmaf(q0, s, -x[i]), inv, q0);  // (this way round, -0 stays -0)
  }
  const uint32_t codes = float8_to_fp4(x);
  int64_t slot;
  int r_in;
  split_row(row, a.page_size, a.page_shift, slot, r_in);
  const int t = r_in & (kFp4TileTokens - 1);
  uint8_t* tile = a.pool + tile_base<D>(slot, r_in, h, a.hkv, a.page_size);
  using L = Fp4Tile<D>;
  // (a branch: the rows of a warp are mostly of one kind, and each side's
  // offsets are a dozen instructions)
  if (is_v) {
    *reinterpret_cast<uint32_t*>(tile + L::v_code(t, part * 4)) = codes;
    if ((part & 1) == 0) tile[L::v_scale(t, part >> 1)] = static_cast<uint8_t>(s8);
  } else {
    *reinterpret_cast<uint32_t*>(tile + L::k_code(t, part * 4)) = codes;
    if ((part & 1) == 0) tile[L::k_scale(t, part >> 1)] = static_cast<uint8_t>(s8);
  }
}

struct GatherFp4Args {
  const uint8_t* pool;
  int64_t pool_rows;
  const int64_t* slot_rows;
  void* k_out;
  int64_t ko_st, ko_sh;
  void* v_out;
  int64_t vo_st, vo_sh;
  int hkv, page_size, page_shift;
  float k_scale, v_scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(kFp4RowWarps * 32) gather_rows_fp4_kernel(const GatherFp4Args a) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tok = blockIdx.x;
  const int part = lane % kLanes;
  const int hr = (blockIdx.y * kFp4RowWarps + warp) * kRows + lane / kLanes;
  if (hr >= 2 * a.hkv) return;
  const bool is_v = hr >= a.hkv;
  const int h = is_v ? hr - a.hkv : hr;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t row = a.slot_rows[tok];
  if (row >= a.pool_rows) {
    if (part == 0) report_status(HELM_DEV_BAD_PAGE);
  } else if (row >= 0) {
    int64_t slot;
    int r_in;
    split_row(row, a.page_size, a.page_shift, slot, r_in);
    const int t = r_in & (kFp4TileTokens - 1);
    const uint8_t* tile = a.pool + tile_base<D>(slot, r_in, h, a.hkv, a.page_size);
    using L = Fp4Tile<D>;
    uint32_t codes, s8;
    if (is_v) {
      codes = *reinterpret_cast<const uint32_t*>(tile + L::v_code(t, part * 4));
      s8 = tile[L::v_scale(t, part >> 1)];
    } else {
      codes = *reinterpret_cast<const uint32_t*>(tile + L::k_code(t, part * 4));
      s8 = tile[L::k_scale(t, part >> 1)];
    }
    const uint32_t sh = e4m3x2_to_half2(s8);
    const float s = __low2float(*reinterpret_cast<const __half2*>(&sh)) *
                    (is_v ? a.v_scale : a.k_scale);
    uint32_t hv[4];
    fp4x8_to_half(codes, hv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hv[i]));
      x[2 * i] = f.x * s;
      x[2 * i + 1] = f.y * s;
    }
  }
  T* dst = is_v ? static_cast<T*>(a.v_out) + tok * a.vo_st + h * a.vo_sh
                : static_cast<T*>(a.k_out) + tok * a.ko_st + h * a.ko_sh;
  store8<T>(dst + part * 8, x);
}

// Rows of 16-bit values moved with 16-byte accesses.
bool rows16_misaligned(const void* p, std::initializer_list<int64_t> strides) {
  if (p == nullptr) return false;
  if (reinterpret_cast<uintptr_t>(p) & 15) return true;
  for (int64_t st : strides)
    if (st % 8) return true;
  return false;
}

// One block of kFp4RowWarps warps per token and run of head rows.
dim3 fp4_row_grid(int tokens, int rows, int head_dim) {
  const int per_block = kFp4RowWarps * 32 / (head_dim / 8);
  return dim3(static_cast<unsigned>(tokens), static_cast<unsigned>((rows + per_block - 1) / per_block));
}

template <typename T>
cudaError_t launch_append_fp4(int head_dim, int tokens, const AppendFp4Args& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = fp4_row_grid(tokens, a.hq + 2 * a.hkv, head_dim);
  cfg.blockDim = dim3(kFp4RowWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  switch (head_dim) {
    case 64:
      return cudaLaunchKernelEx(&cfg, kv_append_fp4_kernel<T, 64>, a);
    case 128:
      return cudaLaunchKernelEx(&cfg, kv_append_fp4_kernel<T, 128>, a);
    default:
      return cudaLaunchKernelEx(&cfg, kv_append_fp4_kernel<T, 256>, a);
  }
}

template <typename T>
cudaError_t launch_gather_fp4(int head_dim, int tokens, const GatherFp4Args& a, cudaStream_t s) {
  const dim3 grid = fp4_row_grid(tokens, 2 * a.hkv, head_dim), block(kFp4RowWarps * 32);
  switch (head_dim) {
    case 64:
      gather_rows_fp4_kernel<T, 64><<<grid, block, 0, s>>>(a);
      break;
    case 128:
      gather_rows_fp4_kernel<T, 128><<<grid, block, 0, s>>>(a);
      break;
    default:
      gather_rows_fp4_kernel<T, 256><<<grid, block, 0, s>>>(a);
  }
  return cudaGetLastError();
}

// Checks shared by the two entry points.
int fp4_rows_check(const void* pool, int64_t pool_pages, const void* slot_rows, int num_tokens,
                   int num_kv_heads, int head_dim, int page_size, int dtype, float k_scale,
                   float v_scale) {
  if (num_tokens < 0 || num_kv_heads <= 0 || page_size <= 0 || pool_pages <= 0)
    return HELM_ERR_INVALID_ARGUMENT;
  if (pool == nullptr || slot_rows == nullptr) return HELM_ERR_INVALID_ARGUMENT;
  if (!fp4_scale_ok(k_scale) || !fp4_scale_ok(v_scale)) return HELM_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return HELM_ERR_UNSUPPORTED;
  if (page_size % kFp4TileTokens != 0) return HELM_ERR_UNSUPPORTED;
  if (dtype != HELM_DTYPE_BF16 && dtype != HELM_DTYPE_FP16) return HELM_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(pool) & 15) return HELM_ERR_ALIGNMENT;
  return HELM_OK;
}

// The run of head rows is a grid's second dimension.
bool fp4_grid_fits(int64_t rows, int head_dim) {
  return rows < (int64_t(1) << 30) && fp4_row_grid(1, static_cast<int>(rows), head_dim).y <= 65535;
}

}  // namespace
}  // namespace helm

extern "C" int64_t helm_fp4_page_bytes(int num_kv_heads, int page_size, int head_dim) {
  if (num_kv_heads <= 0 || page_size <= 0 || page_size % helm::kFp4TileTokens != 0 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return -1;
  return static_cast<int64_t>(num_kv_heads) * (page_size / helm::kFp4TileTokens) * 18 * head_dim;
}

extern "C" int helm_kv_append_fp4(const void* q, int64_t q_stride_t, int64_t q_stride_h,
                                  const void* k, int64_t k_stride_t, int64_t k_stride_h,
                                  const void* v, int64_t v_stride_t, int64_t v_stride_h,
                                  const void* q_norm_w, const void* k_norm_w, float eps,
                                  const void* cos, const void* sin, int64_t rope_stride_t,
                                  void* q_out, int64_t q_out_stride_t, int64_t q_out_stride_h,
                                  void* kv_pool, int64_t pool_pages, const int64_t* slot_rows,
                                  int num_tokens, int num_q_heads, int num_kv_heads, int head_dim,
                                  int page_size, int dtype, float k_scale, float v_scale,
                                  void* stream) {
  using namespace helm;
  const int rc = fp4_rows_check(kv_pool, pool_pages, slot_rows, num_tokens, num_kv_heads, head_dim,
                                page_size, dtype, k_scale, v_scale);
  if (rc != HELM_OK) return rc;
  if (num_q_heads < 0 || k == nullptr || v == nullptr || (q == nullptr) != (q_out == nullptr) ||
      (cos == nullptr) != (sin == nullptr) || (q_norm_w != nullptr && q == nullptr))
    return HELM_ERR_INVALID_ARGUMENT;
  if (q != nullptr && num_q_heads == 0) return HELM_ERR_INVALID_ARGUMENT;
  if (rows16_misaligned(q, {q_stride_t, q_stride_h}) ||
      rows16_misaligned(k, {k_stride_t, k_stride_h}) ||
      rows16_misaligned(v, {v_stride_t, v_stride_h}) ||
      rows16_misaligned(q_out, {q_out_stride_t, q_out_stride_h}) ||
      rows16_misaligned(cos, {rope_stride_t}) || rows16_misaligned(sin, {rope_stride_t}) ||
      rows16_misaligned(q_norm_w, {}) || rows16_misaligned(k_norm_w, {}))
    return HELM_ERR_ALIGNMENT;
  if (num_tokens == 0) return HELM_OK;
  AppendFp4Args a;
  a.src[0] = q;
  a.st[0] = q_stride_t;
  a.sh[0] = q_stride_h;
  a.src[1] = k;
  a.st[1] = k_stride_t;
  a.sh[1] = k_stride_h;
  a.src[2] = v;
  a.st[2] = v_stride_t;
  a.sh[2] = v_stride_h;
  a.weight[0] = q_norm_w;
  a.weight[1] = k_norm_w;
  a.weight[2] = nullptr;
  a.eps = eps;
  a.cos = cos;
  a.sin = sin;
  a.rope_st = rope_stride_t;
  a.q_out = q_out;
  a.qo_st = q_out_stride_t;
  a.qo_sh = q_out_stride_h;
  a.pool = static_cast<uint8_t*>(kv_pool);
  a.pool_rows = pool_pages * page_size;
  a.slot_rows = slot_rows;
  a.hq = q != nullptr ? num_q_heads : 0;
  a.hkv = num_kv_heads;
  a.page_size = page_size;
  a.page_shift = shift_of(page_size);
  a.inv[0] = 1.f;
  a.inv[1] = 1.f / k_scale;
  a.inv[2] = 1.f / v_scale;
  if (!fp4_grid_fits(static_cast<int64_t>(a.hq) + 2 * static_cast<int64_t>(a.hkv), head_dim))
    return HELM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == HELM_DTYPE_BF16
                            ? launch_append_fp4<__nv_bfloat16>(head_dim, num_tokens, a, s)
                            : launch_append_fp4<__half>(head_dim, num_tokens, a, s);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}

extern "C" int helm_gather_kv_rows_fp4(const void* kv_pool, int64_t pool_pages,
                                       const int64_t* slot_rows, void* k_out,
                                       int64_t k_out_stride_t, int64_t k_out_stride_h, void* v_out,
                                       int64_t v_out_stride_t, int64_t v_out_stride_h,
                                       int num_tokens, int num_kv_heads, int head_dim,
                                       int page_size, int dtype, float k_scale, float v_scale,
                                       void* stream) {
  using namespace helm;
  const int rc = fp4_rows_check(kv_pool, pool_pages, slot_rows, num_tokens, num_kv_heads, head_dim,
                                page_size, dtype, k_scale, v_scale);
  if (rc != HELM_OK) return rc;
  if (k_out == nullptr || v_out == nullptr) return HELM_ERR_INVALID_ARGUMENT;
  if (rows16_misaligned(k_out, {k_out_stride_t, k_out_stride_h}) ||
      rows16_misaligned(v_out, {v_out_stride_t, v_out_stride_h}))
    return HELM_ERR_ALIGNMENT;
  if (num_tokens == 0) return HELM_OK;
  GatherFp4Args a;
  a.pool = static_cast<const uint8_t*>(kv_pool);
  a.pool_rows = pool_pages * page_size;
  a.slot_rows = slot_rows;
  a.k_out = k_out;
  a.ko_st = k_out_stride_t;
  a.ko_sh = k_out_stride_h;
  a.v_out = v_out;
  a.vo_st = v_out_stride_t;
  a.vo_sh = v_out_stride_h;
  a.hkv = num_kv_heads;
  a.page_size = page_size;
  a.page_shift = shift_of(page_size);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  if (!fp4_grid_fits(2 * static_cast<int64_t>(num_kv_heads), head_dim)) return HELM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == HELM_DTYPE_BF16
                            ? launch_gather_fp4<__nv_bfloat16>(head_dim, num_tokens, a, s)
                            : launch_gather_fp4<__half>(head_dim, num_tokens, a, s);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}
