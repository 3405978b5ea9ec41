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
  const void* q;
  int64_t q_st, q_sh;
  const void* k;
  int64_t k_st, k_sh;
  const void* v;
  int64_t v_st, v_sh;
  const void* qw;
  const void* kw;
  float eps;
  const void* cos;
  const void* sin;
  int64_t rope_st;
  void* q_out;
  int64_t qo_st, qo_sh;
  uint8_t* pool;
  int64_t pool_rows;  // pool_pages * page_size
  const int64_t* slot_rows;
  int64_t num_rows;   // tokens * (hq + 2 hkv)
  int hq, hkv, page_size;
  float k_inv, v_inv;  // 1 / cache scale (a power of two)
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_float<T>(x[i]);
  *reinterpret_cast<uint4*>(p) = r;
}

// Slot and row inside the page of a pool row (32-bit division where it fits).
__device__ __forceinline__ void split_row(int64_t row, int page_size, int64_t& slot, int& r_in) {
  if (row < (int64_t(1) << 32)) {
    const uint32_t u = static_cast<uint32_t>(row), s = u / static_cast<uint32_t>(page_size);
    slot = s;
    r_in = static_cast<int>(u - s * page_size);
  } else {
    slot = row / page_size;
    r_in = static_cast<int>(row - slot * page_size);
  }
}

// First byte of the tile that holds pool row (slot, r_in) of KV head h.
template <int D>
__device__ __forceinline__ int64_t tile_base(int64_t slot, int r_in, int h, int hkv,
                                             int page_size) {
  return ((slot * hkv + h) * (page_size / kFp4TileTokens) + r_in / kFp4TileTokens) *
         Fp4Tile<D>::kBytes;
}

// One head row of D values on D / 8 lanes, eight values a lane (16-byte loads).
// A quantisation block is two neighbouring lanes.  Rows of different kinds (q,
// k, v) may share a warp, so the shuffles run for every lane and the results
// are selected.  HBM bound: per token 2 (2 Hq + 2 Hkv) D + 1.125 Hkv D bytes.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_append_fp4_kernel(const AppendFp4Args a) {
  // programmatic dependent launch both ways, as kv_append_kernel
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kLanes = D / 8;
  const int64_t idx = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
  const int part = threadIdx.x % kLanes;  // dims [8 part, 8 part + 8)
  const bool live = idx < a.num_rows;
  const int per_tok = a.hq + 2 * a.hkv;
  const int64_t tok = live ? idx / per_tok : 0;
  const int hr = live ? static_cast<int>(idx - tok * per_tok) : 0;
  const bool is_q = hr < a.hq, is_v = hr >= a.hq + a.hkv;
  const int h = is_q ? hr : (is_v ? hr - a.hq - a.hkv : hr - a.hq);
  float x[8];
  const T* src = is_q ? static_cast<const T*>(a.q) + tok * a.q_st + h * a.q_sh
                      : (is_v ? static_cast<const T*>(a.v) + tok * a.v_st + h * a.v_sh
                              : static_cast<const T*>(a.k) + tok * a.k_st + h * a.k_sh);
  load8<T>(src + part * 8, x);
  const T* w = static_cast<const T*>(is_q ? a.qw : (is_v ? nullptr : a.kw));
  if (a.qw != nullptr || a.kw != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
    ss = warp_sum_xor(ss, 1, kLanes / 2);
    if (w != nullptr) {
      const float r = 1.f / sqrtf(ss / static_cast<float>(D) + a.eps);
      float wv[8];
      load8<T>(w + part * 8, wv);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wv[i];
    }
  }
  if (a.cos != nullptr) {
    float other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl_xor_sync(0xffffffffu, x[i], kLanes / 2);
    if (!is_v) {
      float c[8], s[8];
      load8<T>(static_cast<const T*>(a.cos) + tok * a.rope_st + part * 8, c);
      load8<T>(static_cast<const T*>(a.sin) + tok * a.rope_st + part * 8, s);
      const float sign = part < kLanes / 2 ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * c[i] + sign * other[i] * s[i];
    }
  }
  if (is_q) {
    if (live) store8<T>(static_cast<T*>(a.q_out) + tok * a.qo_st + h * a.qo_sh + part * 8, x);
  }
  // ---- quantise (q rows take part in the shuffles only) ----------------------
  const float inv_cache = is_v ? a.v_inv : a.k_inv;
  float amax = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] *= inv_cache;
    nan |= x[i] != x[i];
    amax = fmaxf(amax, fabsf(x[i]));
  }
  if (nan) amax = NAN;  // a NaN marks its whole block
  const float peer = __shfl_xor_sync(0xffffffffu, amax, 1);
  nan = amax != amax || peer != peer;
  amax = fmaxf(amax, peer);
  if (!live || is_q) return;
  const int64_t row = a.slot_rows[tok];
  if (row < 0) return;
  if (row >= a.pool_rows) {
    if (part == 0) report_status(HELM_DEV_BAD_PAGE);
    return;
  }
  const uint32_t s8 = nan ? 0x7fu : float_to_e4m3(amax / 6.f);
  const uint32_t sh = e4m3x2_to_half2(s8);
  const float s = __low2float(*reinterpret_cast<const __half2*>(&sh));
  // x / s correctly rounded: one Newton step on the product with the rounded
  // reciprocal (s has four significant bits), so a value on the border between
  // two codes is seen on the border
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = fminf(fmaxf(x[i], -3.0e38f), 3.0e38f);  // infinities saturate
    const float q0 = y * inv;
    x[i] = copysignf(fmaf(fmaf(-q0, s, y), inv, q0), y);  // -0 stays -0
  }
  const uint32_t codes = float8_to_fp4(x);
  int64_t slot;
  int r_in;
  split_row(row, a.page_size, slot, r_in);
  const int t = r_in & (kFp4TileTokens - 1);
  uint8_t* tile = a.pool + tile_base<D>(slot, r_in, h, a.hkv, a.page_size);
  using L = Fp4Tile<D>;
  *reinterpret_cast<uint32_t*>(tile + (is_v ? L::v_code(t, part * 4) : L::k_code(t, part * 4))) =
      codes;
  if ((part & 1) == 0)
    tile[is_v ? L::v_scale(t, part >> 1) : L::k_scale(t, part >> 1)] = static_cast<uint8_t>(s8);
}

struct GatherFp4Args {
  const uint8_t* pool;
  int64_t pool_rows;
  const int64_t* slot_rows;
  void* k_out;
  int64_t ko_st, ko_sh;
  void* v_out;
  int64_t vo_st, vo_sh;
  int64_t num_rows;  // tokens * 2 hkv
  int hkv, page_size;
  float k_scale, v_scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(256) gather_rows_fp4_kernel(const GatherFp4Args a) {
  constexpr int kLanes = D / 8;
  const int64_t idx = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
  const int part = threadIdx.x % kLanes;
  if (idx >= a.num_rows) return;
  const int64_t tok = idx / (2 * a.hkv);
  const int hr = static_cast<int>(idx - tok * (2 * a.hkv));
  const bool is_v = hr >= a.hkv;
  const int h = is_v ? hr - a.hkv : hr;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t row = a.slot_rows[tok];
  if (row >= a.pool_rows) {
    if (part == 0) report_status(HELM_DEV_BAD_PAGE);
  } else if (row >= 0) {
    int64_t slot;
    int r_in;
    split_row(row, a.page_size, slot, r_in);
    const int t = r_in & (kFp4TileTokens - 1);
    const uint8_t* tile = a.pool + tile_base<D>(slot, r_in, h, a.hkv, a.page_size);
    using L = Fp4Tile<D>;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(
        tile + (is_v ? L::v_code(t, part * 4) : L::k_code(t, part * 4)));
    const uint32_t s8 = tile[is_v ? L::v_scale(t, part >> 1) : L::k_scale(t, part >> 1)];
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

template <typename T>
cudaError_t launch_append_fp4(int head_dim, const AppendFp4Args& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  const int64_t threads = a.num_rows * (head_dim / 8);
  cfg.gridDim = dim3(static_cast<unsigned>((threads + 255) / 256));
  cfg.blockDim = dim3(256);
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
cudaError_t launch_gather_fp4(int head_dim, const GatherFp4Args& a, cudaStream_t s) {
  const int64_t threads = a.num_rows * (head_dim / 8);
  const unsigned grid = static_cast<unsigned>((threads + 255) / 256);
  switch (head_dim) {
    case 64:
      gather_rows_fp4_kernel<T, 64><<<grid, 256, 0, s>>>(a);
      break;
    case 128:
      gather_rows_fp4_kernel<T, 128><<<grid, 256, 0, s>>>(a);
      break;
    default:
      gather_rows_fp4_kernel<T, 256><<<grid, 256, 0, s>>>(a);
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

// Threads of a launch must fit a 31-bit grid of 256-thread blocks.
bool fp4_grid_fits(int64_t rows, int head_dim) {
  return rows <= (int64_t(1) << 38) && (rows * (head_dim / 8) + 255) / 256 < (int64_t(1) << 31);
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
  a.q = q;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k = k;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v = v;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.qw = q_norm_w;
  a.kw = k_norm_w;
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
  a.num_rows = static_cast<int64_t>(num_tokens) * (a.hq + 2 * a.hkv);
  a.page_size = page_size;
  a.k_inv = 1.f / k_scale;
  a.v_inv = 1.f / v_scale;
  if (!fp4_grid_fits(a.num_rows, head_dim)) return HELM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == HELM_DTYPE_BF16 ? launch_append_fp4<__nv_bfloat16>(head_dim, a, s)
                                                 : launch_append_fp4<__half>(head_dim, a, s);
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
  a.num_rows = static_cast<int64_t>(num_tokens) * 2 * num_kv_heads;
  a.hkv = num_kv_heads;
  a.page_size = page_size;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  if (!fp4_grid_fits(a.num_rows, head_dim)) return HELM_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == HELM_DTYPE_BF16 ? launch_gather_fp4<__nv_bfloat16>(head_dim, a, s)
                                                 : launch_gather_fp4<__half>(head_dim, a, s);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}
