// Block tables, slot rows and positions of one step of a continuous batch,
// built on the device from the requests' lengths.
//
// The reference keeps this on the host, page by page (KVAllocator.allocate /
// free, helm/runtime/kv_allocator.py:36-93, and KVCacheManager.append_decode /
// append_prefill, helm/runtime/kv_cache.py:113-171); a captured decode step
// cannot.  Integer work on a few bytes per request and per token: bound by
// launch and memory latency, so it is one launch.  The grid is ONE cluster: its
// barrier orders the three phases (lengths read; tables and stack written;
// rows read back from the tables), every CTA holding the prefix sums of all
// requests in its shared memory.
#include <cooperative_groups.h>

#include "common.cuh"

namespace helm {
namespace {

constexpr int kStepThreads = 512;
constexpr int kStepCluster = 8;            // CTAs when there are many tokens
constexpr int kStepMaxRequests = 8192;     // four int32 arrays in shared memory
constexpr int kStepTokensPerCta = 2048;    // tokens one CTA serves alone

struct StepArgs {
  const int32_t* past_lens;
  const int32_t* new_lens;
  int32_t* page_table;
  int64_t pt_sb;
  int max_pages;
  int32_t* free_pages;
  int free_capacity;
  const int32_t* free_count;
  int32_t* free_count_out;
  int32_t* kv_lens;
  int32_t* cu_tokens;
  int32_t* seq_ids;
  int32_t* positions;
  int64_t* slot_rows;
  int batch, page_size, num_rows;
};

__device__ __forceinline__ int block_scan_incl(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int off = 1; off < 32; off <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += n;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kStepThreads / 32; ++w) {
    const int x = s_warp[w];
    if (w < warp) before += x;
    total += x;
  }
  __syncthreads();
  return v + before;
}

// Largest b in [0, n) with prefix[b] <= x, for a nondecreasing prefix with
// prefix[0] = 0 (of equal entries the last: requests that own nothing are skipped).
__device__ __forceinline__ int owner_of(const int* prefix, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kStepThreads) step_tables_kernel(const StepArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ int s_mem[];
  __shared__ int s_warp[kStepThreads / 32];
  int* s_cu = s_mem;                  // [batch + 1] tokens before request b
  int* s_want = s_cu + a.batch + 1;   // [batch + 1] pages asked for before b
  int* s_give = s_want + a.batch + 1; // [batch + 1] pages given back before b
  int* s_past = s_give + a.batch + 1; // [batch] past length, top bit: the request leaves
  cg::cluster_group cluster = cg::this_cluster();
  const int P = a.page_size;

  auto pages = [&](int64_t tokens) { return (tokens + P - 1) / P; };
  // ---- prefix sums over the requests (every CTA, from the same inputs) -------
  int c_cu = 0, c_want = 0, c_give = 0;
  bool refused = false;
  for (int base = 0; base < a.batch; base += kStepThreads) {
    const int b = base + threadIdx.x;
    int n = 0, want = 0, give = 0, past = 0;
    bool leaves = false;
    if (b < a.batch) {
      past = max(a.past_lens[b], 0);
      n = a.new_lens[b];
      leaves = n < 0;
      n = max(n, 0);
      const int64_t held = pages(past), all = pages(static_cast<int64_t>(past) + n);
      if (leaves)
        give = static_cast<int>(min(held, static_cast<int64_t>(a.max_pages)));
      else if (all <= a.max_pages)
        want = static_cast<int>(all - held);
      else
        refused = true;
    }
    int t0, t1, t2;
    const int i0 = block_scan_incl(n, s_warp, t0);
    const int i1 = block_scan_incl(want, s_warp, t1);
    const int i2 = block_scan_incl(give, s_warp, t2);
    if (b < a.batch) {
      s_cu[b + 1] = c_cu + i0;
      s_want[b + 1] = c_want + i1;
      s_give[b + 1] = c_give + i2;
      s_past[b] = past | (leaves ? 0x80000000 : 0);
    }
    c_cu += t0;
    c_want += t1;
    c_give += t2;
  }
  if (threadIdx.x == 0) s_cu[0] = s_want[0] = s_give[0] = 0;
  const int count = min(max(*a.free_count, 0), a.free_capacity);
  __syncthreads();
  cluster.sync();  // every CTA has read the inputs: outputs may overwrite them
  const int tid = static_cast<int>(cluster.block_rank()) * kStepThreads + threadIdx.x;
  const int nthreads = static_cast<int>(cluster.num_blocks()) * kStepThreads;
  const int64_t top = static_cast<int64_t>(count) + c_give;

  auto granted = [&](int b) {  // request b keeps its place and gets its pages
    const int sp = s_past[b];
    if (sp < 0) return false;
    if (pages(static_cast<int64_t>(sp) + (s_cu[b + 1] - s_cu[b])) > a.max_pages) return false;
    return s_want[b + 1] == s_want[b] || s_want[b + 1] <= top;
  };
  // page r of those given back in this step
  auto given_page = [&](int r) {
    const int b = owner_of(s_give, a.batch, r);
    return a.page_table[static_cast<int64_t>(b) * a.pt_sb + (r - s_give[b])];
  };

  // ---- tables, stack, lengths -------------------------------------------------
  for (int b = tid; b < a.batch; b += nthreads) {
    const int sp = s_past[b], n = s_cu[b + 1] - s_cu[b];
    const bool ok = granted(b);
    if (sp >= 0 && !ok) refused = true;
    a.kv_lens[b] = sp < 0 ? 0 : (ok ? sp + n : sp);
    a.cu_tokens[b + 1] = s_cu[b + 1];
  }
  for (int j = tid; j < c_want; j += nthreads) {  // fresh page j: popped from the top
    const int64_t at = top - 1 - j;
    if (at < 0) break;
    const int b = owner_of(s_want, a.batch, j);
    if (!granted(b)) continue;
    const int page = at < count ? a.free_pages[at] : given_page(static_cast<int>(at - count));
    const int64_t i = pages(s_past[b]) + (j - s_want[b]);
    a.page_table[static_cast<int64_t>(b) * a.pt_sb + i] = page;
  }
  for (int r = tid; r < c_give; r += nthreads) {  // pushed on the stack, request by request
    if (static_cast<int64_t>(count) + r < a.free_capacity)
      a.free_pages[count + r] = given_page(r);
    else
      refused = true;  // more pages than the stack holds
  }
  if (tid == 0) {
    a.cu_tokens[0] = 0;
    // pages taken: the longest run of requests whose wants fit
    int taken = 0;
    if (c_want > 0) {
      const int b = owner_of(s_want, a.batch + 1,
                             static_cast<int>(min(top, static_cast<int64_t>(0x7fffffff))));
      taken = s_want[b];
    }
    *a.free_count_out =
        static_cast<int>(min(top - taken, static_cast<int64_t>(a.free_capacity)));
  }
  if (refused) report_status(HELM_DEV_NO_PAGES);
  cluster.sync();  // the tables are written

  // ---- tokens -----------------------------------------------------------------
  for (int t = tid; t < a.num_rows; t += nthreads) {
    int seq = -1, pos = 0;
    int64_t row = -1;
    if (t < c_cu) {
      const int b = owner_of(s_cu, a.batch, t);
      seq = b;
      pos = (s_past[b] & 0x7fffffff) + (t - s_cu[b]);
      if (granted(b)) {
        const int page = pos / P;
        const int slot = __ldcg(a.page_table + static_cast<int64_t>(b) * a.pt_sb + page);
        if (slot >= 0)
          row = static_cast<int64_t>(slot) * P + (pos - page * P);
        else
          report_status(HELM_DEV_BAD_PAGE);
      }
    }
    a.slot_rows[t] = row;
    if (a.positions != nullptr) a.positions[t] = pos;
    if (a.seq_ids != nullptr) a.seq_ids[t] = seq;
  }
}

}  // namespace
}  // namespace helm

extern "C" int helm_build_step_tables(const int32_t* past_lens, const int32_t* new_lens,
                                      int32_t* page_table, int64_t pt_stride_b, int max_pages,
                                      int32_t* free_pages, int free_capacity,
                                      const int32_t* free_count, int32_t* free_count_out,
                                      int32_t* kv_lens, int32_t* cu_tokens, int32_t* seq_ids,
                                      int32_t* positions, int64_t* slot_rows, int batch,
                                      int page_size, int num_rows, void* stream) {
  using namespace helm;
  if (past_lens == nullptr || new_lens == nullptr || page_table == nullptr ||
      free_pages == nullptr || free_count == nullptr || free_count_out == nullptr ||
      kv_lens == nullptr || cu_tokens == nullptr || (slot_rows == nullptr && num_rows > 0))
    return HELM_ERR_INVALID_ARGUMENT;
  if (batch <= 0 || page_size <= 0 || max_pages <= 0 || free_capacity < 0 || num_rows < 0 ||
      pt_stride_b < max_pages)
    return HELM_ERR_INVALID_ARGUMENT;
  if (batch > kStepMaxRequests) return HELM_ERR_UNSUPPORTED;
  // page counts of all requests together, and positions, are 32-bit
  if (static_cast<int64_t>(batch) * max_pages >= (int64_t(1) << 31) ||
      static_cast<int64_t>(max_pages) * page_size >= (int64_t(1) << 31))
    return HELM_ERR_UNSUPPORTED;
  const StepArgs a = {past_lens, new_lens,  page_table, pt_stride_b, max_pages, free_pages,
                      free_capacity, free_count, free_count_out, kv_lens, cu_tokens, seq_ids,
                      positions, slot_rows, batch,     page_size,  num_rows};
  const size_t smem = (static_cast<size_t>(batch) * 4 + 3) * sizeof(int);
  cudaError_t e = cudaSuccess;
  static unsigned long long configured = 0;  // one bit per device
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(configured & (1ull << dev)))) {
    e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (kStepMaxRequests * 4 + 3) * static_cast<int>(sizeof(int)));
    if (e == cudaSuccess && dev < 64) configured |= 1ull << dev;
  }
  if (e == cudaSuccess) {
    const unsigned ctas =
        num_rows <= kStepTokensPerCta && batch <= kStepThreads ? 1 : kStepCluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kStepThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, step_tables_kernel, a);
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}
