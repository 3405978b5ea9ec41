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

constexpr int kStepThreads = 1024;
constexpr int kStepWarps = kStepThreads / 32;
// CTAs when there are many tokens: sixteen where the device places such a cluster.
// Few SMs then write all rows, 16 bytes a token; 131k tokens took 14.6 us with
// half-sector stores from eight SMs.
constexpr int kStepCluster = 16, kStepPortableCluster = 8;
constexpr int kStepMaxRequests = 8192;     // four int32 arrays and a byte in shared memory
constexpr int kStepTokensPerCta = 2048;    // tokens one CTA serves alone
constexpr int kStepRun = 4;                // consecutive pages of a thread: one search for them
constexpr int kStepTokens = 4;             // consecutive tokens of a thread, when there are many

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
  int page_shift;  // page_size = 1 << page_shift, or -1
  int wide;        // seq_ids and positions are 16-byte aligned, slot_rows 32
};

constexpr uint8_t kStepLeaves = 1, kStepTooLong = 2;

// Sum of two token counts, saturating: the running sums stay in order whatever
// the lengths are.  (Page counts are bounded by batch * max_pages.)
__device__ __forceinline__ int token_sum(int a, int b) {
  return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), 0x7fffffffu));
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
  __shared__ int s_warp[3][kStepWarps];
  int* s_cu = s_mem;                   // [batch + 1] tokens before request b
  int* s_want = s_cu + a.batch + 1;    // [batch + 1] pages asked for before b
  int* s_give = s_want + a.batch + 1;  // [batch + 1] pages given back before b
  int* s_past = s_give + a.batch + 1;  // [batch] past length
  uint8_t* s_flag = reinterpret_cast<uint8_t*>(s_past + a.batch);  // [batch]
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned P = static_cast<unsigned>(a.page_size);

  auto page_of = [&](unsigned token) { return a.page_shift >= 0 ? token >> a.page_shift : token / P; };
  auto pages = [&](unsigned tokens) {  // ceil, without overflow
    return tokens == 0 ? 0u : page_of(tokens - 1) + 1;
  };
  // ---- prefix sums over the requests (every CTA, from the same inputs): a
  // thread takes consecutive requests, one scan of three values does the rest
  const int per = (a.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min(a.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.batch, b0 + per);
  int sum[3] = {0, 0, 0};
  bool refused = false;
  for (int b = b0; b < b1; ++b) {
    const unsigned past = static_cast<unsigned>(max(a.past_lens[b], 0));
    const int n = a.new_lens[b];
    const unsigned held = pages(past), all = pages(past + static_cast<unsigned>(max(n, 0)));
    uint8_t flag = 0;
    s_cu[b] = sum[0];
    s_want[b] = sum[1];
    s_give[b] = sum[2];
    if (n < 0) {
      flag = kStepLeaves;
      sum[2] += min(held, static_cast<unsigned>(a.max_pages));
    } else if (all <= static_cast<unsigned>(a.max_pages)) {
      sum[0] = token_sum(sum[0], n);
      sum[1] += all - held;
    } else {
      sum[0] = token_sum(sum[0], n);
      flag = kStepTooLong;
    }
    s_past[b] = static_cast<int>(past);
    s_flag[b] = flag;
  }
  const int count = min(max(*a.free_count, 0), a.free_capacity);
  int before[3], total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int v = sum[i];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v = i == 0 ? token_sum(v, x) : v + x;
    }
    if (lane == 31) s_warp[i][warp] = v;
    v = __shfl_up_sync(0xffffffffu, v, 1);
    before[i] = lane ? v : 0;
  }
  __syncthreads();
  const int warps = (blockDim.x + 31) / 32;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const int w = lane < warps ? s_warp[i][lane] : 0;
    int v = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v = i == 0 ? token_sum(v, x) : v + x;
    }
    total[i] = __shfl_sync(0xffffffffu, v, 31);
    const int warps_before = __shfl_sync(0xffffffffu, v, max(warp - 1, 0));
    if (warp > 0) before[i] = i == 0 ? token_sum(before[i], warps_before) : before[i] + warps_before;
  }
  for (int b = b0; b < b1; ++b) {
    s_cu[b] = token_sum(s_cu[b], before[0]);
    s_want[b] += before[1];
    s_give[b] += before[2];
  }
  if (threadIdx.x == 0) {
    s_cu[a.batch] = total[0];
    s_want[a.batch] = total[1];
    s_give[a.batch] = total[2];
  }
  __syncthreads();
  cluster.sync();  // every CTA has read the inputs: outputs may overwrite them
  const int tid = static_cast<int>(cluster.block_rank() * blockDim.x + threadIdx.x);
  const int nthreads = static_cast<int>(cluster.num_blocks() * blockDim.x);
  const int64_t top = static_cast<int64_t>(count) + total[2];

  // request b keeps its place and gets its pages
  auto granted = [&](int b) {
    return s_flag[b] == 0 && (s_want[b + 1] == s_want[b] || s_want[b + 1] <= top);
  };
  // Entry of page r of those given back in this step; b: a request at or before
  // its owner, moved on to it.
  auto given_entry = [&](int r, int& b) {
    while (s_give[b + 1] <= r) ++b;
    return a.page_table + static_cast<int64_t>(b) * a.pt_sb + (r - s_give[b]);
  };

  // ---- tables, stack, lengths -------------------------------------------------
  for (int b = tid; b < a.batch; b += nthreads) {
    const int past = s_past[b], n = s_cu[b + 1] - s_cu[b];
    const bool leaves = s_flag[b] & kStepLeaves, ok = granted(b);
    refused |= !leaves && !ok;
    a.kv_lens[b] = leaves ? 0 : (ok ? past + n : past);
    a.cu_tokens[b + 1] = s_cu[b + 1];
  }
  // Pages go in runs of consecutive ones, too: one search, their loads together.
  for (int j0 = tid * kStepRun; j0 < total[1]; j0 += nthreads * kStepRun) {  // fresh: popped
    const int n = min(kStepRun, total[1] - j0);
    int b = owner_of(s_want, a.batch, j0);
    // page j is entry top - 1 - j of the stack; those from `count` up are given back
    const int64_t at = top - 1 - j0;
    if (at < 0) break;
    int page[kStepRun];
    int g = at >= count ? owner_of(s_give, a.batch,
                                   static_cast<int>(max(at - (n - 1), static_cast<int64_t>(count)) - count))
                        : 0;
#pragma unroll
    for (int i = kStepRun - 1; i >= 0; --i) {  // upwards in the stack
      const int64_t e = at - i;
      page[i] = -1;
      if (i < n && e >= 0)
        page[i] = e < count ? a.free_pages[e] : *given_entry(static_cast<int>(e - count), g);
    }
#pragma unroll
    for (int i = 0; i < kStepRun; ++i) {
      if (i >= n || at - i < 0) break;
      const int j = j0 + i;
      while (s_want[b + 1] <= j) ++b;
      if (granted(b))
        a.page_table[static_cast<int64_t>(b) * a.pt_sb + pages(s_past[b]) + (j - s_want[b])] =
            page[i];
    }
  }
  for (int r0 = tid * kStepRun; r0 < total[2]; r0 += nthreads * kStepRun) {  // given back: pushed
    const int n = min(kStepRun, total[2] - r0);
    int b = owner_of(s_give, a.batch, r0);
    int page[kStepRun];
#pragma unroll
    for (int i = 0; i < kStepRun; ++i)
      if (i < n) page[i] = *given_entry(r0 + i, b);
#pragma unroll
    for (int i = 0; i < kStepRun; ++i) {
      if (i >= n) break;
      if (static_cast<int64_t>(count) + r0 + i < a.free_capacity)
        a.free_pages[count + r0 + i] = page[i];
      else
        refused = true;  // more pages than the stack holds
    }
  }
  if (tid == 0) {
    a.cu_tokens[0] = 0;
    // pages taken: the longest run of requests whose wants fit
    const int b = owner_of(s_want, a.batch + 1,
                           static_cast<int>(min(top, static_cast<int64_t>(0x7fffffff))));
    *a.free_count_out =
        static_cast<int>(min(top - s_want[b], static_cast<int64_t>(a.free_capacity)));
  }
  if (refused) report_status(HELM_DEV_NO_PAGES);
  cluster.sync();  // the tables are written

  // ---- tokens -------------------------------------------------------------------
  auto put = [&](int t, int seq, int pos, int64_t row) {
    if (a.seq_ids != nullptr) a.seq_ids[t] = seq;
    if (a.positions != nullptr) a.positions[t] = pos;
    a.slot_rows[t] = row;
  };
  auto slot_of = [&](int b, int page) {
    return __ldcg(a.page_table + static_cast<int64_t>(b) * a.pt_sb + page);
  };
  auto row_of = [&](int slot, int pos, int page) {
    if (slot < 0) {
      report_status(HELM_DEV_BAD_PAGE);
      return static_cast<int64_t>(-1);
    }
    return static_cast<int64_t>(slot) * P + (pos - page * static_cast<int>(P));
  };
  // one token of request b
  auto token = [&](int t, int b) {
    const int pos = s_past[b] + (t - s_cu[b]);
    int64_t row = -1;
    if (granted(b)) {
      const int page = static_cast<int>(page_of(pos));
      row = row_of(slot_of(b, page), pos, page);
    }
    put(t, b, pos, row);
  };
  if (a.num_rows <= nthreads) {  // a token each
    if (tid < a.num_rows) {
      if (tid < total[0])
        token(tid, owner_of(s_cu, a.batch, tid));
      else
        put(tid, -1, 0, -1);
    }
    return;
  }
  for (int t0 = tid * kStepTokens; t0 < a.num_rows; t0 += nthreads * kStepTokens) {
    const int t1 = min(t0 + kStepTokens, a.num_rows);
    int b = t0 < total[0] ? owner_of(s_cu, a.batch, t0) : 0;
    if (a.wide && t0 + kStepTokens <= min(s_cu[b + 1], a.num_rows) && P >= kStepTokens) {
      // the whole run belongs to one request: two pages at most, wide stores
      const int pos = s_past[b] + (t0 - s_cu[b]);
      const bool ok = granted(b);
      const int p0 = static_cast<int>(page_of(pos)), p1 = static_cast<int>(page_of(pos + kStepTokens - 1));
      int slot0 = 0, slot1 = 0;
      if (ok) {
        slot0 = slot_of(b, p0);
        slot1 = slot_of(b, p1);
      }
      const int64_t row0 = ok ? row_of(slot0, pos, p0) : -1;
      // row of the second page's first token; tokens before it stay in the first
      const int cut = p1 != p0 ? p1 * static_cast<int>(P) - pos : kStepTokens;
      const int64_t row1 = ok ? row_of(slot1, p1 * static_cast<int>(P), p1) : -1;
      if (a.seq_ids != nullptr) *reinterpret_cast<int4*>(a.seq_ids + t0) = make_int4(b, b, b, b);
      if (a.positions != nullptr)
        *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos, pos + 1, pos + 2, pos + 3);
      int64_t r[kStepTokens];
#pragma unroll
      for (int k = 0; k < kStepTokens; ++k) {
        const bool first = k < cut;
        const int64_t from = first ? row0 : row1;
        r[k] = from < 0 ? -1 : from + (first ? k : k - cut);
      }
      static_assert(kStepTokens == 4, "one 32-byte store");
      asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(a.slot_rows + t0), "l"(r[0]),
                   "l"(r[1]), "l"(r[2]), "l"(r[3])
                   : "memory");
      continue;
    }
    for (int t = t0; t < t1; ++t) {
      if (t >= total[0]) {
        put(t, -1, 0, -1);
        continue;
      }
      while (s_cu[b + 1] <= t) ++b;  // total > t: there is one
      token(t, b);
    }
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
      (free_pages == nullptr && free_capacity > 0) || free_count == nullptr ||
      free_count_out == nullptr ||
      kv_lens == nullptr || cu_tokens == nullptr || (slot_rows == nullptr && num_rows > 0))
    return HELM_ERR_INVALID_ARGUMENT;
  if (batch <= 0 || page_size <= 0 || max_pages <= 0 || free_capacity < 0 || num_rows < 0 ||
      pt_stride_b < max_pages)
    return HELM_ERR_INVALID_ARGUMENT;
  if (batch > kStepMaxRequests) return HELM_ERR_UNSUPPORTED;
  // positions are 32-bit; so are the counts of pages and tokens, and a stride of all
  // threads beyond them
  static_assert(kStepCluster * kStepThreads * std::max(kStepRun, kStepTokens) < 1 << 17, "");
  constexpr int64_t kMost = (int64_t(1) << 31) - (1 << 17);
  if (static_cast<int64_t>(batch) * max_pages > kMost || num_rows > kMost ||
      static_cast<int64_t>(max_pages) * page_size >= (int64_t(1) << 31))
    return HELM_ERR_UNSUPPORTED;
  int shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    while ((1 << ++shift) < page_size) {
    }
  const int wide =
      ((reinterpret_cast<uintptr_t>(seq_ids) | reinterpret_cast<uintptr_t>(positions)) & 15) == 0 &&
      (reinterpret_cast<uintptr_t>(slot_rows) & 31) == 0;
  const StepArgs a = {past_lens, new_lens,  page_table, pt_stride_b, max_pages, free_pages,
                      free_capacity, free_count, free_count_out, kv_lens, cu_tokens, seq_ids,
                      positions, slot_rows, batch,     page_size,  num_rows, shift, wide};
  const size_t smem = (static_cast<size_t>(batch) * 4 + 3) * sizeof(int) + batch;
  cudaError_t e = cudaSuccess;
  static int cluster_of[64] = {0};  // CTAs of a large step, by device
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev >= 64) return HELM_ERR_UNSUPPORTED;
  constexpr int kMostSmem =
      (kStepMaxRequests * 4 + 3) * static_cast<int>(sizeof(int)) + kStepMaxRequests;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (e == cudaSuccess && cluster_of[dev] == 0) {
    e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kMostSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) {
      int clusters = 0;
      cfg.gridDim = dim3(kStepCluster);
      cfg.blockDim = dim3(kStepThreads);
      cfg.dynamicSmemBytes = kMostSmem;
      attr[0].val.clusterDim.x = kStepCluster;
      const cudaError_t o = cudaOccupancyMaxActiveClusters(&clusters, step_tables_kernel, &cfg);
      if (o != cudaSuccess) (void)cudaGetLastError();
      cluster_of[dev] = o == cudaSuccess && clusters > 0 ? kStepCluster : kStepPortableCluster;
    }
  }
  if (e == cudaSuccess) {
    // one CTA for a step of single tokens; its threads follow the work, barriers
    // being most of what it does
    const bool small = num_rows <= kStepTokensPerCta && batch <= kStepThreads;
    const unsigned ctas = small ? 1 : static_cast<unsigned>(cluster_of[dev]);
    const int work = std::max(batch, num_rows);
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(small ? std::min(kStepThreads, std::max(128, (work + 31) / 32 * 32))
                              : kStepThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    attr[0].val.clusterDim.x = ctas;
    e = cudaLaunchKernelEx(&cfg, step_tables_kernel, a);
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return HELM_ERR_CUDA;
  }
  return HELM_OK;
}
