// paged_plan.cu - pages, positions and cache slots of one step from the
// requests' lengths (vvli_cuda_paged_plan).
//
// Every output is a function of prefix sums over the requests: the rows'
// (cu_new) and the lacking pages'.  One thread-block cluster does it in one
// launch: every CTA computes both sums over all requests for itself (a few
// block scans; the lengths are read by all CTAs, and the cluster barrier
// between the reads and the first write lets owned / owned_out and the free
// count be the same memory), keeps them in shared memory, and then takes its
// share of the rows and of the taken pages, each finding its request by a
// binary search in shared memory.  Bound by latency: one dependent read, the
// scans, the searches; a second launch or a workspace for the sums would cost
// more than the repeated scan.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "op_common.cuh"

using namespace vvli;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxRequests = 8192;
constexpr int kPlanCluster = 8;  // CTAs of a large step

struct PlanShared {  // per request; 4 arrays of `requests` ints
  int* first_row;    // cu_new
  int* first_page;   // taken pages before this request's
  int* context;
  int* owned;        // owned pages, -1 - owned for an unserved request
};

// Inclusive sum over the CTA of one value a thread; all threads get `total`.
VVLI_DEV long long block_scan(long long v, long long* part, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += a;
  }
  __syncthreads();  // the previous scan's readers of `part` are done
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    long long p = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += a;
    }
    part[lane] = p;
  }
  __syncthreads();
  total = part[31];
  return v + (warp ? part[warp - 1] : 0);
}

// Last index i in [0, n) with a[i] <= x (a does not decrease, a[0] <= x).
VVLI_DEV int last_at_most(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const vvli_paged_plan_args p, int shift) {
  extern __shared__ int plan_smem[];
  __shared__ long long part[32];
  const int B = static_cast<int>(p.requests), P = 1 << shift, tid = threadIdx.x;
  const int nt = gridDim.x * kPlanThreads, gt = blockIdx.x * kPlanThreads + tid;
  PlanShared s{plan_smem, plan_smem + B, plan_smem + 2 * B, plan_smem + 3 * B};
  const long long cap = static_cast<long long>(p.max_tokens), width = static_cast<long long>(p.table_width);
  const long long free0 = min(max(0LL, static_cast<long long>(*p.free_count)), static_cast<long long>(p.free_entries));
  long long rows = 0, lacking = 0, taken = 0;  // sums over the requests before this chunk
  const bool writer = blockIdx.x == 0;
  // what the writer CTA writes per request once every CTA has read its inputs
  int w_cu[kPlanMaxRequests / kPlanThreads], w_len[kPlanMaxRequests / kPlanThreads];
  int w_own[kPlanMaxRequests / kPlanThreads], w_st[kPlanMaxRequests / kPlanThreads];
#pragma unroll
  for (int c = 0; c < kPlanMaxRequests / kPlanThreads; ++c) {
    const int b = c * kPlanThreads + tid;
    if (c * kPlanThreads >= B) break;  // uniform
    long long ctx = 0, add = 0, own = 0, total;
    if (b < B) ctx = max(0, p.context[b]), add = max(0, p.new_tokens[b]), own = max(0, p.owned[b]);
    const long long end = rows + block_scan(add, part, total);
    rows += total;
    const long long pages = (ctx + add + P - 1) >> shift;
    long long need = max(0LL, pages - own);
    int st = end > cap && add > 0 && cap > 0 ? 3 : pages > width || ctx + add > INT_MAX ? 2 : 0;
    if (st) need = 0;
    const long long upto = lacking + block_scan(need, part, total);
    lacking += total;
    if (need > 0 && upto > free0) st = 1, need = 0;
    const long long have = taken + block_scan(need, part, total);
    taken += total;
    w_cu[c] = static_cast<int>(min(end, static_cast<long long>(INT_MAX)));
    w_len[c] = st ? 0 : static_cast<int>(ctx + add);
    w_own[c] = static_cast<int>(own + need);
    w_st[c] = st;
    if (b < B) {
      s.first_row[b] = static_cast<int>(min(end - add, static_cast<long long>(INT_MAX)));
      s.first_page[b] = static_cast<int>(have - need);
      s.context[b] = static_cast<int>(ctx);
      s.owned[b] = st ? -1 - static_cast<int>(own) : static_cast<int>(own);
    }
  }
  if (gridDim.x > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __syncthreads();  // the sums are in shared memory, and every CTA has read the state
  if (writer) {
#pragma unroll
    for (int c = 0; c < kPlanMaxRequests / kPlanThreads; ++c) {
      const int b = c * kPlanThreads + tid;
      if (b >= B) break;
      p.cu_new[b + 1] = w_cu[c];
      p.seq_len[b] = w_len[c];
      p.owned_out[b] = w_own[c];
      p.status[b] = w_st[c];
    }
    if (tid == 0) {
      p.cu_new[0] = 0;
      *p.free_count_out = static_cast<int>(free0 - taken);
    }
  }
  // A served request takes free_pages[free0 - 1 - n] as its n-th of all taken
  // pages.  Requests that take none share their first_page with the next one
  // that does, and the search finds the last, so it never finds them unless no
  // later request takes any (then n >= taken).
  for (long long n = gt; n < taken; n += nt) {
    const int b = last_at_most(s.first_page, B, static_cast<int>(n));
    const size_t at = static_cast<size_t>(s.owned[b]) + static_cast<size_t>(n - s.first_page[b]);
    p.block_table[static_cast<size_t>(b) * p.table_width + at] = p.free_pages[free0 - 1 - n];
  }
  const long long shown = min(rows, cap);
  for (long long t = gt; t < cap; t += nt) {
    int pos = 0, slot = -1;
    if (t < shown) {
      const int b = last_at_most(s.first_row, B, static_cast<int>(t));
      const long long at = static_cast<long long>(s.context[b]) + (t - s.first_row[b]);
      pos = static_cast<int>(min(at, static_cast<long long>(INT_MAX)));
      const int own = s.owned[b];
      if (own >= 0) {
        const long long page = at >> shift;
        const int id = page < own ? p.block_table[static_cast<size_t>(b) * p.table_width + page]
                                  : p.free_pages[free0 - 1 - (s.first_page[b] + (page - own))];
        if (id >= 0 && id <= (INT_MAX - (P - 1)) >> shift) slot = (id << shift) + static_cast<int>(at & (P - 1));
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

std::string check_plan(const vvli_paged_plan_args* a) {
  if (!a) return "null arguments";
  if (a->requests < 1 || a->requests > kPlanMaxRequests)
    return "requests must be in [1, " + std::to_string(kPlanMaxRequests) + "]";
  const std::string page = check_page_size(a->page_size);
  if (!page.empty()) return page;
  if (a->free_entries < 1 || a->free_entries > INT_MAX) return "free_entries must be in [1, 2^31)";
  if (a->table_width < 1 || a->table_width > INT_MAX) return "table_width must be in [1, 2^31)";
  if (a->max_tokens > INT_MAX) return "max_tokens must be below 2^31";
  const void* need[] = {a->context,    a->new_tokens, a->owned,     a->block_table,    a->free_pages, a->free_count,
                        a->cu_new,     a->seq_len,    a->owned_out, a->free_count_out, a->status};
  for (const void* q : need) {
    if (!q) return "null pointer";
    if (!aligned_to(q, 4)) return "pointers must be 4-byte aligned";
  }
  if (a->max_tokens && (!a->positions || !a->slots)) return "null pointer";
  if (!aligned_to(a->positions, 4) || !aligned_to(a->slots, 4)) return "pointers must be 4-byte aligned";
  return "";
}

cudaError_t queue_plan(int device, const vvli_paged_plan_args& a, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(a.requests) * 4 * sizeof(int);  // <= 128 KB
  static SetupOnce setup[kOpMaxDevices];
  if (device < 0 || device >= kOpMaxDevices) return cudaErrorInvalidDevice;
  const cudaError_t e = setup[device]([] {
    return cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kPlanMaxRequests * 4 * sizeof(int));
  });
  if (e != cudaSuccess) return e;
  // One CTA while its threads take at most two rows each; the cluster beyond.
  const unsigned ctas = a.max_tokens <= 2 * kPlanThreads ? 1 : kPlanCluster;
  int shift = 4;
  while ((1u << shift) < a.page_size) ++shift;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_plan_kernel, a, shift);
}

}  // namespace

extern "C" int vvli_cuda_paged_plan(int device, const vvli_paged_plan_args* args, void* stream) {
  return run_op(
      "paged_plan", device, [&] { return check_plan(args); },
      [&] { return queue_plan(device, *args, static_cast<cudaStream_t>(stream)); });
}
