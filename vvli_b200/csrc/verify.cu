// verify.cu - verification of drafted tokens against the target's
// probabilities, with given random numbers (vvli_cuda_verify_drafts).
//
// The rejection rule of speculative sampling: draft x with target probability
// p(x) and draft probability q(x) is accepted when u q(x) < p(x), i.e. with
// probability min(1, p / q); the first rejected position draws from
// max(0, p - q), which makes every emitted token distributed as p.
// The sampler's vvli_cuda_sample draws one token; this is its form for several.
//
// One thread-block cluster per request.  Every CTA works the accepted count
// out for itself (two gathered floats a draft), then the cluster sums the
// weights of the one row that is drawn from, a contiguous slice per CTA and
// per warp, in 64 bits: a cumulative sum of 10^5 fp32 terms rounded to 32 bits
// would move the drawn index.  The CTAs exchange their slice sums through
// distributed shared memory, and the CTA with the threshold goes over the one
// warp slice that holds it once more (from L2), a short run per thread.  Bound: HBM, one row of the target and,
// when a draft was rejected, one of the draft model per request.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "op_common.cuh"

using namespace vvli;

namespace {

constexpr int kVerThreads = 256;
constexpr int kVerWarps = kVerThreads / 32;
constexpr int kVerCluster = 8;
constexpr int kVerRun = 12;  // values of a thread's run held in registers: the whole run up to 196,608 tokens
constexpr int kVerUnroll = 4;  // loads in flight per lane and row

VVLI_DEV uint32_t ver_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
VVLI_DEV void ver_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
VVLI_DEV double ld_cluster_f64(const double* p, uint32_t rank) {
  uint32_t a;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a));
  return v;
}

// The weights a token is drawn from: max(0, t - d), t alone (d null), and 0 at `skip`.
struct Weights {
  const float* t;
  const float* d;
  int skip;
  VVLI_DEV double of(float a, float b, int i) const {
    const double w = static_cast<double>(a) - static_cast<double>(b);
    return w > 0.0 && i != skip ? w : 0.0;  // NaN: 0
  }
  VVLI_DEV double at(int i) const { return of(t[i], d ? d[i] : 0.f, i); }
};

// This lane's share of the weights [s0, s1): whole batches of kVerUnroll loads
// without a branch between them, so that all are in flight, then the rest.
template <int VEC, bool DRAFT>
VVLI_DEV double slice_sum(const Weights& w, int s0, int s1) {
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
  int i = s0 + VEC * lane;
  if constexpr (VEC == 4) {
    for (; i + 128 * (kVerUnroll - 1) + 4 <= s1; i += 128 * kVerUnroll) {
      float4 x[kVerUnroll], y[kVerUnroll];
#pragma unroll
      for (int u = 0; u < kVerUnroll; ++u) {
        x[u] = *reinterpret_cast<const float4*>(w.t + i + 128 * u);
        y[u] = DRAFT ? *reinterpret_cast<const float4*>(w.d + i + 128 * u) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < kVerUnroll; ++u) {
        const int k = i + 128 * u;
        sum += (w.of(x[u].x, y[u].x, k) + w.of(x[u].y, y[u].y, k + 1)) +
               (w.of(x[u].z, y[u].z, k + 2) + w.of(x[u].w, y[u].w, k + 3));
      }
    }
    for (; i < s1; i += 128)
      for (int k = i; k < min(i + 4, s1); ++k) sum += w.of(w.t[k], DRAFT ? w.d[k] : 0.f, k);
  } else {
    for (; i + 32 * (kVerUnroll - 1) < s1; i += 32 * kVerUnroll) {
      float x[kVerUnroll], y[kVerUnroll];
#pragma unroll
      for (int u = 0; u < kVerUnroll; ++u) x[u] = w.t[i + 32 * u], y[u] = DRAFT ? w.d[i + 32 * u] : 0.f;
#pragma unroll
      for (int u = 0; u < kVerUnroll; ++u) sum += w.of(x[u], y[u], i + 32 * u);
    }
    for (; i < s1; i += 32) sum += w.of(w.t[i], DRAFT ? w.d[i] : 0.f, i);
  }
  return sum;
}

VVLI_DEV double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// VEC: 4 when every row starts on a 16-byte boundary, else 1.
template <int VEC>
__global__ void __launch_bounds__(kVerThreads, 4) verify_kernel(const vvli_verify_args p) {
  __shared__ double warp_part[kVerWarps];
  __shared__ double scan_part[kVerWarps];
  __shared__ double cta_part[2];  // this CTA's slice sum, by attempt (read by the cluster)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / kVerCluster;
  const uint32_t rank = ver_cluster_rank();
  const int V = static_cast<int>(p.vocab);
  const int r0 = min(max(0, p.cu_rows[b]), static_cast<int>(p.rows));
  const int r1 = min(max(r0, p.cu_rows[b + 1]), static_cast<int>(p.rows));
  if (r0 == r1) {  // uniform over the cluster
    if (rank == 0 && tid == 0) p.accepted[b] = 0;
    return;
  }
  // accepted drafts: every warp of the cluster finds the same count
  const int drafts = r1 - r0 - 1;
  int acc = 0;
  for (;;) {
    const int i = acc + lane;
    bool ok = false;
    if (i < drafts) {
      const int x = p.tokens[r0 + i + 1];
      if (x >= 0 && x < V) {
        const double pt = p.target[static_cast<size_t>(r0 + i) * p.target_stride + x];
        const double qd = p.draft ? p.draft[static_cast<size_t>(r0 + i) * p.draft_stride + x] : 1.0f;
        ok = static_cast<double>(p.u_accept[r0 + i]) * qd < pt;
      }
    }
    const unsigned yes = __ballot_sync(0xffffffffu, ok);
    const int run = yes == 0xffffffffu ? 32 : __ffs(~yes) - 1;
    acc += run;
    if (run < 32) break;
  }
  const int row = r0 + acc;
  const bool rejected = acc < drafts;
  if (rank == 0) {
    if (tid == 0) p.accepted[b] = acc;
    for (int r = r0 + tid; r < r1; r += kVerThreads)
      if (r != row) p.out_tokens[r] = r < row ? p.tokens[r + 1] : -1;
  }
  Weights w{p.target + static_cast<size_t>(row) * p.target_stride, nullptr, -1};
  if (rejected) {
    if (p.draft)
      w.d = p.draft + static_cast<size_t>(row) * p.draft_stride;
    else
      w.skip = p.tokens[row + 1];
  }
  // contiguous slices: CTA `rank` of the cluster, warp `warp` of the CTA
  const int per_warp = ((V + kVerCluster * kVerWarps - 1) / (kVerCluster * kVerWarps) + 3) & ~3;  // V <= 2^30
  const long long first = static_cast<long long>(rank * kVerWarps + warp) * per_warp;
  const int s0 = static_cast<int>(min(first, static_cast<long long>(V)));
  const int s1 = static_cast<int>(min(first + per_warp, static_cast<long long>(V)));
  double before = 0.0, total = 0.0, mine = 0.0, slice = 0.0;
  int chosen = -1;  // CTA that holds the threshold
  double thr = 0.0;
  for (int attempt = 0; attempt < 2; ++attempt) {
    const double sum = w.d ? slice_sum<VEC, true>(w, s0, s1) : slice_sum<VEC, false>(w, s0, s1);
    mine = warp_sum_f64(sum);
    if (lane == 0) warp_part[warp] = mine;
    __syncthreads();
    slice = 0.0;
#pragma unroll
    for (int u = 0; u < kVerWarps; ++u) slice += warp_part[u];
    if (tid == 0) cta_part[attempt] = slice;
    ver_cluster_sync();
    double part[kVerCluster];
    total = 0.0;
#pragma unroll
    for (int c = 0; c < kVerCluster; ++c) total += part[c] = ld_cluster_f64(&cta_part[attempt], c);
    if (!(total > 0.0) && rejected && attempt == 0) {  // nothing of p is above q: draw from p (uniform)
      w.d = nullptr, w.skip = -1;
      continue;
    }
    thr = static_cast<double>(p.u_sample[b]) * total;
    double run = 0.0;
    int last = 0;  // last slice with any weight: takes the draw when rounding or u >= 1 leaves none
    double last_before = 0.0;
#pragma unroll
    for (int c = 0; c < kVerCluster; ++c) {
      if (part[c] > 0.0) last = c, last_before = run;
      if (chosen < 0 && part[c] > 0.0 && run + part[c] > thr) chosen = c, before = run;
      run += part[c];
    }
    if (chosen < 0) chosen = last, before = last_before;
    break;
  }
  ver_cluster_sync();  // no CTA leaves while its sum may still be read
  if (static_cast<int>(rank) != chosen) return;
  int cw = -1, last = 0;
  double run = before, wb = before, last_before = before;
#pragma unroll
  for (int u = 0; u < kVerWarps; ++u) {
    const double part = warp_part[u];
    if (part > 0.0) last = u, last_before = run;
    if (cw < 0 && part > 0.0 && run + part > thr) cw = u, wb = run;
    run += part;
  }
  if (cw < 0) cw = last, wb = last_before;
  // That slice again, by the whole CTA: a contiguous run per thread, its sum, a
  // scan over the CTA, and the thread whose run holds the threshold walks it.
  const long long c_first = static_cast<long long>(rank * kVerWarps + cw) * per_warp;
  const int c0 = static_cast<int>(min(c_first, static_cast<long long>(V)));
  const int c1 = static_cast<int>(min(c_first + per_warp, static_cast<long long>(V)));
  const int per = (c1 - c0 + kVerThreads - 1) / kVerThreads;
  const int b0 = min(c0 + tid * per, c1), b1 = min(b0 + per, c1);
  double sum = 0.0;
  float x[kVerRun], y[kVerRun];  // the run, or its last values where it is longer
  for (int i0 = b0; i0 < b1; i0 += kVerRun) {
#pragma unroll
    for (int u = 0; u < kVerRun; ++u) {
      const int i = i0 + u;
      x[u] = i < b1 ? w.t[i] : 0.f, y[u] = w.d && i < b1 ? w.d[i] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kVerRun; ++u) sum += w.of(x[u], y[u], i0 + u);
  }
  double c = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, c, o);
    if (lane >= o) c += y;
  }
  if (lane == 31) scan_part[warp] = c;
  __syncthreads();
  double lead = wb;
#pragma unroll
  for (int u = 0; u < kVerWarps; ++u)
    if (u < warp) lead += scan_part[u];
  // the first thread whose run passes the threshold, else the last with any weight
  __shared__ int hit_s[kVerWarps], any_s[kVerWarps];
  const unsigned hit = __ballot_sync(0xffffffffu, sum > 0.0 && lead + c > thr);
  const unsigned any = __ballot_sync(0xffffffffu, sum > 0.0);
  if (lane == 0) {
    hit_s[warp] = hit ? warp * 32 + __ffs(hit) - 1 : INT_MAX;
    any_s[warp] = any ? warp * 32 + 31 - __clz(any) : -1;
  }
  __syncthreads();
  int owner = INT_MAX, some = -1;
#pragma unroll
  for (int u = 0; u < kVerWarps; ++u) owner = min(owner, hit_s[u]), some = max(some, any_s[u]);
  if (owner == INT_MAX) owner = max(some, 0);
  if (tid != owner) return;
  int best = c0;  // no weight at all: the slice's first index (0: the draw falls to the first slice)
  run = lead + c - sum;
  bool over = false;
  if (per <= kVerRun) {
#pragma unroll
    for (int u = 0; u < kVerRun; ++u) {
      const double v = w.of(x[u], y[u], b0 + u);
      if (v > 0.0 && !over) best = b0 + u, run += v, over = run > thr;
    }
  } else {
    for (int i = b0; i < b1 && !over; ++i) {
      const double v = w.at(i);
      if (v > 0.0) best = i, run += v, over = run > thr;
    }
  }
  p.out_tokens[row] = best;
}

std::string check_verify(const vvli_verify_args* a) {
  if (!a) return "null arguments";
  if (a->requests < 1 || a->requests > 65535) return "requests must be in [1, 65535]";
  if (a->rows > INT_MAX) return "rows must be below 2^31";
  if (a->vocab < 1 || a->vocab > (1u << 30)) return "vocab must be in [1, 2^30]";
  if (a->target_stride < a->vocab || a->target_stride > (1ull << 40) ||
      (a->draft && (a->draft_stride < a->vocab || a->draft_stride > (1ull << 40))))
    return "strides must be at least vocab";
  const void* need[] = {a->target, a->tokens, a->cu_rows, a->u_accept, a->u_sample, a->accepted, a->out_tokens};
  for (const void* q : need) {
    if (!q) return "null pointer";
    if (!aligned_to(q, 4)) return "pointers must be 4-byte aligned";
  }
  if (!aligned_to(a->draft, 4)) return "pointers must be 4-byte aligned";
  return "";
}

cudaError_t queue_verify(const vvli_verify_args& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kVerCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(a.requests) * kVerCluster);
  cfg.blockDim = dim3(kVerThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool vec = aligned_to(a.target, 16) && a.target_stride % 4 == 0 &&
                   (!a.draft || (aligned_to(a.draft, 16) && a.draft_stride % 4 == 0));
  return vec ? cudaLaunchKernelEx(&cfg, verify_kernel<4>, a) : cudaLaunchKernelEx(&cfg, verify_kernel<1>, a);
}

}  // namespace

extern "C" int vvli_cuda_verify_drafts(int device, const vvli_verify_args* args, void* stream) {
  return run_op(
      "verify_drafts", device, [&] { return check_verify(args); },
      [&] { return queue_verify(*args, static_cast<cudaStream_t>(stream)); });
}
