// qk_rope.cu - RMSNorm of q and k, rotary positions and the paged cache
// write of a step's tokens, in one pass (vvli_cuda_qk_rope_write).
//
// Bound: HBM (every 16-bit value of q, k and v is read once and written once;
// about two FMAs a value).  A thread takes the two 16-byte chunks that hold
// eight rotary pairs of a head, so a pair never leaves its thread: chunks j
// and j + rotary_pairs / 8 for split halves, 2 j and 2 j + 1 for interleaved
// pairs and for the part of a head that is not turned.  head_dim / 16 threads
// side by side own a head and meet in shuffles for its mean square; a CTA owns
// a few tokens, so that the 64-bit angles of a token are worked out once for
// all its heads, in shared memory.
//   angle: positions[t] * inv_freq[i] in turns, reduced to [-1/2, 1/2] in 64
//   bits before the fp32 sine and cosine, so far positions lose nothing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "op_common.cuh"

using namespace vvli;

namespace {

constexpr int kQkMaxThreads = 256;
constexpr int kQkMaxTokens = 8;  // tokens of a CTA
// Tokens in flight, and CTAs per SM: 16,384 tokens of 48 heads of 128 took 73.6 us so,
// 75 with five ahead, 80 to 82 with two CTAs or four (registers), 84 loading one ahead
// into registers.
constexpr int kQkAhead = 3;
constexpr int kQkPerSm = 3;
constexpr int kQkStages = kQkAhead + 1;

template <class T>
struct Pair16;
template <>
struct Pair16<__nv_bfloat16> {
  static VVLI_DEV float2 load(uint32_t w) { return make_float2(bf16_lo(w), bf16_hi(w)); }
  static VVLI_DEV uint32_t store(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Pair16<__half> {
  static VVLI_DEV float2 load(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static VVLI_DEV uint32_t store(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

template <class T>
VVLI_DEV void unpack8(const uint4& w, float* v) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Pair16<T>::load(u[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
template <class T>
VVLI_DEV uint4 pack8(const float* v) {
  return make_uint4(Pair16<T>::store(v[0], v[1]), Pair16<T>::store(v[2], v[3]), Pair16<T>::store(v[4], v[5]),
                    Pair16<T>::store(v[6], v[7]));
}
VVLI_DEV uint4 ld16(const void* p) { return *reinterpret_cast<const uint4*>(p); }
VVLI_DEV void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
VVLI_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
VVLI_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}
VVLI_DEV void st16(void* p, const uint4& v) { *reinterpret_cast<uint4*>(p) = v; }

struct QkDev {
  int tokens, hq, hk, d, pairs, shift;  // page_size = 1 << shift
  int per_cta;                          // tokens of a CTA
  unsigned slots_end;                   // pages << shift
  long long page_stride, q_stride, k_stride, v_stride, out_stride;
  float eps, q_share, k_share;  // 1 over the values of a mean
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_cache, *v_cache;
  const uint16_t *q_weight, *k_weight;
  const int *positions, *slots;
  const double* inv_freq;
};

// PAIRED: interleaved pairs.  NORM: enum vvli_qk_norm.  LANES: threads of a
// head, head_dim / 16 rounded up to a power of two (LANES <= 16, so a head stays
// in a warp).  CTA (x, y): tokens x * per_cta .. and part y of the heads;
// a thread keeps its head and chunks, hence its weights, for all tokens.
template <class T, int NORM, int LANES, bool PAIRED>
__global__ void __launch_bounds__(kQkMaxThreads, kQkPerSm) qk_rope_kernel(const QkDev p) {
  extern __shared__ __align__(16) float2 turn[];  // [tokens of the CTA][pairs] cosine, sine
  uint4* ring = reinterpret_cast<uint4*>(turn + ((p.per_cta * p.pairs + 1) & ~1));  // [kQkStages][2][threads]
  __shared__ unsigned slots[kQkMaxTokens];
  __shared__ float row_sum[2][kQkMaxTokens][kQkMaxThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int t0 = blockIdx.x * p.per_cta, nt = min(p.per_cta, p.tokens - t0);
  const int j = tid % LANES, chunks = p.d >> 4;  // chunk pair within the head
  const bool turned = 8 * j < p.pairs;
  // chunk c0 and its partner; the part past 2 * pairs starts at an even chunk
  const int c0 = 8 * (!PAIRED && turned ? j : 2 * j);
  const int c1 = 8 * (!PAIRED && turned ? j + (p.pairs >> 3) : 2 * j + 1);
  // Parts of the heads: one per CTA, or all in turn where a norm over the row
  // needs every head before any is written (q_out may be q).
  for (int part = blockIdx.y; part * (threads / LANES) < p.hq + 2 * p.hk; part += gridDim.y) {
    const int head = part * (threads / LANES) + tid / LANES;
    const int kind = head < p.hq ? 0 : head < p.hq + p.hk ? 1 : 2;  // q, k, v
    const int g = head - (kind == 0 ? 0 : kind == 1 ? p.hq : p.hq + p.hk);
    const bool live = head < p.hq + 2 * p.hk && j < chunks;
    const uint16_t* src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const long long step = kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride;
    src += t0 * step + g * p.d;
    // A thread's own chunks of the next kQkAhead tokens are on their way to its
    // own places of shared memory, so that they take no registers.
    auto ahead = [&](int t) {
      if (live && t < nt) {
        uint4* at = ring + (t % kQkStages) * 2 * threads + tid;
        cp_async16(at, src + t * step + c0);
        cp_async16(at + threads, src + t * step + c1);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int t = 0; t < kQkAhead; ++t) ahead(t);
    uint4 wa, wb;  // this thread's weights
    if constexpr (NORM != VVLI_NORM_NONE) {
      const uint16_t* wp = kind == 1 ? p.k_weight : p.q_weight;
      const uint32_t one = Pair16<T>::store(1.f, 1.f);
      wa = wb = make_uint4(one, one, one, one);
      if (wp && live && kind < 2) {
        if (NORM == VVLI_NORM_ROW) wp += g * p.d;
        wa = ld16(wp + c0), wb = ld16(wp + c1);
      }
    }
    if (part == static_cast<int>(blockIdx.y)) {
      if (tid < nt) slots[tid] = static_cast<unsigned>(p.slots[t0 + tid]);
      for (int i = tid; i < nt * p.pairs; i += threads) {
        const int t = i / p.pairs, f = i - t * p.pairs;
        constexpr double kInvTwoPi = 0.15915494309189533576888;
        const double turns = static_cast<double>(p.positions[t0 + t]) * p.inv_freq[f] * kInvTwoPi;
        float s, c;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
        turn[i] = make_float2(c, s);
      }
      if constexpr (NORM == VVLI_NORM_ROW) {
        // square sums over all q heads and over all k heads of each token (whatever heads this CTA has)
        for (int t = 0; t < nt; ++t) {
          float ss[2] = {0.f, 0.f};
          for (int h = tid / LANES; h < p.hq + p.hk; h += threads / LANES) {
            if (j >= chunks) continue;
            const uint16_t* row = h < p.hq ? p.q + (t0 + t) * p.q_stride + h * p.d
                                           : p.k + (t0 + t) * p.k_stride + (h - p.hq) * p.d;
            float v[16];
            unpack8<T>(ld16(row + c0), v);
            unpack8<T>(ld16(row + c1), v + 8);
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sq = fmaf(v[i], v[i], sq);
            ss[h >= p.hq] += sq;
          }
          ss[0] = warp_sum(ss[0]), ss[1] = warp_sum(ss[1]);
          if (lane == 0) row_sum[0][t][warp] = ss[0], row_sum[1][t][warp] = ss[1];
        }
      }
      __syncthreads();
    }

    // the head's own threads: other heads of the warp may be values, which skip the sums
    const unsigned head_mask = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
    uint16_t* const out = p.q_out + t0 * p.out_stride + g * p.d;
    uint16_t* const cache = kind == 1 ? p.k_cache : p.v_cache;
    for (int t = 0; t < nt; ++t) {
      cp_async_wait<kQkAhead - 1>();
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (live) {
        const uint4* at = ring + (t % kQkStages) * 2 * threads + tid;
        a = at[0], b = at[threads];
      }
      ahead(t + kQkAhead);  // into the place of token t - 1
      const unsigned slot = live && kind ? slots[t] : 0u;
      uint16_t* dst = nullptr;
      if (live && kind == 0)
        dst = out + t * p.out_stride;
      else if (live && slot < p.slots_end)  // -1 is past the end too
        dst = cache + static_cast<long long>(slot >> p.shift) * p.page_stride +
              ((static_cast<long long>(g) << p.shift) + (slot & ((1u << p.shift) - 1))) * p.d;
      if (kind < 2) {
        float x[16];
        unpack8<T>(a, x);
        unpack8<T>(b, x + 8);
        if constexpr (NORM != VVLI_NORM_NONE) {
          float ms = 0.f;
          if constexpr (NORM == VVLI_NORM_HEAD) {
#pragma unroll
            for (int i = 0; i < 16; ++i) ms = fmaf(x[i], x[i], ms);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ms += __shfl_xor_sync(head_mask, ms, o);
          } else {
            for (int u = 0; u < threads / 32; ++u) ms += row_sum[kind][t][u];
          }
          const float scale = rsqrtf(fmaf(ms, kind == 1 ? p.k_share : p.q_share, p.eps));
          float w[16];
          unpack8<T>(wa, w);
          unpack8<T>(wb, w + 8);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= scale * w[i];
        }
        if (turned) {
          const float4* cs = reinterpret_cast<const float4*>(turn + t * p.pairs + 8 * j);  // two pairs each
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 w2 = cs[i >> 1];
            const float cw = i & 1 ? w2.z : w2.x, sw = i & 1 ? w2.w : w2.y;
            float& xa = x[PAIRED ? 2 * i : i];
            float& xb = x[PAIRED ? 2 * i + 1 : i + 8];
            const float ra = xa * cw - xb * sw, rb = xb * cw + xa * sw;
            xa = ra, xb = rb;
          }
        }
        a = pack8<T>(x), b = pack8<T>(x + 8);
      }
      if (dst) st16(dst + c0, a), st16(dst + c1, b);
    }
  }
}

std::string check_qk(const vvli_qk_rope_args* a) {
  if (!a) return "null arguments";
  if (a->tokens > INT_MAX) return "tokens must be below 2^31";
  if (a->q_heads < 1 || a->q_heads > 512 || a->kv_heads < 1 || a->kv_heads > 512)
    return "q_heads and kv_heads must be in [1, 512]";
  if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 16) return "head_dim must be a multiple of 16 in [16, 256]";
  if (a->rotary_pairs % 8 || 2 * a->rotary_pairs > a->head_dim || a->rotary_pairs > 128)
    return "rotary_pairs must be a multiple of 8 of at most head_dim / 2";
  const std::string page = check_page_size(a->page_size);
  if (!page.empty()) return page;
  if (a->pages < 1 || a->pages > static_cast<uint64_t>(INT_MAX) / a->page_size)
    return "pages must be at least 1 with pages * page_size < 2^31";
  if (a->page_stride % 8 || a->page_stride < a->kv_heads * a->page_size * a->head_dim || a->page_stride > (1ull << 40))
    return "page_stride must be a multiple of 8 and at least kv_heads * page_size * head_dim";
  const uint64_t qw = a->q_heads * a->head_dim, kw = a->kv_heads * a->head_dim;
  const uint64_t strides[] = {a->q_stride, a->k_stride, a->v_stride, a->out_stride};
  for (int i = 0; i < 4; ++i)
    if (strides[i] % 8 || strides[i] < (i == 1 || i == 2 ? kw : qw) || strides[i] > (1ull << 31))
      return "strides must be multiples of 8 and at least a row";
  if (a->dtype != VVLI_BF16 && a->dtype != VVLI_FP16) return "dtype must be VVLI_BF16 or VVLI_FP16";
  if (a->norm < VVLI_NORM_NONE || a->norm > VVLI_NORM_ROW) return "norm must be VVLI_NORM_NONE, _HEAD or _ROW";
  if (!(a->eps >= 0.f)) return "eps must be >= 0";
  const void* wide[] = {a->q, a->k, a->v, a->q_out, a->k_cache, a->v_cache};
  for (const void* q : wide) {
    if (!q) return "null pointer";
    if (!aligned_to(q, 16)) return "16-bit pointers must be 16-byte aligned";
  }
  if (!aligned_to(a->q_weight, 16) || !aligned_to(a->k_weight, 16)) return "16-bit pointers must be 16-byte aligned";
  if (!a->slots || (a->rotary_pairs && (!a->positions || !a->inv_freq))) return "null pointer";
  if (!aligned_to(a->slots, 4) || !aligned_to(a->positions, 4) || !aligned_to(a->inv_freq, 8))
    return "positions and slots must be 4-byte aligned, inv_freq 8-byte";
  return "";
}

template <class T, int NORM, bool PAIRED>
cudaError_t queue_lanes(const QkDev& p, size_t smem, cudaStream_t s) {
  int lanes = 1;
  while (lanes < p.d >> 4) lanes *= 2;
  // all heads in one CTA if it can hold them, else in CTAs of equal shares
  const int heads = p.hq + 2 * p.hk, most = kQkMaxThreads / lanes;
  const int parts = (heads + most - 1) / most, each = (heads + parts - 1) / parts;
  const int threads = (each * lanes + 31) & ~31;
  smem += static_cast<size_t>(kQkStages) * 2 * threads * sizeof(uint4);  // <= 8 + 32 KB
  const dim3 grid((static_cast<unsigned>(p.tokens) + p.per_cta - 1) / p.per_cta, NORM == VVLI_NORM_ROW ? 1 : (heads + threads / lanes - 1) / (threads / lanes));
  switch (lanes) {
    case 1: qk_rope_kernel<T, NORM, 1, PAIRED><<<grid, threads, smem, s>>>(p); break;
    case 2: qk_rope_kernel<T, NORM, 2, PAIRED><<<grid, threads, smem, s>>>(p); break;
    case 4: qk_rope_kernel<T, NORM, 4, PAIRED><<<grid, threads, smem, s>>>(p); break;
    case 8: qk_rope_kernel<T, NORM, 8, PAIRED><<<grid, threads, smem, s>>>(p); break;
    default: qk_rope_kernel<T, NORM, 16, PAIRED><<<grid, threads, smem, s>>>(p); break;
  }
  return cudaGetLastError();
}

template <class T, bool PAIRED>
cudaError_t queue_norm(const QkDev& p, int norm, size_t smem, cudaStream_t s) {
  return norm == VVLI_NORM_NONE   ? queue_lanes<T, VVLI_NORM_NONE, PAIRED>(p, smem, s)
         : norm == VVLI_NORM_HEAD ? queue_lanes<T, VVLI_NORM_HEAD, PAIRED>(p, smem, s)
                                  : queue_lanes<T, VVLI_NORM_ROW, PAIRED>(p, smem, s);
}

cudaError_t queue_qk(const vvli_qk_rope_args& a, cudaStream_t s) {
  if (a.tokens == 0) return cudaSuccess;
  QkDev p{};
  p.tokens = static_cast<int>(a.tokens), p.hq = static_cast<int>(a.q_heads), p.hk = static_cast<int>(a.kv_heads);
  p.d = static_cast<int>(a.head_dim), p.pairs = static_cast<int>(a.rotary_pairs);
  p.shift = 4;
  while ((1u << p.shift) < a.page_size) ++p.shift;
  p.slots_end = static_cast<unsigned>(a.pages) << p.shift;
  p.page_stride = static_cast<long long>(a.page_stride), p.q_stride = static_cast<long long>(a.q_stride);
  p.k_stride = static_cast<long long>(a.k_stride), p.v_stride = static_cast<long long>(a.v_stride);
  p.out_stride = static_cast<long long>(a.out_stride);
  p.eps = a.eps;
  const bool row = a.norm == VVLI_NORM_ROW;
  p.q_share = 1.0f / static_cast<float>(row ? p.hq * p.d : p.d);
  p.k_share = 1.0f / static_cast<float>(row ? p.hk * p.d : p.d);
  p.q = static_cast<const uint16_t*>(a.q), p.k = static_cast<const uint16_t*>(a.k);
  p.v = static_cast<const uint16_t*>(a.v), p.q_out = static_cast<uint16_t*>(a.q_out);
  p.k_cache = static_cast<uint16_t*>(a.k_cache), p.v_cache = static_cast<uint16_t*>(a.v_cache);
  p.q_weight = static_cast<const uint16_t*>(a.q_weight), p.k_weight = static_cast<const uint16_t*>(a.k_weight);
  p.positions = a.positions, p.slots = a.slots, p.inv_freq = a.inv_freq;
  // Few tokens are spread over the SMs; many share a CTA's table and prologue.
  p.per_cta = p.tokens <= 256 ? 1 : p.tokens <= 1024 ? 2 : kQkMaxTokens;
  const size_t smem = static_cast<size_t>((p.per_cta * p.pairs + 1) & ~1) * sizeof(float2);
  if (a.dtype == VVLI_BF16)
    return a.interleaved ? queue_norm<__nv_bfloat16, true>(p, a.norm, smem, s)
                         : queue_norm<__nv_bfloat16, false>(p, a.norm, smem, s);
  return a.interleaved ? queue_norm<__half, true>(p, a.norm, smem, s) : queue_norm<__half, false>(p, a.norm, smem, s);
}

}  // namespace

extern "C" int vvli_cuda_qk_rope_write(int device, const vvli_qk_rope_args* args, void* stream) {
  return run_op(
      "qk_rope_write", device, [&] { return check_qk(args); },
      [&] { return queue_qk(*args, static_cast<cudaStream_t>(stream)); });
}
