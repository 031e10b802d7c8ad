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

constexpr int kQkThreads = 256;
constexpr int kQkMaxTokens = 8;  // tokens of a CTA

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
VVLI_DEV void st16(void* p, const uint4& v) { *reinterpret_cast<uint4*>(p) = v; }

struct QkDev {
  int tokens, hq, hk, d, pairs, shift;  // page_size = 1 << shift
  int per_cta;                          // tokens of a CTA
  int interleaved;
  unsigned slots_end;                   // pages << shift
  long long page_stride, q_stride, k_stride, v_stride, out_stride;
  float eps;
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_cache, *v_cache;
  const uint16_t *q_weight, *k_weight;
  const int *positions, *slots;
  const double* inv_freq;
};

// NORM: enum vvli_qk_norm.  LANES: threads of a head, head_dim / 16 rounded up
// to a power of two (LANES <= 16, so a head stays in a warp).
template <class T, int NORM, int LANES>
__global__ void __launch_bounds__(kQkThreads) qk_rope_kernel(const QkDev p) {
  extern __shared__ float2 turn[];  // [tokens of the CTA][pairs] cosine, sine
  __shared__ float row_sum[2][kQkMaxTokens][kQkThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t0 = blockIdx.x * p.per_cta, nt = min(p.per_cta, p.tokens - t0);
  const int j = tid % LANES;  // chunk pair within the head
  const int heads = p.hq + 2 * p.hk, chunks = p.d >> 4;
  const int c0 = !p.interleaved && 8 * j < p.pairs ? j : 2 * j;
  // chunk c's partner; the part past 2 * pairs starts at an even chunk
  const int c1 = !p.interleaved && 8 * j < p.pairs ? j + (p.pairs >> 3) : 2 * j + 1;
  const bool turned = 8 * j < p.pairs;

  for (int i = tid; i < nt * p.pairs; i += kQkThreads) {
    const int t = i / p.pairs, f = i - t * p.pairs;
    constexpr double kInvTwoPi = 0.15915494309189533576888;
    const double turns = static_cast<double>(p.positions[t0 + t]) * p.inv_freq[f] * kInvTwoPi;
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    turn[i] = make_float2(c, s);
  }
  if constexpr (NORM == VVLI_NORM_ROW) {
    // mean squares over all q heads and over all k heads of each token
    for (int t = 0; t < nt; ++t) {
      float ss[2] = {0.f, 0.f};
      for (int h = tid / LANES; h < p.hq + p.hk; h += kQkThreads / LANES) {
        if (j >= chunks) continue;
        const uint16_t* src = h < p.hq ? p.q + (t0 + t) * p.q_stride + h * p.d
                                       : p.k + (t0 + t) * p.k_stride + (h - p.hq) * p.d;
        float v[16];
        unpack8<T>(ld16(src + 8 * c0), v);
        unpack8<T>(ld16(src + 8 * c1), v + 8);
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) a = fmaf(v[i], v[i], a);
        ss[h >= p.hq] += a;
      }
      ss[0] = warp_sum(ss[0]), ss[1] = warp_sum(ss[1]);
      if (lane == 0) row_sum[0][t][warp] = ss[0], row_sum[1][t][warp] = ss[1];
    }
  }
  __syncthreads();

  const int total = nt * heads;  // (token, head) items, LANES threads each
  const int rounds = (total + kQkThreads / LANES - 1) / (kQkThreads / LANES);
  for (int r = 0; r < rounds; ++r) {  // uniform: the head sums below are warp-wide
    const int item = r * (kQkThreads / LANES) + tid / LANES;
    const bool live = item < total && j < chunks;
    const int t = live ? item / heads : 0, h = live ? item - t * heads : 0;
    const long long tok = t0 + t;
    const int kind = h < p.hq ? 0 : h < p.hq + p.hk ? 1 : 2;  // q, k, v
    const int g = kind == 0 ? h : kind == 1 ? h - p.hq : h - p.hq - p.hk;
    const uint16_t* src = kind == 0   ? p.q + tok * p.q_stride
                          : kind == 1 ? p.k + tok * p.k_stride
                                      : p.v + tok * p.v_stride;
    src += g * p.d;
    uint16_t* dst = nullptr;
    if (live) {
      if (kind == 0) {
        dst = p.q_out + tok * p.out_stride + g * p.d;
      } else {
        const unsigned slot = static_cast<unsigned>(p.slots[tok]);  // -1 is past the end too
        if (slot < p.slots_end)
          dst = (kind == 1 ? p.k_cache : p.v_cache) + static_cast<long long>(slot >> p.shift) * p.page_stride +
                ((static_cast<long long>(g) << p.shift) + (slot & ((1u << p.shift) - 1))) * p.d;
      }
    }
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (live) a = ld16(src + 8 * c0), b = ld16(src + 8 * c1);
    if (kind == 2) {
      if (dst) st16(dst + 8 * c0, a), st16(dst + 8 * c1, b);
    }
    float x[16];
    unpack8<T>(a, x);
    unpack8<T>(b, x + 8);
    if constexpr (NORM != VVLI_NORM_NONE) {
      float ms;
      if constexpr (NORM == VVLI_NORM_HEAD) {
        ms = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ms = fmaf(x[i], x[i], ms);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ms += __shfl_xor_sync(0xffffffffu, ms, o);
        ms /= static_cast<float>(p.d);
      } else {
        ms = 0.f;
#pragma unroll
        for (int w = 0; w < kQkThreads / 32; ++w) ms += row_sum[kind == 1][t][w];
        ms /= static_cast<float>(kind == 1 ? p.hk : p.hq) * p.d;
      }
      const float scale = 1.0f / sqrtf(ms + p.eps);
      const uint16_t* w = kind == 1 ? p.k_weight : p.q_weight;
      if (NORM == VVLI_NORM_ROW && w) w += g * p.d;
      float y[16];
      if (w && live && kind != 2) {
        unpack8<T>(ld16(w + 8 * c0), y);
        unpack8<T>(ld16(w + 8 * c1), y + 8);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = x[i] * scale * y[i];
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= scale;
      }
    }
    if (!dst || kind == 2) continue;  // the rest has no warp-wide step
    if (turned) {
      const float2* cs = turn + t * p.pairs + 8 * j;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 w = cs[i];
        const float xa = p.interleaved ? x[2 * i] : x[i], xb = p.interleaved ? x[2 * i + 1] : x[i + 8];
        const float ra = xa * w.x - xb * w.y, rb = xb * w.x + xa * w.y;
        if (p.interleaved)
          x[2 * i] = ra, x[2 * i + 1] = rb;
        else
          x[i] = ra, x[i + 8] = rb;
      }
    }
    st16(dst + 8 * c0, pack8<T>(x));
    st16(dst + 8 * c1, pack8<T>(x + 8));
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

template <class T, int NORM>
cudaError_t queue_lanes(const QkDev& p, unsigned grid, size_t smem, cudaStream_t s) {
  const int chunks = p.d >> 4;
  if (chunks <= 1)
    qk_rope_kernel<T, NORM, 1><<<grid, kQkThreads, smem, s>>>(p);
  else if (chunks <= 2)
    qk_rope_kernel<T, NORM, 2><<<grid, kQkThreads, smem, s>>>(p);
  else if (chunks <= 4)
    qk_rope_kernel<T, NORM, 4><<<grid, kQkThreads, smem, s>>>(p);
  else if (chunks <= 8)
    qk_rope_kernel<T, NORM, 8><<<grid, kQkThreads, smem, s>>>(p);
  else
    qk_rope_kernel<T, NORM, 16><<<grid, kQkThreads, smem, s>>>(p);
  return cudaGetLastError();
}

template <class T>
cudaError_t queue_norm(const QkDev& p, int norm, unsigned grid, size_t smem, cudaStream_t s) {
  return norm == VVLI_NORM_NONE   ? queue_lanes<T, VVLI_NORM_NONE>(p, grid, smem, s)
         : norm == VVLI_NORM_HEAD ? queue_lanes<T, VVLI_NORM_HEAD>(p, grid, smem, s)
                                  : queue_lanes<T, VVLI_NORM_ROW>(p, grid, smem, s);
}

cudaError_t queue_qk(const vvli_qk_rope_args& a, cudaStream_t s) {
  if (a.tokens == 0) return cudaSuccess;
  QkDev p{};
  p.tokens = static_cast<int>(a.tokens), p.hq = static_cast<int>(a.q_heads), p.hk = static_cast<int>(a.kv_heads);
  p.d = static_cast<int>(a.head_dim), p.pairs = static_cast<int>(a.rotary_pairs);
  p.shift = 4;
  while ((1u << p.shift) < a.page_size) ++p.shift;
  p.interleaved = a.interleaved != 0;
  p.slots_end = static_cast<unsigned>(a.pages) << p.shift;
  p.page_stride = static_cast<long long>(a.page_stride), p.q_stride = static_cast<long long>(a.q_stride);
  p.k_stride = static_cast<long long>(a.k_stride), p.v_stride = static_cast<long long>(a.v_stride);
  p.out_stride = static_cast<long long>(a.out_stride);
  p.eps = a.eps;
  p.q = static_cast<const uint16_t*>(a.q), p.k = static_cast<const uint16_t*>(a.k);
  p.v = static_cast<const uint16_t*>(a.v), p.q_out = static_cast<uint16_t*>(a.q_out);
  p.k_cache = static_cast<uint16_t*>(a.k_cache), p.v_cache = static_cast<uint16_t*>(a.v_cache);
  p.q_weight = static_cast<const uint16_t*>(a.q_weight), p.k_weight = static_cast<const uint16_t*>(a.k_weight);
  p.positions = a.positions, p.slots = a.slots, p.inv_freq = a.inv_freq;
  p.per_cta = 1;
  const unsigned grid = static_cast<unsigned>((p.tokens + p.per_cta - 1) / p.per_cta);
  const size_t smem = static_cast<size_t>(p.per_cta) * p.pairs * sizeof(float2);
  return a.dtype == VVLI_BF16 ? queue_norm<__nv_bfloat16>(p, a.norm, grid, smem, s)
                              : queue_norm<__half>(p, a.norm, grid, smem, s);
}

}  // namespace

extern "C" int vvli_cuda_qk_rope_write(int device, const vvli_qk_rope_args* args, void* stream) {
  return run_op(
      "qk_rope_write", device, [&] { return check_qk(args); },
      [&] { return queue_qk(*args, static_cast<cudaStream_t>(stream)); });
}
