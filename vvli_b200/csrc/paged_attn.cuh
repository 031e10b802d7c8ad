// paged_attn.cuh - what the two kernels of vvli_cuda_paged_attention share: the
// work schedule, the split parts and the score arithmetic.
//
// Work.  A request's query rows of one kv head are packed: row r is the new
// token r / G and the group's q head r % G.  An item is (request, kv head,
// block of ROWS packed rows); it counts the KT-key tiles that any of its rows
// sees, and EXTRA units more, which stand for its start and end (q in, sums
// out) and come first.  The units of all items in order (request, head, block, tile)
// form one line that is cut into equal shares, one per CTA, whatever the
// lengths: a CTA's share is a run of segments, each a range of one item's
// tiles.  A segment that is a whole item writes its output; the others (at most
// the first and the last of a CTA) leave unnormalised sums and their running
// maximum in the workspace, two slots per CTA, and the combine kernel adds an
// item's parts in tile order.  The lengths stay on the device: every CTA sums
// the units over the requests for itself.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

#include "common.cuh"
#include "op_common.cuh"

namespace vvli {

constexpr int kPaMaxCtas = 160;    // CTAs of a launch at most: the workspace is sized for them
constexpr int kPaMaxRows = 256;    // rows of an item at most

struct PaDesc {  // what the combine kernel needs of a CTA
  int finish;    // its first segment ends an item that another CTA began
  int h, blk;    // that item: kv head, block
  int row0;      // first q row of its request
  int rows;      // its packed rows
  int first;     // the CTA that began it; its part is in slot `slot`, the later CTAs' in slot 0
  int slot;
  int pad;
};

struct PaParams {
  int B, T, hq, hk, G, shift, pages, width;  // page_size = 1 << shift
  int longest;                               // what a table row holds: seq_len is cut there
  uint32_t g_mul, g_shift;                   // x / G = x * g_mul >> g_shift for 0 <= x < 2^31
  int window;                                // 0: none
  float scale_log2;                          // scale * log2(e); its magnitude without a feature, then
  int negate;                                // the sign goes into q
  float cap_y, cap_log2;                     // softcap: scale / cap; cap * log2(e), 0 without
  long long q_stride, out_stride;
  const uint16_t* q;
  const uint16_t* v;                         // the value cache, pages page_stride elements apart
  long long page_stride;
  uint16_t* out;
  float* lse;
  const float* alibi;
  const int *table, *cu, *seq;
  // workspace
  int* err;
  PaDesc* desc;    // [kPaMaxCtas]
  float* part_ml;  // [kPaMaxCtas][2][kPaMaxRows][2] reference (the maximum, but see pa_lift; log2 units) and sum
  float* part_o;   // [kPaMaxCtas][2] sums of an item's rows: [rows][D], or [D / 4][rows][4] (256 rows, a thread each)
};

inline size_t pa_workspace_bytes(int d) {
  const size_t slots = static_cast<size_t>(kPaMaxCtas) * 2 * kPaMaxRows;
  return 256 + kPaMaxCtas * sizeof(PaDesc) + slots * 2 * sizeof(float) + slots * d * sizeof(float);
}

// Variants of the score arithmetic.  Without either, exp's argument is one FMA
// of the raw score; a scale too small for that (0 among them) takes the ALiBi
// form, with slopes of 0.
enum : int { kPaCap = 1, kPaAlibi = 2 };
inline int pa_features(const PaParams& p) {
  return p.cap_log2 > 0.f ? kPaCap | (p.alibi ? kPaAlibi : 0) : p.alibi || !(p.scale_log2 > 1e-30f) ? kPaAlibi : 0;
}

// ---------------------------------------------------------------- schedule

struct PaReq {
  int row0;  // first row of q
  int n;     // rows of q (tokens)
  int pos0;  // position of the first (may be negative)
};

VVLI_DEV PaReq pa_request(const PaParams& p, int b) {
  const int c0 = min(max(p.cu[b], 0), p.T), c1 = max(p.cu[b + 1], c0);
  PaReq r;
  r.row0 = c0;
  r.n = min(c1, p.T) - c0;
  r.pos0 = max(min(p.seq[b], p.longest), 0) - (c1 - c0);
  return r;
}

// g_mul = ceil(2^g_shift / G), g_shift = 31 + ceil(log2 G): exact, since x * (g_mul G - 2^g_shift) < 2^g_shift.
VVLI_DEV int pa_div_g(const PaParams& p, int x) {
  return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * p.g_mul >> p.g_shift);
}
// a / b of small or large counts.
VVLI_DEV long long pa_div(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

template <int ROWS>
VVLI_DEV int pa_blocks(const PaParams& p, const PaReq& r) {
  return (r.n * p.G + ROWS - 1) / ROWS;
}

// Keys [lo, hi) that rows of block blk see, and its tiles [t0, t1), one at least.
struct PaItem {
  int rows;     // rows of the block
  int lo, hi;
  int t0, t1;
};
template <int ROWS, int KT>
VVLI_DEV PaItem pa_item(const PaParams& p, const PaReq& r, int blk) {
  PaItem it;
  it.rows = min(ROWS, r.n * p.G - blk * ROWS);
  const int first = r.pos0 + pa_div_g(p, blk * ROWS), last = r.pos0 + pa_div_g(p, blk * ROWS + it.rows - 1);
  it.hi = max(0, last + 1);
  it.lo = p.window && first >= p.window ? first + 1 - p.window : 0;
  it.t0 = it.lo / KT;
  it.t1 = max(it.t0 + 1, (it.hi + KT - 1) / KT);
  return it;
}

struct PaShare {
  long long each, more;     // units of a CTA; the first `more` CTAs have one more
  long long u0, u1;         // this CTA's
  int active;               // CTAs with a share
  int b, h, blk, off;       // where u0 lies: item and unit of it
  long long item_first;     // first unit of that item
};

// Sum over the CTA (NT threads, a multiple of 32) of one value a thread, and the sum before it.
template <int NT>
VVLI_DEV long long pa_scan(long long v, long long* part, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += a;
  }
  __syncthreads();
  if (lane == 31) part[warp] = s;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w == warp) before = total;
    total += part[w];
  }
  return before + s - v;
}

// Units of one kv head of request b over all its blocks; a warp works out requests of many blocks together.
template <int ROWS, int KT, int EXTRA>
VVLI_DEV long long pa_units(const PaParams& p, int b, bool live) {
  PaReq r{0, 0, 0};
  int nb = 0;
  if (live) r = pa_request(p, b), nb = pa_blocks<ROWS>(p, r);
  long long u = 0;
  if (nb <= 2) {
    for (int i = 0; i < nb; ++i) {
      const PaItem it = pa_item<ROWS, KT>(p, r, i);
      u += it.t1 - it.t0 + EXTRA;
    }
  }
  unsigned big = __ballot_sync(0xffffffffu, nb > 2);
  while (big) {
    const int src = __ffs(big) - 1;
    big &= big - 1;
    PaReq o;
    o.row0 = 0, o.n = __shfl_sync(0xffffffffu, r.n, src), o.pos0 = __shfl_sync(0xffffffffu, r.pos0, src);
    const int n = __shfl_sync(0xffffffffu, nb, src);
    long long s = 0;
    for (int i = threadIdx.x & 31; i < n; i += 32) {
      const PaItem it = pa_item<ROWS, KT>(p, o, i);
      s += it.t1 - it.t0 + EXTRA;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if ((threadIdx.x & 31) == src) u = s;
  }
  return u;
}

VVLI_DEV long long pa_start(const PaShare& s, long long i) { return s.each * i + min(i, s.more); }

template <int NT>
struct PaScratch {
  long long part[NT / 32];
  long long units[NT];  // of one kv head of each request
};

// Units of requests b0 .. b0 + NT: thread t gets request b0 + t's, those of one
// head, and the units of all heads of the requests before it.  Neighbouring
// requests go to different warps, which share the ones of many blocks.
template <int ROWS, int KT, int EXTRA, int NT>
VVLI_DEV long long pa_count(const PaParams& p, int b0, PaScratch<NT>* sc, long long& units, long long& before) {
  const int at = (threadIdx.x & 31) * (NT / 32) + (threadIdx.x >> 5);
  __syncthreads();
  sc->units[at] = pa_units<ROWS, KT, EXTRA>(p, b0 + at, b0 + at < p.B);
  __syncthreads();
  units = sc->units[threadIdx.x];
  long long total;
  before = pa_scan<NT>(units * p.hk, sc->part, total);
  return total;
}

// This CTA's share, worked out by all its NT threads; valid in `out` (shared) after the call.
template <int ROWS, int KT, int EXTRA, int NT>
VVLI_DEV void pa_schedule(const PaParams& p, PaShare* out, PaScratch<NT>* sc) {
  const int tid = threadIdx.x;
  long long total = 0, before, units;
  for (int b0 = 0; b0 < p.B; b0 += NT) total += pa_count<ROWS, KT, EXTRA, NT>(p, b0, sc, units, before);
  const int active = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  PaShare s;
  s.each = active ? pa_div(total, active) : 0, s.more = total - s.each * active;
  s.active = active;
  const bool idle = static_cast<int>(blockIdx.x) >= active;
  const long long u0 = idle ? 0 : pa_start(s, blockIdx.x), u1 = idle ? 0 : pa_start(s, blockIdx.x + 1);
  if (tid == 0) out->each = s.each, out->more = s.more, out->active = active, out->u0 = u0, out->u1 = u1;
  long long done = 0;
  for (int b0 = 0; b0 < p.B && u0 < u1; b0 += NT) {
    long long t = total;
    if (p.B > NT) t = pa_count<ROWS, KT, EXTRA, NT>(p, b0, sc, units, before);  // more requests than threads: again
    const long long lead = done + before;
    if (units > 0 && lead <= u0 && u0 < lead + units * p.hk) {
      out->b = b0 + tid;
      out->h = static_cast<int>(pa_div(u0 - lead, units));
      out->item_first = lead + out->h * units;  // first unit of the head, for now
    }
    done += t;
    if (done > u0) break;  // uniform
  }
  __syncthreads();
  if (tid < 32 && u0 < u1) {  // the block of the head and the tile of the block
    const PaReq r = pa_request(p, out->b);
    const int nb = pa_blocks<ROWS>(p, r);
    long long at = out->item_first;
    for (int k0 = 0; k0 < nb; k0 += 32) {
      const int k = k0 + tid;
      int n = 0;
      if (k < nb) {
        const PaItem it = pa_item<ROWS, KT>(p, r, k);
        n = it.t1 - it.t0 + EXTRA;
      }
      long long s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, s, o);
        if (tid >= o) s += a;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, at + s > u0 && at + s - n <= u0 && n > 0);
      if (hit) {
        if (tid == __ffs(hit) - 1) out->blk = k, out->item_first = at + s - n, out->off = static_cast<int>(u0 - (at + s - n));
        break;
      }
      at += __shfl_sync(0xffffffffu, s, 31);
    }
  }
  __syncthreads();
}

// A run of tiles of one item.
struct PaSeg {
  int b, h, blk;
  PaReq r;
  PaItem it;
  int t0, t1;        // tiles of this segment
  bool starts, ends;  // the item's first / last tile among them
  bool at_start;     // the CTA's first segment
  long long item_first;
};

template <int ROWS, int KT, int EXTRA>
struct PaWalk {
  long long u, u1, item_first;
  int b, h, blk, off;
  bool first;
  VVLI_DEV explicit PaWalk(const PaShare& s)
      : u(s.u0), u1(s.u1), item_first(s.item_first), b(s.b), h(s.h), blk(s.blk), off(s.off), first(true) {}
  VVLI_DEV bool next(const PaParams& p, PaSeg& s) {
    if (u >= u1) return false;
    s.r = pa_request(p, b);
    while (s.r.n <= 0) s.r = pa_request(p, ++b);  // some later request has the unit u
    s.b = b, s.h = h, s.blk = blk;
    s.it = pa_item<ROWS, KT>(p, s.r, blk);
    s.item_first = item_first;
    s.at_start = first;
    const int left = s.it.t1 - s.it.t0 + EXTRA - off;
    const int n = static_cast<int>(min(static_cast<long long>(left), u1 - u));
    s.t0 = s.it.t0 + max(0, off - EXTRA);
    s.t1 = s.it.t0 + max(0, off + n - EXTRA);
    if (s.t1 == s.t0) return false;  // the share ends before the item's first tile
    s.starts = s.t0 == s.it.t0;
    s.ends = n == left;
    first = false;
    u += n;
    if (s.ends) {
      item_first += s.it.t1 - s.it.t0 + EXTRA;
      off = 0;
      if (++blk >= pa_blocks<ROWS>(p, s.r)) {
        blk = 0;
        if (++h >= p.hk) h = 0, ++b;
      }
    } else {
      off += n;
    }
    return true;
  }
};

// Workspace slot of a segment that is not a whole item.
VVLI_DEV int pa_slot(const PaSeg& s) { return s.at_start ? 0 : 1; }

// Called by one thread per CTA: what the combine kernel does for it.
template <int EXTRA>
VVLI_DEV void pa_describe(const PaParams& p, const PaShare& sh, const PaSeg* s) {
  PaDesc d{};
  if (s && !s->starts && s->ends) {
    const long long tile = s->item_first + EXTRA, wide = sh.more * (sh.each + 1);  // the unit of the item's first tile
    const long long j = tile < wide ? pa_div(tile, sh.each + 1) : sh.more + pa_div(tile - wide, sh.each);
    d.finish = 1, d.h = s->h, d.blk = s->blk, d.row0 = s->r.row0, d.rows = s->it.rows;
    d.first = static_cast<int>(j), d.slot = pa_start(sh, j) >= s->item_first ? 0 : 1;  // its second slot unless its share starts there
  }
  p.desc[blockIdx.x] = d;
}

// ---------------------------------------------------------------- scores
// In log2 units, so that exp is one ex2: x = s * scale * log2(e), or with a
// softcap cap * log2(e) * tanh(y), y = s * scale / cap.  tanh.approx is off by
// 2^-11 (a capped score of 50 by 0.02); here tanh(y) = 1 - 2 / (1 + e^2y), and for
// |y| <= 0.4, where that would lose the leading digits, y times the degree-3
// minimax fit of tanh(y) / y in y^2 (relative error 1e-7).
VVLI_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
VVLI_DEV float pa_capped(float s, const PaParams& p) {
  const float y = s * p.cap_y, u = y * y;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(y * 2.885390081777927f)));  // 2 log2(e)
  float q = fmaf(-0.04755360336859857f, u, 0.13270976752811006f);
  q = fmaf(fmaf(q, u, -0.3333136245857671f), u, 0.9999999019009012f);
  return p.cap_log2 * (fabsf(y) <= 0.4f ? q * y : fmaf(-2.0f, r, 1.0f));
}

// Probabilities are 2^(x - reference), and enter the second product rounded to
// the 16-bit type (half a step of each, on top of the output's own rounding).  A
// second product with what the rounding leaves would make them exact to 2^-17:
// against 64 bits, the output's error is 1.07 to 1.41 times that of rounding the
// output alone without it, 1.00 times with it.  It is left out because it costs
// 359 -> 504 us at 4,096 rows over 8,192 keys (8B heads), 24.7 -> 28 us at 48
// requests x 5 rows (0.5B heads), 75 -> 97 us for 16 mixed requests with a cap, and
// 285.5 -> 290.5 us in the streaming kernel at 16 x 24,000 to 32,767 keys, where
// infinite values times what is left (0 or less) would have to be kept out as
// well.  Scores, maxima, sums and parts are fp32.
// bf16 has fp32's exponents; fp16 loses bits below 2^-14 and holds nothing below
// 2^-25, so there the reference is `fp16_bits` (log2) below the row's maximum: with
// it at the maximum, 30,000 keys 18 (natural units) below a few dominant ones
// vanished from the output while the sum counted them.  The sums and the
// log-sum-exp are relative to the same reference.  2^fp16_bits times what a
// maximum may rise before the reference follows stays below 2^16, fp16's end;
// for maxima from 2^22 on the difference would round, and the reference is the maximum.
template <class T>
constexpr float pa_lift(float fp16_bits) {
  return std::is_same<T, __half>::value ? fp16_bits : 0.f;
}
VVLI_DEV float pa_reference(float m, float lift) { return fabsf(m) < 4194304.f ? m - lift : m; }

template <class T>
VVLI_DEV uint32_t pa_pack(float a, float b);
template <>
VVLI_DEV uint32_t pa_pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
VVLI_DEV uint32_t pa_pack<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// TMA load of a box of the cache's 4-D map {64 elements, rows of a page, 64-element slices, pages}.
VVLI_DEV void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// The table entry of page pg of request b, or one past the cache (which a TMA load fills with zeros).
VVLI_DEV int pa_page(const PaParams& p, int b, int pg) {
  int id = -1;
  if (pg < p.width) id = __ldg(p.table + static_cast<size_t>(b) * p.width + pg);
  return id >= 0 && id < p.pages ? id : p.pages;
}

// ---------------------------------------------------------------- values that are not finite
// The second product multiplies a row's zeros with the values it does not see,
// and 0 times an infinity or NaN is no 0.  Where the rows of an item see
// different keys of a tile, such values are therefore taken out of the tile in
// shared memory, the tiles that had any are kept as a range, and what a row does
// see of them is added to its sums at the end, from the cache.
template <class T>
VVLI_DEV uint32_t pa_not_finite(uint32_t w) {  // 0xffff in each half that is an infinity or NaN
  const uint32_t m = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(w & m, m);
}
template <class T>
VVLI_DEV float pa_half(uint32_t w, int i) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return i ? bf16_hi(w) : bf16_lo(w);
  const __half2 v = *reinterpret_cast<const __half2*>(&w);
  return i ? __high2float(v) : __low2float(v);
}
// Adds what the row at position pos sees of them in key tiles [f0, f1] of request b, N dims from e0 on.
template <class T, int D, int KT, int N>
VVLI_DEV void pa_add_not_finite(const PaParams& p, const PaSeg& s, int pos, int e0, int f0, int f1, float* o) {
  const int end = min(pos + 1, min((f1 + 1) * KT, s.it.hi));
#pragma unroll 1
  for (int key = max(f0 * KT, p.window ? pos + 1 - p.window : 0); key < end; ++key) {
    const int page = pa_page(p, s.b, key >> p.shift);
    if (page == p.pages) continue;
    const uint16_t* v = p.v + page * p.page_stride +
                        ((static_cast<long long>(s.h) << p.shift) + (key & ((1 << p.shift) - 1))) * D + e0;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(v + i), m = pa_not_finite<T>(w);
      if (m & 0xffffu) o[i] += pa_half<T>(w, 0);
      if (m >> 16) o[i + 1] += pa_half<T>(w, 1);
    }
  }
}

// ---------------------------------------------------------------- host
template <class K>
cudaError_t allow_smem(K kernel, size_t bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}
cudaError_t pa_tensor_map(CUtensorMap* map, const void* cache, const vvli_paged_attn_args& a, uint32_t box_rows,
                          uint32_t box_slices);
// The tensor-core kernel (paged_attn_tc.cu) and, for either, the combine kernel (paged_attn.cu).
template <class T, int D>
cudaError_t pa_set_up_tc();
template <class T, int D>
cudaError_t pa_queue_tc(const PaParams& p, const vvli_paged_attn_args& a, int ctas, cudaStream_t s);
template <class T, int D, int ROWS>
cudaError_t pa_queue_combine(const PaParams& p, int ctas, cudaStream_t s);

}  // namespace vvli
