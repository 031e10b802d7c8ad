// paged_attn.cu - attention of the new tokens over a paged 16-bit cache
// (vvli_cuda_paged_attention): the C entry, the kernel for steps of few rows
// per request (decode tokens, drafts), and the kernel that adds split parts.
//
// paged_short_kernel.  Bound: HBM, every visible key and value once (two to
// four FLOP a byte at 1 to 8 rows per kv head).  One CTA per SM takes its share
// of the 64-key tiles (paged_attn.cuh), so the lengths need not be even or
// many.  A producer warp streams the tiles through a 128 KB ring of shared
// memory with TMA, one box per page of keys and of values, as far ahead as the
// ring reaches and across segment borders; a page outside the cache is a box
// outside the tensor map, which arrives as zeros.  Eight consumer warps each
// take 16 keys of a tile: S = Q K^T and O += P V are mma.sync.m16n8k16 (16
// packed rows fill M; a tcgen05 MMA has 128 rows, seven eighths of them
// padding at 16, and both are far from being the bound), the running maximum
// and sum are the warp's own, so nothing is exchanged until the segment ends
// and the warps' parts meet in shared memory.  With up to 16 rows the two
// halves of the warps take tiles in turn; with up to 32 each half takes 16 rows
// of every tile; longer requests take several blocks.
#include "paged_attn.cuh"

#include <algorithm>
#include <cmath>
#include <mutex>

namespace vvli {
namespace {

constexpr int kShKeys = 64;                       // keys of a tile
constexpr int kShConsumers = 256;                 // 8 warps
constexpr int kShThreads = kShConsumers + 32;     // and the producer
// An item's start and end count as this many tiles (64 requests of 100 to 2,000 tokens
// at head_dim 64: 44 us with none, 34 with 1, 28 with 3 or 6).
constexpr int kShExtra = 3;
constexpr int kShBarrier = 1;                     // named barrier of the consumers

template <int D>
struct ShLayout {
  static constexpr uint32_t kv = kShKeys * D * 2;       // bytes of a tile's keys (or values)
  static constexpr uint32_t stage = 2 * kv;
  static constexpr uint32_t stages = 131072 / stage;    // 4 at D 128, 8 at D 64
  static constexpr uint32_t o_ld = D + 4;               // floats of a merge row
  static constexpr uint32_t merge = stages * stage;     // [8 warps][16 rows][o_ld]
  static constexpr uint32_t ml = merge + 8 * 16 * o_ld * 4;  // [8][16][2]
  static constexpr uint32_t bars = ml + 8 * 16 * 2 * 4;
  static constexpr uint32_t share = bars + 2 * stages * 8;
  static constexpr uint32_t odd = share + 64;           // ranges of tiles with values that are not finite, [2][2]
  static constexpr uint32_t part = odd + 64;          // schedule scratch
  static constexpr uint32_t smem = part + sizeof(PaScratch<kShThreads>) + 1024;  // + alignment slack
};
static_assert(sizeof(PaShare) <= 64, "the share fits its space");

VVLI_DEV void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
VVLI_DEV void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <class T>
VVLI_DEV void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
VVLI_DEV void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
VVLI_DEV void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// RG: 16-row groups of a block.  FEAT: softcap or ALiBi.
template <class T, int D, int RG, bool FEAT>
__global__ void __launch_bounds__(kShThreads, 1)
    paged_short_kernel(const PaParams p, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
  using L = ShLayout<D>;
  constexpr int ROWS = 16 * RG;
  constexpr int ST = L::stages;
  extern __shared__ uint8_t sh_raw[];
  const uint32_t raw = smem_u32(sh_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;  // swizzled boxes want 1024-byte alignment
  uint8_t* sm = sh_raw + (base - raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* empty = full + ST;
  PaShare* share = reinterpret_cast<PaShare*>(sm + L::share);
  int* odd = reinterpret_cast<int*>(sm + L::odd);  // first and last tile, by the segment's parity
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  grid_launch_dependents();  // the combine kernel waits for this grid's completion before reading
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], RG == 1 ? 4 : 8);  // the warps that read a stage
    }
    odd[0] = odd[2] = INT_MAX, odd[1] = odd[3] = -1;
    fence_barrier_init();
  }
  pa_schedule<ROWS, kShKeys, kShExtra, kShThreads>(p, share, reinterpret_cast<PaScratch<kShThreads>*>(sm + L::part));
  PaWalk<ROWS, kShKeys, kShExtra> walk(*share);
  PaSeg sg;
  const int rows_page = min(1 << p.shift, kShKeys);  // key rows of a box
  bool dead = false;  // a wait gave up: the rest is skipped

  if (warp == 8) {  // ---- producer
    int it = 0;
    const int per_tile = kShKeys >> (p.shift < 6 ? p.shift : 6);  // boxes of a tile
    bool any = false;
    while (walk.next(p, sg)) {
      if (!any && lane == 0) pa_describe<kShExtra>(p, *share, &sg);
      any = true;
      const int pg0 = (sg.t0 * kShKeys) >> p.shift;
      int chunk = 0;  // lane l holds the pages pg0 + 32 chunk + l, and those 32 further
      int ids = pa_page(p, sg.b, pg0 + lane), ids2 = pa_page(p, sg.b, pg0 + 32 + lane);
      for (int t = sg.t0; t < sg.t1; ++t, ++it) {
        const int s = it % ST;
        if (it >= ST && !dead) dead = !mbar_wait(&empty[s], ((it / ST) - 1) & 1, p.err);
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        // boxes with a visible key; a tile without any arrives at once
        const int key0 = t * kShKeys;
        const int boxes = min(per_tile, (sg.it.hi - key0 + rows_page - 1) / rows_page);
        if (lane == 0) mbar_arrive_expect_tx(&full[s], max(boxes, 0) * 2 * rows_page * D * 2);
        __syncwarp();
        const int first = (key0 >> p.shift) - pg0;
        if (first >= 32 * (chunk + 1)) {
          ++chunk;
          ids = ids2;
          ids2 = pa_page(p, sg.b, pg0 + 32 * (chunk + 1) + lane);
        }
        // a tile's pages lie in one chunk: 32 is a multiple of the boxes of a tile, but
        // the segment's first page need not be, so the next chunk may hold the last ones
        const int j = first - 32 * chunk + lane;
        const int a = __shfl_sync(0xffffffffu, ids, j & 31), c = __shfl_sync(0xffffffffu, ids2, j & 31);
        if (lane < boxes) {
          const int id = j < 32 ? a : c;
          const uint32_t dst = base + s * L::stage + lane * rows_page * D * 2;
          const int y = (sg.h << p.shift) + (key0 & ((1 << p.shift) - 1));
          tma_load_4d(dst, &kmap, 0, y, 0, id, &full[s]);
          tma_load_4d(dst + L::kv, &vmap, 0, y, 0, id, &full[s]);
        }
      }
      if (dead) break;
    }
    if (!any && lane == 0) pa_describe<kShExtra>(p, *share, nullptr);
    // no copy of this CTA is in flight when it ends
    for (int k = max(0, it - ST); k < it; ++k) mbar_wait(&full[k % ST], (k / ST) & 1, p.err);
    return;
  }

  // ---- consumers: warp w takes keys 16 (w % 4) .. of a tile
  const int kq = warp & 3, half = warp >> 2;
  const int g = lane >> 2, t4 = lane & 3;
  const int rg0 = RG == 2 ? 16 * half : 0;  // this warp's rows of the block
  float* mo = reinterpret_cast<float*>(sm + L::merge);
  float* mml = reinterpret_cast<float*>(sm + L::ml);
  // ldmatrix: byte offset of this lane's row within the K and V tile, before the 16-byte chunk
  const int kkey = 16 * kq + (lane >> 4) * 8 + (lane & 7);          // K: key of matrix lane / 16
  const int vkey = 16 * kq + ((lane >> 3) & 1) * 8 + (lane & 7);    // V
  const int rp_shift = min(p.shift, 6);
  const uint32_t slice = rows_page * 128;  // bytes of a box's 64-element slice
  auto row_off = [&](int key) {
    return static_cast<uint32_t>((key >> rp_shift) * rows_page * D * 2 + (key & (rows_page - 1)) * 128);
  };
  const uint32_t krow = row_off(kkey), vrow = L::kv + row_off(vkey);

  int it = 0, seg = 0;
  for (; walk.next(p, sg); ++seg) {
    uint32_t qf[D / 16][4];
    int pos[2];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, slope[2] = {0.f, 0.f};
    float o[D / 8][4];
    {
      const uint32_t sign = p.negate ? 0x80008000u : 0u;
      const uint16_t* src[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = rg0 + g + 8 * i;
        const int pr = sg.blk * ROWS + r, tok = pa_div_g(p, pr), head = sg.h * p.G + pr - tok * p.G;
        const bool live = r < sg.it.rows;
        pos[i] = live ? sg.r.pos0 + tok : -1;
        src[i] = live ? p.q + (sg.r.row0 + tok) * p.q_stride + static_cast<long long>(head) * D : nullptr;
        if (FEAT && p.alibi && live) slope[i] = p.alibi[head] * 1.44269504088896340736f;
      }
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint16_t* a = src[j & 1];
          qf[ks][j] = a ? *reinterpret_cast<const uint32_t*>(a + 16 * ks + 8 * (j >> 1) + 2 * t4) ^ sign : 0u;
        }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    }
    const int min_pos = sg.r.pos0 + pa_div_g(p, sg.blk * ROWS);  // of the block's first row
    for (int t = sg.t0; t < sg.t1; ++t, ++it) {
      if (RG == 1 && (it & 1) != half) continue;
      const int s = it % ST;
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(&full[s], (it / ST) & 1, p.err));
      if (dead) continue;
      const uint32_t kv = base + s * L::stage;
      const int key0 = t * kShKeys + 16 * kq;
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t kf[4];
        const int c = 2 * ks + ((lane >> 3) & 1);
        ldsm4(kv + krow + (c >> 3) * slice + (((c & 7) ^ (kkey & 7)) << 4), kf);
        mma16816<T>(sc[0], qf[ks], kf[0], kf[1]);
        mma16816<T>(sc[1], qf[ks], kf[2], kf[3]);
      }
      // whether some row of the block does not see some of these keys
      const bool border = key0 + 15 > min_pos || (p.window && key0 <= sg.it.hi - 1 - p.window);
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = j >> 1, key = key0 + 8 * nb + 2 * t4 + (j & 1);
          float x = sc[nb][j];
          if constexpr (FEAT) {
            x = p.cap_log2 > 0.f ? pa_capped(x, p) : x * p.scale_log2;
            x = fmaf(slope[i], static_cast<float>(key - pos[i]), x);
          } else {
            x *= p.scale_log2;
          }
          if (border && (key > pos[i] || (p.window && key <= pos[i] - p.window))) x = -INFINITY;
          sc[nb][j] = x;
          mx[i] = fmaxf(mx[i], x);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          alpha[i] = m[i] == -INFINITY ? 0.f : ex2(m[i] - mx[i]);
          m[i] = mx[i];
          l[i] *= alpha[i];
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= alpha[0], o[i][1] *= alpha[0];
          o[i][2] *= alpha[1], o[i][3] *= alpha[1];
        }
      }
      constexpr float kLift = pa_lift<T>(15.f);
      const float mu[2] = {m[0] == -INFINITY ? 0.f : pa_reference(m[0], kLift),
                           m[1] == -INFINITY ? 0.f : pa_reference(m[1], kLift)};
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sc[nb][j] = ex2(sc[nb][j] - mu[j >> 1]);
          l[j >> 1] += sc[nb][j];
        }
      const uint32_t pf[4] = {pa_pack<T>(sc[0][0], sc[0][1]), pa_pack<T>(sc[0][2], sc[0][3]),
                              pa_pack<T>(sc[1][0], sc[1][1]), pa_pack<T>(sc[1][2], sc[1][3])};
      // Values no row sees may be anything (0 times infinity is no 0): cleared, by pairs of keys
      const bool cut = key0 + 16 > sg.it.hi || key0 < sg.it.lo;
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (cut) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = key0 + 8 * i + 2 * t4;
          keep[i] = (key >= sg.it.lo && key < sg.it.hi ? 0xffffu : 0u) |
                    (key + 1 >= sg.it.lo && key + 1 < sg.it.hi ? 0xffff0000u : 0u);
        }
      }
      const bool uneven = border && min_pos < sg.it.hi - 1;  // some row sees keys here that another does not
      uint32_t bad = 0;
#pragma unroll
      for (int jj = 0; jj < D / 16; ++jj) {
        uint32_t vf[4];
        const int c = 2 * jj + (lane >> 4);
        ldsm4_t(kv + vrow + (c >> 3) * slice + (((c & 7) ^ (vkey & 7)) << 4), vf);
        if (cut) vf[0] &= keep[0], vf[1] &= keep[1], vf[2] &= keep[0], vf[3] &= keep[1];
        if (uneven) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t b = pa_not_finite<T>(vf[i]);
            vf[i] &= ~b, bad |= b;
          }
        }
        mma16816<T>(o[2 * jj], pf, vf[0], vf[1]);
        mma16816<T>(o[2 * jj + 1], pf, vf[2], vf[3]);
      }
      if (__any_sync(0xffffffffu, bad != 0) && lane == 0) {
        atomicMin(&odd[2 * (seg & 1)], t);
        atomicMax(&odd[2 * (seg & 1) + 1], t);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    // ---- the segment's end: the warps' parts meet
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      if (t4 == 0) {
        mml[(warp * 16 + g + 8 * i) * 2] = pa_reference(m[i], pa_lift<T>(15.f));
        mml[(warp * 16 + g + 8 * i) * 2 + 1] = l[i];
      }
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      float* at = mo + (warp * 16 + g) * L::o_ld + 8 * i + 2 * t4;
      *reinterpret_cast<float2*>(at) = make_float2(o[i][0], o[i][1]);
      *reinterpret_cast<float2*>(at + 8 * L::o_ld) = make_float2(o[i][2], o[i][3]);
    }
    named_barrier(kShBarrier, kShConsumers);
    const int odd0 = odd[2 * (seg & 1)], odd1 = odd[2 * (seg & 1) + 1];
    if (tid == 0) odd[2 * (~seg & 1)] = INT_MAX, odd[2 * (~seg & 1) + 1] = -1;  // the next segment's
    constexpr int PER = ROWS * D / kShConsumers;  // dims of a row a thread adds up
    constexpr int PARTS = 8 / RG;
    const int r = tid / (D / PER), e0 = tid % (D / PER) * PER;
    if (r < sg.it.rows && !dead) {
      const int w0 = RG == 2 ? 4 * (r >> 4) : 0, rr = r & 15;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < PARTS; ++w) M = fmaxf(M, mml[((w0 + w) * 16 + rr) * 2]);
      const float mu = M == -INFINITY ? 0.f : M;
      float Ls = 0.f, acc[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
      for (int w = 0; w < PARTS; ++w) {
        const float f = ex2(mml[((w0 + w) * 16 + rr) * 2] - mu);
        Ls = fmaf(f, mml[((w0 + w) * 16 + rr) * 2 + 1], Ls);
        const float* src = mo + ((w0 + w) * 16 + rr) * L::o_ld + e0;
#pragma unroll
        for (int e = 0; e < PER; e += 4) {
          const float4 v = *reinterpret_cast<const float4*>(src + e);
          acc[e] = fmaf(f, v.x, acc[e]), acc[e + 1] = fmaf(f, v.y, acc[e + 1]);
          acc[e + 2] = fmaf(f, v.z, acc[e + 2]), acc[e + 3] = fmaf(f, v.w, acc[e + 3]);
        }
      }
      const int pr = sg.blk * ROWS + r, tok = pa_div_g(p, pr), head = sg.h * p.G + pr - tok * p.G;
      if (odd1 >= odd0) pa_add_not_finite<T, D, kShKeys, PER>(p, sg, sg.r.pos0 + tok, e0, odd0, odd1, acc);
      if (sg.starts && sg.ends) {
        const float inv = Ls > 0.f ? 1.0f / Ls : 0.f;
        uint16_t* dst = p.out + (sg.r.row0 + tok) * p.out_stride + static_cast<long long>(head) * D + e0;
#pragma unroll
        for (int e = 0; e < PER; e += 4)
          *reinterpret_cast<uint2*>(dst + e) = make_uint2(pa_pack<T>(acc[e] * inv, acc[e + 1] * inv),
                                                          pa_pack<T>(acc[e + 2] * inv, acc[e + 3] * inv));
        if (p.lse && e0 == 0)
          p.lse[static_cast<long long>(sg.r.row0 + tok) * p.hq + head] =
              Ls == 0.f ? -INFINITY : (M + log2f(Ls)) * 0.69314718055994530942f;
      } else {
        const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + pa_slot(sg);
        float* dst = p.part_o + (slot * ROWS + r) * D + e0;
#pragma unroll
        for (int e = 0; e < PER; e += 4)
          *reinterpret_cast<float4*>(dst + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
        if (e0 == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * ROWS + r) * 2) = make_float2(M, Ls);
      }
    }
    named_barrier(kShBarrier, kShConsumers);  // the parts are read before the next segment's overwrite them
  }
}

// Adds the parts of the item that CTA blockIdx.x of the first kernel finished
// for others, in tile order; 4 or 8 output values a thread.
template <int N, int F4>
struct CombineState {
  float M = -INFINITY, L = 0.f;
  float4 acc[F4] = {};
  // Parts j0 .. j0 + N (past `last`: the last again, with no weight), loaded
  // together: one by one, nine parts took 9 us of dependent loads.
  VVLI_DEV void add(const float2* mls, const float4* parts, const PaDesc& d, int j0, int last, int rows, size_t floats4,
                    int apart) {
    float2 ml[N];
    float4 v[N][F4];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int j = min(j0 + u, last);
      const size_t slot = static_cast<size_t>(j) * 2 + (j == d.first ? d.slot : 0);
      ml[u] = mls[slot * rows];
#pragma unroll
      for (int f = 0; f < F4; ++f) v[u][f] = parts[slot * floats4 + f * apart];
      if (j0 + u > last) ml[u].y = 0.f;
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (ml[u].y == 0.f) continue;  // no such part, or no visible key among its tiles
      const float m = fmaxf(M, ml[u].x), fa = ex2(M - m), fb = ex2(ml[u].x - m);  // M = -inf: 0
      M = m;
      L = L * fa + ml[u].y * fb;
#pragma unroll
      for (int f = 0; f < F4; ++f) {
        acc[f].x = acc[f].x * fa + v[u][f].x * fb, acc[f].y = acc[f].y * fa + v[u][f].y * fb;
        acc[f].z = acc[f].z * fa + v[u][f].z * fb, acc[f].w = acc[f].w * fa + v[u][f].w * fb;
      }
    }
  }
};

template <class T, int D, int ROWS>
__global__ void __launch_bounds__(256, ROWS == kPaMaxRows ? 4 : 2) paged_combine_kernel(const PaParams p) {
  grid_dependency_wait();
  const PaDesc d = p.desc[blockIdx.x];
  if (!d.finish) return;
  constexpr bool kByDims = ROWS == kPaMaxRows;  // the layout of the parts
  constexpr int F4 = kByDims ? 2 : 1;           // float4s of a thread
  const int at = blockIdx.y * 256 + threadIdx.x;
  // by dims: four threads side by side have 32 dims of a row, so that reads and writes are runs of 64 bytes or more
  const int r = kByDims ? at / 4 % ROWS : at / (D / 4);
  const int e4 = kByDims ? (at % 4 + at / (4 * ROWS) * 4) * 2 : at % (D / 4);
  if (r >= d.rows) return;
  const float4* parts = reinterpret_cast<const float4*>(p.part_o) + (kByDims ? e4 * ROWS + r : r * (D / 4) + e4);
  const float2* mls = reinterpret_cast<const float2*>(p.part_ml) + r;
  const int last = blockIdx.x;
  constexpr int N = kByDims ? 4 : 8;  // a chunk's item has two or three parts, a lone decode token one per CTA
  CombineState<N, F4> s;
  for (int j0 = d.first; j0 <= last; j0 += N) s.add(mls, parts, d, j0, last, ROWS, ROWS * D / 4, ROWS);
  const int pr = d.blk * ROWS + r, tok = pa_div_g(p, pr), head = d.h * p.G + pr - tok * p.G;
  const float inv = s.L == 0.f ? 0.f : 1.0f / s.L;
  uint16_t* dst = p.out + (d.row0 + tok) * p.out_stride + static_cast<long long>(head) * D + 4 * e4;
  uint32_t o[2 * F4];
#pragma unroll
  for (int f = 0; f < F4; ++f) {
    o[2 * f] = pa_pack<T>(s.acc[f].x * inv, s.acc[f].y * inv);
    o[2 * f + 1] = pa_pack<T>(s.acc[f].z * inv, s.acc[f].w * inv);
  }
  if constexpr (kByDims)
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
  else
    *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
  if (p.lse && e4 == 0)
    p.lse[static_cast<long long>(d.row0 + tok) * p.hq + head] =
        s.L == 0.f ? -INFINITY : (s.M + log2f(s.L)) * 0.69314718055994530942f;
}

template <class T, int D, int RG, bool FEAT>
cudaError_t launch_short(const PaParams& p, const vvli_paged_attn_args& a, int ctas, cudaStream_t s) {
  CUtensorMap km, vm;
  const uint32_t rows = static_cast<uint32_t>(std::min<uint64_t>(a.page_size, kShKeys));
  cudaError_t e = pa_tensor_map(&km, a.k_cache, a, rows, D / 64);
  if (e == cudaSuccess) e = pa_tensor_map(&vm, a.v_cache, a, rows, D / 64);
  if (e != cudaSuccess) return e;
  paged_short_kernel<T, D, RG, FEAT><<<ctas, kShThreads, ShLayout<D>::smem, s>>>(p, km, vm);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return pa_queue_combine<T, D, 16 * RG>(p, ctas, s);
}

// Blocks of 16 or 32 rows while they hold a request's rows; beyond, every block of
// 32 would stream the request's keys again, and the tensor-core kernel's blocks
// have 256 rows.
template <class T, int D>
cudaError_t queue_variant(const PaParams& p, const vvli_paged_attn_args& a, int ctas, cudaStream_t s) {
  const bool feat = pa_features(p) != 0;
  if (a.max_new <= 16u / p.G)
    return feat ? launch_short<T, D, 1, true>(p, a, ctas, s) : launch_short<T, D, 1, false>(p, a, ctas, s);
  if (a.max_new <= 32u / p.G)
    return feat ? launch_short<T, D, 2, true>(p, a, ctas, s) : launch_short<T, D, 2, false>(p, a, ctas, s);
  return pa_queue_tc<T, D>(p, a, ctas, s);
}

// Every kernel of a type and head_dim, loaded and allowed its shared memory.
template <class T, int D>
cudaError_t set_up_variants() {
  cudaError_t e = allow_smem(paged_short_kernel<T, D, 1, false>, ShLayout<D>::smem);
  if (e == cudaSuccess) e = allow_smem(paged_short_kernel<T, D, 1, true>, ShLayout<D>::smem);
  if (e == cudaSuccess) e = allow_smem(paged_short_kernel<T, D, 2, false>, ShLayout<D>::smem);
  if (e == cudaSuccess) e = allow_smem(paged_short_kernel<T, D, 2, true>, ShLayout<D>::smem);
  if (e == cudaSuccess) e = pa_set_up_tc<T, D>();
  cudaFuncAttributes loaded;
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&loaded, paged_combine_kernel<T, D, 16>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&loaded, paged_combine_kernel<T, D, 32>);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&loaded, paged_combine_kernel<T, D, kPaMaxRows>);
  return e;
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encode = nullptr;  // set by the first setup

// Once per device, for all types and head_dims: a call that is captured into a
// graph then does no more than launch.
cudaError_t set_up_device(int device, int* sms) {
  cudaError_t e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device);
  cudaDriverEntryPointQueryResult found;
  void* f = nullptr;
  if (e == cudaSuccess) e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found);
  if (e == cudaSuccess && found != cudaDriverEntryPointSuccess) e = cudaErrorNotSupported;
  if (e == cudaSuccess) e = set_up_variants<__nv_bfloat16, 64>();
  if (e == cudaSuccess) e = set_up_variants<__nv_bfloat16, 128>();
  if (e == cudaSuccess) e = set_up_variants<__half, 64>();
  if (e == cudaSuccess) e = set_up_variants<__half, 128>();
  if (e == cudaSuccess) {
    static std::once_flag once;  // devices are set up side by side
    std::call_once(once, [&] { tensor_map_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f); });
  }
  return e;
}

constexpr double kLog2e = 1.44269504088896340736;

std::string check_attn(const vvli_paged_attn_args* a) {
  if (!a) return "null arguments";
  if (a->requests < 1 || a->requests > 65536) return "requests must be in [1, 65536]";
  if (a->head_dim != 64 && a->head_dim != 128) return "head_dim must be 64 or 128";
  if (a->kv_heads < 1 || a->q_heads < 1 || a->q_heads > 512 || a->q_heads % a->kv_heads)
    return "q_heads must be a multiple of kv_heads in [1, 512]";
  if (a->tokens > (INT_MAX - 1024) / a->q_heads) return "tokens * q_heads must be at most 2^31 - 1025";
  const std::string page = check_page_size(a->page_size);
  if (!page.empty()) return page;
  if (a->pages < 1 || a->pages > static_cast<uint64_t>(INT_MAX) / a->page_size)
    return "pages must be at least 1 with pages * page_size < 2^31";
  if (a->page_stride % 8 || a->page_stride < a->kv_heads * a->page_size * a->head_dim || a->page_stride >= (1ull << 38))
    return "page_stride must be a multiple of 8 and at least kv_heads * page_size * head_dim";
  if (a->table_width < 1 || a->table_width > INT_MAX) return "table_width must be in [1, 2^31)";
  const uint64_t row = a->q_heads * a->head_dim;
  if (a->q_stride % 8 || a->out_stride % 8 || a->q_stride < row || a->out_stride < row || a->q_stride > (1ull << 31) ||
      a->out_stride > (1ull << 31))
    return "strides must be multiples of 8 and at least a row";
  if (a->window > INT_MAX) return "window must be below 2^31";
  if (a->dtype != VVLI_BF16 && a->dtype != VVLI_FP16) return "dtype must be VVLI_BF16 or VVLI_FP16";
  if (!std::isfinite(a->scale) || !(a->softcap >= 0.f) || std::isinf(a->softcap))
    return "scale must be finite, softcap finite and >= 0";
  if (std::isinf(static_cast<float>(a->scale * kLog2e)) ||
      (a->softcap > 0.f && (std::isinf(a->scale / a->softcap) || std::isinf(static_cast<float>(a->softcap * kLog2e)))))
    return "scale, scale / softcap and softcap are too large or too small for fp32";
  const void* need[] = {a->q, a->k_cache, a->v_cache, a->out, a->block_table, a->cu_new, a->seq_len, a->workspace};
  for (int i = 0; i < 8; ++i) {
    if (!need[i] && !(a->tokens == 0 && (i == 0 || i == 3))) return "null pointer";
    if (!aligned_to(need[i], i < 4 ? 16 : 4))
      return i < 4 ? "16-bit pointers must be 16-byte aligned" : "32-bit pointers must be 4-byte aligned";
  }
  if (!aligned_to(a->lse, 4) || !aligned_to(a->alibi, 4)) return "32-bit pointers must be 4-byte aligned";
  if (!aligned_to(a->workspace, 256)) return "workspace must be 256-byte aligned";
  if (a->workspace_bytes < pa_workspace_bytes(static_cast<int>(a->head_dim)))
    return "workspace_bytes " + std::to_string(a->workspace_bytes) + " < " +
           std::to_string(pa_workspace_bytes(static_cast<int>(a->head_dim))) + " (vvli_cuda_paged_attn_workspace_bytes)";
  return "";
}

cudaError_t queue_attn(int device, const vvli_paged_attn_args& a, cudaStream_t s) {
  if (a.tokens == 0) return cudaSuccess;
  if (device < 0 || device >= kOpMaxDevices) return cudaErrorInvalidDevice;
  static SetupOnce setup[kOpMaxDevices];
  static int sms[kOpMaxDevices];
  const cudaError_t e = setup[device]([&] { return set_up_device(device, &sms[device]); });
  if (e != cudaSuccess) return e;
  const int ctas = std::min(sms[device], kPaMaxCtas);
  PaParams p{};
  p.B = static_cast<int>(a.requests), p.T = static_cast<int>(a.tokens);
  p.hq = static_cast<int>(a.q_heads), p.hk = static_cast<int>(a.kv_heads), p.G = p.hq / p.hk;
  p.g_shift = 31;
  while ((1 << (p.g_shift - 31)) < p.G) ++p.g_shift;
  p.g_mul = static_cast<uint32_t>(((1ull << p.g_shift) + p.G - 1) / p.G);
  p.shift = 4;
  while ((1u << p.shift) < a.page_size) ++p.shift;
  p.pages = static_cast<int>(a.pages), p.width = static_cast<int>(a.table_width);
  p.window = static_cast<int>(a.window);
  p.longest = static_cast<int>(std::min<uint64_t>(a.table_width * a.page_size, INT_MAX - 1024));
  p.negate = a.scale < 0.f && !(a.softcap > 0.f) && !a.alibi;
  p.scale_log2 = static_cast<float>((p.negate ? -a.scale : a.scale) * kLog2e);
  if (a.softcap > 0.f) {
    p.cap_y = a.scale / a.softcap;
    p.cap_log2 = static_cast<float>(a.softcap * kLog2e);
  }
  p.q_stride = static_cast<long long>(a.q_stride), p.out_stride = static_cast<long long>(a.out_stride);
  p.q = static_cast<const uint16_t*>(a.q), p.out = static_cast<uint16_t*>(a.out);
  p.lse = a.lse, p.alibi = a.alibi;
  p.v = static_cast<const uint16_t*>(a.v_cache), p.page_stride = static_cast<long long>(a.page_stride);
  p.table = a.block_table, p.cu = a.cu_new, p.seq = a.seq_len;
  char* ws = static_cast<char*>(a.workspace);
  p.err = reinterpret_cast<int*>(ws);
  p.desc = reinterpret_cast<PaDesc*>(ws + 256);
  p.part_ml = reinterpret_cast<float*>(ws + 256 + kPaMaxCtas * sizeof(PaDesc));
  p.part_o = p.part_ml + static_cast<size_t>(kPaMaxCtas) * 2 * kPaMaxRows * 2;
  static_assert((256 + kPaMaxCtas * sizeof(PaDesc)) % 16 == 0, "the parts are 16-byte aligned");
  if (a.dtype == VVLI_BF16)
    return a.head_dim == 64 ? queue_variant<__nv_bfloat16, 64>(p, a, ctas, s)
                            : queue_variant<__nv_bfloat16, 128>(p, a, ctas, s);
  return a.head_dim == 64 ? queue_variant<__half, 64>(p, a, ctas, s) : queue_variant<__half, 128>(p, a, ctas, s);
}

}  // namespace

// ---------------------------------------------------------------- shared with the other kernel
template <class T, int D, int ROWS>
cudaError_t pa_queue_combine(const PaParams& p, int ctas, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), ROWS == kPaMaxRows ? D / 8 : (ROWS * D / 4 + 255) / 256);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_combine_kernel<T, D, ROWS>, p);
}

cudaError_t pa_tensor_map(CUtensorMap* map, const void* cache, const vvli_paged_attn_args& a, uint32_t box_rows,
                          uint32_t box_slices) {
  const cuuint64_t dims[4] = {64, a.kv_heads * a.page_size, a.head_dim / 64, a.pages};
  const cuuint64_t strides[3] = {a.head_dim * 2, 128, a.page_stride * 2};
  const cuuint32_t box[4] = {64, box_rows, box_slices, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      tensor_map_encode(map, a.dtype == VVLI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(cache), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template cudaError_t pa_queue_combine<__nv_bfloat16, 64, kPaMaxRows>(const PaParams&, int, cudaStream_t);
template cudaError_t pa_queue_combine<__nv_bfloat16, 128, kPaMaxRows>(const PaParams&, int, cudaStream_t);
template cudaError_t pa_queue_combine<__half, 64, kPaMaxRows>(const PaParams&, int, cudaStream_t);
template cudaError_t pa_queue_combine<__half, 128, kPaMaxRows>(const PaParams&, int, cudaStream_t);

}  // namespace vvli

extern "C" uint64_t vvli_cuda_paged_attn_workspace_bytes(uint64_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? vvli::pa_workspace_bytes(static_cast<int>(head_dim)) : 0;
}

extern "C" int vvli_cuda_paged_attention(int device, const vvli_paged_attn_args* args, void* stream) {
  return vvli::run_op(
      "paged_attention", device, [&] { return vvli::check_attn(args); },
      [&] { return vvli::queue_attn(device, *args, static_cast<cudaStream_t>(stream)); });
}
