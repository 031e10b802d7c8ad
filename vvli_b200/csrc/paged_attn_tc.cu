// paged_attn_tc.cu - vvli_cuda_paged_attention for requests with many new
// tokens (prompt chunks, alone or among decoding requests), on the tensor
// cores (tcgen05, TMEM).
//
// A CTA works on 256 packed rows (two tiles of 128, the M of every MMA) and
// 128-key tiles.  Bound: at head_dim 128 the two products of a 128 x 128 tile
// take about 1,020 tensor cycles per SM and its 16,384 exponentials 1,024
// cycles of the SM's 16-lane exponential unit, so the two must run side by
// side: while the softmax of one row tile runs, the MMAs of the other do.
//   * S_t = Q_t K^T (128 x 128) lands in TMEM columns 128 t; a thread owns a
//     row (a TMEM lane), so the online softmax needs no shuffles.  P, rounded
//     to the 16-bit type, goes back over the same columns, from where it is the
//     A operand of O_t += P_t V; O_t stays in TMEM.  A row's O is rescaled only
//     when its maximum rises by more than 2^8 (P then stays below 2^8; in fp16
//     2^6 and 2^15), which after a row's first tiles is rare.
//   * K and V tiles come by TMA, a box per page and 64-element slice, into a
//     128 KB ring in the 128-byte-swizzled layout; V is read as it lies (keys by
//     rows) through an MN-major descriptor, so nothing is transposed.
//   * MMAs are issued in the order P_0 V_j, S_0 of j + 1, P_1 V_j, S_1 of
//     j + 1; they run in that order, so S of a tile may overwrite the P before
//     it, and a softmax thread that sees S of j + 1 knows P V of j is done.
//   * An item of at most 128 rows is worked on by both tiles, alternate key tiles
//     each.
//   * Warps 0-3 and 4-7: softmax of tile 0 and 1, loading Q and writing the
//     output; warp 8 issues the MMAs, warp 9 the copies, warp 10 clears the
//     values past the last visible key in shared memory (they may be anything,
//     and 0 times infinity is no 0).  Every wait is bounded.
#include "paged_attn.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace vvli {
namespace {

constexpr int kTcKeys = 128;     // keys of a tile
constexpr int kTcTile = 128;     // rows of a tile: M
constexpr int kTcRows = 256;     // rows of an item
constexpr int kTcThreads = 384;
constexpr int kTcOdd = 8;        // segments of a row tile whose key tiles with values that are not finite are kept
// An item's start and end count as this many tiles (4,096 new tokens at head_dim 64:
// 172 us with none, 155 with 1, 134 with 2, 127 with 3; others alike from 2 on).
constexpr int kTcExtra = 3;
// A row maximum's rise (log2) that rescales its output: 2^8, in fp16 2^6 above a
// maximum 2^9 above the reference (paged_attn.cuh).  4,096 rows over 8,192 keys in
// fp16: 389 us with 2^8 and 2^7, 386 so, 391 with 2^5 and 2^10, 411 with 2^4 and 2^11.
template <class T>
constexpr float kTcRise = std::is_same<T, __half>::value ? 6.0f : 8.0f;

template <int D>
struct TcaLayout {
  static constexpr uint32_t q_tile = kTcTile * D * 2;  // D / 64 slices of 128 rows of 128 bytes
  static constexpr uint32_t kv = kTcKeys * D * 2;
  static constexpr uint32_t stages = 131072 / kv;      // 4 at D 128, 8 at D 64; keys and values in turn
  static constexpr uint32_t ring = 2 * q_tile;
  static constexpr uint32_t bars = ring + stages * kv;
  static constexpr uint32_t odd = bars + 320;            // after 3 stages + 11 barriers and the TMEM address
  static constexpr uint32_t share = odd + 16 * kTcOdd;   // [2][kTcOdd] first and last tile with values that are not finite
  static constexpr uint32_t part = share + 64;
  static constexpr uint32_t smem = part + sizeof(PaScratch<kTcThreads>) + 1024;  // + alignment slack
  static constexpr uint32_t o_col = 256;               // S_0 at column 0, S_1 at 128, O_t at 256 + D t
  static constexpr uint32_t slice = 128 * 128;         // bytes of a 64-element slice of a 128-row tile
  static_assert((3 * stages + 11) * 8 + 4 <= odd - bars, "the barriers and the TMEM address fit");
  static_assert(stages / 2 + 2 <= kTcOdd, "no range is overwritten before it is read");
};

// K-major operands have both descriptors' defaults (tc_ptx.cuh); this one is
// MN-major with the 128-byte swizzle: 64 elements of N by 8 of K per 1,024
// bytes, the next 8 of K after 1,024, the next 64 of N after a slice.
VVLI_DEV uint64_t tca_mn_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>((128 * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
template <class T>
constexpr uint32_t tca_idesc(int N, bool b_mn) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (b_mn ? 1u << 16 : 0u) | ((static_cast<uint32_t>(N) >> 3) << 17) |
         ((128u >> 4) << 24);
}
// The MMA warp runs as one (so that ptxas keeps addresses and descriptors in
// uniform registers: with one thread branched off, an MMA took about 90 cycles
// to issue and 64 to run), and one elected lane issues.
VVLI_DEV void tca_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D += A B with A in TMEM (rows = lanes, two 16-bit elements a column).
VVLI_DEV void tca_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
VVLI_DEV void tca_commit(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}

#define TCA_REGS                                                                                                  \
  "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29," \
  "%30,%31"

// 32 columns of this thread's lane; not to be used before tca_ld_done and tca_pin.
VVLI_DEV void tca_ld32(uint32_t taddr, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {" TCA_REGS "}, [%32];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                 "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                 "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]),
                 "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]),
                 "=f"(v[30]), "=f"(v[31])
               : "r"(taddr));
}
VVLI_DEV void tca_ld_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps the compiler from moving uses of v above an earlier tca_ld_done.
VVLI_DEV void tca_pin(float* v) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31]));
}
VVLI_DEV void tca_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {" TCA_REGS "};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
               "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
               "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
               "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
               : "memory");
}
VVLI_DEV void tca_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
VVLI_DEV void tca_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Pairs of fp32 operations in one instruction.
VVLI_DEV uint64_t f2_bits(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
VVLI_DEV float2 f2_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
VVLI_DEV float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return f2_of(r);
}
VVLI_DEV float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
VVLI_DEV float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
VVLI_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The capped scores of a row, in log2 units.  tanh by its formula takes two
// exponential-unit operations a score beside the softmax's one, on the unit
// that bounds this kernel; scores are mostly well below the cap, and there
// tanh(y) = y P(y^2) on the FMA units: P is the minimax fit of tanh(y) / y, of
// degree 3 on y <= 0.4 and 5 on y <= 0.75, found by iterated reweighted least
// squares (relative errors below 1.3e-7 and 3e-8).  One branch per warp and tile.
VVLI_DEV void tca_cap(const PaParams& p, float* s) {
  float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 128; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) big[k] = max3(big[k], fabsf(s[i + 2 * k]), fabsf(s[i + 2 * k + 1]));
  const float y = max3(fmaxf(big[0], big[1]), big[2], big[3]) * fabsf(p.cap_y);
  if (__any_sync(0xffffffffu, !(y <= 0.75f))) {
#pragma unroll
    for (int i = 0; i < 128; ++i) s[i] = pa_capped(s[i], p);
    return;
  }
  const float c = p.cap_log2;
  // the short one takes the raw score, with its factors' powers (up to the 7th) in the coefficients
  const float k_abs = fabsf(p.cap_y);
  if (k_abs > 1e-5f && k_abs < 1e5f && !__any_sync(0xffffffffu, y > 0.4f)) {
    const float k = c * p.cap_y, k2 = p.cap_y * p.cap_y;
    const float2 a0 = make_float2(k * 0.9999999019009012f, k * 0.9999999019009012f);
    const float2 a1 = make_float2(k * k2 * -0.3333136245857671f, k * k2 * -0.3333136245857671f);
    const float2 a2 = make_float2(k * k2 * k2 * 0.13270976752811006f, k * k2 * k2 * 0.13270976752811006f);
    const float2 a3 = make_float2(k * k2 * k2 * k2 * -0.04755360336859857f, k * k2 * k2 * k2 * -0.04755360336859857f);
#pragma unroll
    for (int i = 0; i < 128; i += 2) {
      const float2 v = make_float2(s[i], s[i + 1]), u = mul2(v, v);
      float2 r = fma2(a3, u, a2);
      r = fma2(r, u, a1);
      r = mul2(fma2(r, u, a0), v);
      s[i] = r.x, s[i + 1] = r.y;
    }
    return;
  }
  const float2 in = make_float2(p.cap_y, p.cap_y);
  const float2 c0 = make_float2(c * 0.9999999710138239f, c * 0.9999999710138239f);
  const float2 c1 = make_float2(c * -0.3333295887885829f, c * -0.3333295887885829f);
  const float2 c2 = make_float2(c * 0.13325406008965843f, c * 0.13325406008965843f);
  const float2 c3 = make_float2(c * -0.05334442971164088f, c * -0.05334442971164088f);
  const float2 c4 = make_float2(c * 0.019582907313611682f, c * 0.019582907313611682f);
  const float2 c5 = make_float2(c * -0.004716256631635093f, c * -0.004716256631635093f);
#pragma unroll
  for (int i = 0; i < 128; i += 2) {
    const float2 v = mul2(make_float2(s[i], s[i + 1]), in), u = mul2(v, v);
    float2 r = fma2(c5, u, c4);
    r = fma2(r, u, c3);
    r = fma2(r, u, c2);
    r = fma2(r, u, c1);
    r = mul2(fma2(r, u, c0), v);
    s[i] = r.x, s[i + 1] = r.y;
  }
}

// The bounded wait, out of line: the MMA warp's loop stays short.
__device__ __noinline__ bool tca_wait_long(uint64_t* bar, uint32_t parity, int* err) { return mbar_wait(bar, parity, err); }

// An item of at most 128 rows would leave one row tile idle and the other
// waiting for its own MMAs: both tiles then hold the same rows and take the key
// tiles in turn (twins), and tile 1's sums are added to tile 0's at the end.
// That reads two tiles ahead, which the ring's four stages at head_dim 128 do not
// reach: 16 requests of 16,000 keys and 48 rows took 114 us against 164 at
// head_dim 64, but 268 against 197 at 128.
template <int D>
VVLI_DEV bool tca_twins(const PaSeg& s) {
  return D == 64 && s.it.rows <= kTcTile;
}

// Key tiles of this segment that row tile t works on (its rows see no later key).
template <int D>
VVLI_DEV int tca_tiles(const PaParams& p, const PaSeg& s, int t) {
  if (tca_twins<D>(s)) return (s.t1 - s.t0 + 1 - t) >> 1;
  const int rows = min(kTcTile, s.it.rows - t * kTcTile);
  if (rows <= 0) return 0;
  const int last = s.r.pos0 + pa_div_g(p, s.blk * kTcRows + t * kTcTile + rows - 1);
  const int end = max(s.it.t0 + 1, (max(0, last + 1) + kTcKeys - 1) / kTcKeys);
  return max(0, min(s.t1, end) - s.t0);
}

template <class T, int D, int FEAT>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_tc_kernel(const PaParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using L = TcaLayout<D>;
  constexpr int ST = L::stages;
  extern __shared__ uint8_t tca_raw[];
  const uint32_t raw = smem_u32(tca_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = tca_raw + (base - raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::bars);  // [ST] a stage's copies have arrived
  uint64_t* empty = full + ST;                                 // [ST] the MMAs that read it are done
  uint64_t* v_ready = empty + ST;                              // [ST] a stage's values, cleared where nothing is seen
  uint64_t* q_full = v_ready + ST;                             // [2] Q_t is in shared memory
  uint64_t* s_full = q_full + 2;                               // [2] S_t is in TMEM (and the P V before it done)
  uint64_t* p_half = q_full + 4;                               // [2] P_t of the first 64 keys is in TMEM (and O_t rescaled)
  uint64_t* p_full = q_full + 6;                               // [2] all of P_t is
  uint64_t* o_full = q_full + 8;                               // [2] the segment's last P_t V is done
  uint64_t* drained = q_full + 10;                             // every MMA is done
  uint32_t* holder = reinterpret_cast<uint32_t*>(q_full + 11);
  PaShare* share = reinterpret_cast<PaShare*>(sm + L::share);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  grid_launch_dependents();  // the combine kernel waits for this grid's completion before reading
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1), mbar_init(&v_ready[s], 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], kTcTile), mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], kTcTile), mbar_init(&p_full[t], kTcTile), mbar_init(&o_full[t], 1);
    }
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  pa_schedule<kTcRows, kTcKeys, kTcExtra, kTcThreads>(p, share, reinterpret_cast<PaScratch<kTcThreads>*>(sm + L::part));  // has barriers
  tc_fence_after();
  const uint32_t tmem = *holder;
  PaWalk<kTcRows, kTcKeys, kTcExtra> walk(*share);
  PaSeg sg;
  bool dead = false;  // a wait gave up: the rest is skipped

  // The register file's 384 x 168 are split anew: 256 x 200 for the softmax, 128 x 104 for the rest.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 9) {  // ---- copies
      int n = 0;      // copies into the ring so far
      const int rows_page = 1 << p.shift;
      const int per_tile = kTcKeys >> p.shift;
      bool any = false;
      while (!dead && walk.next(p, sg)) {
        if (!any && lane == 0) pa_describe<kTcExtra>(p, *share, &sg);
        any = true;
        const int pg0 = (sg.t0 * kTcKeys) >> p.shift;
        int chunk = 0;  // lane l holds page pg0 + 32 chunk + l, and the one 32 further
        int ids = pa_page(p, sg.b, pg0 + lane), ids2 = pa_page(p, sg.b, pg0 + 32 + lane);
        for (int t = sg.t0; t < sg.t1 && !dead; ++t) {
          const int key0 = t * kTcKeys;
          const int boxes = max(0, min(per_tile, (sg.it.hi - key0 + rows_page - 1) >> p.shift));
          const int first = (key0 >> p.shift) - pg0;
          if (first >= 32 * (chunk + 1)) {
            ++chunk;
            ids = ids2;
            ids2 = pa_page(p, sg.b, pg0 + 32 * (chunk + 1) + lane);
          }
          const int box = lane % per_tile, z = lane / per_tile;  // page of the tile, 64-element slice
          const int j = first - 32 * chunk + box;  // a tile's pages lie in one chunk: both start at a multiple of per_tile
          const int id = __shfl_sync(0xffffffffu, ids, j & 31);
          const uint32_t off = z * L::slice + box * rows_page * 128;
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv, ++n) {
            const int s = n % ST;
            if (n >= ST) dead = !__all_sync(0xffffffffu, mbar_wait(&empty[s], ((n / ST) - 1) & 1, p.err));
            if (dead) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[s], boxes * rows_page * D * 2);
            __syncwarp();
            if (box < boxes && z < D / 64)
              tma_load_4d(base + L::ring + s * L::kv + off, kv ? &vmap : &kmap, 0, sg.h << p.shift, z, id, &full[s]);
          }
        }
      }
      if (!any && lane == 0) pa_describe<kTcExtra>(p, *share, nullptr);
      // no copy of this CTA is in flight when it ends
      for (int k = max(0, n - ST); k < n; ++k) mbar_wait(&full[k % ST], (k / ST) & 1, p.err);
    } else if (warp == 10) {  // ---- clears the values past the visible keys, and hands every V tile on
      int n = 0;
      // A segment's range is written before its V tiles are handed on and read
      // after their MMAs, by each row tile that works on it; a row tile counts the
      // segments that it works on, and has kTcOdd places for them.  When this warp
      // comes to a row tile's segment W, the MMAs are done with all but the last
      // stages / 2 tiles before it, so with its segment W - 1 - stages / 2, whose
      // queries the row tile hands over after reading the range of the one before.
      int worked[2] = {0, 0};
      while (!dead && walk.next(p, sg)) {
        int* odd[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          odd[t] = tca_tiles<D>(p, sg, t) > 0 ? reinterpret_cast<int*>(sm + L::odd) + 2 * (t * kTcOdd + worked[t]++ % kTcOdd) : nullptr;
          if (odd[t] && lane == 0) odd[t][0] = INT_MAX, odd[t][1] = -1;
        }
        const int first_pos = sg.r.pos0 + pa_div_g(p, sg.blk * kTcRows), last_pos = sg.it.hi - 1;
        for (int t = sg.t0; t < sg.t1; ++t, n += 2) {
          const int s = (n + 1) % ST;
          dead = !__all_sync(0xffffffffu, mbar_wait(&full[s], ((n + 1) / ST) & 1, p.err));
          if (dead) break;
          if ((t + 1) * kTcKeys > sg.it.hi || t * kTcKeys < sg.it.lo) {
            uint8_t* v = sm + L::ring + s * L::kv;
            for (int i = lane; i < kTcKeys * (D / 8); i += 32) {  // 16 bytes each, of key i / (D / 8)
              const int key = i / (D / 8), c = i % (D / 8), at = t * kTcKeys + key;
              if (at < sg.it.lo || at >= sg.it.hi)
                *reinterpret_cast<uint4*>(v + (c >> 3) * L::slice + key * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            tca_fence_async();
            __syncwarp();
          }
          // some row sees keys here that another does not
          if (first_pos < last_pos && ((t + 1) * kTcKeys - 1 > first_pos || (p.window && t * kTcKeys <= last_pos - p.window))) {
            uint4* v = reinterpret_cast<uint4*>(sm + L::ring + s * L::kv);
            uint32_t any = 0;
#pragma unroll 4
            for (int i = lane; i < kTcKeys * (D / 8); i += 32) {
              uint4 w = v[i];
              const uint4 b = make_uint4(pa_not_finite<T>(w.x), pa_not_finite<T>(w.y), pa_not_finite<T>(w.z), pa_not_finite<T>(w.w));
              if (b.x | b.y | b.z | b.w) v[i] = make_uint4(w.x & ~b.x, w.y & ~b.y, w.z & ~b.z, w.w & ~b.w), any = 1;
            }
            if (__any_sync(0xffffffffu, any)) {
              tca_fence_async();
#pragma unroll
              for (int i = 0; i < 2; ++i)
                if (odd[i] && lane == 0) odd[i][0] = min(odd[i][0], t), odd[i][1] = t;
              __syncwarp();
            }
          }
          if (lane == 0) mbar_arrive(&v_ready[s]);
        }
      }
    } else if (warp == 8) {  // ---- MMAs
      constexpr uint32_t s_idesc = tca_idesc<T>(kTcKeys, false), o_idesc = tca_idesc<T>(D, true);
      const uint64_t dq = umma_desc(base), dk = umma_desc(base + L::ring), dv = tca_mn_desc(base + L::ring);
      uint32_t n = 0;                                          // stages used before this segment
      uint32_t q_par0 = 0, q_par1 = 0, p_par0 = 0, p_par1 = 0;  // parities of the next waits on q_full, p_half / p_full
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity & 1)) && !dead)
          dead = !__all_sync(0xffffffffu, tca_wait_long(bar, parity & 1, p.err));
      };
      auto issue_s = [&](int t, uint32_t stage) {
        const uint64_t a = dq + ((t * L::q_tile) >> 4), b = dk + stage * (L::kv >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t o = ((ks >> 2) * L::slice + (ks & 3) * 32) >> 4;
          tca_mma(tmem + t * 128, a + o, b + o, s_idesc, ks != 0);
        }
        tca_commit(&s_full[t]);
      };
      auto issue_pv = [&](int t, uint32_t stage, int half, uint32_t more) {  // 64 of the tile's keys
        const uint64_t b = dv + stage * (L::kv >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ks = 4 * half + i;
          tca_mma_ts(tmem + L::o_col + t * D, tmem + t * 128 + ks * 8, b + ((ks * 16 * 128) >> 4), o_idesc, more | ks);
        }
      };
      // P V of tile j and S of tile j + 1
      auto step = [&](int t, int j, int nt, uint32_t& par, uint32_t vs, uint32_t ks) {
        if (j < nt) {
          wait(&p_half[t], par);
          tc_fence_after();
          if (!dead) issue_pv(t, vs, 0, j);
          wait(&p_full[t], par);
          tc_fence_after();
          par ^= 1;
          if (!dead) issue_pv(t, vs, 1, j);
          if (!dead && j + 1 == nt) tca_commit(&o_full[t]);
        }
        if (!dead && j + 1 < nt) issue_s(t, ks);
      };
      while (!dead && walk.next(p, sg)) {
        const int N = sg.t1 - sg.t0;
        if (tca_twins<D>(sg)) {
          for (int j = 0; j < min(N, 2) && !dead; ++j) {
            const uint32_t k = n + 2 * j;
            wait(&full[k % ST], k / ST);
            wait(&q_full[j], j ? q_par1 : q_par0);
            if (dead) break;
            issue_s(j, k % ST);
            tca_commit(&empty[k % ST]);
          }
          q_par0 ^= 1;
          if (N > 1) q_par1 ^= 1;
          for (int j = 0; j < N && !dead; ++j) {
            const int t = j & 1;
            const uint32_t v = n + 2 * j + 1, k = v + 3, par = t ? p_par1 : p_par0;
            wait(&v_ready[v % ST], v / ST);
            if (j + 2 < N) wait(&full[k % ST], k / ST);
            wait(&p_half[t], par);
            tc_fence_after();
            if (!dead) issue_pv(t, v % ST, 0, j >> 1);
            wait(&p_full[t], par);
            tc_fence_after();
            if (dead) break;
            issue_pv(t, v % ST, 1, j >> 1);
            if (t)
              p_par1 ^= 1;
            else
              p_par0 ^= 1;
            if (j + 2 >= N) tca_commit(&o_full[t]);
            if (j + 2 < N) {
              issue_s(t, k % ST);
              tca_commit(&empty[k % ST]);
            }
            tca_commit(&empty[v % ST]);
          }
          n += 2 * N;
          continue;
        }
        const int nt0 = tca_tiles<D>(p, sg, 0), nt1 = tca_tiles<D>(p, sg, 1);
        wait(&full[n % ST], n / ST);
        if (nt0) {
          wait(&q_full[0], q_par0);
          q_par0 ^= 1;
          if (!dead) issue_s(0, n % ST);
        }
        if (nt1) {
          wait(&q_full[1], q_par1);
          q_par1 ^= 1;
          if (!dead) issue_s(1, n % ST);
        }
        if (!dead) tca_commit(&empty[n % ST]);
        for (int j = 0; j < N && !dead; ++j) {
          const uint32_t v = n + 2 * j + 1, k = v + 1;
          wait(&v_ready[v % ST], v / ST);
          if (j + 1 < N) wait(&full[k % ST], k / ST);
          step(0, j, nt0, p_par0, v % ST, k % ST);
          step(1, j, nt1, p_par1, v % ST, k % ST);
          if (dead) break;
          tca_commit(&empty[v % ST]);
          if (j + 1 < N) tca_commit(&empty[k % ST]);
        }
        n += 2 * N;
      }
      tca_commit(drained);
      mbar_wait(drained, 0, p.err);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---- softmax of row tile t: thread = row
    const int t = warp >> 2, lane_row = 32 * (warp & 3) + lane;  // TMEM lane
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + L::o_col + t * D;
    // where twins' tile 1 leaves its sums: O over both tiles' q, [D / 4][128][4], and (m, l) over the schedule's scratch
    float4* twin_o = reinterpret_cast<float4*>(sm) + lane_row;
    float2* twin_ml = reinterpret_cast<float2*>(sm + L::part) + lane_row;
    uint32_t ss = 0, os = 0;  // waits on s_full, o_full so far
    auto wait = [&](uint64_t* bar, uint32_t parity) {  // warp-wide: what follows is
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity & 1, p.err));
      tc_fence_after();
    };
    int worked = 0;           // segments that this tile has worked on
    while (walk.next(p, sg)) {  // after a wait gave up too: the tiles' barriers below need all threads
      const int nt = tca_tiles<D>(p, sg, t);
      const bool twins = tca_twins<D>(sg);
      const int row0 = twins ? 0 : t * kTcTile, R = row0 + lane_row;  // row of the item
      const int pr = sg.blk * kTcRows + R, tok = pa_div_g(p, pr), head = sg.h * p.G + pr - tok * p.G;
      const bool live = R < sg.it.rows;
      const int pos = live ? sg.r.pos0 + tok : -1;
      const int first_pos = sg.r.pos0 + pa_div_g(p, sg.blk * kTcRows + row0);  // of this tile's first row
      const int last_pos = sg.it.hi - 1;
      constexpr float kLift = pa_lift<T>(9.f);
      float m = -INFINITY, l = 0.f;  // the row's reference, and its sum relative to it
      const float slope = (FEAT & kPaAlibi) && p.alibi && live ? p.alibi[head] * 1.44269504088896340736f : 0.f;
      if (nt > 0 && !dead) {
        // D / 8 lanes side by side read a row: 16-byte chunk c of rows i * (256 / D) + lane / (D / 8) of the warp's 32
        const uint32_t sign = p.negate ? 0x80008000u : 0u;
        const int c = lane % (D / 8), w0 = 32 * (warp & 3), pr0 = sg.blk * kTcRows + row0 + w0;
        uint8_t* dst = sm + t * L::q_tile + (c >> 3) * L::slice;
        uint4 v[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const int row = i * (256 / D) + lane / (D / 8), rp = pr0 + row, rt = pa_div_g(p, rp);
          v[i] = make_uint4(0, 0, 0, 0);
          if (row0 + w0 + row < sg.it.rows)
            v[i] = *reinterpret_cast<const uint4*>(p.q + (sg.r.row0 + rt) * p.q_stride +
                                                   static_cast<long long>(sg.h * p.G + rp - rt * p.G) * D + 8 * c);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const int row = w0 + i * (256 / D) + lane / (D / 8);
          *reinterpret_cast<uint4*>(dst + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
              make_uint4(v[i].x ^ sign, v[i].y ^ sign, v[i].z ^ sign, v[i].w ^ sign);
        }
        tca_fence_async();
        mbar_arrive(&q_full[t]);
      }
      for (int j = 0; j < nt && !dead; ++j) {
        wait(&s_full[t], ss++);
        if (dead) break;
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tca_ld32(ts + 32 * c, s + 32 * c);
        tca_ld_done();
#pragma unroll
        for (int c = 0; c < 4; ++c) tca_pin(s + 32 * c);
        const int key0 = (sg.t0 + (twins ? 2 * j + t : j)) * kTcKeys;
        const int lim = pos - key0;  // columns up to here are visible
        const bool border = key0 + kTcKeys - 1 > first_pos || (p.window && key0 <= last_pos - p.window);  // uniform over the warp
        const int low = p.window ? lim - p.window : -1;  // columns up to here are before the window
        if constexpr (FEAT & kPaCap) {
          if (border) {  // what is not visible (old shared memory past the last key) must not choose the formula
#pragma unroll
            for (int i = 0; i < 128; ++i) s[i] = i <= lim && i > low ? s[i] : 0.f;
          }
          tca_cap(p, s);
        }
        if constexpr (FEAT & kPaAlibi) {
          const float2 sl = make_float2(slope, slope), at = make_float2(-static_cast<float>(lim), -static_cast<float>(lim));
          const float2 unit2 = make_float2(p.scale_log2, p.scale_log2);
#pragma unroll
          for (int i = 0; i < 128; i += 2) {
            const float2 d = add2(make_float2(i, i + 1), at);  // key - query position, exact below 2^24
            float2 x = make_float2(s[i], s[i + 1]);
            if constexpr (!(FEAT & kPaCap)) x = mul2(x, unit2);
            x = fma2(sl, d, x);
            s[i] = x.x, s[i + 1] = x.y;
          }
        }
        if (border) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] = i <= lim && i > low ? s[i] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < 124; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], s[i + 2 * k], s[i + 2 * k + 1]);
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], s[124 + k]);
        const float unit = FEAT ? 1.0f : p.scale_log2;  // s * unit is in log2 units; > 0
        const float mt = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * unit;
        const bool rise = mt - m > kTcRise<T> + kLift;  // m = -inf: any finite mt; a difference, which is exact for large ones
        if (__any_sync(0xffffffffu, rise)) {
          const float low_mt = pa_reference(mt, kLift);
          const float alpha = rise ? ex2(m - low_mt) : 1.0f;  // m = -inf: 0
          if (rise) m = low_mt;
          l *= alpha;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tca_ld32(to + 32 * c, o);
              tca_ld_done();
              tca_pin(o);
              uint32_t w[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(o[i] * alpha);
              tca_st32(to + 32 * c, w);
            }
          }
        }
        const float mu = m == -INFINITY ? 0.f : m;
        const float2 unit2 = make_float2(unit, unit), low2 = make_float2(-mu, -mu);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float2 x = fma2(make_float2(s[64 * h + 2 * i], s[64 * h + 2 * i + 1]), unit2, low2);
            x.x = ex2(x.x), x.y = ex2(x.y);
            sum[i & 1] = add2(sum[i & 1], x);
            w[i] = pa_pack<T>(x.x, x.y);
          }
          tca_st32(ts + 32 * h, w);
          tca_st_done();
          tc_fence_before();
          mbar_arrive(h == 0 ? &p_half[t] : &p_full[t]);
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      if (nt > 0 && !dead) wait(&o_full[t], os++);
      float fold = 0.f, other = 0.f;  // twins: factors of this tile's and the other's sums
      if (twins && sg.t1 - sg.t0 > 1) {
        named_barrier(1, 2 * kTcTile);  // both tiles' MMAs are done: q is free
        if (t == 1) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tca_ld32(to + 32 * c, o);
            tca_ld_done();
            tca_pin(o);
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              twin_o[(32 * c + i) / 4 * kTcTile] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
          *twin_ml = make_float2(m, l);
        }
        named_barrier(1, 2 * kTcTile);
        if (t == 0) {
          const float2 ml = *twin_ml;
          const float both = fmaxf(m, ml.x), mu = both == -INFINITY ? 0.f : both;
          fold = ex2(m - mu), other = ex2(ml.x - mu);
          m = both;
          l = l * fold + ml.y * other;
        }
      }
      const bool whole = sg.starts && sg.ends, mine = !dead && !(twins && t == 1);
      const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + pa_slot(sg);
      const float inv = l == 0.f ? 0.f : 1.0f / l;  // no visible key: zeros
      const int2 odd = *reinterpret_cast<const int2*>(sm + L::odd + 8 * (t * kTcOdd + worked % kTcOdd));
      worked += nt > 0;
      if (live && mine) {
        if (whole) {
          if (p.lse)
            p.lse[static_cast<long long>(sg.r.row0 + tok) * p.hq + head] =
                l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
        } else {
          *reinterpret_cast<float2*>(p.part_ml + (slot * kTcRows + R) * 2) = make_float2(m, l);
        }
      }
      if (nt > 0 && mine) {
        uint16_t* dst = p.out + (sg.r.row0 + tok) * p.out_stride + static_cast<long long>(head) * D;
        float4* part = reinterpret_cast<float4*>(p.part_o) + slot * (kTcRows * D / 4) + R;  // four dims of all rows together
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          tca_ld32(to + 32 * c, o);
          tca_ld_done();
          tca_pin(o);
          if (!live) continue;  // the loads are warp-wide
          if (other != 0.f || fold != 0.f) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 v = twin_o[(32 * c + i) / 4 * kTcTile];
              o[i] = o[i] * fold + v.x * other, o[i + 1] = o[i + 1] * fold + v.y * other;
              o[i + 2] = o[i + 2] * fold + v.z * other, o[i + 3] = o[i + 3] * fold + v.w * other;
            }
          }
          if (odd.y >= odd.x) pa_add_not_finite<T, D, kTcKeys, 32>(p, sg, pos, 32 * c, odd.x, odd.y, o);
          if (whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(dst + 32 * c + i) =
                  make_uint4(pa_pack<T>(o[i] * inv, o[i + 1] * inv), pa_pack<T>(o[i + 2] * inv, o[i + 3] * inv),
                             pa_pack<T>(o[i + 4] * inv, o[i + 5] * inv), pa_pack<T>(o[i + 6] * inv, o[i + 7] * inv));
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              part[(32 * c + i) / 4 * kTcRows] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      if (twins && sg.t1 - sg.t0 > 1) named_barrier(1, 2 * kTcTile);  // tile 1's sums are read before q is written again
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <class T, int D, int FEAT>
cudaError_t launch_tc(const PaParams& p, const vvli_paged_attn_args& a, int ctas, cudaStream_t s) {
  CUtensorMap km, vm;
  cudaError_t e = pa_tensor_map(&km, a.k_cache, a, static_cast<uint32_t>(a.page_size), 1);
  if (e == cudaSuccess) e = pa_tensor_map(&vm, a.v_cache, a, static_cast<uint32_t>(a.page_size), 1);
  if (e != cudaSuccess) return e;
  paged_tc_kernel<T, D, FEAT><<<ctas, kTcThreads, TcaLayout<D>::smem, s>>>(p, km, vm);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return pa_queue_combine<T, D, kTcRows>(p, ctas, s);
}

}  // namespace

template <class T, int D>
cudaError_t pa_set_up_tc() {
  cudaError_t e = allow_smem(paged_tc_kernel<T, D, 0>, TcaLayout<D>::smem);
  if (e == cudaSuccess) e = allow_smem(paged_tc_kernel<T, D, kPaCap>, TcaLayout<D>::smem);
  if (e == cudaSuccess) e = allow_smem(paged_tc_kernel<T, D, kPaAlibi>, TcaLayout<D>::smem);
  if (e == cudaSuccess) e = allow_smem(paged_tc_kernel<T, D, kPaCap | kPaAlibi>, TcaLayout<D>::smem);
  return e;
}
template <class T, int D>
cudaError_t pa_queue_tc(const PaParams& p, const vvli_paged_attn_args& a, int ctas, cudaStream_t s) {
  switch (pa_features(p)) {
    case 0: return launch_tc<T, D, 0>(p, a, ctas, s);
    case kPaCap: return launch_tc<T, D, kPaCap>(p, a, ctas, s);
    case kPaAlibi: return launch_tc<T, D, kPaAlibi>(p, a, ctas, s);
    default: return launch_tc<T, D, kPaCap | kPaAlibi>(p, a, ctas, s);
  }
}
template cudaError_t pa_set_up_tc<__nv_bfloat16, 64>();
template cudaError_t pa_queue_tc<__nv_bfloat16, 64>(const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);
template cudaError_t pa_set_up_tc<__nv_bfloat16, 128>();
template cudaError_t pa_queue_tc<__nv_bfloat16, 128>(const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);
template cudaError_t pa_set_up_tc<__half, 64>();
template cudaError_t pa_queue_tc<__half, 64>(const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);
template cudaError_t pa_set_up_tc<__half, 128>();
template cudaError_t pa_queue_tc<__half, 128>(const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);

}  // namespace vvli
