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
//     when its maximum rises by more than 2^8 (P then stays below 2^8), which
//     after a row's first tiles is rare.
//   * K and V tiles come by TMA, a box per page and 64-element slice, into a
//     128 KB ring in the 128-byte-swizzled layout; V is read as it lies (keys by
//     rows) through an MN-major descriptor, so nothing is transposed.
//   * MMAs are issued in the order P_0 V_j, S_0 of j + 1, P_1 V_j, S_1 of
//     j + 1; they run in that order, so S of a tile may overwrite the P before
//     it, and a softmax thread that sees S of j + 1 knows P V of j is done.
//   * Warps 0-3 and 4-7: softmax of tile 0 and 1, loading Q and writing the
//     output; warp 8 issues the MMAs, warp 9 the copies, warp 10 clears the
//     values past the last visible key in shared memory (they may be anything,
//     and 0 times infinity is no 0).  Every wait is bounded.
#include "paged_attn.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace vvli {
namespace {

constexpr int kTcKeys = 128;     // keys of a tile
constexpr int kTcTile = 128;     // rows of a tile: M
constexpr int kTcRows = 256;     // rows of an item
constexpr int kTcThreads = 384;
constexpr float kTcRise = 8.0f;  // a row maximum's rise (log2) that rescales its output

template <int D>
struct TcaLayout {
  static constexpr uint32_t q_tile = kTcTile * D * 2;  // D / 64 slices of 128 rows of 128 bytes
  static constexpr uint32_t kv = kTcKeys * D * 2;
  static constexpr uint32_t stages = 131072 / kv;      // 4 at D 128, 8 at D 64; keys and values in turn
  static constexpr uint32_t ring = 2 * q_tile;
  static constexpr uint32_t bars = ring + stages * kv;
  static constexpr uint32_t share = bars + 320;        // 3 stages + 9 barriers and the TMEM address
  static constexpr uint32_t part = share + 64;
  static constexpr uint32_t smem = part + 128 + 1024;  // + alignment slack
  static constexpr uint32_t o_col = 256;               // S_0 at column 0, S_1 at 128, O_t at 256 + D t
  static constexpr uint32_t slice = 128 * 128;         // bytes of a 64-element slice of a 128-row tile
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
// D += A B with A in TMEM (rows = lanes, two 16-bit elements a column).
VVLI_DEV void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
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

// Tiles of this segment that row tile t works on (its rows see no later key).
VVLI_DEV int tca_tiles(const PaParams& p, const PaSeg& s, int t) {
  const int rows = min(kTcTile, s.it.rows - t * kTcTile);
  if (rows <= 0) return 0;
  const int last = s.r.pos0 + (s.blk * kTcRows + t * kTcTile + rows - 1) / p.G;
  const int end = max(s.it.t0 + 1, (max(0, last + 1) + kTcKeys - 1) / kTcKeys);
  return max(0, min(s.t1, end) - s.t0);
}

template <class T, int D, bool FEAT>
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
  uint64_t* p_full = q_full + 4;                               // [2] P_t is in TMEM (and O_t rescaled)
  uint64_t* o_full = q_full + 6;                               // [2] the segment's last P_t V is done
  uint64_t* drained = q_full + 8;                              // every MMA is done
  uint32_t* holder = reinterpret_cast<uint32_t*>(q_full + 9);
  PaShare* share = reinterpret_cast<PaShare*>(sm + L::share);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  grid_launch_dependents();  // the combine kernel waits for this grid's completion before reading
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1), mbar_init(&v_ready[s], 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], kTcTile), mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], kTcTile), mbar_init(&o_full[t], 1);
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
  pa_schedule<kTcRows, kTcKeys, kTcThreads>(p, share, reinterpret_cast<long long*>(sm + L::part));  // has barriers
  tc_fence_after();
  const uint32_t tmem = *holder;
  PaWalk<kTcRows, kTcKeys> walk(*share);
  PaSeg sg;
  bool dead = false;  // a wait gave up: the rest is skipped

  // The register file's 384 x 168 are split anew: 256 x 208 for the softmax, 128 x 88 for the rest.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 9) {  // ---- copies
      int n = 0;      // copies into the ring so far
      const int rows_page = 1 << p.shift;
      const int per_tile = kTcKeys >> p.shift;
      bool any = false;
      while (!dead && walk.next(p, sg)) {
        if (!any && lane == 0) pa_describe(p, *share, &sg);
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
      if (!any && lane == 0) pa_describe(p, *share, nullptr);
      // no copy of this CTA is in flight when it ends
      for (int k = max(0, n - ST); k < n; ++k) mbar_wait(&full[k % ST], (k / ST) & 1, p.err);
    } else if (warp == 10) {  // ---- clears the values past the visible keys, and hands every V tile on
      int n = 0;
      while (!dead && walk.next(p, sg)) {
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
          if (lane == 0) mbar_arrive(&v_ready[s]);
        }
      }
    } else if (warp == 8) {  // ---- MMAs, by one thread
      if (lane == 0) {
        constexpr uint32_t s_idesc = tca_idesc<T>(kTcKeys, false), o_idesc = tca_idesc<T>(D, true);
        const uint64_t dq = umma_desc(base), dk = umma_desc(base + L::ring), dv = tca_mn_desc(base + L::ring);
        int n = 0;                                // stages used before this segment
        uint32_t qs[2] = {0, 0}, ps[2] = {0, 0};  // waits on q_full, p_full so far
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          if (!dead) dead = !mbar_wait(bar, parity & 1, p.err);
          tc_fence_after();
        };
        while (!dead && walk.next(p, sg)) {
          const int N = sg.t1 - sg.t0;
          const int nt[2] = {tca_tiles(p, sg, 0), tca_tiles(p, sg, 1)};
          auto issue_s = [&](int t, int j) {
            const int s = (n + 2 * j) % ST;
            const uint64_t a = dq + ((t * L::q_tile) >> 4), b = dk + ((s * L::kv) >> 4);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t o = ((ks >> 2) * L::slice + (ks & 3) * 32) >> 4;
              umma_bf16(tmem + t * 128, a + o, b + o, s_idesc, ks != 0);
            }
            umma_commit(&s_full[t]);
          };
          auto issue_pv = [&](int t, int j) {
            const int s = (n + 2 * j + 1) % ST;
            const uint64_t b = dv + ((s * L::kv) >> 4);
#pragma unroll
            for (int ks = 0; ks < kTcKeys / 16; ++ks)
              umma_ts(tmem + L::o_col + t * D, tmem + t * 128 + ks * 8, b + ((ks * 16 * 128) >> 4), o_idesc, (j | ks) != 0);
          };
          wait(&full[n % ST], n / ST);
          for (int t = 0; t < 2; ++t) {
            if (nt[t] == 0) continue;
            wait(&q_full[t], qs[t]++);
            if (!dead) issue_s(t, 0);
          }
          if (!dead) umma_commit(&empty[n % ST]);
          for (int j = 0; j < N && !dead; ++j) {
            const int vs = n + 2 * j + 1, ks = vs + 1;
            const bool next = j + 1 < N;
            wait(&v_ready[vs % ST], vs / ST);
            bool k_in = false;
            for (int t = 0; t < 2; ++t) {
              if (j < nt[t]) {
                wait(&p_full[t], ps[t]++);
                if (!dead) issue_pv(t, j);
                if (!dead && j + 1 == nt[t]) umma_commit(&o_full[t]);
              }
              if (j + 1 < nt[t]) {
                if (!k_in) wait(&full[ks % ST], ks / ST), k_in = true;
                if (!dead) issue_s(t, j + 1);
              }
            }
            if (!dead) umma_commit(&empty[vs % ST]);
            if (next && !k_in) wait(&full[ks % ST], ks / ST);
            if (next && !dead) umma_commit(&empty[ks % ST]);
          }
          n += 2 * N;
        }
        umma_commit(drained);
        mbar_wait(drained, 0, p.err);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax of row tile t: thread = row
    const int t = warp >> 2, R = kTcTile * t + 32 * (warp & 3) + lane;  // row of the item
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + L::o_col + t * D;
    uint8_t* qrow = sm + t * L::q_tile + (R & 127) * 128;
    uint32_t ss = 0, os = 0;  // waits on s_full, o_full so far
    auto wait = [&](uint64_t* bar, uint32_t parity) {  // warp-wide: what follows is
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity & 1, p.err));
      tc_fence_after();
    };
    while (!dead && walk.next(p, sg)) {
      const int nt = tca_tiles(p, sg, t);
      const int pr = sg.blk * kTcRows + R, tok = pr / p.G, head = sg.h * p.G + pr - tok * p.G;
      const bool live = R < sg.it.rows;
      const int pos = live ? sg.r.pos0 + tok : -1;
      const int first_pos = sg.r.pos0 + (sg.blk * kTcRows + t * kTcTile) / p.G;  // of this tile's first row
      const int last_pos = sg.it.hi - 1;
      float m = -INFINITY, l = 0.f;
      const float slope = FEAT && p.alibi && live ? p.alibi[head] * 1.44269504088896340736f : 0.f;
      if (nt > 0) {
        const uint16_t* src = p.q + (sg.r.row0 + tok) * p.q_stride + static_cast<long long>(head) * D;
        uint4 v[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          v[c] = live ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          if (p.negate) v[c].x ^= 0x80008000u, v[c].y ^= 0x80008000u, v[c].z ^= 0x80008000u, v[c].w ^= 0x80008000u;
          *reinterpret_cast<uint4*>(qrow + (c >> 3) * L::slice + (((c & 7) ^ (R & 7)) << 4)) = v[c];
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
        const int key0 = (sg.t0 + j) * kTcKeys;
        const int lim = pos - key0;  // columns up to here are visible
        if constexpr (FEAT) {
#pragma unroll
          for (int i = 0; i < 128; ++i) {
            const float x = p.cap_log2 > 0.f ? pa_capped(s[i], p) : s[i] * p.scale_log2;
            s[i] = fmaf(slope, static_cast<float>(i - lim), x);
          }
        }
        if (key0 + kTcKeys - 1 > first_pos || (p.window && key0 <= last_pos - p.window)) {  // uniform over the warp
          const int low = p.window ? lim - p.window : -1;  // columns up to here are before the window
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] = i <= lim && i > low ? s[i] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
        const float unit = FEAT ? 1.0f : p.scale_log2;  // s * unit is in log2 units; > 0
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * unit;
        const bool rise = mt > m + kTcRise;  // m = -inf: any finite mt
        if (__any_sync(0xffffffffu, rise)) {
          const float alpha = rise ? ex2(m - mt) : 1.0f;  // m = -inf: 0
          if (rise) m = mt;
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
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float a = ex2(fmaf(s[64 * h + 2 * i], unit, -mu)), b = ex2(fmaf(s[64 * h + 2 * i + 1], unit, -mu));
            sum[(2 * i) & 3] += a, sum[(2 * i + 1) & 3] += b;
            w[i] = pa_pack<T>(a, b);
          }
          tca_st32(ts + 32 * h, w);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tca_st_done();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (dead) break;
      if (nt > 0) wait(&o_full[t], os++);
      if (dead) break;
      const bool whole = sg.starts && sg.ends;
      const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + pa_slot(sg);
      const float inv = l > 0.f ? 1.0f / l : (l == l ? 0.f : l);
      if (live) {
        if (whole) {
          if (p.lse)
            p.lse[static_cast<long long>(sg.r.row0 + tok) * p.hq + head] =
                m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
        } else {
          *reinterpret_cast<float2*>(p.part_ml + (slot * kTcRows + R) * 2) = make_float2(m, l);
        }
      }
      if (nt > 0) {
        uint16_t* dst = p.out + (sg.r.row0 + tok) * p.out_stride + static_cast<long long>(head) * D;
        float* part = p.part_o + (slot * kTcRows + R) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          tca_ld32(to + 32 * c, o);
          tca_ld_done();
          tca_pin(o);
          if (!live) continue;  // the loads are warp-wide
          if (whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(dst + 32 * c + i) =
                  make_uint4(pa_pack<T>(o[i] * inv, o[i + 1] * inv), pa_pack<T>(o[i + 2] * inv, o[i + 3] * inv),
                             pa_pack<T>(o[i + 4] * inv, o[i + 5] * inv), pa_pack<T>(o[i + 6] * inv, o[i + 7] * inv));
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(part + 32 * c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <class T, int D, bool FEAT>
cudaError_t launch_tc(int device, const PaParams& p, const vvli_paged_attn_args& a, int ctas, cudaStream_t s) {
  static std::once_flag once[kOpMaxDevices];
  static cudaError_t ready[kOpMaxDevices];
  std::call_once(once[device], [&] {
    ready[device] = cudaFuncSetAttribute(paged_tc_kernel<T, D, FEAT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         TcaLayout<D>::smem);
  });
  cudaError_t e = ready[device];
  CUtensorMap km, vm;
  if (e == cudaSuccess) e = pa_tensor_map(&km, a.k_cache, a, static_cast<uint32_t>(a.page_size), 1);
  if (e == cudaSuccess) e = pa_tensor_map(&vm, a.v_cache, a, static_cast<uint32_t>(a.page_size), 1);
  if (e != cudaSuccess) return e;
  paged_tc_kernel<T, D, FEAT><<<ctas, kTcThreads, TcaLayout<D>::smem, s>>>(p, km, vm);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return pa_queue_combine<T, D, kTcRows>(p, ctas, s);
}

}  // namespace

template <class T, int D>
cudaError_t pa_queue_tc(int device, const PaParams& p, const vvli_paged_attn_args& a, int ctas, cudaStream_t s) {
  return pa_featured(p) ? launch_tc<T, D, true>(device, p, a, ctas, s) : launch_tc<T, D, false>(device, p, a, ctas, s);
}
template cudaError_t pa_queue_tc<__nv_bfloat16, 64>(int, const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);
template cudaError_t pa_queue_tc<__nv_bfloat16, 128>(int, const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);
template cudaError_t pa_queue_tc<__half, 64>(int, const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);
template cudaError_t pa_queue_tc<__half, 128>(int, const PaParams&, const vvli_paged_attn_args&, int, cudaStream_t);

}  // namespace vvli
