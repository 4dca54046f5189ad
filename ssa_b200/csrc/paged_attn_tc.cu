// Attention of chunks over the paged cache on the 5th-generation tensor cores:
// bf16 / fp16, head size 64 or 128, pages of a power of two of at least 8 slots.
//
// A CTA (one per SM) holds 256 query rows of one item (the g heads of a KV
// group at floor(256 / g) tokens) as two streams of 128 rows, and walks key
// tiles of 128 slots.  Per tile and stream: S = Q K^T (tcgen05, fp32 in TMEM),
// the online softmax of a row by the thread that owns its TMEM lane, P written
// back to TMEM over S in the input type, O += P V (tcgen05, A from TMEM).
// While one stream is in its softmax the tensor cores work for the other: a
// tile costs them 4 * 128 * 128 * d flops and the MUFU 128 * 128 exponentials,
// about 1000 clocks each at d = 128.  Neither bounds it (each is busy 48% of the
// time): a stream's softmax, 2100 clocks, and the two products of its next tile
// follow one another.  2048 tokens x 32 heads over 32768 slots, bf16: 1154 us a
// call, 0.92 PFLOP/s (1022 in a replayed graph; it runs at the power limit, and a tenth
// more or less from box to box).  Slower on that call, beside 978 us in the same run:
// tiles of 64 slots with two S buffers each (1349), two threads a row (1148), a quarter
// of the exponentials as polynomials (2%).
//
//   warps 0-3   stream A: loads its Q rows, softmax, epilogue (a row per thread)
//   warps 4-7   stream B
//   warp 8      TMEM allocation, single-thread MMA issue
//   warp 9      TMA producer: a lane per page box, K and V tiles in a ring
//   warps 10-11 look through V for non-finite values
//
// TMEM (512 columns): S_A, S_B (128 each; P in the first 64), O_A, O_B (d each).
//
// The running maximum that scales a row's exponentials is raised only when a
// tile exceeds it by more than 2^8 (O, in TMEM, is then multiplied by the
// quotient): exponentials stay below 2^8, sums in fp32.  P is rounded to the
// input type, as the tensor cores take it (relative error at most 2^-8 / 2^-11 of
// each weight); the row sum adds the unrounded values.  (P in two terms, as for single
// tokens, lengthens the chain by the split and by a second product: 1040 -> 1490 us on
// the call above, 311 -> 402 for 24 mixed sequences.)  For fp16 every exponential
// carries a factor 2^7, so that weights down to 2^-21 of the largest stay
// normal numbers.
//
// Hidden slots (past a row's position, or past the sequence in the last page)
// have P = 0, and so have small weights rounded to fp16 (below 2^-31 of the largest), but
// 0 times an infinite or NaN value is NaN.  So two warps look through V as it comes, for
// bf16 on the tiles that some row does not see whole, for fp16 on all: the product of a
// tile with a non-finite value is made on the CUDA cores over the visible slots alone,
// in fp16 with P in fp32.
//
// Every wait is bounded (about one second); on expiry the CTA records
// SSA_DEVICE_TIMEOUT, waits (bounded) for its copies and MMAs in flight, frees
// TMEM and exits.
#include <type_traits>

#include "common.cuh"
#include "mma_utils.cuh"
#include "paged.cuh"
#include "paged_join.cuh"
#include "paged_tma.cuh"
#include "tc_utils.cuh"

namespace ssa {
namespace ptc {

using namespace tc;

constexpr int kRows = 256;         // rows of an item
constexpr int kKT = 128;           // slots per key tile
constexpr int kExtra = 4;          // units an item costs besides its tiles
constexpr int kLeast = 1;          // units a CTA takes at least
constexpr int kLookers = 2;        // warps that look through V, half a tile each
constexpr int kThreads = 32 * (10 + kLookers);
constexpr float kSlack = 8.f;      // how far (log2) a tile may exceed the running maximum

template <int D>
struct Geo {
  static constexpr int kTileBytes = kKT * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr size_t kSmem = 1024 + 2 * kTileBytes + static_cast<size_t>(kStages) * kTileBytes + 640;
};

// A from TMEM, B from shared memory.
__device__ __forceinline__ void mma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bd), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The tile's O += P V for this thread's row over its first `see` slots, on the
// CUDA cores (P in TMEM over S, packed in T or in fp32; V swizzled in shared memory).
// `fresh`: O holds nothing yet.  The whole stream calls it.
template <typename T, int D, bool kPacked>
__device__ __forceinline__ void visible_product(uint32_t s_addr, uint32_t o_addr, const unsigned char* v, int see,
                                             bool fresh) {
#pragma unroll 1
  for (int c0 = 0; c0 < D; c0 += 16) {
    uint32_t o[16];
    if (!fresh) {
      tmem_ld16_async(o_addr + c0, o);
      tmem_wait();
    }
    float acc[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) acc[x] = fresh ? 0.f : __uint_as_float(o[x]);
    constexpr int kSlots = kPacked ? 32 : 16;            // of 16 columns
#pragma unroll 1
    for (int j0 = 0; j0 < kKT; j0 += kSlots) {
      uint32_t pk[16];
      tmem_ld16_async(s_addr + j0 * 16 / kSlots, pk);
      tmem_wait();
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const float2 two = unpack2<T>(pk[j * 16 / kSlots]);
        const float pj = !kPacked ? __uint_as_float(pk[j * 16 / kSlots]) : (j & 1) ? two.y : two.x;
        if (j0 + j < see) {
          const unsigned char* row = v + (c0 / 64) * (kKT * 128) + (j0 + j) * 128;
#pragma unroll
          for (int x = 0; x < 16; x += 8) {
            const int piece = ((c0 % 64) + x) / 8;
            const uint4 w = *reinterpret_cast<const uint4*>(row + ((piece ^ ((j0 + j) & 7)) << 4));
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack2<T>(ww[e]);
              acc[x + 2 * e] = fmaf(pj, f.x, acc[x + 2 * e]);
              acc[x + 2 * e + 1] = fmaf(pj, f.y, acc[x + 2 * e + 1]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(acc[x]);
    tmem_st16(o_addr + c0, o);
    tmem_wait_st();
  }
}
// The row's exponentials of the first `see` slots in fp32, over the scores; their sum.
__device__ __forceinline__ float wide_exps(uint32_t s_addr, int see, float c, float off) {
  float sum = 0.f;
#pragma unroll 1
  for (int j0 = 0; j0 < kKT; j0 += 16) {
    uint32_t u[16];
    tmem_ld16_async(s_addr + j0, u);
    tmem_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float e = j0 + j < see ? ex2_approx(fmaf(__uint_as_float(u[j]), c, -off)) : 0.f;
      sum += e;
      u[j] = __float_as_uint(e);
    }
    tmem_st16(s_addr + j0, u);
    tmem_wait_st();
  }
  return sum;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                                                              const __grid_constant__ CUtensorMap vmap,
                                                              PagedAttnParams p, MapOrder mo) {
  using G = Geo<D>;
  constexpr bool kBf = std::is_same<T, __nv_bfloat16>::value;
  constexpr float kShift = kBf ? 0.f : 7.f;              // factor 2^kShift on every exponential
  // weights that fp32 holds but fp16 rounds to 0: V matters where every row sees it too
  constexpr bool kLookAll = !kBf;
  constexpr uint32_t kIdS = idesc_f16(128, kKT, kBf);
  constexpr uint32_t kIdO = idesc_f16(128, D, kBf) | (1u << 16);   // B (= V) is MN-major
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* q_tile = base;                          // [2][D / 64][128][128 B], SWIZZLE_128B
  unsigned char* ring = base + 2 * G::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + G::kStages * G::kTileBytes);
  const uint32_t full = smem_u32(bars), empty = full + 8 * G::kStages, seen = empty + 8 * G::kStages;
  const uint32_t q_full = seen + 8 * G::kStages, s_full = q_full + 16, p_full = s_full + 16, o_full = p_full + 32;
  const uint32_t drain = o_full + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * G::kStages + 11);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd_half = abort_flag + 1;               // [stage][looker] the half of V holds a non-finite value
  volatile int* made = odd_half + 2 * G::kStages;        // [stream] it makes the tile's product itself
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int tt = tile_tokens(kRows, p.group);

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1 + kLookers);
      mbar_init(seen + 8 * s, kLookers);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(q_full + 8 * x, 4);
      mbar_init(s_full + 8 * x, 1);
      mbar_init(p_full + 16 * x, 4);                     // P of slots 0-63, and of 64-127
      mbar_init(p_full + 16 * x + 8, 4);
      mbar_init(o_full + 8 * x, 1);
      made[x] = 0;
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  PagedStart& start = *reinterpret_cast<PagedStart*>(bars + 4 * G::kStages + 14);
  paged_start(p, tt, kKT, kExtra, kLeast, &start);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  PagedWalk w = start.w;
  const bool any = start.any;
  if (threadIdx.x == 0) p.split[blockIdx.x] = any ? paged_split(p, w, tt, kExtra) : PagedSplit{};
  auto fail = [&]() {
    *abort_flag = 1;
    paged_error(p.c, SSA_DEVICE_TIMEOUT);
  };

  // V of the next tile: its ring entry and phase (every tile takes two entries, K's and V's)
  auto next_entries = [](int& st, uint32_t& par) {
    st += 2;
    if (st >= G::kStages) {
      st -= G::kStages;
      par ^= 1u;
    }
  };

  if (any && warp == 9) {
    // ---------------- TMA producer ----------------
    // lane i < boxes copies 64 columns of one page piece; the page of the next
    // tile is looked up before this tile's ring entries are waited for
    const int piece_rows = min(p.c.page_size, kKT), pieces = kKT / piece_rows, boxes = pieces * (D / 64);
    const int piece = lane & (pieces - 1), half = lane / pieces;
    const uint32_t box_at = half * (kKT * 128) + piece * piece_rows * 128;
    int64_t g = 0;
    int st = 0;
    uint32_t par = 1;
    bool stop = false;
    for (bool going = true; going && !stop; going = !stop && paged_advance(p, tt, kKT, kExtra, w)) {
      const PagedSegment seg = paged_segment(w, kExtra);
      if (seg.first == seg.last) continue;
      const int last_tok = min(w.tile * tt + tt, w.n) - 1;
      const int lim = p.causal ? max(w.len - w.n + last_tok + 1, 0) : w.len;
      int j = seg.first * kKT + piece * piece_rows;
      PageSpot next = page_spot(p.c, w.seq, j, lane < boxes ? lim : 0);
      for (int t = seg.first; t < seg.last && !stop; ++t) {
        const PageSpot at = next;
        j += kKT;
        if (t + 1 < seg.last) next = page_spot(p.c, w.seq, j, lane < boxes ? lim : 0);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++g) {
          if (!__all_sync(0xffffffffu, mbar_wait_or(empty + 8 * st, par, abort_flag))) {
            stop = true;
            fail();
            break;
          }
          if (lane == 0) mbar_expect_tx(full + 8 * st, G::kTileBytes);
          __syncwarp();
          if (lane < boxes)
            tma_load_4d(smem_u32(ring) + st * G::kTileBytes + box_at, kv ? &vmap : &kmap, half * 64,
                        mo.head_first ? w.head : at.row, mo.head_first ? at.row : w.head, at.page, full + 8 * st);
          if (++st == G::kStages) {
            st = 0;
            par ^= 1u;
          }
        }
      }
    }
    // every issued copy lands before the CTA exits
    if (lane == 0)
      for (int64_t r = g - 1; r >= 0 && r >= g - G::kStages; --r)
        mbar_wait(full + 8 * static_cast<int>(r % G::kStages), static_cast<uint32_t>((r / G::kStages) & 1));
  } else if (any && warp == 8) {
    // ---------------- MMA issuer: the warp decides, one lane issues ----------------
    constexpr uint32_t kTileDesc = G::kTileBytes >> 4, kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
    const uint32_t q_lo = smem_u32(q_tile) >> 4, ring_lo = smem_u32(ring) >> 4;
    // descriptors: SWIZZLE_128B, groups of 8 rows 1024 bytes apart; V (MN-major): 64-column chunks 16 KB apart
    auto desc = [](uint32_t lo) { return (static_cast<uint64_t>(kDescHi) << 32) | (lo & 0x3fffu); };
    auto desc_v = [](uint32_t lo) {
      return (static_cast<uint64_t>(kDescHi) << 32) | ((kKT * 128u >> 4) << 16) | (lo & 0x3fffu);
    };
    uint32_t p_ph = 0, q_ph = 0;                         // bit x: stream x
    int ks = 0;                               // ring entry of the current unit's K
    uint32_t kpar = 0;
    bool stop = false;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!stop && !__all_sync(0xffffffffu, mbar_wait_or(bar, parity, abort_flag))) {
        fail();
        stop = true;
      }
      fence_after();
      return !stop;
    };
    auto scores = [&](int x, int st) {                   // S_x = Q_x K^T, K in ring entry st
      if (elect_one()) {
        const uint32_t kb = ring_lo + st * kTileDesc, qb = q_lo + x * kTileDesc;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k / 4) * (kKT * 128) + (k % 4) * 32) >> 4;
          mma_f16(tmem + x * 128, desc(qb + off), desc(kb + off), kIdS, k > 0);
        }
        mma_commit(s_full + 8 * x);
      }
      __syncwarp();
    };
    auto release = [&](int st) {
      if (elect_one()) mma_commit(empty + 8 * st);
      __syncwarp();
    };
    for (bool going = true; going && !stop; going = !stop && paged_advance(p, tt, kKT, kExtra, w)) {
      const PagedSegment seg = paged_segment(w, kExtra);
      const int units = __shfl_sync(0xffffffffu, seg.last - seg.first, 0);
      if (units == 0) continue;
      const int rows = min(tt, w.n - w.tile * tt) * p.group;
      const int streams = __shfl_sync(0xffffffffu, rows > 128 ? 2 : 1, 0);
      uint32_t fresh = 3;
      wait(full + 8 * ks, kpar);
      for (int x = 0; x < streams && !stop; ++x) {
        if (!wait(q_full + 8 * x, (q_ph >> x) & 1u)) break;
        q_ph ^= 1u << x;
        scores(x, ks);
      }
      if (stop) break;
      release(ks);
      for (int i = 0; i < units && !stop; ++i) {
        int vs = ks + 1;
        uint32_t vpar = kpar;
        if (vs == G::kStages) { vs = 0; vpar ^= 1u; }
        int ns = vs + 1;                                 // the next unit's K
        uint32_t npar = vpar;
        if (ns == G::kStages) { ns = 0; npar ^= 1u; }
        const bool more = i + 1 < units;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (x >= streams) break;
          if (x == 0) wait(full + 8 * vs, vpar);
          const uint32_t pp = (p_ph >> x) & 1u;
          if (!wait(p_full + 16 * x, pp)) break;
          p_ph ^= 1u << x;
          const bool done = __shfl_sync(0xffffffffu, made[x], 0) != 0;    // by the stream
          const uint32_t vb = ring_lo + vs * kTileDesc, acc = ((fresh >> x) & 1u) ^ 1u;
          auto product = [&](int k0) {                   // four steps of 16 slots
#pragma unroll
            for (int k = k0; k < k0 + 4; ++k)
              mma_f16_ta(tmem + 256 + x * D, tmem + x * 128 + k * 8, desc_v(vb + (k * 2048 >> 4)), kIdO, k > 0 ? 1u : acc);
          };
          if (!done && elect_one()) product(0);
          __syncwarp();
          if (!wait(p_full + 16 * x + 8, pp)) break;
          if (elect_one()) {
            if (!done) product(4);
            if (x == streams - 1) mma_commit(empty + 8 * vs);
            if (!more) mma_commit(o_full + 8 * x);
          }
          __syncwarp();
          fresh &= ~(1u << x);
          if (more) {
            if (x == 0 && !wait(full + 8 * ns, npar)) break;
            scores(x, ns);
            if (x == streams - 1) release(ns);
          }
        }
        ks = ns;
        kpar = npar;
      }
    }
    // after a failed wait: the commit arrives once every MMA issued before it is done
    if (stop) {
      if (elect_one()) mma_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0);
    }
  } else if (any && warp < 8) {
    // ---------------- softmax and epilogue of stream x ----------------
    const int x = warp >> 2, r = (warp & 3) * 32 + lane;  // row of the stream, its TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + x * 128, o_addr = tmem + lane_base + 256 + x * D;
    // the warp's rows of its stream's Q tile: 16-byte piece pc of row rr
    constexpr int kPieces = D / 8;
    unsigned char* stage = q_tile + x * G::kTileBytes + (warp & 3) * 32 * 128;
    auto stage_at = [](int rr, int pc) { return (pc / 8) * (kKT * 128) + rr * 128 + (((pc % 8) ^ (rr & 7)) << 4); };
    const float c = p.inv_scale * kLog2e;
    uint32_t s_ph = 0, o_ph = 0, vpar = 0;
    int vs = 1;
    bool stop = false;
    // the same answer in every lane: what follows is done by whole warps
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!__all_sync(0xffffffffu, mbar_wait_or(bar, parity, abort_flag))) {
        fail();
        stop = true;
      }
      fence_after();
      return !stop;
    };
    auto arrive = [&](uint32_t bar) {                     // once a warp
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    bool going = true;
    for (int slot = 0; going && !stop; slot = 1, going = !stop && paged_advance(p, tt, kKT, kExtra, w)) {
      const PagedSegment seg = paged_segment(w, kExtra);
      const int units = seg.last - seg.first;
      if (units == 0) continue;
      const int tok0 = w.tile * tt, rows = min(tt, w.n - tok0) * p.group;
      const bool whole = seg.whole;
      if (x == 1 && rows <= 128) {                        // nothing for this stream here
        for (int i = 0; i < units; ++i) next_entries(vs, vpar);
        continue;
      }
      const int row = x * 128 + r;
      const bool live = row < rows;
      const int tok = tok0 + min(row, rows - 1) / p.group, head = w.head * p.group + row % p.group;
      const int lim = p.causal ? max(w.len - w.n + tok + 1, 0) : w.len;     // slots this row sees
      const int lim0 = p.causal ? max(w.len - w.n + tok0 + (x * 128) / p.group + 1, 0) : w.len;   // the stream's first row
      // ---- Q: a warp brings its own 32 rows, whole rows side by side ----
      const int64_t q_at = (w.q0 + tok) * p.q_sn + static_cast<int64_t>(head) * p.q_sh;
      const unsigned alive = __ballot_sync(0xffffffffu, live);
#pragma unroll
      for (int it = 0; it < kPieces; ++it) {
        const int rr = it * (32 / kPieces) + lane / kPieces, pc = lane % kPieces;
        const T* src = static_cast<const T*>(p.q) + __shfl_sync(0xffffffffu, q_at, rr) + pc * 8;
        unsigned char* dst = stage + stage_at(rr, pc);
        if ((alive >> rr) & 1u) cp_async16(smem_u32(dst), src);
        else *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
      }
      cp_commit();
      cp_wait<0>();
      fence_proxy_async();
      fence_before();
      arrive(q_full + 8 * x);
      if (r == 0) made[x] = 0;                            // tiles that are not looked at come first
      float m = -INFINITY, l = 0.f;
      int k0 = seg.first * kKT;
      for (int i = 0; i < units; ++i, k0 += kKT, next_entries(vs, vpar)) {
        if (!wait(s_full + 8 * x, s_ph)) break;
        s_ph ^= 1u;
        const bool masked = k0 + kKT > lim0;              // the same for the whole stream
        const int see = masked ? lim - k0 : kKT;
        uint32_t v[2][32];
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        tmem_ld32_async(s_addr, v[0]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          tmem_wait();
          tmem_ld32_async(s_addr + 32 * ((q + 1) & 3), v[(q + 1) & 1]);
          uint32_t (&u)[32] = v[q & 1];
          if (masked) {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] = 32 * q + j < see ? u[j] : __float_as_uint(-INFINITY);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(u[j + e]), __uint_as_float(u[j + 4 + e]));
        }
        const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * c;
        const bool raise = top > m + kSlack;
        if (__any_sync(0xffffffffu, raise)) {
          const float mn = raise ? top : m;
          const float f = m == -INFINITY ? 0.f : ex2_approx(m - mn);       // 1 where the row keeps its maximum
          m = mn;
          l *= f;
          if (i > 0) {                               // the PV of the tile before is done: S of this one came after it
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += 16) {
              uint32_t o[16];
              tmem_ld16_async(o_addr + c0, o);
              tmem_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(o_addr + c0, o);
            }
            tmem_wait_st();
          }
        }
        // V holds a non-finite value: the product is made here, over the slots a row sees
        auto odd = [&]() {
          const bool is = wait(seen + 8 * vs, vpar) && (odd_half[2 * vs] | odd_half[2 * vs + 1]) != 0;
          if (r == 0) made[x] = is;                       // before the MMA warp is told of P
          return is;
        };
        const float off = (m == -INFINITY ? 0.f : m) - kShift;
        const uint64_t c2 = pair(c, c), off2 = pair(-off, -off);
        uint64_t sum[2] = {0, 0};
        auto exps = [&](auto masked_tile) {
          constexpr bool kMasked = decltype(masked_tile)::value;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            tmem_wait();
            if (q < 3) tmem_ld32_async(s_addr + 32 * (q + 1), v[(q + 1) & 1]);
            uint32_t (&u)[32] = v[q & 1];
            if (kMasked) {
#pragma unroll
              for (int j = 0; j < 32; ++j) u[j] = 32 * q + j < see ? u[j] : __float_as_uint(-INFINITY);
            }
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float a, b;
              unpair(fma_pair(pair(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1])), c2, off2), a, b);
              a = ex2_approx(a);
              b = ex2_approx(b);
              sum[j & 1] = add_pair(sum[j & 1], pair(a, b));
              pk[j] = pack2<T>(a, b);
            }
            tmem_st16(s_addr + 16 * q, pk);
            if (!kMasked && q == 1) {                     // the tensor cores may begin
              tmem_wait_st();
              fence_before();
              arrive(p_full + 16 * x);
            }
          }
        };
        const unsigned char* v_tile = ring + vs * G::kTileBytes;
        if (kLookAll && odd()) {
          l += wide_exps(s_addr, see, c, off);
          visible_product<T, D, false>(s_addr, o_addr, v_tile, see, i == 0);
          fence_before();
          arrive(p_full + 16 * x);
        } else {
          if (masked) exps(std::true_type{});
          else exps(std::false_type{});
          float a, b;
          unpair(add_pair(sum[0], sum[1]), a, b);
          l += a + b;
          tmem_wait_st();
          if (!kLookAll && masked && odd()) visible_product<T, D, true>(s_addr, o_addr, v_tile, see, i == 0);
          fence_before();
          if (masked) arrive(p_full + 16 * x);
        }
        if (stop) break;
        arrive(p_full + 16 * x + 8);
      }
      if (stop) break;
      // ---- epilogue ----
      if (!wait(o_full + 8 * x, o_ph)) break;
      o_ph ^= 1u;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // through the warp's own rows of the Q tile, which no product reads any
      // more, so that whole rows are stored side by side
      const int64_t o_at = (w.q0 + tok) * p.o_sn + static_cast<int64_t>(head) * p.o_sh;
      float* part = p.part + (static_cast<int64_t>(blockIdx.x * 2 + slot) * kRows + row) * (D + 4);
      if (whole) {
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          tmem_ld32_async(o_addr + c0, o);
          tmem_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 f;
            f.x = pack2<T>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
            f.y = pack2<T>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            f.z = pack2<T>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
            f.w = pack2<T>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
            *reinterpret_cast<uint4*>(stage + stage_at(lane, (c0 + e) / 8)) = f;
          }
        }
        __syncwarp();
#pragma unroll
        for (int it = 0; it < kPieces; ++it) {
          const int rr = it * (32 / kPieces) + lane / kPieces, pc = lane % kPieces;
          T* dst = static_cast<T*>(p.out) + __shfl_sync(0xffffffffu, o_at, rr) + pc * 8;
          if ((alive >> rr) & 1u) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(stage + stage_at(rr, pc));
        }
        __syncwarp();
      } else {
        // D / 2 columns in fp32 fill a staged row
        float* rows0 = part - static_cast<int64_t>(lane) * (D + 4);
#pragma unroll
        for (int h0 = 0; h0 < D; h0 += D / 2) {
#pragma unroll
          for (int c0 = 0; c0 < D / 2; c0 += 32) {
            uint32_t o[32];
            tmem_ld32_async(o_addr + h0 + c0, o);
            tmem_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(stage + stage_at(lane, (c0 + e) / 4)) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
          __syncwarp();
#pragma unroll
          for (int it = 0; it < kPieces; ++it) {
            const int rr = it * (32 / kPieces) + lane / kPieces, pc = lane % kPieces;
            if ((alive >> rr) & 1u)
              *reinterpret_cast<uint4*>(rows0 + rr * (D + 4) + h0 + pc * 4) =
                  *reinterpret_cast<const uint4*>(stage + stage_at(rr, pc));
          }
          __syncwarp();
        }
      }
      if (live) {
        if (whole) {
          store_lse(p, w.q0 + tok, head, m - kShift, l);
        } else {
          part[D] = m - kShift;
          part[D + 1] = l;
        }
      }
    }
  } else if (any) {
    // ---------------- lookers: does V hold a non-finite value? ----------------
    // They pass every entry, K's too, before it is filled again: so each sees every
    // phase of its barrier.
    const int half = warp - 10;
    int st = 0;
    uint32_t par = 0;
    bool stop = false;
    for (bool going = true; going && !stop; going = !stop && paged_advance(p, tt, kKT, kExtra, w)) {
      const PagedSegment seg = paged_segment(w, kExtra);
      // as the streams: the first row's slots
      const int lim0 = p.causal ? max(w.len - w.n + w.tile * tt + 1, 0) : w.len;
      for (int t = seg.first; t < seg.last && !stop; ++t) {
        const bool look = kLookAll || t * kKT + kKT > lim0;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (!__all_sync(0xffffffffu, mbar_wait_or(full + 8 * st, par, abort_flag))) {
            stop = true;
            fail();
            break;
          }
          if (kv == 1 && look) {
            const uint4* v = reinterpret_cast<const uint4*>(ring + st * G::kTileBytes + half * (G::kTileBytes / 2)) + lane;
            uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 8
            for (int y = 0; y < G::kTileBytes / 1024; ++y) {
              const uint4 a = v[32 * y];
              z.x = times_zero<T>(a.x, z.x);
              z.y = times_zero<T>(a.y, z.y);
              z.z = times_zero<T>(a.z, z.z);
              z.w = times_zero<T>(a.w, z.w);
            }
            const bool found = __any_sync(0xffffffffu, odd_bits<T>(z.x | z.y | z.z | z.w) != 0);
            if (lane == 0) odd_half[2 * st + half] = found;
          }
          if (lane == 0) {
            mbar_arrive(seen + 8 * st);
            mbar_arrive(empty + 8 * st);
          }
          __syncwarp();
          if (++st == G::kStages) {
            st = 0;
            par ^= 1u;
          }
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 8) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <typename T, int D>
cudaError_t launch_t(const PagedAttnParams& p, ssa_dtype dt, int grid, cudaStream_t st) {
  CUtensorMap km, vm;
  MapOrder mo, vo;
  if (!page_map(p.c, p.c.k, p.c.k_sp, p.c.k_sn, p.c.k_sh, dt, kKT, &km, &mo) ||
      !page_map(p.c, p.c.v, p.c.v_sp, p.c.v_sn, p.c.v_sh, dt, kKT, &vm, &vo) || mo.head_first != vo.head_first)
    return cudaErrorInvalidValue;
  auto kern = attn_tc_kernel<T, D>;
  static SmemOptIn opt_in;
  const cudaError_t e = opt_in(reinterpret_cast<const void*>(kern), Geo<D>::kSmem);
  if (e != cudaSuccess) return e;
  kern<<<grid, kThreads, Geo<D>::kSmem, st>>>(km, vm, p, mo);
  return cudaGetLastError();
}

}  // namespace ptc

cudaError_t launch_paged_attn_tc(const PagedAttnParams& p, ssa_dtype dt, int grid, cudaStream_t st) {
  if (dt == SSA_BF16)
    return p.c.d == 128 ? ptc::launch_t<__nv_bfloat16, 128>(p, dt, grid, st) : ptc::launch_t<__nv_bfloat16, 64>(p, dt, grid, st);
  return p.c.d == 128 ? ptc::launch_t<__half, 128>(p, dt, grid, st) : ptc::launch_t<__half, 64>(p, dt, grid, st);
}

}  // namespace ssa
