// Slot weights of chunks on the 5th-generation tensor cores: bf16 / fp16, head
// size 64 or 128, page tiles (paged_tma.cuh).
//
//   w_j += sum_i exp2(s_ij log2 e - lse2_i) over the rows i that see slot j,
//
// with lse2_i from the attention kernel.  The scores are made again, transposed:
// S^T = K Q^T puts a slot in every TMEM lane and the rows in its columns, so
// the sum over rows is a thread's own, with no exchange between lanes.
//
// An item is 256 slots of one (sequence, KV head): two streams of 128 slots
// share every tile of Q rows (the g heads of a group at floor(128 / g) tokens).
// The row tiles of all items are shared out evenly (SlotCosts, paged.cuh); the
// slot sums of an item that is cut are joined by the last of its CTAs, in CTA order.
// Per row tile and stream the tensor cores do 128 x 128 x d products, the MUFU
// 128 x 128 exponentials, which bound it (1024 clocks against 512 at d = 128);
// a quarter of them is made on the FMA pipe instead (4% faster; a half, no more).
// 2 x 1024 tokens x 32 heads over 8192 slots, bf16: 225 us, 570 TFLOP/s (whole
// items in turn: 235; 4 x 1618 tokens x 8 heads of 64 over 3529: 12% of the call
// gained; items of two row tiles lose 5% by the join).  Two threads a slot (16
// warps) took the same time.
//
//   warps 0-3, 4-7  streams: a slot per thread; scores from TMEM, two buffers each
//   warp 8          TMEM allocation, single-thread MMA issue
//   warp 9          TMA producer: K (two items deep), Q rows and their lse2 (ring of 3)
//
// Every wait is bounded (about one second); on expiry the CTA records
// SSA_DEVICE_TIMEOUT and runs to its end without further waits or copies.
#include <type_traits>

#include "common.cuh"
#include "mma_utils.cuh"
#include "paged.cuh"
#include "paged_tma.cuh"
#include "tc_utils.cuh"

namespace ssa {
namespace pwt {

using namespace tc;

constexpr int kSlots = 128;        // of a stream
constexpr int kRows = 128;         // of a Q tile
constexpr int kThreads = 320;
constexpr int kGrid = 148;
constexpr int kExtra = 2;          // units an item costs besides its row tiles
constexpr int kLeast = 1;          // units a CTA takes at least
static_assert(kGrid * 8 * 4 <= SSA_PAGED_ZEROED, "a counter for every warp of the streams of a CTA");
constexpr int kQStages = 3;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Geo {
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr size_t kSmem = 1024 + (4 + kQStages) * static_cast<size_t>(kTileBytes) + kQStages * kRows * 4 + kRows * 2 + 160 + sizeof(PagedStart);
};

struct QueryMap {
  int tokens;                      // per Q tile
  int head_first;                  // row r of a tile: token r / g, head r % g; else token r % tokens, head r / tokens
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) weights_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                 const __grid_constant__ CUtensorMap qmap,
                                                                 PagedAttnParams p, MapOrder mo, QueryMap qm) {
  using G = Geo<D>;
  constexpr uint32_t kId = idesc_f16(128, kRows, std::is_same<T, __nv_bfloat16>::value);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* q_ring = base + 4 * G::kTileBytes;      // base: K [2 items][2 streams]
  float* z_ring = reinterpret_cast<float*>(q_ring + kQStages * G::kTileBytes);
  short* row_token = reinterpret_cast<short*>(z_ring + kQStages * kRows);   // token of a row in its tile
  uint64_t* bars = reinterpret_cast<uint64_t*>(row_token + kRows);
  const uint32_t k_full = smem_u32(bars), k_empty = k_full + 16, q_full = k_empty + 16, q_empty = q_full + 8 * kQStages;
  const uint32_t s_full = q_empty + 8 * kQStages, s_empty = s_full + 32;     // [stream][buffer]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 + 2 * kQStages + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  PagedStart& start = *reinterpret_cast<PagedStart*>(bars + 4 + 2 * kQStages + 10);
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int g = p.group, tt = qm.tokens;

  // rows of a Q slot that no box fills (tokens * g < 128) read as zero queries
  for (int i = threadIdx.x; i < kQStages * G::kTileBytes / 16; i += kThreads)
    reinterpret_cast<uint4*>(q_ring)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (threadIdx.x < kRows) {
    const int row = threadIdx.x, a = qm.head_first ? row / g : row % tt, h = qm.head_first ? row % g : row / tt;
    row_token[row] = static_cast<short>(h < g && a < tt ? a : kRows);       // kRows: no row
  }
  fence_proxy_async();
  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(k_full + 8 * b, 1);
      mbar_init(k_empty + 8 * b, 1);
    }
    for (int s = 0; s < kQStages; ++s) {
      mbar_init(q_full + 8 * s, 1 + 32);                 // the copies' bytes, and the lse2 of 32 lanes
      mbar_init(q_empty + 8 * s, 1 + 8);                 // the MMAs, and the streams' warps
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(s_full + 8 * b, 1);
      mbar_init(s_empty + 8 * b, 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&qmap);
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  paged_start<SlotCosts>(p, tt, 2 * kSlots, kExtra, kLeast, &start);
  fence_before();
  __syncthreads();
  fence_after();
  paged_after();                                         // lse2
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (!mbar_wait_or(bar, parity, abort_flag) && !*abort_flag) {
      *abort_flag = 1;
      paged_error(p.c, SSA_DEVICE_TIMEOUT);
    }
  };
  PagedWalk w = start.w;
  const bool any = start.any;
  auto advance = [&]() { return paged_advance<SlotCosts>(p, tt, 2 * kSlots, kExtra, w); };
  // the current item's part of this CTA: row tiles [first, last)
  auto row_tiles = [&]() {
    PagedSegment s = paged_segment(w, kExtra);
    const int r0 = SlotCosts(w.n, w.len, tt, 2 * kSlots, kExtra, p.causal).first_row_tile(w.tile);
    s.first += r0;
    s.last += r0;
    return s;
  };
  int64_t t = 0, n = 0;                                  // Q tiles and items so far

  if (any && warp == 9) {
    // ---------------- producer ----------------
    const int piece_rows = min(p.c.page_size, kSlots), pieces = kSlots / piece_rows, boxes = pieces * (D / 64);
    const int piece = lane & (pieces - 1), half = lane / pieces;
    const int64_t h_q = static_cast<int64_t>(p.c.h_kv) * g;
    // token and head of this lane's four rows of a Q tile (token `kRows`: no row)
    int row_tok[4], row_head[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = lane + 32 * e;
      row_tok[e] = qm.head_first ? row / g : row % tt;
      row_head[e] = qm.head_first ? row % g : row / tt;
      if (row_head[e] >= g || row_tok[e] >= tt) row_tok[e] = kRows;
    }
    const uint32_t q_bytes = static_cast<uint32_t>(tt * g) * 128 * (D / 64);
    bool stop = false;
    for (bool going = true; going && !stop; going = !stop && advance()) {
      const PagedSegment seg = row_tiles();
      if (seg.first == seg.last) continue;
      const int head = w.head, k0 = w.tile * 2 * kSlots;
      const int b = static_cast<int>(n & 1);
      wait(k_empty + 8 * b, static_cast<uint32_t>((n >> 1) & 1) ^ 1u);
      stop = __any_sync(0xffffffffu, *abort_flag);
      if (stop) break;
      if (lane == 0) mbar_expect_tx(k_full + 8 * b, 2 * G::kTileBytes);
      __syncwarp();
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (lane < boxes) {
          const PageSpot at = page_spot(p.c, w.seq, k0 + x * kSlots + piece * piece_rows, w.len);
          tma_load_4d(smem_u32(base) + (2 * b + x) * G::kTileBytes + half * (kSlots * 128) + piece * piece_rows * 128,
                      &kmap, half * 64, mo.head_first ? head : at.row, mo.head_first ? at.row : head, at.page,
                      k_full + 8 * b);
        }
      // lse2 of the next tile's rows is on its way while this tile's ring entry
      // is waited for
      float z[4];
      auto fetch = [&](int tile) {
        const int64_t tok = w.q0 + static_cast<int64_t>(tile) * tt;
        const int tokens = min(tt, w.n - tile * tt);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          z[e] = row_tok[e] < tokens ? __ldcg(p.lse2 + (tok + row_tok[e]) * h_q + head * g + row_head[e]) : INFINITY;
      };
      fetch(seg.first);
      for (int r = seg.first; r < seg.last; ++r, ++t) {
        const int s = static_cast<int>(t % kQStages);
        wait(q_empty + 8 * s, static_cast<uint32_t>((t / kQStages) & 1) ^ 1u);
        stop = __any_sync(0xffffffffu, *abort_flag);
        if (stop) break;
        if (lane == 0) mbar_expect_tx(q_full + 8 * s, q_bytes);
        __syncwarp();
        if (lane < D / 64) {
          const int y = head * g, zc = static_cast<int>(w.q0) + r * tt;
          tma_load_3d(smem_u32(q_ring + s * G::kTileBytes) + lane * (kRows * 128), &qmap, lane * 64,
                      qm.head_first ? y : zc, qm.head_first ? zc : y, q_full + 8 * s);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) z_ring[s * kRows + lane + 32 * e] = z[e];   // exp2(s - inf) = 0 where there is no row
        mbar_arrive(q_full + 8 * s);
        if (r + 1 < seg.last) fetch(r + 1);
      }
      ++n;
    }
    // every issued copy lands before the CTA exits
    for (int64_t r = n - 1; lane == 0 && r >= 0 && r >= n - 2; --r) mbar_wait(k_full + 8 * static_cast<int>(r & 1), static_cast<uint32_t>((r >> 1) & 1));
    for (int64_t r = t - 1; lane == 0 && r >= 0 && r >= t - kQStages; --r)
      mbar_wait(q_full + 8 * static_cast<int>(r % kQStages), static_cast<uint32_t>((r / kQStages) & 1));
  } else if (any && warp == 8) {
    // ---------------- MMA issuer: the warp decides, one lane issues ----------------
    constexpr uint32_t kTileDesc = G::kTileBytes >> 4, kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
    const uint32_t k_lo = smem_u32(base) >> 4, q_lo = smem_u32(q_ring) >> 4;
    auto desc = [](uint32_t lo) { return (static_cast<uint64_t>(kDescHi) << 32) | (lo & 0x3fffu); };
    int s = 0;
    uint32_t qpar = 0;
    for (bool going = true; going && !__any_sync(0xffffffffu, *abort_flag); going = advance()) {
      const PagedSegment seg = row_tiles();
      const int b = static_cast<int>(n & 1), tiles = __shfl_sync(0xffffffffu, seg.last - seg.first, 0);
      if (tiles == 0) continue;
      wait(k_full + 8 * b, static_cast<uint32_t>((n >> 1) & 1));
      for (int j = 0; j < tiles; ++j, ++t) {
        const int sb = static_cast<int>(t & 1);
        wait(q_full + 8 * s, qpar);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          wait(s_empty + 8 * (2 * x + sb), static_cast<uint32_t>((t >> 1) & 1) ^ 1u);
          __syncwarp();
          fence_after();
          if (elect_one()) {
            const uint32_t kb = k_lo + (2 * b + x) * kTileDesc, qb = q_lo + s * kTileDesc;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t off = ((k / 4) * (128 * 128) + (k % 4) * 32) >> 4;
              mma_f16(tmem + (2 * x + sb) * 128, desc(kb + off), desc(qb + off), kId, k > 0);
            }
            mma_commit(s_full + 8 * (2 * x + sb));
            if (x == 1) mma_commit(q_empty + 8 * s);
          }
          __syncwarp();
        }
        if (++s == kQStages) {
          s = 0;
          qpar ^= 1u;
        }
      }
      if (elect_one()) mma_commit(k_empty + 8 * b);
      __syncwarp();
      ++n;
    }
    // the last commits arrive once every MMA is done; both buffers of K are
    // then free (an item's k_empty is its n-th phase)
    for (int64_t r = n - 1; r >= 0 && r >= n - 2; --r)
      mbar_wait(k_empty + 8 * static_cast<int>(r & 1), static_cast<uint32_t>((r >> 1) & 1));
  } else if (any) {
    // ---------------- stream x: a slot per thread ----------------
    const int x = warp >> 2, r0 = (warp & 3) * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c = p.inv_scale * kLog2e;
    const uint64_t c2 = pair(c, c);
    const int rows = tt * g;                             // of a Q tile that boxes fill
    bool going = true;
    for (int second = 0; going && !__any_sync(0xffffffffu, *abort_flag); second = 1, going = advance()) {
      const PagedSegment seg = row_tiles();
      if (seg.first == seg.last) continue;
      const int k0 = w.tile * 2 * kSlots, slot = k0 + x * kSlots + r0;
      float total = 0.f;
      for (int r = seg.first; r < seg.last; ++r, ++t) {
        const int s = static_cast<int>(t % kQStages), sb = static_cast<int>(t & 1);
        wait(q_full + 8 * s, static_cast<uint32_t>((t / kQStages) & 1));   // lse2 of the rows
        wait(s_full + 8 * (2 * x + sb), static_cast<uint32_t>((t >> 1) & 1));
        __syncwarp();
        fence_after();
        const int64_t lim0 = p.causal ? static_cast<int64_t>(w.len) - w.n + r * tt + 1 : w.len;
        const bool masked = lim0 < k0 + (x + 1) * kSlots || w.n - r * tt < tt;
        const float4* zs = reinterpret_cast<const float4*>(z_ring + s * kRows);
        const uint32_t ta = tmem + lane_base + (2 * x + sb) * 128;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t v[2][32];
        tmem_ld32_async(ta, v[0]);
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          tmem_wait();
          if (q4 < 3) tmem_ld32_async(ta + 32 * (q4 + 1), v[(q4 + 1) & 1]);
          if (q4 == 3 && rows < kRows) {
            // rows that no box fills, fewer than g: zero queries, whose score with an
            // infinite key is NaN
#pragma unroll
            for (int j = 16; j < 32; ++j) v[q4 & 1][j] = 96 + j < rows ? v[q4 & 1][j] : 0u;
          }
          if (!masked) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 z = zs[q4 * 8 + j];
              float e0, e1, e2, e3;
              unpair(fma_pair(pair(__uint_as_float(v[q4 & 1][4 * j]), __uint_as_float(v[q4 & 1][4 * j + 1])), c2,
                              pair(-z.x, -z.y)), e0, e1);
              unpair(fma_pair(pair(__uint_as_float(v[q4 & 1][4 * j + 2]), __uint_as_float(v[q4 & 1][4 * j + 3])), c2,
                              pair(-z.z, -z.w)), e2, e3);
              if (j % 2 == 0) {                            // a quarter of the exponentials off the MUFU
                exp2_pair(e0, e1);
              } else {
                e0 = ex2_approx(e0);
                e1 = ex2_approx(e1);
              }
              sum[0] += e0;
              sum[1] += e1;
              sum[2] += ex2_approx(e2);
              sum[3] += ex2_approx(e3);
            }
          } else {
            // a row of token a sees the slot from token `from` on
            const short4* ts = reinterpret_cast<const short4*>(row_token);
            const int from = p.causal ? slot - (w.len - w.n) - r * tt : -1, tokens = min(tt, w.n - r * tt);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 z = zs[q4 * 8 + j];
              const short4 a = ts[q4 * 8 + j];
              const float e0 = ex2_approx(fmaf(__uint_as_float(v[q4 & 1][4 * j]), c, -z.x));
              const float e1 = ex2_approx(fmaf(__uint_as_float(v[q4 & 1][4 * j + 1]), c, -z.y));
              const float e2 = ex2_approx(fmaf(__uint_as_float(v[q4 & 1][4 * j + 2]), c, -z.z));
              const float e3 = ex2_approx(fmaf(__uint_as_float(v[q4 & 1][4 * j + 3]), c, -z.w));
              sum[0] += a.x >= from && a.x < tokens ? e0 : 0.f;
              sum[1] += a.y >= from && a.y < tokens ? e1 : 0.f;
              sum[2] += a.z >= from && a.z < tokens ? e2 : 0.f;
              sum[3] += a.w >= from && a.w < tokens ? e3 : 0.f;
            }
          }
        }
        total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(s_empty + 8 * (2 * x + sb));
          mbar_arrive(q_empty + 8 * s);
        }
        __syncwarp();
      }
      bool mine = true;
      if (!seg.whole) {
        // a warp's slots are joined by the last of the item's CTAs, in CTA order
        // (the counter is zero before the launch and after it)
        const int a = unit_cta(w, w.item_first + kExtra), parts = unit_cta(w, w.item_first + w.units - 1) - a + 1;
        const int at = x * kSlots + r0;
        p.part[(2 * blockIdx.x + second) * 2 * kSlots + at] = total;
        __threadfence();
        __syncwarp();
        int counted = 0;
        if (lane == 0) {
          counted = atomicAdd(p.counters + a * 8 + warp, 1);
          if (counted == parts - 1) p.counters[a * 8 + warp] = 0;
        }
        mine = __shfl_sync(0xffffffffu, counted, 0) == parts - 1;
        if (mine) {
          __threadfence();
          // the item is the second of CTA a's two parts if a's share starts before it
          const int in_a = mul_div(a, w.total, w.ctas) < w.item_first ? 1 : 0;
          total = 0.f;
          for (int i = 0; i < parts; ++i)
            total += __ldcg(p.part + (2 * (a + i) + (i == 0 ? in_a : 0)) * 2 * kSlots + at);
        }
      }
      if (mine && slot < w.len) {
        int page, row;
        page_of(p.c, slot, page, row);
        const int64_t pg = physical_page(p.c, p.c.table, p.c.table_stride, w.seq, page);
        if (pg >= 0) atomicAdd(&p.c.w[pg * p.c.w_sp + row * p.c.w_sn + w.head * p.c.w_sh], total);
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

// q as a 3-D tensor (d, heads and tokens by ascending stride), boxes of 64
// columns x the g heads of a group x `tokens` tokens.
bool query_map(const PagedAttnParams& p, ssa_dtype dt, CUtensorMap* map, QueryMap* qm) {
  auto enc = tensor_map_encoder();
  if (!enc || !p.q) return false;
  const int64_t h_q = static_cast<int64_t>(p.c.h_kv) * p.group;
  int64_t sh = p.q_sh, sn = p.q_sn;
  if (h_q == 1) sh = p.c.d;
  if (p.rows == 1 && sn < sh * h_q) sn = sh * h_q;
  qm->tokens = kRows / p.group;
  qm->head_first = sh < sn;
  const int64_t s1 = qm->head_first ? sh : sn, s2 = qm->head_first ? sn : sh;
  const int64_t n1 = qm->head_first ? h_q : p.rows, n2 = qm->head_first ? p.rows : h_q;
  if (s1 < p.c.d || s2 < s1 * n1 || s2 * 2 >= (1ll << 40)) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.c.d), static_cast<cuuint64_t>(n1), static_cast<cuuint64_t>(n2)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(s1) * 2, static_cast<cuuint64_t>(s2) * 2};
  const cuuint32_t gh = p.group, tk = qm->tokens;
  const cuuint32_t box[3] = {64, qm->head_first ? gh : tk, qm->head_first ? tk : gh};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType t = dt == SSA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, t, 3, const_cast<void*>(p.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t launch_t(const PagedAttnParams& p, ssa_dtype dt, cudaStream_t st) {
  CUtensorMap km, qm;
  MapOrder mo;
  QueryMap qo;
  if (!page_map(p.c, p.c.k, p.c.k_sp, p.c.k_sn, p.c.k_sh, dt, kSlots, &km, &mo) || !query_map(p, dt, &qm, &qo))
    return cudaErrorInvalidValue;
  auto kern = weights_tc_kernel<T, D>;
  static SmemOptIn opt_in;
  const cudaError_t e = opt_in(reinterpret_cast<const void*>(kern), Geo<D>::kSmem);
  if (e != cudaSuccess) return e;
  return launch_after(kern, dim3(kGrid), dim3(kThreads), Geo<D>::kSmem, st, km, qm, p, mo, qo);
}

}  // namespace pwt

bool paged_weights_tc_supported(const PagedAttnParams& p, ssa_dtype dt) {
  CUtensorMap m;
  pwt::QueryMap q;
  return page_tiles_supported(p, dt) && pwt::query_map(p, dt, &m, &q);
}

cudaError_t launch_paged_weights_tc(const PagedAttnParams& p, ssa_dtype dt, cudaStream_t st) {
  if (dt == SSA_BF16)
    return p.c.d == 128 ? pwt::launch_t<__nv_bfloat16, 128>(p, dt, st) : pwt::launch_t<__nv_bfloat16, 64>(p, dt, st);
  return p.c.d == 128 ? pwt::launch_t<__half, 128>(p, dt, st) : pwt::launch_t<__half, 64>(p, dt, st);
}

}  // namespace ssa
