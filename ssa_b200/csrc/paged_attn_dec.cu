// Attention of a few rows over the paged cache (single tokens): bf16 / fp16,
// head size 64 or 128, pages of a power of two of at least 8 slots.
//
// Bound by reading K and V once.  An item is 16 rows (the g heads of a KV
// group at floor(16 / g) tokens); its key tiles of 64 slots come by TMA into
// a ring (a producer warp, one lane per page box), which a CTA on every SM
// keeps in flight across the items it walks.  Two groups of four warps take the
// tiles in turn, a warp 16 slots of each, with its own running maximum, sum and
// output (mma.sync m16n8k16, Q as A in registers, K and V by ldmatrix), so the
// warps meet only where an item ends.  mma.sync suffices: 16 x 64 x d products
// a tile are a few hundred clocks against about 1400 to fetch its 32 KB at
// d = 128.  (One group of four warps was 8% slower, bound by its own steps; a
// ring of 96 KB is as fast as one of 192 KB.)  32 tokens x 32 heads over 8192
// slots each, bf16: 1.07 GB in 174 us, 6.2 TB/s.  One token over 1024 slots:
// 12 us, all of it latency.
//
// P enters the product with V as two 16-bit terms (p = hi + lo, off by 2^-17),
// sums and outputs are fp32.  Slots hidden from a row have p = 0, and so has lo at
// many others: 0 times infinity is NaN.  So two more warps look through V as it comes,
// and a tile that holds a non-finite value has its product made on the CUDA cores, over
// the visible slots and with p in fp32.
//
// Every wait is bounded (about one second); on expiry the CTA records
// SSA_DEVICE_TIMEOUT and runs to its end without further waits.
#include <type_traits>

#include "common.cuh"
#include "mma_utils.cuh"
#include "paged.cuh"
#include "paged_join.cuh"
#include "paged_tma.cuh"
#include "tc_utils.cuh"

namespace ssa {
namespace pdec {

using namespace tc;

constexpr int kRows = 16;
constexpr int kKT = 64;
constexpr int kExtra = 4;          // units an item costs besides its tiles
constexpr int kLeast = 4;          // units a CTA takes at least (1: 9.8 us, 4: 8.4 us, 8: 11.3 us at 128 slots)
constexpr int kWarps = 8;          // consumers: two groups of four, 16 slots of a tile each
constexpr int kLookers = 2;        // warps that look through V, the tiles of one group each
constexpr int kThreads = 32 * (kWarps + 1 + kLookers);

template <int D>
struct Geo {
  static constexpr int kTileBytes = kKT * D * 2;                    // of K, and of V
  static constexpr int kStages = D == 128 ? 4 : 8;
  // a stage always serves the same group: its warps then see every phase of
  // the stage's barrier, and a wait by parity means the phase it should
  static_assert(kStages % 2 == 0, "stages alternate between the two groups");
  static constexpr int kJoinRow = D + 4;                            // floats
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * 2 * kTileBytes +
                                  kWarps * kRows * kJoinRow * 4 + 28 * kStages + 16 + sizeof(PagedStart);
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) attn_dec_kernel(const __grid_constant__ CUtensorMap kmap,
                                                               const __grid_constant__ CUtensorMap vmap,
                                                               PagedAttnParams p, MapOrder mo) {
  using G = Geo<D>;
  constexpr int KS = D / 16, NT = D / 8;
  constexpr int64_t kPartFloats = kRows * (D + 4);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* join = reinterpret_cast<float*>(base + G::kStages * 2 * G::kTileBytes);   // [warp][row][D + 4]
  uint64_t* bars = reinterpret_cast<uint64_t*>(join + kWarps * kRows * G::kJoinRow);
  const uint32_t ring = smem_u32(base), full = smem_u32(bars), empty = full + 8 * G::kStages, seen = empty + 8 * G::kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 3 * G::kStages);
  volatile int* last = abort_flag + 1;
  volatile int* odd_tile = abort_flag + 2;               // [kStages] V of the stage holds a non-finite value
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int tt = tile_tokens(kRows, p.group);
  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, kWarps / 2);
      mbar_init(seen + 8 * s, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  PagedStart& start = *reinterpret_cast<PagedStart*>(bars + 3 * G::kStages + 1 + G::kStages / 2);
  paged_start(p, tt, kKT, kExtra, kLeast, &start);
  __syncthreads();
  PagedWalk w = start.w;
  if (!start.any) return;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (!mbar_wait_or(bar, parity, abort_flag) && !*abort_flag) {
      *abort_flag = 1;
      paged_error(p.c, SSA_DEVICE_TIMEOUT);
    }
  };

  if (warp == kWarps) {
    // ---------------- TMA producer ----------------
    // lane i copies 64 columns of one page piece of K or of V; the page of the
    // next tile is looked up before this tile's ring entry is waited for
    const int piece_rows = min(p.c.page_size, kKT), pieces = kKT / piece_rows, boxes = pieces * (D / 64);
    const int kv = lane / boxes, box = lane - kv * boxes, piece = box & (pieces - 1), half = box / pieces;
    const uint32_t box_at = ring + kv * G::kTileBytes + half * (kKT * 128) + piece * piece_rows * 128;
    int64_t g = 0;
    bool going = true;
    for (; going; going = going && paged_advance(p, tt, kKT, kExtra, w)) {
      const PagedSegment seg = paged_segment(w, kExtra);
      if (seg.first == seg.last) continue;
      const int last_tok = min(w.tile * tt + tt, w.n) - 1;
      const int lim = p.causal ? max(w.len - w.n + last_tok + 1, 0) : w.len;
      int j = seg.first * kKT + piece * piece_rows;
      PageSpot next = page_spot(p.c, w.seq, j, kv < 2 ? lim : 0);
      for (int t = seg.first; t < seg.last; ++t, ++g) {
        const PageSpot at = next;
        j += kKT;
        if (t + 1 < seg.last) next = page_spot(p.c, w.seq, j, kv < 2 ? lim : 0);
        const int s = static_cast<int>(g % G::kStages);
        wait(empty + 8 * s, static_cast<uint32_t>((g / G::kStages) & 1) ^ 1u);
        if (__any_sync(0xffffffffu, *abort_flag)) {
          going = false;
          break;
        }
        if (lane == 0) mbar_expect_tx(full + 8 * s, 2 * G::kTileBytes);
        __syncwarp();
        if (kv < 2)
          tma_load_4d(box_at + 2 * s * G::kTileBytes, kv ? &vmap : &kmap, half * 64, mo.head_first ? w.head : at.row,
                      mo.head_first ? at.row : w.head, at.page, full + 8 * s);
      }
    }
    // every issued copy lands before the CTA exits
    if (lane == 0)
      for (int64_t r = g - 1; r >= 0 && r >= g - G::kStages; --r)
        mbar_wait(full + 8 * static_cast<int>(r % G::kStages), static_cast<uint32_t>((r / G::kStages) & 1));
    return;
  }

  if (warp > kWarps) {
    // ---------------- lookers: does V of a tile hold a non-finite value? ----------------
    const int mine = warp - kWarps - 1;
    int64_t g = 0;
    for (bool going = true; going; going = paged_advance(p, tt, kKT, kExtra, w)) {
      const PagedSegment seg = paged_segment(w, kExtra);
      for (int t = seg.first; t < seg.last; ++t, ++g) {
        if ((g & 1) != mine) continue;
        const int st = static_cast<int>(g % G::kStages);
        wait(full + 8 * st, static_cast<uint32_t>((g / G::kStages) & 1));
        const uint4* v = reinterpret_cast<const uint4*>(base + (2 * st + 1) * G::kTileBytes) + lane;
        uint4 odd = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 8
        for (int x = 0; x < G::kTileBytes / 512; ++x) {
          const uint4 a = v[32 * x];
          odd.x = times_zero<T>(a.x, odd.x);
          odd.y = times_zero<T>(a.y, odd.y);
          odd.z = times_zero<T>(a.z, odd.z);
          odd.w = times_zero<T>(a.w, odd.w);
        }
        const bool any = __any_sync(0xffffffffu, odd_bits<T>(odd.x | odd.y | odd.z | odd.w) != 0);
        if (lane == 0) {
          odd_tile[st] = any;
          mbar_arrive(seen + 8 * st);
        }
        __syncwarp();
      }
    }
    return;
  }

  // ---------------- consumers ----------------
  const int gr = lane >> 2, gc = lane & 3;               // rows gr, gr + 8; column pairs 2 gc of a fragment
  const float c = p.inv_scale * kLog2e;
  const int64_t cap = score_stride(p.c);
  // ldmatrix rows of this lane: K (slots x 16 columns), V transposed (16 slots x columns)
  const int kk = (lane >> 4) * 8 + (lane & 7), kp = (lane >> 3) & 1;
  const int vk = ((lane >> 3) & 1) * 8 + (lane & 7), vp = lane >> 4;
  int64_t g = 0;
  bool going = true;
  for (int slot = 0; going; slot = 1, going = paged_advance(p, tt, kKT, kExtra, w)) {
    const PagedSegment seg = paged_segment(w, kExtra);
    if (seg.first == seg.last) continue;
    const int tok0 = w.tile * tt, rows = min(tt, w.n - tok0) * p.group;
    uint32_t q[KS][4];
    int lim[2];
    float* sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = min(gr + 8 * i, rows - 1), tok = tok0 + r / p.group, head = w.head * p.group + r % p.group;
      const T* src = static_cast<const T*>(p.q) + (w.q0 + tok) * p.q_sn + static_cast<int64_t>(head) * p.q_sh + 2 * gc;
      const bool live = gr + 8 * i < rows;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[ks][i] = live ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * ks)) : 0u;
        q[ks][i + 2] = live ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * ks + 8)) : 0u;
      }
      lim[i] = p.causal ? max(w.len - w.n + tok + 1, 0) : w.len;
      sc[i] = p.scores && live
                  ? p.scores + ((w.q0 + tok) * (static_cast<int64_t>(p.c.h_kv) * p.group) + head) * cap : nullptr;
    }
    const int lim0 = p.causal ? max(w.len - w.n + tok0 + 1, 0) : w.len;    // the first row's
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][e] = 0.f;
    for (int t = seg.first; t < seg.last; ++t, ++g) {
      if ((g & 1) != (warp >> 2)) continue;
      const int st = static_cast<int>(g % G::kStages);
      const int k0 = t * kKT + (warp & 3) * 16;
      wait(full + 8 * st, static_cast<uint32_t>((g / G::kStages) & 1));
      __syncwarp();
      const uint32_t kb = ring + 2 * st * G::kTileBytes, vb = kb + G::kTileBytes;
      float s[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
      {
        const int key = (warp & 3) * 16 + kk;
        const uint32_t row = kb + key * 128;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4(row + (ks / 4) * (kKT * 128) + ((((ks % 4) * 2 + kp) ^ (key & 7)) << 4), b0, b1, b2, b3);
          mma16816<T>(s[0], q[ks], b0, b1);
          mma16816<T>(s[1], q[ks], b2, b3);
        }
      }
      const bool masked = k0 + 16 > lim0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[t][2 * i] *= c;
          s[t][2 * i + 1] *= c;
          const int j = k0 + 8 * t + 2 * gc;
          if (sc[i] && j < cap) *reinterpret_cast<float2*>(sc[i] + j) = make_float2(s[t][2 * i], s[t][2 * i + 1]);
          if (masked) {
            if (j >= lim[i]) s[t][2 * i] = -INFINITY;
            if (j + 1 >= lim[i]) s[t][2 * i + 1] = -INFINITY;
          }
        }
      float f[2];
      bool raise = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[i], mx);
        f[i] = mn == -INFINITY ? 1.f : ex2_approx(m[i] - mn);
        raise |= mn > m[i];
        m[i] = mn;
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[i] *= f[i];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            o[t][2 * i] *= f[i];
            o[t][2 * i + 1] *= f[i];
          }
        }
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float off = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          s[t][2 * i] = ex2_approx(s[t][2 * i] - off);
          s[t][2 * i + 1] = ex2_approx(s[t][2 * i + 1] - off);
          l[i] += s[t][2 * i] + s[t][2 * i + 1];         // this lane's columns; joined at the end
          split2<T>(s[t][2 * i], s[t][2 * i + 1], hi[2 * t + i], lo[2 * t + i]);
        }
      }
      const int key = (warp & 3) * 16 + vk;
      const uint32_t row = vb + key * 128;
      auto v_at = [&](int t) { return row + (t / 4) * (kKT * 128) + ((((t % 4) * 2 + vp) ^ (key & 7)) << 4); };
      wait(seen + 8 * st, static_cast<uint32_t>((g / G::kStages) & 1));
      if (__any_sync(0xffffffffu, odd_tile[st])) {
        for (int j = 0; j < 16; ++j) {
          // p of rows gr, gr + 8 at slot j: fragment t = j / 8, lane column (j % 8) / 2
          const int src = (lane & 28) + ((j & 7) >> 1);
          float pj[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x0 = __shfl_sync(0xffffffffu, s[0][2 * i], src), x1 = __shfl_sync(0xffffffffu, s[0][2 * i + 1], src);
            const float y0 = __shfl_sync(0xffffffffu, s[1][2 * i], src), y1 = __shfl_sync(0xffffffffu, s[1][2 * i + 1], src);
            pj[i] = j < 8 ? ((j & 1) ? x1 : x0) : ((j & 1) ? y1 : y0);
          }
          const int slot_row = (warp & 3) * 16 + j;
          const unsigned char* vr = base + (2 * st + 1) * G::kTileBytes + slot_row * 128;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(vr + (t / 8) * (kKT * 128) +
                                                                  (((t % 8) ^ (slot_row & 7)) << 4) + gc * 4);
            const float2 two = unpack2<T>(x);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (k0 + j < lim[i]) {
                o[t][2 * i] = fmaf(pj[i], two.x, o[t][2 * i]);
                o[t][2 * i + 1] = fmaf(pj[i], two.y, o[t][2 * i + 1]);
              }
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT / 2; ++t) {
          uint32_t v[4];
          ldsm_x4_t(v_at(t), v[0], v[1], v[2], v[3]);
          mma16816<T>(o[2 * t], hi, v[0], v[1]);
          mma16816<T>(o[2 * t + 1], hi, v[2], v[3]);
          mma16816<T>(o[2 * t], lo, v[0], v[1]);
          mma16816<T>(o[2 * t + 1], lo, v[2], v[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * st);
    }
    // ---- join the warps ----
    float* mine = join + warp * kRows * G::kJoinRow;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      float* dst = mine + (gr + 8 * i) * G::kJoinRow;
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<float2*>(dst + 8 * t + 2 * gc) = make_float2(o[t][2 * i], o[t][2 * i + 1]);
      if (gc == 0) {
        dst[D] = m[i];
        dst[D + 1] = l[i];
      }
    }
    asm volatile("barrier.cta.sync 1, 256;" ::: "memory");
    const int r = threadIdx.x >> 4, x0 = (threadIdx.x & 15) * (D / 16);
    const bool whole = seg.whole;
    if (r < rows) {
      float mx = -INFINITY;
#pragma unroll
      for (int y = 0; y < kWarps; ++y) mx = fmaxf(mx, join[(y * kRows + r) * G::kJoinRow + D]);
      const float off = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, fy[kWarps];
#pragma unroll
      for (int y = 0; y < kWarps; ++y) {
        const float* src = join + (y * kRows + r) * G::kJoinRow;
        fy[y] = ex2_approx(src[D] - off);
        sum = fmaf(fy[y], src[D + 1], sum);
      }
      const int tok = tok0 + r / p.group, head = w.head * p.group + r % p.group;
      const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      T* out = static_cast<T*>(p.out) + (w.q0 + tok) * p.o_sn + static_cast<int64_t>(head) * p.o_sh + x0;
      float* part = p.part + (blockIdx.x * 2 + slot) * kPartFloats + r * (D + 4);
#pragma unroll
      for (int x = 0; x < D / 16; x += 4) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int y = 0; y < kWarps; ++y) {
          const float4 u = *reinterpret_cast<const float4*>(join + (y * kRows + r) * G::kJoinRow + x0 + x);
          a.x = fmaf(fy[y], u.x, a.x);
          a.y = fmaf(fy[y], u.y, a.y);
          a.z = fmaf(fy[y], u.z, a.z);
          a.w = fmaf(fy[y], u.w, a.w);
        }
        if (whole) {
          uint2 pk;
          pk.x = pack2<T>(a.x * inv, a.y * inv);
          pk.y = pack2<T>(a.z * inv, a.w * inv);
          *reinterpret_cast<uint2*>(out + x) = pk;
        } else {
          *reinterpret_cast<float4*>(part + x0 + x) = a;
        }
      }
      if ((threadIdx.x & 15) == 0) {
        if (whole) {
          store_lse(p, w.q0 + tok, head, mx, sum);
        } else {
          part[D] = mx;
          part[D + 1] = sum;
        }
      }
    }
    if (!whole) __threadfence();                         // the part, before this CTA counts itself in
    asm volatile("barrier.cta.sync 1, 256;" ::: "memory");   // also: before the next item's partials overwrite these
    if (!whole) {
      // the last of the item's CTAs joins it, a warp per row
      const int a = unit_cta(w, w.item_first + kExtra), parts = unit_cta(w, w.item_first + w.units - 1) - a + 1;
      if (threadIdx.x == 0) {
        const bool is = atomicAdd(p.counters + a, 1) == parts - 1;
        if (is) p.counters[a] = 0;
        *last = is;
      }
      asm volatile("barrier.cta.sync 1, 256;" ::: "memory");
      if (*last) {
        __threadfence();
        // the item is the second of CTA a's two parts if a's share starts before it
        const int second = mul_div(a, w.total, w.ctas) < w.item_first ? 1 : 0;
        const float* first = p.part + 2 * static_cast<int64_t>(a) * kPartFloats;
        for (int r = warp; r < rows; r += kWarps)
          write_joined<T, 8>(p, [&](int i) { return first + (2 * i + (i == 0 ? second : 0)) * kPartFloats + r * (D + 4); },
                             parts, w.q0 + tok0, w.head, r);
      }
    }
  }
}

// Slot weights from the scores the attention kernel left: w_j += sum over the
// rows that see j of exp2(s_ij - lse2_i).  A thread takes four slots of one KV
// head; the additions of a slot are in row order.  It reads 4 bytes a score, 1/32 of
// the cache's bytes at four heads a group and d = 128: 6 us for 16 tokens over up
// to 8192 slots, most of it launch and latency.
__global__ void __launch_bounds__(256) weights_dec_kernel(PagedAttnParams p) {
  paged_after();
  const int seq = blockIdx.z, head = blockIdx.y;
  const PagedSeq q = paged_seq(p.c, p.q_starts, p.rows, seq);
  const int j0 = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (q.n == 0 || j0 >= q.len) return;
  const int64_t cap = score_stride(p.c);
  const int h_q = p.c.h_kv * p.group;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < q.n; ++i) {
    const int lim = p.causal ? q.len - q.n + i + 1 : q.len;
    if (j0 >= lim) continue;
    const int64_t r0 = (q.q0 + i) * h_q + head * p.group;
#pragma unroll 4
    for (int e = 0; e < p.group; ++e) {
      const float z = p.lse2[r0 + e];
      const float4 s = *reinterpret_cast<const float4*>(p.scores + (r0 + e) * cap + j0);
      a[0] += ex2_approx(s.x - z);
      if (j0 + 1 < lim) a[1] += ex2_approx(s.y - z);
      if (j0 + 2 < lim) a[2] += ex2_approx(s.z - z);
      if (j0 + 3 < lim) a[3] += ex2_approx(s.w - z);
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (j0 + x >= q.len) break;
    int page, row;
    page_of(p.c, j0 + x, page, row);
    const int64_t pg = physical_page(p.c, p.c.table, p.c.table_stride, seq, page);
    if (pg >= 0) atomicAdd(&p.c.w[pg * p.c.w_sp + row * p.c.w_sn + head * p.c.w_sh], a[x]);
  }
}

template <typename T, int D>
cudaError_t launch_t(const PagedAttnParams& p, ssa_dtype dt, int grid, cudaStream_t st) {
  CUtensorMap km, vm;
  MapOrder mo, vo;
  if (!page_map(p.c, p.c.k, p.c.k_sp, p.c.k_sn, p.c.k_sh, dt, kKT, &km, &mo) ||
      !page_map(p.c, p.c.v, p.c.v_sp, p.c.v_sn, p.c.v_sh, dt, kKT, &vm, &vo) || mo.head_first != vo.head_first)
    return cudaErrorInvalidValue;
  auto kern = attn_dec_kernel<T, D>;
  static SmemOptIn opt_in;
  const cudaError_t e = opt_in(reinterpret_cast<const void*>(kern), Geo<D>::kSmem);
  if (e != cudaSuccess) return e;
  kern<<<grid, kThreads, Geo<D>::kSmem, st>>>(km, vm, p, mo);
  return cudaGetLastError();
}

}  // namespace pdec

cudaError_t launch_paged_attn_dec(const PagedAttnParams& p, ssa_dtype dt, int grid, cudaStream_t st) {
  if (dt == SSA_BF16)
    return p.c.d == 128 ? pdec::launch_t<__nv_bfloat16, 128>(p, dt, grid, st)
                        : pdec::launch_t<__nv_bfloat16, 64>(p, dt, grid, st);
  return p.c.d == 128 ? pdec::launch_t<__half, 128>(p, dt, grid, st) : pdec::launch_t<__half, 64>(p, dt, grid, st);
}

cudaError_t launch_paged_weights_dec(const PagedAttnParams& p, cudaStream_t st) {
  const int64_t slots = static_cast<int64_t>(p.c.max_pages) * p.c.page_size;
  if (slots == 0) return cudaSuccess;
  return launch_after(pdec::weights_dec_kernel, dim3(static_cast<unsigned>(cdiv(slots, 1024)), p.c.h_kv, p.c.batch),
                      dim3(256), 0, st, p);
}

}  // namespace ssa
