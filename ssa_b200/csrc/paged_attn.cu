// Attention over the paged cache on the CUDA cores: every type, head size up
// to 256 and page size, in fp32 throughout; the join of split items; and the
// slot weights.
//
//   s_ij = (q_i . k_j) / scale,  p_ij = exp(s_ij - m_i),  out_i = sum_j p_ij v_j / sum_j p_ij
//
// with the running maximum m_i and sum of the online softmax, in base 2
// (s * log2 e is folded into q when it is loaded).  One CTA holds a tile of R
// query rows (the g heads of a KV group at R / g consecutive tokens) and walks
// key tiles of 64 slots: 256 threads form a 16 x 16 grid, a thread owns R / 16
// rows and every 16th key (scores) or column quad (output).  A warp none of whose
// rows exists only loads: it would take its share of shared memory's bandwidth
// (16 tokens x 32 heads of 128 over 4000 slots, fp32: 325 us with it, 145 without,
// 3.6 TB/s).
//
// Tiles of 64 rows are bound by what shared memory returns: a step of four columns
// is 64 FMAs a thread, 16 clocks of the SM for every warp, and eight 16-byte loads, 32
// clocks.  fp32, 6 x 191 tokens x 28 heads of 128 over 4430 slots: 2.36 ms, 30
// TFLOP/s.  Small calls are bound by latency: 3 chunks of up to 129 tokens x 8 heads of
// 64 over up to 1500 slots take 29 us and 6 us for the join.
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "paged_join.cuh"
#include "paged_tma.cuh"

namespace ssa {
namespace {

constexpr int kKT = 64;            // slots per key tile
constexpr int kThreads = 256;
constexpr int kExtra = 1;          // units an item costs besides its tiles
constexpr int kLeast = 1;          // units a CTA takes at least

// Rows of the item's tile: row r is token tile * tt + r / g, head h * g + r % g.
struct TileRows {
  int tok0, rows;
};
__device__ __forceinline__ TileRows tile_rows(const PagedWalk& w, int tt, int group) {
  TileRows t;
  t.tok0 = w.tile * tt;
  t.rows = min(tt, w.n - t.tok0) * group;
  return t;
}
// Slots the row of token `tok` sees.
__device__ __forceinline__ int seen_slots(const PagedAttnParams& p, int n, int len, int tok) {
  return p.causal ? max(len - n + tok + 1, 0) : len;
}

template <typename T>
__device__ __forceinline__ void load_rows(const PagedAttnParams& p, int64_t q0, int head, const TileRows& t, int R,
                                          int stride, float* qs) {
  const int d = p.c.d, vecs = d / 8;
  const float c = p.inv_scale * kLog2e;
  for (int e = threadIdx.x; e < R * vecs; e += kThreads) {
    const int r = e / vecs, x = (e - r * vecs) * 8;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < t.rows) {
      const T* src = static_cast<const T*>(p.q) + (q0 + t.tok0 + r / p.group) * p.q_sn +
                     static_cast<int64_t>(head * p.group + r % p.group) * p.q_sh + x;
      load8<T>(src, f);
    }
    *reinterpret_cast<float4*>(qs + r * stride + x) = make_float4(f[0] * c, f[1] * c, f[2] * c, f[3] * c);
    *reinterpret_cast<float4*>(qs + r * stride + x + 4) = make_float4(f[4] * c, f[5] * c, f[6] * c, f[7] * c);
  }
}

// s[i][j] = q_{ty + 16 i} . k_{tx + 16 j}
template <int RI>
__device__ __forceinline__ void scores(const float* qs, const float* ks, int d, int stride, int tx, int ty,
                                       float (&s)[RI][4]) {
#pragma unroll
  for (int i = 0; i < RI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 2
  for (int x = 0; x < d; x += 4) {
    float4 a[RI], b[4];
#pragma unroll
    for (int i = 0; i < RI; ++i) a[i] = *reinterpret_cast<const float4*>(qs + (ty + 16 * i) * stride + x);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * stride + x);
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fmaf(a[i].x, b[j].x, s[i][j]);
        s[i][j] = fmaf(a[i].y, b[j].y, s[i][j]);
        s[i][j] = fmaf(a[i].z, b[j].z, s[i][j]);
        s[i][j] = fmaf(a[i].w, b[j].w, s[i][j]);
      }
  }
}

template <int R, int DP>
struct SimtGeo {
  static constexpr int QS = DP + 4, PS = kKT + 4;          // row strides: 16-byte rows on shifted banks
  // Q, a key tile, a value tile, P
  static constexpr size_t kSmem = sizeof(float) * (R * QS + 2 * kKT * QS + R * PS);
};

// This thread's row of a key tile (four threads a row): its element offsets in
// the pages, -1 past `lim` or where the page is bad.
struct RowOffsets {
  int64_t k, v;
};
__device__ __forceinline__ RowOffsets row_offsets(const PagedCacheParams& c, int seq, int head, int j, int lim) {
  RowOffsets o{-1, -1};
  if (j < lim) {
    int page, row;
    page_of(c, j, page, row);
    const int64_t pg = physical_page(c, c.table, c.table_stride, seq, page);
    if (pg >= 0) {
      o.k = pg * c.k_sp + row * c.k_sn + static_cast<int64_t>(head) * c.k_sh;
      o.v = pg * c.v_sp + row * c.v_sn + static_cast<int64_t>(head) * c.v_sh;
    }
  }
  return o;
}
// Its quarter of the row on the way to shared memory as fp32 (asynchronously
// where the cache is fp32); columns d .. dpad and rows without a slot are zero.
template <typename T>
__device__ __forceinline__ void bring_row(const void* base, int64_t off, int d, int dpad, float* dst) {
  for (int x = (threadIdx.x & 3) * 8; x < dpad; x += 32) {
    if (off < 0 || x >= d) {
      *reinterpret_cast<float4*>(dst + x) = make_float4(0.f, 0.f, 0.f, 0.f);
      *reinterpret_cast<float4*>(dst + x + 4) = make_float4(0.f, 0.f, 0.f, 0.f);
    } else if constexpr (sizeof(T) == 4) {
      const T* src = static_cast<const T*>(base) + off + x;
      const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst + x));
      cp_async16(to, src);
      cp_async16(to + 16, src + 4);
    } else {
      float f[8];
      load8<T>(static_cast<const T*>(base) + off + x, f);
      *reinterpret_cast<float4*>(dst + x) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(dst + x + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
}

template <typename T, int R, int DP>
__global__ void __launch_bounds__(kThreads) attn_simt_kernel(PagedAttnParams p) {
  using G = SimtGeo<R, DP>;
  constexpr int RI = R / 16, CI = DP / 64;
  extern __shared__ __align__(16) float smem[];
  float* qs = smem;
  float* ks = qs + R * G::QS;
  float* vs = ks + kKT * G::QS;
  float* ps = vs + kKT * G::QS;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int tt = tile_tokens(R, p.group), d = p.c.d;
  const int64_t cap = score_stride(p.c);
  __shared__ PagedStart start;
  __shared__ bool last_part;
  paged_start(p, tt, kKT, kExtra, kLeast, &start);
  __syncthreads();
  PagedWalk w = start.w;
  if (tid == 0) p.split[blockIdx.x] = start.any ? paged_split(p, w, tt, kExtra) : PagedSplit{};
  if (!start.any) return;
  float* const krow = ks + (tid >> 2) * G::QS;
  float* const vrow = vs + (tid >> 2) * G::QS;
  bool going = true;
  for (int slot = 0; going; slot = 1, going = paged_advance(p, tt, kKT, kExtra, w)) {
    const PagedSegment seg = paged_segment(w, kExtra);
    if (seg.first == seg.last) continue;
    const TileRows t = tile_rows(w, tt, p.group);
    const bool live = tid / kWarp * 2 < t.rows;                // the warp has a row (its first is row 2 * warp)
    const int tile_min = seen_slots(p, w.n, w.len, t.tok0);                              // every row sees these
    const int tile_max = seen_slots(p, w.n, w.len, t.tok0 + t.rows / p.group - 1);       // some row sees these
    __syncthreads();
    RowOffsets off = row_offsets(p.c, w.seq, w.head, seg.first * kKT + (tid >> 2), tile_max);
    bring_row<T>(p.c.k, off.k, d, d, krow);
    cp_commit();
    bring_row<T>(p.c.v, off.v, d, DP, vrow);
    cp_commit();
    load_rows<T>(p, w.q0, w.head, t, R, G::QS, qs);
    float m[RI], l[RI], o[RI][CI][4];
    int lim[RI];
    float* sc[RI];
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = ty + 16 * i;
      m[i] = -INFINITY;
      l[i] = 0.f;
      lim[i] = seen_slots(p, w.n, w.len, t.tok0 + min(r / p.group, tt - 1));
      sc[i] = p.scores && r < t.rows
                  ? p.scores + ((w.q0 + t.tok0 + r / p.group) * (static_cast<int64_t>(p.c.h_kv) * p.group) +
                                w.head * p.group + r % p.group) * cap : nullptr;
#pragma unroll
      for (int c = 0; c < CI; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
    }
    for (int kt = seg.first; kt < seg.last; ++kt) {
      const int k0 = kt * kKT;
      const bool more = kt + 1 < seg.last;
      // the next tile's page is looked up now, its keys come during this tile's
      // product and its values during the next tile's scores
      if (more) off = row_offsets(p.c, w.seq, w.head, k0 + kKT + (tid >> 2), tile_max);
      cp_wait<1>();                                          // the keys
      __syncthreads();
      float s[RI][4];
      if (live) scores<RI>(qs, ks, d, G::QS, tx, ty, s);
#pragma unroll
      for (int i = 0; live && i < RI; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = k0 + tx + 16 * j;
          if (sc[i] && at < cap) sc[i][at] = s[i][j];
          if (at >= lim[i]) s[i][j] = -INFINITY;
          mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int x = 8; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        const float mn = fmaxf(m[i], mx);
        const float base = mn == -INFINITY ? 0.f : mn;       // a row that has seen nothing: p = 0, no NaN
        const float r = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = exp2f(s[i][j] - base);
          sum += e;
          ps[(ty + 16 * i) * G::PS + tx + 16 * j] = e;
        }
        l[i] = l[i] * r + sum;                               // this thread's keys only; joined at the end
        m[i] = mn;
#pragma unroll
        for (int c = 0; c < CI; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][c][e] *= r;
      }
      cp_wait<0>();                                          // the values
      __syncthreads();
      if (more) bring_row<T>(p.c.k, off.k, d, d, krow);
      cp_commit();
      // a tile that some row does not see whole: if it holds a non-finite value,
      // hidden slots are left out one by one (0 * inf would be NaN)
      bool odd = false;
      if (k0 + kKT > tile_min) {
        for (int x = (tid & 3) * 8; x < d; x += 32)
#pragma unroll
          for (int e = 0; e < 8; ++e) odd |= !isfinite(vrow[x + e]);
        odd = __syncthreads_or(odd);
      }
      if (!live) {
        // nothing to add
      } else if (!odd) {
#pragma unroll 4
        for (int j = 0; j < kKT; j += 4) {
          float4 pr[RI];
#pragma unroll
          for (int i = 0; i < RI; ++i) pr[i] = *reinterpret_cast<const float4*>(ps + (ty + 16 * i) * G::PS + j);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int c = 0; c < CI; ++c) {
              const float4 v = *reinterpret_cast<const float4*>(vs + (j + jj) * G::QS + 64 * c + 4 * tx);
#pragma unroll
              for (int i = 0; i < RI; ++i) {
                const float e = jj == 0 ? pr[i].x : jj == 1 ? pr[i].y : jj == 2 ? pr[i].z : pr[i].w;
                o[i][c][0] = fmaf(e, v.x, o[i][c][0]);
                o[i][c][1] = fmaf(e, v.y, o[i][c][1]);
                o[i][c][2] = fmaf(e, v.z, o[i][c][2]);
                o[i][c][3] = fmaf(e, v.w, o[i][c][3]);
              }
            }
        }
      } else {
        for (int j = 0; j < kKT; ++j)
#pragma unroll
          for (int c = 0; c < CI; ++c) {
            const float4 v = *reinterpret_cast<const float4*>(vs + j * G::QS + 64 * c + 4 * tx);
#pragma unroll
            for (int i = 0; i < RI; ++i) {
              const float e = ps[(ty + 16 * i) * G::PS + j];
              if (k0 + j < lim[i]) {
                o[i][c][0] = fmaf(e, v.x, o[i][c][0]);
                o[i][c][1] = fmaf(e, v.y, o[i][c][1]);
                o[i][c][2] = fmaf(e, v.z, o[i][c][2]);
                o[i][c][3] = fmaf(e, v.w, o[i][c][3]);
              }
            }
          }
      }
      __syncthreads();
      if (more) bring_row<T>(p.c.v, off.v, d, DP, vrow);
      cp_commit();
    }
    const int64_t one = static_cast<int64_t>(R) * (d + 4);
#pragma unroll
    for (int i = 0; i < RI; ++i) {
#pragma unroll
      for (int x = 8; x; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
      const int r = ty + 16 * i;
      if (r >= t.rows) continue;
      if (seg.whole) {
        const int64_t tok = w.q0 + t.tok0 + r / p.group;
        const int head = w.head * p.group + r % p.group;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        T* dst = static_cast<T*>(p.out) + tok * p.o_sn + static_cast<int64_t>(head) * p.o_sh;
#pragma unroll
        for (int c = 0; c < CI; ++c)
          if (64 * c + 4 * tx < d)
            store4(dst + 64 * c + 4 * tx, make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]), inv);
        if (tx == 0) store_lse(p, tok, head, m[i], l[i]);
      } else {
        float* dst = p.part + (blockIdx.x * 2 + slot) * one + r * (d + 4);
#pragma unroll
        for (int c = 0; c < CI; ++c)
          if (64 * c + 4 * tx < d)
            *reinterpret_cast<float4*>(dst + 64 * c + 4 * tx) =
                make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
        if (tx == 0) {
          dst[d] = m[i];
          dst[d + 1] = l[i];
        }
      }
    }
    if (R == 16 && !seg.whole) {
      // few rows: the last of the item's CTAs joins it, a warp per row
      const int a = unit_cta(w, w.item_first + kExtra), parts = unit_cta(w, w.item_first + w.units - 1) - a + 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        last_part = atomicAdd(p.counters + a, 1) == parts - 1;
        if (last_part) p.counters[a] = 0;
      }
      __syncthreads();
      if (last_part) {
        __threadfence();
        // the item is the second of CTA a's two parts if a's share starts before it
        const int second = mul_div(a, w.total, w.ctas) < w.item_first ? 1 : 0;
        const float* first = p.part + 2 * static_cast<int64_t>(a) * one;
        for (int r = tid / kWarp; r < t.rows; r += kThreads / kWarp)
          write_joined<T, 8>(p, [&](int i) { return first + (2 * i + (i == 0 ? second : 0)) * one + r * (d + 4); },
                             parts, w.q0 + t.tok0, w.head, r);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// join of the items cut by CTA boundaries.  Block b looks at the boundary
// before CTA b + 1: if it is the first one inside its item, the blocks (b, y) join
// the item's rows, a warp per row, over the CTAs that hold parts of it, in CTA
// order, in one pass with a running maximum.  A matter of latency: everything
// it needs to find its rows is in the two split records, and the parts of a
// row are loaded four at a time.  Up to 147 boundaries of 256 rows of 528 bytes, twice:
// 17 us with a cold L2 after the chunks of 2 x 1024 tokens over 8192 slots.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(PagedAttnParams p, int R) {
  paged_after();
  const int b = blockIdx.x + 1;
  const PagedSplit it = p.split[b];
  const int64_t before = p.split[b - 1].item_first;
  // the item starts before this CTA, and in the CTA before it
  if (!it.valid || it.cta_first != b - 1) return;
  const int pd = p.c.d + 4, parts = it.cta_last - b + 2;            // CTAs b - 1 .. cta_last
  const int slot0 = before == it.item_first ? 0 : 1;                // CTA b - 1: is it also that CTA's first item
  const int64_t one = static_cast<int64_t>(R) * pd;
  const float* first = p.part + static_cast<int64_t>(b - 1) * 2 * one;
  const int warps = blockDim.x / kWarp;
  for (int r = blockIdx.y * warps + threadIdx.x / kWarp; r < it.rows; r += gridDim.y * warps)
    write_joined<T, 4>(p, [&](int i) { return first + (2 * i + (i == 0 ? slot0 : 0)) * one + r * pd; }, parts, it.tok0,
                       it.head, r);
}

// ---------------------------------------------------------------------------
// slot weights: w_j += sum over the rows i of the group that see j of
// exp2(s_ij - lse2_i).  One CTA per (64 slots, KV head, sequence) walks the row
// tiles that see its slots; every slot is added to once per call, so without
// shared pages the sums do not depend on timing.
// ---------------------------------------------------------------------------
template <typename T, int R, int DP>
__global__ void __launch_bounds__(kThreads) weights_simt_kernel(PagedAttnParams p) {
  paged_after();
  using G = SimtGeo<R, DP>;
  constexpr int RI = R / 16;
  extern __shared__ __align__(16) float smem[];
  float* qs = smem;
  float* ks = qs + R * G::QS;
  float* ps = ks + 2 * kKT * G::QS;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int seq = blockIdx.z, head = blockIdx.y, k0 = blockIdx.x * kKT;
  const int tt = tile_tokens(R, p.group), d = p.c.d;
  const PagedSeq q = paged_seq(p.c, p.q_starts, p.rows, seq);
  if (q.n == 0 || k0 >= q.len) return;
  bring_row<T>(p.c.k, row_offsets(p.c, seq, head, k0 + (tid >> 2), q.len).k, d, d, ks + (tid >> 2) * G::QS);
  cp_commit();
  cp_wait<0>();
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < q.n; t0 += tt) {
    const TileRows t{t0, min(tt, q.n - t0) * p.group};
    if (seen_slots(p, q.n, q.len, t0 + t.rows / p.group - 1) <= k0) continue;
    __syncthreads();
    load_rows<T>(p, q.q0, head, t, R, G::QS, qs);
    __syncthreads();
    float s[RI][4];
    scores<RI>(qs, ks, d, G::QS, tx, ty, s);
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = ty + 16 * i;
      if (r >= t.rows) continue;
      const int lim = seen_slots(p, q.n, q.len, t0 + r / p.group);
      const float z = p.lse2[(q.q0 + t0 + r / p.group) * (static_cast<int64_t>(p.c.h_kv) * p.group) +
                             head * p.group + r % p.group];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k0 + tx + 16 * j < lim) sum[j] += exp2f(s[i][j] - z);
    }
  }
  // over the 16 row groups of the CTA, in a fixed order
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) ps[ty * G::PS + tx + 16 * j] = sum[j];
  __syncthreads();
  if (tid < kKT && k0 + tid < q.len) {
    float a = 0.f;
    for (int y = 0; y < 16; ++y) a += ps[y * G::PS + tid];
    int page, row;
    page_of(p.c, k0 + tid, page, row);
    const int64_t pg = physical_page(p.c, p.c.table, p.c.table_stride, seq, page);
    if (pg >= 0) atomicAdd(&p.c.w[pg * p.c.w_sp + row * p.c.w_sn + head * p.c.w_sh], a);
  }
}

// Runs f(type tag, head size class) for the call's type and head size.
template <typename F>
cudaError_t by_type_and_size(const PagedAttnParams& p, ssa_dtype dt, F&& f) {
  auto sized = [&](auto zero) {
    if (p.c.d <= 64) return f(zero, std::integral_constant<int, 64>{});
    if (p.c.d <= 128) return f(zero, std::integral_constant<int, 128>{});
    return f(zero, std::integral_constant<int, 256>{});
  };
  if (dt == SSA_F32) return sized(float{});
  if (dt == SSA_BF16) return sized(__nv_bfloat16{});
  return sized(__half{});
}

template <int R>
cudaError_t launch_simt(const PagedAttnParams& p, ssa_dtype dt, int grid, cudaStream_t st) {
  return by_type_and_size(p, dt, [&](auto zero, auto size) {
    using T = decltype(zero);
    constexpr int DP = decltype(size)::value;
    auto kern = attn_simt_kernel<T, R, DP>;
    static SmemOptIn opt_in;
    const cudaError_t e = opt_in(reinterpret_cast<const void*>(kern), SimtGeo<R, DP>::kSmem);
    if (e != cudaSuccess) return e;
    kern<<<grid, kThreads, SimtGeo<R, DP>::kSmem, st>>>(p);
    return cudaGetLastError();
  });
}

cudaError_t launch_weights_simt(const PagedAttnParams& p, ssa_dtype dt, cudaStream_t st) {
  const int64_t slots = static_cast<int64_t>(p.c.max_pages) * p.c.page_size;
  if (slots == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>(cdiv(slots, kKT)), p.c.h_kv, p.c.batch);
  return by_type_and_size(p, dt, [&](auto zero, auto size) {
    using T = decltype(zero);
    constexpr int DP = decltype(size)::value;
    auto kern = weights_simt_kernel<T, 64, DP>;
    static SmemOptIn opt_in;
    const cudaError_t e = opt_in(reinterpret_cast<const void*>(kern), SimtGeo<64, DP>::kSmem);
    if (e != cudaSuccess) return e;
    return launch_after(kern, grid, dim3(kThreads), SimtGeo<64, DP>::kSmem, st, p);
  });
}

// CTAs of the CUDA-core kernel that an SM's shared memory holds, two at most (a
// share of the work for more than are resident cost 3% to 6%).
int simt_resident(int rows, int d) {
  auto bytes = [&](auto size) {
    constexpr int DP = decltype(size)::value;
    return rows == 64 ? SimtGeo<64, DP>::kSmem : rows == 32 ? SimtGeo<32, DP>::kSmem : SimtGeo<16, DP>::kSmem;
  };
  const size_t one = d <= 64 ? bytes(std::integral_constant<int, 64>{})
                     : d <= 128 ? bytes(std::integral_constant<int, 128>{}) : bytes(std::integral_constant<int, 256>{});
  return 2 * (one + 2048) <= 228 * 1024 ? 2 : 1;       // with what a CTA takes besides
}

// Kept scores take as much as the table could hold, whatever is filled: with wide
// tables (131072 slots, 32 heads: 17 MB a row) more than a serving cache leaves free.
// Beyond this they are made again for the weights, which takes twice the time of
// the call (32 tokens x 32 heads over 8192 slots: 195 us kept, 418 made again).
constexpr size_t kMostScores = static_cast<size_t>(4) << 30;

// The kernel that serves a call, its tile rows and grid, and the workspace.
enum class AttnKernel { kSimt, kTokens, kChunks };
struct AttnPlan {
  AttnKernel kernel;
  int rows, grid;
  size_t part, split, lse2, scores, total;
};

// More than 16 rows (new tokens x heads of a group) per sequence on average
// take tiles of many rows; 16-bit caches that page tiles fit, the tensor cores
// (24 x 5 tokens over 8000 slots, four heads a group: 167 us, and 249 with tiles of
// 16 rows; one such sequence over 2000: 18.0 and 15.8).  Both are measured for equal
// sequences: many single tokens beside one chunk may take either.
// On the CUDA cores a tile costs its rows whether they are used or not, and a
// row of a 32-row tile about 5/4 of one of a 64-row tile.
AttnPlan attn_plan(const PagedAttnParams& p, ssa_dtype dt) {
  AttnPlan a{};
  if (p.rows == 0 || p.c.batch == 0) {       // nothing is launched: the zeroed head alone
    a.total = SSA_PAGED_ZEROED;
    return a;
  }
  const bool chunks = p.rows * p.group > 16ll * p.c.batch;
  a.kernel = !page_tiles_supported(p, dt) ? AttnKernel::kSimt : chunks ? AttnKernel::kChunks : AttnKernel::kTokens;
  const int64_t mean = (p.rows * p.group + p.c.batch - 1) / p.c.batch, padded64 = (mean + 63) / 64 * 64,
                padded32 = (mean + 31) / 32 * 32;
  a.rows = !chunks ? 16 : a.kernel == AttnKernel::kChunks ? 256 : 4 * padded64 <= 5 * padded32 ? 64 : 32;
  a.grid = a.kernel == AttnKernel::kSimt ? 148 * simt_resident(a.rows, p.c.d) : 148;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t lines = static_cast<size_t>(p.rows) * p.c.h_kv * p.group;
  a.part = SSA_PAGED_ZEROED;                 // after the counters, whose place never changes
  a.split = a.part + up(static_cast<size_t>(a.grid) * 2 * a.rows * (p.c.d + 4) * 4);
  a.lse2 = a.split + up(a.grid * sizeof(PagedSplit));
  a.scores = a.lse2 + (p.c.w ? up(lines * 4) : 0);
  a.total = a.scores;
  if (p.c.w && a.rows == 16) {
    const size_t bytes = lines * score_stride(p.c) * 4;
    if (bytes <= kMostScores) a.total += up(bytes);
  }
  return a;
}

}  // namespace

size_t paged_attn_workspace(const PagedAttnParams& p, ssa_dtype dt) { return attn_plan(p, dt).total; }

cudaError_t launch_paged_attn(PagedAttnParams p, ssa_dtype dt, void* ws, cudaStream_t st) {
  const AttnPlan a = attn_plan(p, dt);
  char* at = static_cast<char*>(ws);
  p.counters = reinterpret_cast<int32_t*>(at);
  p.part = reinterpret_cast<float*>(at + a.part);
  p.split = reinterpret_cast<PagedSplit*>(at + a.split);
  p.lse2 = p.c.w ? reinterpret_cast<float*>(at + a.lse2) : nullptr;
  p.scores = a.total > a.scores ? reinterpret_cast<float*>(at + a.scores) : nullptr;
  cudaError_t e;
  switch (a.kernel) {
    case AttnKernel::kChunks: e = launch_paged_attn_tc(p, dt, a.grid, st); break;
    case AttnKernel::kTokens: e = launch_paged_attn_dec(p, dt, a.grid, st); break;
    default:
      e = a.rows == 64   ? launch_simt<64>(p, dt, a.grid, st)
          : a.rows == 32 ? launch_simt<32>(p, dt, a.grid, st)
                         : launch_simt<16>(p, dt, a.grid, st);
  }
  if (e != cudaSuccess) return e;
  if (a.rows > 16) {
    // one wave of blocks, a row or four for every warp
    const dim3 grid(a.grid - 1, 8);
    switch (dt) {
      case SSA_F32: e = launch_after(combine_kernel<float>, grid, dim3(256), 0, st, p, a.rows); break;
      case SSA_BF16: e = launch_after(combine_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p, a.rows); break;
      default: e = launch_after(combine_kernel<__half>, grid, dim3(256), 0, st, p, a.rows); break;
    }
  }
  if (e != cudaSuccess || !p.c.w) return e;
  if (p.scores) return launch_paged_weights_dec(p, st);
  if (a.kernel != AttnKernel::kSimt && paged_weights_tc_supported(p, dt)) return launch_paged_weights_tc(p, dt, st);
  return launch_weights_simt(p, dt, st);
}

}  // namespace ssa
