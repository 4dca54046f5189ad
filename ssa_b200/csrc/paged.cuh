// The paged key/value cache: parameter blocks, launchers, and the division of
// attention work over CTAs that its kernels share.  Internal.
//
// Attention work is a line of units.  An item is (sequence, KV head, tile of
// query rows): the g heads of a KV group at `tokens` consecutive new tokens
// are the rows of one tile.  Its units are the key tiles of KT slots its last
// row sees (one where it sees none, so that its zero rows are written), after
// `extra` units that stand for what an item costs besides its tiles (its query
// rows, its results, the pipeline's first and last steps): without them a CTA
// whose share is many short items would run long.
// Items follow one another by sequence, head, tile.  CTA c of G takes units
// [c W / G, (c + 1) W / G) of the W there are, whatever the lengths of the
// batch: ragged batches and long contexts of few rows spread evenly, with no
// plan made on the host.  An item cut by a CTA boundary leaves partial results
// (running maximum, sum, unnormalised rows) that are joined in CTA order, so
// results do not depend on timing (paged_join.cuh).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"

namespace ssa {

struct PagedCacheParams {
  const void* k; int64_t k_sp, k_sn, k_sh;
  const void* v; int64_t v_sp, v_sn, v_sh;
  float* w; int64_t w_sp, w_sn, w_sh;
  const int32_t* table; int64_t table_stride;
  const int32_t* kv_lens;
  int32_t* status;
  int64_t num_pages;
  int batch, max_pages, page_size, page_shift, h_kv, d;   // page_shift: log2(page_size), -1 if no power of two
};

struct PagedAppendParams {
  PagedCacheParams c;
  const int32_t* q_starts;
  const void* k_new; int64_t kn_sn, kn_sh;
  const void* v_new; int64_t vn_sn, vn_sh;
  int64_t rows;
};

// What a CTA leaves about the item its first unit belongs to.
struct PagedSplit {
  int64_t item_first;              // the item's first unit
  int64_t tok0;                    // row (of q) of the tile's first token
  int32_t head, rows;              // KV head, rows of the tile
  int32_t cta_first, cta_last;     // the CTAs that hold its first and its last unit
  int32_t valid;                   // 0: the CTA had no unit
};

struct PagedAttnParams {
  PagedCacheParams c;
  const int32_t* q_starts;
  const void* q; int64_t q_sn, q_sh;
  void* out; int64_t o_sn, o_sh;
  float* lse;                      // [rows, h_q] or NULL
  float* lse2;                     // [rows, h_q] row log2-sum-exp2 for the weights pass, or NULL
  float* part;                     // [grid][2][tile rows][d + 4]: unnormalised row, maximum (log2), sum, -
  PagedSplit* split;               // [grid]
  int32_t* counters;               // [grid], zero before and after a launch
  float* scores;                   // [rows, h_q, slots of a table row] scaled logits (base 2), or NULL
  int64_t rows;
  int group, causal;
  float inv_scale;
};

struct PagedEvictParams {
  PagedCacheParams c;
  const int32_t* new_table; int64_t new_table_stride;
  int32_t* kept;
  int32_t* new_lens;
  int new_max_pages, budget, recent;
};

// A run-time error word: plain stores, so that it may be mapped host memory, of
// the byte that the kind of error has to itself, so that none hides another.
__device__ __forceinline__ void paged_error(const PagedCacheParams& c, uint32_t bits) {
  static_assert(SSA_DEVICE_BAD_PAGE < 0x100 && SSA_DEVICE_TIMEOUT == 0x100 && SSA_DEVICE_BAD_LENGTH == 0x10000, "a byte each");
  const int at = bits >= 0x10000u ? 2 : bits >= 0x100u ? 1 : 0;
  if (c.status) reinterpret_cast<volatile uint8_t*>(c.status)[at] = static_cast<uint8_t>(bits >> (8 * at));
}

__device__ __forceinline__ void page_of(const PagedCacheParams& c, int slot, int& page, int& row) {
  if (c.page_shift >= 0) {
    page = slot >> c.page_shift;
    row = slot & (c.page_size - 1);
  } else {
    page = slot / c.page_size;
    row = slot - page * c.page_size;
  }
}

// Elements from row to row of the kept scores: the slots a table row holds, in
// whole 16-byte vectors.
__host__ __device__ inline int64_t score_stride(const PagedCacheParams& c) {
  return (static_cast<int64_t>(c.max_pages) * c.page_size + 3) / 4 * 4;
}

// Page of a slot below the sequence's length; -1 where the table is wrong.
__device__ __forceinline__ int64_t physical_page(const PagedCacheParams& c, const int32_t* table, int64_t stride,
                                                 int seq, int page) {
  const int32_t pg = table[static_cast<int64_t>(seq) * stride + page];
  if (pg < 0 || pg >= c.num_pages) {
    paged_error(c, SSA_DEVICE_BAD_PAGE);
    return -1;
  }
  return pg;
}

// The same without a branch, for loops that keep many loads in flight: page 0
// and `bad` where the table is wrong (paged_len lets no slot of an empty cache by).
__device__ __forceinline__ int64_t page_or_zero(const PagedCacheParams& c, const int32_t* table, int64_t stride,
                                                int seq, int page, bool& bad) {
  const int32_t pg = table[static_cast<int64_t>(seq) * stride + page];
  const bool ok = pg >= 0 && pg < c.num_pages;
  bad |= !ok;
  return ok ? pg : 0;
}

// New rows [q0, q0 + n) and length of a sequence; n = 0 where they are wrong.
struct PagedSeq {
  int64_t q0;
  int n, len;
};
__device__ __forceinline__ int paged_len(const PagedCacheParams& c, int s) {
  const int len = c.kv_lens[s];
  if (len < 0 || len > static_cast<int64_t>(c.max_pages) * c.page_size) {
    paged_error(c, SSA_DEVICE_BAD_LENGTH);
    return -1;
  }
  if (len > 0 && c.num_pages == 0) {
    paged_error(c, SSA_DEVICE_BAD_PAGE);
    return -1;
  }
  return len;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedCacheParams& c, const int32_t* q_starts, int64_t rows,
                                              int s) {
  const int q0 = q_starts[s], q1 = q_starts[s + 1];
  PagedSeq r;
  r.len = paged_len(c, s);
  if (q0 < 0 || q1 < q0 || q1 > rows) {
    paged_error(c, SSA_DEVICE_BAD_LENGTH);
    r.len = -1;
  }
  r.q0 = q0;
  r.n = r.len < 0 ? 0 : q1 - q0;
  return r;
}

// sum_{i < n} floor((a i + b) / m) for m > 0 and a n + b < 2^32: the lattice points
// under a line, whole parts taken out and the axes exchanged in turn as in Euclid's
// algorithm (the reciprocity of floor sums: Graham, Knuth, Patashnik, Concrete
// Mathematics, section 3.5; 32-bit divisions: every CTA starts with a few of these).
__host__ __device__ inline int64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  int64_t ans = 0;
  while (n > 0) {
    if (a >= m) {
      const uint32_t q = a / m;
      ans += static_cast<int64_t>(n) * (n - 1) / 2 * q;
      a -= q * m;
    }
    if (b >= m) {
      const uint32_t q = b / m;
      ans += static_cast<int64_t>(n) * q;
      b -= q * m;
    }
    const uint32_t y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y - n * m;
    const uint32_t t = m;
    m = a;
    a = t;
  }
  return ans;
}
// a * b / c, a * b mostly below 2^32
__host__ __device__ inline int64_t mul_div(int64_t a, int64_t b, int64_t c) {
  const int64_t x = a * b;
  return x < (1ll << 32) ? static_cast<uint32_t>(x) / static_cast<uint32_t>(c) : x / c;
}

// The tiles of one sequence: `tiles` of them, `tt` tokens each, and their units.
struct TileCosts {
  int n, len, tt, kt, more, causal, tiles;
  __host__ __device__ TileCosts(int n_, int len_, int tt_, int kt_, int extra, int causal_)
      : n(n_), len(len_), tt(tt_), kt(kt_), more(extra), causal(causal_), tiles(n_ > 0 ? static_cast<int>((static_cast<uint32_t>(n_) + tt_ - 1) / static_cast<uint32_t>(tt_)) : 0) {}
  // slots the tile's last row sees
  __host__ __device__ int seen(int r) const {
    if (!causal) return len;
    const int64_t last = static_cast<int64_t>(r + 1) * tt < n ? static_cast<int64_t>(r + 1) * tt : n;
    const int64_t e = static_cast<int64_t>(len) - n + last;
    return e > 0 ? static_cast<int>(e) : 0;
  }
  // its key tiles, and its units
  __host__ __device__ int key_tiles(int r) const {
    const int u = static_cast<int>((static_cast<uint32_t>(seen(r)) + kt - 1) / static_cast<uint32_t>(kt));
    return u > 0 ? u : 1;
  }
  __host__ __device__ int units(int r) const { return key_tiles(r) + more; }
  // units of tiles 0 .. r-1
  __host__ __device__ int64_t before(int r) const { return key_tiles_before(r) + static_cast<int64_t>(r) * more; }
  __host__ __device__ int64_t key_tiles_before(int r) const {
    if (!causal) return static_cast<int64_t>(r) * key_tiles(0);
    int64_t extra = 0;
    if (r == tiles && r > 0) {                 // the last tile may be short
      extra = key_tiles(r - 1);
      --r;
    }
    // tile i < tiles - 1 sees base + (i + 1) tt slots; one unit while that is at most kt
    const int base = len - n;
    int one = base >= kt ? 0 : static_cast<int>(static_cast<uint32_t>(kt - base) / static_cast<uint32_t>(tt));
    if (one > r) one = r;
    // sum_{i < m} floor((a i + b) / kt); kt is a constant power of two in every
    // kernel, so this first step of floor_sum has no division
    const uint32_t m = r - one, k = kt;
    uint32_t a = tt, b = static_cast<uint32_t>(base + (static_cast<int64_t>(one) + 1) * tt + kt - 1);
    if (m == 0) return extra + one;
    int64_t sum = extra + one + static_cast<int64_t>(m) * (m - 1) / 2 * (a / k) + static_cast<int64_t>(m) * (b / k);
    a %= k;
    b %= k;
    const uint32_t y = a * m + b;
    return sum + (a && y >= k ? floor_sum(y / k, a, k, y % k) : 0);
  }
};

// The same with the parts exchanged, for the slot weights: a tile is `kt` slots,
// its units the row tiles (of `tt` tokens) that hold a row that sees one of them.
struct SlotCosts {
  int n, len, tt, kt, more, causal, row_tiles, tiles;
  __host__ __device__ SlotCosts(int n_, int len_, int tt_, int kt_, int extra, int causal_)
      : n(n_), len(len_), tt(tt_), kt(kt_), more(extra), causal(causal_),
        row_tiles(static_cast<int>((static_cast<uint32_t>(n_) + tt_ - 1) / static_cast<uint32_t>(tt_))),
        tiles(n_ > 0 ? static_cast<int>((static_cast<uint32_t>(len_) + kt_ - 1) / static_cast<uint32_t>(kt_)) : 0) {}
  // first token that sees the tile (below n: the tile begins below len)
  __host__ __device__ int first_token(int i) const {
    const int64_t t = static_cast<int64_t>(i) * kt - (static_cast<int64_t>(len) - n);
    return causal && t > 0 ? static_cast<int>(t) : 0;
  }
  __host__ __device__ int first_row_tile(int i) const {
    return static_cast<int>(static_cast<uint32_t>(first_token(i)) / static_cast<uint32_t>(tt));
  }
  __host__ __device__ int units(int i) const { return row_tiles - first_row_tile(i) + more; }
  // units of tiles 0 .. i-1
  __host__ __device__ int64_t before(int i) const {
    const int64_t all = static_cast<int64_t>(i) * (row_tiles + more), old = static_cast<int64_t>(len) - n;
    if (!causal) return all;
    // tiles from `from` on miss floor((their first slot - old) / tt) row tiles
    const int from = old > 0 ? static_cast<int>((old + kt - 1) / kt) : 0;
    return i > from ? all - floor_sum(i - from, tt, kt, static_cast<uint32_t>(static_cast<int64_t>(from) * kt - old)) : all;
  }
};

// The tile that unit u (of a sequence's units of one head) lies in, and the
// units before it: a 32-way search by a full warp.
template <typename Costs>
__device__ inline int find_tile(const Costs& t, int64_t u, int64_t& first) {
  const int lane = threadIdx.x & 31;
  int lo = 0, width = t.tiles;                 // the tile is in [lo, lo + width)
  first = 0;
  while (width > 1) {
    const int step = (width + 31) / 32;
    const int64_t b = lane * step < width ? t.before(lo + lane * step) : u + 1;
    const int hit = 31 - __clz(__ballot_sync(0xffffffffu, b <= u));
    first = __shfl_sync(0xffffffffu, b, hit);
    width = min(step, lo + width - (lo + hit * step));
    lo += hit * step;
  }
  return lo;
}

// A CTA's walk over its units: the current item, and the unit in it.
struct PagedWalk {
  int64_t total, ctas;             // all units, and the CTAs that share them
  int64_t u, end;                  // next unit and the CTA's last + 1
  int64_t item_first;              // first unit of the current item
  int64_t q0;
  int seq, head, tile, n, len, units;   // units: of the current item
};

// Total units, and the walk of CTA `cta` of `grid`; little work is shared by
// fewer CTAs, of `least` units each.  Called by one full warp; every lane gets
// the result.  False: no work.
template <typename Costs = TileCosts>
__device__ inline bool paged_schedule(const PagedAttnParams& p, int tt, int kt, int extra, int least, int64_t cta, int64_t grid,
                                      PagedWalk& w) {
  const int lane = threadIdx.x & 31;
  const int hk = p.c.h_kv;
  // the first 32 sequences stay in registers for the second look
  PagedSeq q_first{0, 0, 0};
  int64_t mine = 0, cost_first = 0;
  for (int s = lane; s < p.c.batch; s += 32) {
    const PagedSeq q = paged_seq(p.c, p.q_starts, p.rows, s);
    const Costs t(q.n, q.len, tt, kt, extra, p.causal);
    const int64_t cost = t.before(t.tiles) * hk;
    if (s < 32) {
      q_first = q;
      cost_first = cost;
    }
    mine += cost;
  }
  int64_t total = mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const int64_t ctas = total >= grid * least ? grid : mul_div(total + least - 1, 1, least);
  w.total = total;
  w.ctas = ctas;
  if (cta >= ctas) return false;
  w.u = mul_div(cta, total, ctas);
  w.end = mul_div(cta + 1, total, ctas);
  // the sequence holding unit w.u: running totals over groups of 32 sequences
  int64_t base = 0;
  for (int s0 = 0;; s0 += 32) {
    const int s = s0 + lane;
    int64_t cost = s0 == 0 ? cost_first : 0;
    PagedSeq q = q_first;
    if (s0 > 0 && s < p.c.batch) {
      q = paged_seq(p.c, p.q_starts, p.rows, s);
      const Costs t(q.n, q.len, tt, kt, extra, p.causal);
      cost = t.before(t.tiles) * hk;
    }
    int64_t incl = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + incl > w.u);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int64_t first = base + incl - cost;
      first = __shfl_sync(0xffffffffu, first, src);
      w.seq = s0 + src;
      w.n = __shfl_sync(0xffffffffu, q.n, src);
      w.len = __shfl_sync(0xffffffffu, q.len, src);
      w.q0 = __shfl_sync(0xffffffffu, q.q0, src);
      const Costs t(w.n, w.len, tt, kt, extra, p.causal);
      const int64_t per = t.before(t.tiles), off = w.u - first;
      w.head = static_cast<int>(mul_div(off, 1, per));
      int64_t in_tiles;
      w.tile = find_tile(t, off - w.head * per, in_tiles);
      w.item_first = first + w.head * per + in_tiles;
      w.units = t.units(w.tile);
      return true;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
    if (s0 + 32 >= p.c.batch) return false;   // not reached: w.u < total
  }
}

// The item after the current one (w.u is its first unit).  Every lane of a
// warp, or a single thread, may call it: no exchange between lanes.
template <typename Costs = TileCosts>
__device__ inline void paged_next_item(const PagedAttnParams& p, int tt, int kt, int extra, PagedWalk& w) {
  w.item_first += w.units;
  Costs t(w.n, w.len, tt, kt, extra, p.causal);
  if (++w.tile >= t.tiles) {
    w.tile = 0;
    if (++w.head >= p.c.h_kv) {
      w.head = 0;
      do {
        if (++w.seq >= p.c.batch) return;
        const PagedSeq q = paged_seq(p.c, p.q_starts, p.rows, w.seq);
        w.n = q.n;
        w.len = q.len;
        w.q0 = q.q0;
        t = Costs(w.n, w.len, tt, kt, extra, p.causal);
      } while (t.tiles == 0);
    }
  }
  w.units = t.units(w.tile);
}

// The same for a whole CTA: warp 0 works it out, the others read it (after a
// __syncthreads that the caller makes in any case).
struct PagedStart {
  PagedWalk w;
  int any;
};
template <typename Costs = TileCosts>
__device__ inline void paged_start(const PagedAttnParams& p, int tt, int kt, int extra, int least, PagedStart* shared) {
  if (threadIdx.x < 32) {
    PagedWalk w{};
    const bool any = paged_schedule<Costs>(p, tt, kt, extra, least, blockIdx.x, gridDim.x, w);
    if (threadIdx.x == 0) {
      shared->w = w;
      shared->any = any;
    }
  }
}

// The CTA that holds unit u: the last c with floor(c W / G) <= u.
__device__ __forceinline__ int unit_cta(const PagedWalk& w, int64_t u) {
  const int64_t x = (u + 1) * w.ctas - 1;
  return static_cast<int>(x < (1ll << 32) ? static_cast<uint32_t>(x) / static_cast<uint32_t>(w.total) : x / w.total);
}
__device__ __forceinline__ PagedSplit paged_split(const PagedAttnParams& p, const PagedWalk& w, int tt, int extra) {
  const int tok0 = w.tile * tt;
  return PagedSplit{w.item_first, w.q0 + tok0, w.head, (w.n - tok0 < tt ? w.n - tok0 : tt) * p.group,
                    unit_cta(w, w.item_first + extra), unit_cta(w, w.item_first + w.units - 1), 1};
}
// The key tiles [first, last) of the current item that are this CTA's (none
// where its share holds only units of `extra`), and whether that is all of them.
struct PagedSegment {
  int first, last;
  bool whole;
};
__device__ __forceinline__ PagedSegment paged_segment(const PagedWalk& w, int extra) {
  const int64_t item_end = w.item_first + w.units, end = w.end < item_end ? w.end : item_end;
  const int64_t a = w.u - w.item_first - extra, b = end - w.item_first - extra;
  PagedSegment s;
  s.first = a > 0 ? static_cast<int>(a) : 0;
  s.last = b > 0 ? static_cast<int>(b) : 0;
  s.whole = s.first == 0 && end == item_end;
  return s;
}
// To the first unit past the current item; false if that is not this CTA's.
template <typename Costs = TileCosts>
__device__ __forceinline__ bool paged_advance(const PagedAttnParams& p, int tt, int kt, int extra, PagedWalk& w) {
  w.u = w.item_first + w.units;
  if (w.u >= w.end) return false;
  paged_next_item<Costs>(p, tt, kt, extra, w);
  return true;
}

__host__ __device__ inline int tile_tokens(int tile_rows, int group) { return tile_rows / group; }

// Allows a kernel its dynamic shared memory, once per device (one of these, static, per kernel).
class SmemOptIn {
 public:
  cudaError_t operator()(const void* kernel, size_t bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done_.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

// Launch of a kernel that follows another of the same op: its CTAs may be set
// up while the other drains, and wait (paged_after) before they read its results.
template <typename... KArgs, typename... Args>
cudaError_t launch_after(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}
// Everything the kernel launched before has written is visible after this.
__device__ __forceinline__ void paged_after() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

cudaError_t launch_paged_append(const PagedAppendParams& p, ssa_dtype dt, cudaStream_t st);
cudaError_t launch_paged_evict(const PagedEvictParams& p, ssa_dtype dt, cudaStream_t st);
// Attention (paged_attn.cu): picks the kernel, joins split items, adds slot weights.
size_t paged_attn_workspace(const PagedAttnParams& p, ssa_dtype dt);
cudaError_t launch_paged_attn(PagedAttnParams p, ssa_dtype dt, void* ws, cudaStream_t st);
// Chunks on the tensor cores (paged_attn_tc.cu), 256 rows an item, one CTA per SM.
cudaError_t launch_paged_attn_tc(const PagedAttnParams& p, ssa_dtype dt, int grid, cudaStream_t st);
// Few rows (paged_attn_dec.cu), 16 an item; the slot weights from the scores it
// leaves, and those of chunks from scores made again (paged_weights_tc.cu).
cudaError_t launch_paged_attn_dec(const PagedAttnParams& p, ssa_dtype dt, int grid, cudaStream_t st);
bool paged_weights_tc_supported(const PagedAttnParams& p, ssa_dtype dt);
cudaError_t launch_paged_weights_tc(const PagedAttnParams& p, ssa_dtype dt, cudaStream_t st);
cudaError_t launch_paged_weights_dec(const PagedAttnParams& p, cudaStream_t st);

}  // namespace ssa
