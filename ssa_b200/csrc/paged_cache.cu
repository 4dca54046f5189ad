// The paged cache's writes: new rows appended to their slots, and eviction.
#include "common.cuh"
#include "paged.cuh"

namespace ssa {
namespace {

// ---------------------------------------------------------------------------
// append: slot (kv_len - n + i) of sequence s <- row q_starts[s] + i.
// Pure data movement, 2 * h_kv * d elements in and out per row.  A block takes
// `per_block` rows: a thread each first finds where they go (the sequence by
// bisection of q_starts, then its length and page: five loads in a row), then
// all threads move 16-byte pieces of K and V, four of each in flight.  (With the
// look-ups made by every thread for its own piece, 75 MB took 16.8 us, now 15.7:
// 4.8 TB/s; 268 MB take 42.5 us, 6.3 TB/s.)
// ---------------------------------------------------------------------------
constexpr int kAppendRows = 64;            // rows of a block at most
__global__ void __launch_bounds__(256) append_kernel(PagedAppendParams p, int elem, int vecs, int per_block) {
  const PagedCacheParams& c = p.c;
  __shared__ int64_t to_k[kAppendRows], to_v[kAppendRows], to_w[kAppendRows];   // element offsets; to_k -1: no place
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * per_block;
  const int rows = static_cast<int>(p.rows - t0 < per_block ? p.rows - t0 : per_block);
  if (static_cast<int>(threadIdx.x) < rows) {
    const int64_t t = t0 + threadIdx.x;
    int lo = 0, hi = c.batch;                       // last s with q_starts[s] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.q_starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    const PagedSeq q = paged_seq(c, p.q_starts, p.rows, lo);
    int64_t k_at = -1, v_at = 0, w_at = 0;
    if (t >= q.q0 && t < q.q0 + q.n) {              // else a skipped sequence, or a row of none
      if (q.n > q.len) {                            // more rows than the sequence holds: none of them is written
        paged_error(c, SSA_DEVICE_BAD_LENGTH);
      } else {
        int page, row;
        page_of(c, q.len - q.n + static_cast<int>(t - q.q0), page, row);
        const int64_t pg = physical_page(c, c.table, c.table_stride, lo, page);
        if (pg >= 0) {
          k_at = pg * c.k_sp + row * c.k_sn;
          v_at = pg * c.v_sp + row * c.v_sn;
          w_at = pg * c.w_sp + row * c.w_sn;
        }
      }
    }
    to_k[threadIdx.x] = k_at;
    to_v[threadIdx.x] = v_at;
    to_w[threadIdx.x] = w_at;
  }
  __syncthreads();
  const uint32_t pieces = static_cast<uint32_t>(c.h_kv) * vecs, total = rows * pieces, one = 16 / elem;
  for (uint32_t e0 = threadIdx.x; e0 < total; e0 += 4 * 256) {
    uint4 kx[4], vx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t e = e0 + i * 256 < total ? e0 + i * 256 : e0, r = e / pieces, x = e - r * pieces;
      const uint32_t h = x / static_cast<uint32_t>(vecs), piece = (x - h * vecs) * one;
      kx[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(p.k_new) +
                                                   ((t0 + r) * p.kn_sn + h * p.kn_sh + piece) * elem));
      vx[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(p.v_new) +
                                                   ((t0 + r) * p.vn_sn + h * p.vn_sh + piece) * elem));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t e = e0 + i * 256;
      if (e >= total) break;
      const uint32_t r = e / pieces, x = e - r * pieces, h = x / static_cast<uint32_t>(vecs), piece = (x - h * vecs) * one;
      if (to_k[r] < 0) continue;
      *reinterpret_cast<uint4*>(static_cast<char*>(const_cast<void*>(c.k)) + (to_k[r] + h * c.k_sh + piece) * elem) = kx[i];
      *reinterpret_cast<uint4*>(static_cast<char*>(const_cast<void*>(c.v)) + (to_v[r] + h * c.v_sh + piece) * elem) = vx[i];
      if (c.w && piece == 0) c.w[to_w[r] + h * c.w_sh] = 0.f;
    }
  }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
// Order-preserving key of a weight; NaN ranks with -inf, below every number.
__device__ __forceinline__ uint32_t weight_key(float w) { return float_key(w != w ? -INFINITY : w); }

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kSelBins = 2048;
constexpr int kSelLoads = 8;       // weights in flight a thread, one by one ...
constexpr int kSelQuads = 4;       // ... and by vectors of four
constexpr int kSelCopies = 4;      // counters of a digit, by lane: equal digits of a warp queue less
constexpr int kSelKeys = 49152;    // keys held in shared memory (192 KB); longer sequences are read again

// The part of the selection that reads keys.  Held: they fit in shared memory;
// Quads: the weights of four slots lie in one aligned vector.
template <bool Held, bool Quads, typename ReadKey, typename ReadQuad>
__device__ __forceinline__ void select_slots(uint32_t* sel_keys, const ReadKey& read_key, const ReadQuad& read_quad, int* hist, int (*wsum)[2],
                                             int* found, int32_t* kept, int len, int older, int n_keep) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto key_of = [&](int j) -> uint32_t { return Held ? sel_keys[j] : read_key(j); };
  uint32_t prefix = 0, known = 0;          // the bits of T found so far, and which
  int left = n_keep;                       // of the keys that agree with them, how many are kept
  // counts a digit of each lane's key (bin -1: none).  Equal weights (a cache's
  // first steps) would queue 32 deep on one counter.
  auto count = [&](int bin) {
    const int one = __shfl_sync(0xffffffffu, bin, 0);
    if (one >= 0 && __all_sync(0xffffffffu, bin == one)) {
      if (lane == 0) atomicAdd(&hist[bin * kSelCopies], 32);
    } else if (bin >= 0) {
      atomicAdd(&hist[bin * kSelCopies + (lane & (kSelCopies - 1))], 1);
    }
  };
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int b = tid; b < kSelBins; b += kSelThreads) reinterpret_cast<int4*>(hist)[b] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (pass == 0 && Quads) {
      // four consecutive slots of a page a load
      for (int j0 = 4 * tid; j0 - 4 * lane < older; j0 += 4 * kSelQuads * kSelThreads) {
        uint4 k[kSelQuads];
#pragma unroll
        for (int e = 0; e < kSelQuads; ++e) k[e] = read_quad(min(j0 + 4 * e * kSelThreads, (older - 1) & ~3));
#pragma unroll
        for (int e = 0; e < kSelQuads; ++e) {
          const int j = j0 + 4 * e * kSelThreads;
          if (j - 4 * lane >= older) break;
          const uint32_t q[4] = {k[e].x, k[e].y, k[e].z, k[e].w};
          if (Held && j < older) *reinterpret_cast<uint4*>(sel_keys + j) = k[e];
#pragma unroll
          for (int x = 0; x < 4; ++x) count(j + x < older ? static_cast<int>(q[x] >> 21) : -1);
        }
      }
    } else if (pass == 0) {
      for (int j0 = tid; j0 - lane < older; j0 += kSelLoads * kSelThreads) {
        uint32_t k[kSelLoads];
#pragma unroll
        for (int e = 0; e < kSelLoads; ++e) k[e] = read_key(min(j0 + e * kSelThreads, older - 1));
#pragma unroll
        for (int e = 0; e < kSelLoads; ++e) {
          const int j = j0 + e * kSelThreads;
          if (Held && j < older) sel_keys[j] = k[e];
          if (j - lane < older) count(j < older ? static_cast<int>(k[e] >> 21) : -1);
        }
      }
    } else {
#pragma unroll 4
      for (int j = tid; j - lane < older; j += kSelThreads) {
        const uint32_t k = j < older ? key_of(j) : 0u;
        const bool in = j < older && (k & known) == prefix;
        if (__any_sync(0xffffffffu, in)) count(in ? static_cast<int>((k >> shift) & (bins - 1)) : -1);
      }
    }
    if (n_keep == 0) break;
    __syncthreads();
    // the largest digit b with (keys of digits >= b) >= left: a thread has two
    // digits, from the top
    const int b0 = kSelBins - 1 - 2 * tid;
    const int4 h0 = reinterpret_cast<const int4*>(hist)[b0], h1 = reinterpret_cast<const int4*>(hist)[b0 - 1];
    const int c0 = h0.x + h0.y + h0.z + h0.w, c1 = h1.x + h1.y + h1.z + h1.w;
    int incl = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) wsum[warp][0] = incl;
    __syncthreads();
    const int above = incl - c0 - c1 + __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane][0] : 0);
    if (above < left && left <= above + c0 + c1) {
      const bool first = left <= above + c0;
      found[0] = first ? b0 : b0 - 1;
      found[1] = first ? left - above : left - above - c0;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found[0]) << shift;
    known |= static_cast<uint32_t>(bins - 1) << shift;
    left = found[1];
  }
  __syncthreads();
  if (n_keep == 0) prefix = 0xffffffffu;   // no key exceeds it, and none that equals it is kept
  // each warp's run of slots: kept if above T, if among the first `left` equal to T, or recent
  const int run = ((len + kSelWarps - 1) / kSelWarps + 31) / 32 * 32, lo = warp * run, hi = min(lo + run, len);
  auto kind = [&](int j, bool& gt, bool& eq) {
    const uint32_t k = j < older ? key_of(j) : 0u;
    gt = j < hi && (j >= older || k > prefix);
    eq = j < hi && j < older && k == prefix;
  };
  int ng = 0, ne = 0;
#pragma unroll 4
  for (int j = lo + lane; j - lane < hi; j += 32) {
    bool gt, eq;
    kind(j, gt, eq);
    ng += gt;
    ne += eq;
  }
  ng = __reduce_add_sync(0xffffffffu, ng);
  ne = __reduce_add_sync(0xffffffffu, ne);
  if (lane == 0) {
    wsum[warp][0] = ng;
    wsum[warp][1] = ne;
  }
  __syncthreads();
  // slots above T, and equal to it, before this warp's run
  int out = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane][0] : 0);
  int equal = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane][1] : 0);
  const unsigned below = (1u << lane) - 1u;
#pragma unroll 4
  for (int j = lo + lane; j - lane < hi; j += 32) {
    bool gt, eq;
    kind(j, gt, eq);
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    const int g0 = out + __popc(bg & below), e0 = equal + __popc(be & below);
    if (gt) kept[g0 + min(e0, left)] = j;
    else if (eq && e0 < left) kept[g0 + e0] = j;
    out += __popc(bg);
    equal += __popc(be);
  }
}

// One CTA per (sequence, KV head).  The n_keep heaviest of the first `older`
// slots are those whose key exceeds the n_keep-th largest, T, and the first
// few that equal it.  The weights are read once into shared memory,
// several loads in flight a thread; T is found from its top bits down in three passes
// of 11, 11 and 10 bits, each counting the next digit of the keys that agree
// with T so far and finding the digit by a sum from the top over the 2048
// counts; then every warp counts and writes the kept slots of its own run of
// slots, in order.  Bound by latency, a dozen block-wide steps: 12.6 us for 64 lists
// of 4352 slots, 32 us for 128 of up to 32768.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(PagedEvictParams p, int held, int quads) {
  asm volatile("griddepcontrol.launch_dependents;");   // the copies of slots that are kept in any case
  const PagedCacheParams& c = p.c;
  const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  extern __shared__ __align__(16) uint32_t sel_keys[];
  __shared__ __align__(16) int hist[kSelBins * kSelCopies];
  __shared__ int wsum[kSelWarps][2];
  __shared__ int found[2];
  const int len = max(paged_len(c, s), 0);
  const int size = min(len, p.budget), recent = min(p.recent, size), older = len - recent, n_keep = size - recent;
  int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.h_kv + h) * p.budget;
  if (tid == 0 && h == 0) p.new_lens[s] = size;
  for (int j = size + tid; j < p.budget; j += kSelThreads) kept[j] = -1;
  if (size == len) {
    for (int j = tid; j < len; j += kSelThreads) kept[j] = j;
    return;
  }
  bool bad = false;
  auto read_key = [&](int j) -> uint32_t {
    int page, row;
    page_of(c, j, page, row);
    const int64_t pg = page_or_zero(c, c.table, c.table_stride, s, page, bad);
    return weight_key(__ldg(c.w + pg * c.w_sp + row * c.w_sn + h * c.w_sh));
  };
  auto read_quad = [&](int j) -> uint4 {
    int page, row;
    page_of(c, j, page, row);
    const int64_t pg = page_or_zero(c, c.table, c.table_stride, s, page, bad);
    const float4 w = __ldg(reinterpret_cast<const float4*>(c.w + pg * c.w_sp + row + h * c.w_sh));
    return make_uint4(weight_key(w.x), weight_key(w.y), weight_key(w.z), weight_key(w.w));
  };
  if (older > held) select_slots<false, false>(sel_keys, read_key, read_quad, hist, wsum, found, kept, len, older, n_keep);
  else if (quads) select_slots<true, true>(sel_keys, read_key, read_quad, hist, wsum, found, kept, len, older, n_keep);
  else select_slots<true, false>(sel_keys, read_key, read_quad, hist, wsum, found, kept, len, older, n_keep);
  if (bad) paged_error(c, SSA_DEVICE_BAD_PAGE);
}

// Kept slots' keys, values and weights to the new pages, a 16-byte piece of K
// and of V per thread and step.  The recent slots (all, where none is evicted)
// need no selection: their copies go on next to it.  (Two or four slots a thread in flight were
// slower: the resident threads are in flight enough.)  8 x 8 lists of 4096 slots of
// 256 + 256 bytes in and out: 48 us, 5.6 TB/s.
__global__ void __launch_bounds__(256) evict_copy_kernel(PagedEvictParams p, int elem, int vecs) {
  const PagedCacheParams& c = p.c;
  const int s = blockIdx.z, h = blockIdx.y;
  const int len = max(paged_len(c, s), 0), size = min(len, p.budget);
  // slots from `sure` on are kept whatever the weights are; slot `to` of them was slot to + len - size
  const int sure = size == len ? 0 : size - p.recent;
  const int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.h_kv + h) * p.budget;
  const int per = 256 / vecs, lane_slot = threadIdx.x / vecs, piece = threadIdx.x - lane_slot * vecs;
  const char* k = static_cast<const char*>(c.k);
  const char* v = static_cast<const char*>(c.v);
  bool bad = false, short_table = false;
  auto copy = [&](int to, int from) {
    int page, row, npage, nrow;
    page_of(c, from, page, row);
    page_of(c, to, npage, nrow);
    if (npage >= p.new_max_pages) {
      short_table = true;
      return;
    }
    bool miss = false;
    const int64_t pg = page_or_zero(c, c.table, c.table_stride, s, page, miss);
    const int64_t ng = page_or_zero(c, p.new_table, p.new_table_stride, s, npage, miss);
    bad |= miss;
    if (miss) return;
    const uint4 kx = reinterpret_cast<const uint4*>(k + (pg * c.k_sp + row * c.k_sn + h * c.k_sh) * elem)[piece];
    const uint4 vx = reinterpret_cast<const uint4*>(v + (pg * c.v_sp + row * c.v_sn + h * c.v_sh) * elem)[piece];
    const float wx = piece == 0 ? c.w[pg * c.w_sp + row * c.w_sn + h * c.w_sh] : 0.f;
    reinterpret_cast<uint4*>(const_cast<char*>(k) + (ng * c.k_sp + nrow * c.k_sn + h * c.k_sh) * elem)[piece] = kx;
    reinterpret_cast<uint4*>(const_cast<char*>(v) + (ng * c.v_sp + nrow * c.v_sn + h * c.v_sh) * elem)[piece] = vx;
    if (piece == 0) c.w[ng * c.w_sp + nrow * c.w_sn + h * c.w_sh] = wx;
  };
  const int first = blockIdx.x * per + lane_slot, step = gridDim.x * per;
  if (lane_slot < per)
    for (int to = sure + first; to < size; to += step) copy(to, to + len - size);
  paged_after();                           // the kept slots
  if (lane_slot < per)
    for (int to = first; to < sure; to += step) copy(to, kept[to]);
  if (bad) paged_error(c, SSA_DEVICE_BAD_PAGE);
  if (short_table) paged_error(c, SSA_DEVICE_BAD_LENGTH);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& p, ssa_dtype dt, cudaStream_t st) {
  const int elem = dt == SSA_F32 ? 4 : 2, vecs = p.c.d * elem / 16;
  // eight pieces of K and of V a thread, in up to kAppendRows rows
  const int64_t pieces = static_cast<int64_t>(p.c.h_kv) * vecs, fit = 8 * 256 / pieces;
  const int per_block = static_cast<int>(fit < 1 ? 1 : fit > kAppendRows ? kAppendRows : fit);
  append_kernel<<<static_cast<unsigned>(cdiv(p.rows, per_block)), 256, 0, st>>>(p, elem, vecs, per_block);
  return cudaGetLastError();
}

cudaError_t launch_paged_evict(const PagedEvictParams& p, ssa_dtype dt, cudaStream_t st) {
  const int elem = dt == SSA_F32 ? 4 : 2, vecs = p.c.d * elem / 16;
  // keys that can occur, up to what shared memory holds
  const int64_t slots = static_cast<int64_t>(p.c.max_pages) * p.c.page_size;
  const int held = static_cast<int>(slots < kSelKeys ? slots : kSelKeys);
  static SmemOptIn opt_in;
  cudaError_t e = opt_in(reinterpret_cast<const void*>(evict_select_kernel), kSelKeys * 4);
  if (e != cudaSuccess) return e;
  const int quads = p.c.w_sn == 1 && p.c.page_size % 4 == 0 && p.c.w_sp % 4 == 0 && p.c.w_sh % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(p.c.w) & 15u) == 0;
  evict_select_kernel<<<dim3(p.c.h_kv, p.c.batch), kSelThreads, (held + 3) / 4 * 16, st>>>(p, held, quads);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // two waves of blocks, which then walk (one: 6% to 11% slower, four and eight: 2% to 11%)
  const int64_t most = cdiv(p.budget, 256 / vecs), wanted = cdiv(148 * 16, static_cast<int64_t>(p.c.h_kv) * p.c.batch);
  const int64_t blocks = most < wanted ? most : wanted;
  return launch_after(evict_copy_kernel, dim3(static_cast<unsigned>(blocks), p.c.h_kv, p.c.batch), dim3(256), 0, st, p,
                      elem, vecs);
}

}  // namespace ssa
