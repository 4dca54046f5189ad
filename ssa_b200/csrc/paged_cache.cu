// The paged cache's writes: new rows appended to their slots, and eviction.
#include "common.cuh"
#include "paged.cuh"

namespace ssa {
namespace {

// ---------------------------------------------------------------------------
// append: slot (kv_len - n + i) of sequence s <- row q_starts[s] + i.
// Pure data movement, 2 * h_kv * d elements in and out per row.  A group of
// `rows_threads` threads moves one (row, K or V) in 16-byte pieces; the
// sequence of a row is found by bisection of q_starts.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) append_kernel(PagedAppendParams p, int elem, int vecs) {
  const PagedCacheParams& c = p.c;
  const int64_t pieces = static_cast<int64_t>(c.h_kv) * vecs;
  const int64_t total = p.rows * pieces;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = e / pieces;
    const int x = static_cast<int>(e - t * pieces);
    const int h = x / vecs, piece = x - h * vecs;
    int lo = 0, hi = c.batch;                       // last s with q_starts[s] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.q_starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    const PagedSeq q = paged_seq(c, p.q_starts, p.rows, lo);
    if (t < q.q0 || t >= q.q0 + q.n) continue;      // a skipped sequence, or a row of none
    const int64_t slot = static_cast<int64_t>(q.len) - q.n + (t - q.q0);
    if (slot < 0) {
      paged_error(c, SSA_DEVICE_BAD_LENGTH);
      continue;
    }
    int page, row;
    page_of(c, static_cast<int>(slot), page, row);
    const int64_t pg = physical_page(c, c.table, c.table_stride, lo, page);
    if (pg < 0) continue;
    const char* ks = static_cast<const char*>(p.k_new) + (t * p.kn_sn + h * p.kn_sh) * elem;
    const char* vs = static_cast<const char*>(p.v_new) + (t * p.vn_sn + h * p.vn_sh) * elem;
    const uint4 kx = __ldg(reinterpret_cast<const uint4*>(ks) + piece);
    const uint4 vx = __ldg(reinterpret_cast<const uint4*>(vs) + piece);
    char* kd = static_cast<char*>(const_cast<void*>(c.k)) + (pg * c.k_sp + row * c.k_sn + h * c.k_sh) * elem;
    char* vd = static_cast<char*>(const_cast<void*>(c.v)) + (pg * c.v_sp + row * c.v_sn + h * c.v_sh) * elem;
    reinterpret_cast<uint4*>(kd)[piece] = kx;
    reinterpret_cast<uint4*>(vd)[piece] = vx;
    if (c.w && piece == 0) c.w[pg * c.w_sp + row * c.w_sn + h * c.w_sh] = 0.f;
  }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
// Order-preserving key of a weight; NaN ranks with -inf, below every number.
__device__ __forceinline__ uint32_t weight_key(float w) { return float_key(w != w ? -INFINITY : w); }

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kSelBins = 2048;
constexpr int kSelLoads = 16;      // weights in flight a thread
constexpr int kSelKeys = 49152;    // keys held in shared memory (192 KB); longer sequences are read again

// One CTA per (sequence, KV head).  The n_keep heaviest of the first `older`
// slots are those whose key exceeds the n_keep-th largest, T, and the first
// few that equal it.  The weights are read once into shared memory,
// sixteen loads in flight a thread; T is found from its top bits down in three passes
// of 11, 11 and 10 bits, each counting the next digit of the keys that agree
// with T so far and finding the digit by a sum from the top over the 2048
// counts; then every warp counts and writes the kept slots of its own run of
// slots, in order.  Bound by latency: a dozen block-wide steps.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(PagedEvictParams p, int held) {
  const PagedCacheParams& c = p.c;
  const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  extern __shared__ uint32_t sel_keys[];
  __shared__ int hist[kSelBins];
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
  auto read_key = [&](int j) -> uint32_t {
    int page, row;
    page_of(c, j, page, row);
    const int64_t pg = physical_page(c, c.table, c.table_stride, s, page);
    return pg < 0 ? 0u : weight_key(c.w[pg * c.w_sp + row * c.w_sn + h * c.w_sh]);
  };
  const bool hold = older <= held;
  uint32_t prefix = 0, known = 0;          // the bits of T found so far, and which
  int left = n_keep;                       // of the keys that agree with them, how many are kept
  // counts a digit of each lane's key (bin -1: none).  Equal weights (a cache's
  // first steps) would queue 32 deep on one counter.
  auto count = [&](int bin) {
    const int one = __shfl_sync(0xffffffffu, bin, 0);
    if (one >= 0 && __all_sync(0xffffffffu, bin == one)) {
      if (lane == 0) atomicAdd(&hist[bin], 32);
    } else if (bin >= 0) {
      atomicAdd(&hist[bin], 1);
    }
  };
  auto key_of = [&](int j) -> uint32_t { return hold ? sel_keys[j] : read_key(j); };
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int b = tid; b < kSelBins; b += kSelThreads) hist[b] = 0;
    __syncthreads();
    if (pass == 0) {
      for (int j0 = tid; j0 - lane < older; j0 += kSelLoads * kSelThreads) {
        uint32_t k[kSelLoads];
#pragma unroll
        for (int e = 0; e < kSelLoads; ++e) k[e] = j0 + e * kSelThreads < older ? read_key(j0 + e * kSelThreads) : 0u;
#pragma unroll
        for (int e = 0; e < kSelLoads; ++e) {
          const int j = j0 + e * kSelThreads;
          if (j < older && hold) sel_keys[j] = k[e];
          if (j - lane < older) count(j < older ? static_cast<int>(k[e] >> 21) : -1);
        }
      }
    } else {
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
    const int b0 = kSelBins - 1 - 2 * tid, c0 = hist[b0], c1 = hist[b0 - 1];
    int incl = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) wsum[warp][0] = incl;
    __syncthreads();
    int above = incl - c0 - c1;
    for (int w = 0; w < warp; ++w) above += wsum[w][0];
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
    gt = eq = false;
    if (j >= hi) return;
    if (j >= older) {
      gt = true;
    } else {
      const uint32_t k = key_of(j);
      gt = k > prefix;
      eq = k == prefix;
    }
  };
  int ng = 0, ne = 0;
  for (int j = lo + lane; j - lane < hi; j += 32) {
    bool gt, eq;
    kind(j, gt, eq);
    ng += gt;
    ne += eq;
  }
  ng = __reduce_add_sync(0xffffffffu, ng);
  ne = __reduce_add_sync(0xffffffffu, ne);
  __syncthreads();
  if (lane == 0) {
    wsum[warp][0] = ng;
    wsum[warp][1] = ne;
  }
  __syncthreads();
  int out = 0, equal = 0;                  // slots above T, and equal to it, before this warp's run
  {
    const int g = lane < warp ? wsum[lane][0] : 0, e = lane < warp ? wsum[lane][1] : 0;
    out = __reduce_add_sync(0xffffffffu, g);
    equal = __reduce_add_sync(0xffffffffu, e);
  }
  const unsigned below = (1u << lane) - 1u;
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

// Kept slots' keys, values and weights to the new pages.  A thread moves one
// 16-byte piece of K and of V of two slots, their loads in flight together
// (the slot, its page and the data are three loads in a row; four slots a
// thread cost more in resident threads than they gained).
constexpr int kCopySlots = 2;
__global__ void __launch_bounds__(256) evict_copy_kernel(PagedEvictParams p, int elem, int vecs) {
  paged_after();                           // the kept slots
  const PagedCacheParams& c = p.c;
  const int s = blockIdx.z, h = blockIdx.y;
  const int size = min(max(paged_len(c, s), 0), p.budget);
  const int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.h_kv + h) * p.budget;
  const int per = 256 / vecs, lane_slot = threadIdx.x / vecs, piece = threadIdx.x - lane_slot * vecs;
  if (lane_slot >= per) return;
  const char* k = static_cast<const char*>(c.k);
  const char* v = static_cast<const char*>(c.v);
  for (int to0 = blockIdx.x * per * kCopySlots + lane_slot; to0 < size; to0 += gridDim.x * per * kCopySlots) {
    int64_t src[kCopySlots], dst[kCopySlots];   // page, and row in the low bits
    uint4 kx[kCopySlots], vx[kCopySlots];
    float wx[kCopySlots];
#pragma unroll
    for (int e = 0; e < kCopySlots; ++e) {
      const int to = to0 + e * per;
      src[e] = dst[e] = -1;
      if (to >= size) continue;
      int page, row, npage, nrow;
      page_of(c, kept[to], page, row);
      page_of(c, to, npage, nrow);
      if (npage >= p.new_max_pages) {
        paged_error(c, SSA_DEVICE_BAD_LENGTH);
        continue;
      }
      const int64_t pg = physical_page(c, c.table, c.table_stride, s, page);
      const int64_t ng = physical_page(c, p.new_table, p.new_table_stride, s, npage);
      if (pg >= 0 && ng >= 0) {
        src[e] = pg << 10 | row;               // page_size <= 1024
        dst[e] = ng << 10 | nrow;
      }
    }
#pragma unroll
    for (int e = 0; e < kCopySlots; ++e) {
      if (src[e] < 0) continue;
      const int64_t pg = src[e] >> 10, row = src[e] & 1023;
      kx[e] = reinterpret_cast<const uint4*>(k + (pg * c.k_sp + row * c.k_sn + h * c.k_sh) * elem)[piece];
      vx[e] = reinterpret_cast<const uint4*>(v + (pg * c.v_sp + row * c.v_sn + h * c.v_sh) * elem)[piece];
      if (piece == 0) wx[e] = c.w[pg * c.w_sp + row * c.w_sn + h * c.w_sh];
    }
#pragma unroll
    for (int e = 0; e < kCopySlots; ++e) {
      if (src[e] < 0) continue;
      const int64_t pg = dst[e] >> 10, row = dst[e] & 1023;
      reinterpret_cast<uint4*>(const_cast<char*>(k) + (pg * c.k_sp + row * c.k_sn + h * c.k_sh) * elem)[piece] = kx[e];
      reinterpret_cast<uint4*>(const_cast<char*>(v) + (pg * c.v_sp + row * c.v_sn + h * c.v_sh) * elem)[piece] = vx[e];
      if (piece == 0) c.w[pg * c.w_sp + row * c.w_sn + h * c.w_sh] = wx[e];
    }
  }
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& p, ssa_dtype dt, cudaStream_t st) {
  const int elem = dt == SSA_F32 ? 4 : 2, vecs = p.c.d * elem / 16;
  const int64_t total = p.rows * p.c.h_kv * vecs;
  int64_t blocks = cdiv(total, 256);
  if (blocks > 148 * 16) blocks = 148 * 16;
  append_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(p, elem, vecs);
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
  evict_select_kernel<<<dim3(p.c.h_kv, p.c.batch), kSelThreads, held * sizeof(uint32_t), st>>>(p, held);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int per = 256 / vecs * kCopySlots;
  int64_t blocks = cdiv(p.budget, per);
  if (blocks > 1024) blocks = 1024;
  return launch_after(evict_copy_kernel, dim3(static_cast<unsigned>(blocks), p.c.h_kv, p.c.batch), dim3(256), 0, st, p,
                      elem, vecs);
}

}  // namespace ssa
