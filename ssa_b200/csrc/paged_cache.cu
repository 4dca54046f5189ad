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

constexpr int kSelThreads = 1024;

// One CTA per (sequence, KV head).  The n_keep heaviest of the first `older`
// slots are those whose key exceeds the n_keep-th largest, T, and the first
// few that equal it: T is found from its top byte down, each pass counting the
// next byte of the keys that agree with T so far; then one pass in slot order
// writes the kept slots.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(PagedEvictParams p) {
  const PagedCacheParams& c = p.c;
  const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int hist[256];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_left;
  __shared__ int wsum[32][2];
  const int len = max(paged_len(c, s), 0);
  const int size = min(len, p.budget), recent = min(p.recent, size), older = len - recent, n_keep = size - recent;
  int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.h_kv + h) * p.budget;
  if (tid == 0 && h == 0) p.new_lens[s] = size;
  auto key_of = [&](int j) -> uint32_t {
    int page, row;
    page_of(c, j, page, row);
    const int64_t pg = physical_page(c, c.table, c.table_stride, s, page);
    return pg < 0 ? 0u : weight_key(c.w[pg * c.w_sp + row * c.w_sn + h * c.w_sh]);
  };
  uint32_t prefix = 0;
  int left = n_keep;                       // of the keys that agree with the prefix, how many are kept
  if (size < len) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int b = tid; b < 256; b += kSelThreads) hist[b] = 0;
      __syncthreads();
      for (int j = tid; j < older; j += kSelThreads) {
        const uint32_t k = key_of(j);
        if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int l = left, b = 255;
        while (b > 0 && hist[b] < l) l -= hist[b--];
        sh_prefix = prefix | (static_cast<uint32_t>(b) << shift);
        sh_left = l;
      }
      __syncthreads();
      prefix = sh_prefix;
      left = sh_left;
      __syncthreads();
    }
  }
  // slots in order: kept if above T, if among the first `left` equal to T, or recent
  int out = 0, equal = 0;
  for (int j0 = 0; j0 < len; j0 += kSelThreads) {
    const int j = j0 + tid;
    bool gt = false, eq = false;
    if (j < len) {
      if (size == len || j >= older) gt = true;
      else {
        const uint32_t k = key_of(j);
        gt = k > prefix;
        eq = k == prefix;
      }
    }
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      wsum[warp][0] = __popc(bg);
      wsum[warp][1] = __popc(be);
    }
    __syncthreads();
    const unsigned below = (1u << lane) - 1u;
    int g0 = out + __popc(bg & below), e0 = equal + __popc(be & below), tg = 0, te = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) {
      if (w < warp) {
        g0 += wsum[w][0];
        e0 += wsum[w][1];
      }
      tg += wsum[w][0];
      te += wsum[w][1];
    }
    if (gt) kept[g0 + min(e0, left)] = j;
    else if (eq && e0 < left) kept[g0 + e0] = j;
    out += tg;
    equal += te;
    __syncthreads();
  }
  for (int j = size + tid; j < p.budget; j += kSelThreads) kept[j] = -1;
}

// Kept slots' keys, values and weights to the new pages: one 16-byte piece of
// K and of V per thread.
__global__ void __launch_bounds__(256) evict_copy_kernel(PagedEvictParams p, int elem, int vecs) {
  const PagedCacheParams& c = p.c;
  const int s = blockIdx.z, h = blockIdx.y;
  const int size = min(max(paged_len(c, s), 0), p.budget);
  const int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.h_kv + h) * p.budget;
  const int64_t total = static_cast<int64_t>(size) * vecs;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int to = static_cast<int>(e / vecs), piece = static_cast<int>(e - static_cast<int64_t>(to) * vecs);
    const int from = kept[to];
    int page, row, npage, nrow;
    page_of(c, from, page, row);
    page_of(c, to, npage, nrow);
    if (npage >= p.new_max_pages) {
      paged_error(c, SSA_DEVICE_BAD_LENGTH);
      continue;
    }
    const int64_t pg = physical_page(c, c.table, c.table_stride, s, page);
    const int64_t ng = physical_page(c, p.new_table, p.new_table_stride, s, npage);
    if (pg < 0 || ng < 0) continue;
    const char* k = static_cast<const char*>(c.k);
    const char* v = static_cast<const char*>(c.v);
    const uint4 kx = reinterpret_cast<const uint4*>(k + (pg * c.k_sp + row * c.k_sn + h * c.k_sh) * elem)[piece];
    const uint4 vx = reinterpret_cast<const uint4*>(v + (pg * c.v_sp + row * c.v_sn + h * c.v_sh) * elem)[piece];
    reinterpret_cast<uint4*>(const_cast<char*>(k) + (ng * c.k_sp + nrow * c.k_sn + h * c.k_sh) * elem)[piece] = kx;
    reinterpret_cast<uint4*>(const_cast<char*>(v) + (ng * c.v_sp + nrow * c.v_sn + h * c.v_sh) * elem)[piece] = vx;
    if (piece == 0)
      c.w[ng * c.w_sp + nrow * c.w_sn + h * c.w_sh] = c.w[pg * c.w_sp + row * c.w_sn + h * c.w_sh];
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
  evict_select_kernel<<<dim3(p.c.h_kv, p.c.batch), kSelThreads, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  int64_t blocks = cdiv(static_cast<int64_t>(p.budget) * vecs, 256 * 4);
  if (blocks > 1024) blocks = 1024;
  evict_copy_kernel<<<dim3(static_cast<unsigned>(blocks), p.c.h_kv, p.c.batch), 256, 0, st>>>(p, elem, vecs);
  return cudaGetLastError();
}

}  // namespace ssa
