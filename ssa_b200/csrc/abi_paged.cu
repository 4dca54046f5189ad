// C-ABI entry points of the paged key/value cache (include/ssa_b200.h).
#include <cmath>

#include "abi_util.cuh"
#include "common.cuh"
#include "paged.cuh"

namespace {

using namespace ssa::abi;

// Largest 1-D extent of launches that put sequences on gridDim.z.
constexpr int kMaxBatch = 65535;

bool aligned_rows(const void* p, int64_t a, int64_t b, ssa_dtype t) {
  return aligned16(p) && stride16(a, t) && stride16(b, t);
}

ssa_status check_cache(const SsaPagedCache* c, ssa::PagedCacheParams& o) {
  if (!c) return fail(SSA_ERR_INVALID_ARG, "cache is NULL");
  if (c->batch < 0 || c->max_pages < 0 || c->num_pages < 0)
    return fail(SSA_ERR_INVALID_ARG, "bad sizes batch=%d max_pages=%d num_pages=%lld", c->batch, c->max_pages,
                static_cast<long long>(c->num_pages));
  if (c->batch > kMaxBatch || c->h_kv > 65535)
    return fail(SSA_ERR_UNSUPPORTED, "batch %d, num_kv_heads %d: at most 65535", c->batch, c->h_kv);
  if (c->page_size < 1 || c->page_size > 1024)
    return fail(SSA_ERR_UNSUPPORTED, "page_size %d: need 1..1024", c->page_size);
  if (c->h_kv < 1) return fail(SSA_ERR_INVALID_ARG, "num_kv_heads %d < 1", c->h_kv);
  if (c->d < 8 || c->d > 256 || c->d % 8 != 0)
    return fail(SSA_ERR_UNSUPPORTED, "head_dim %d: need a multiple of 8 in [8, 256]", c->d);
  if (!valid_dtype(c->dtype)) return fail(SSA_ERR_INVALID_ARG, "bad dtype");
  if (static_cast<int64_t>(c->max_pages) * c->page_size >= (1ll << 31) - (1ll << 17) || c->num_pages >= (1ll << 31))
    return fail(SSA_ERR_UNSUPPORTED, "max_pages * page_size must be < 2^31 - 2^17, num_pages < 2^31");
  if (c->batch > 0 && (!c->kv_lens || (c->max_pages > 0 && !c->page_table)))
    return fail(SSA_ERR_INVALID_ARG, "page_table / kv_lens is NULL");
  if (c->num_pages > 0 && (!c->k_pages || !c->v_pages)) return fail(SSA_ERR_INVALID_ARG, "k_pages / v_pages is NULL");
  if (!aligned_rows(c->k_pages, c->k_stride_n, c->k_stride_h, c->dtype) || !stride16(c->k_stride_p, c->dtype) ||
      !aligned_rows(c->v_pages, c->v_stride_n, c->v_stride_h, c->dtype) || !stride16(c->v_stride_p, c->dtype))
    return fail(SSA_ERR_ALIGNMENT, "k_pages and v_pages must be 16-byte aligned with 16-byte strides");
  o.k = c->k_pages; o.k_sp = c->k_stride_p; o.k_sn = c->k_stride_n; o.k_sh = c->k_stride_h;
  o.v = c->v_pages; o.v_sp = c->v_stride_p; o.v_sn = c->v_stride_n; o.v_sh = c->v_stride_h;
  o.w = c->weights; o.w_sp = c->w_stride_p; o.w_sn = c->w_stride_n; o.w_sh = c->w_stride_h;
  o.table = c->page_table;
  o.table_stride = c->table_stride;
  o.kv_lens = c->kv_lens;
  o.status = c->status;
  o.num_pages = c->num_pages;
  o.batch = c->batch;
  o.max_pages = c->max_pages;
  o.page_size = c->page_size;
  o.page_shift = -1;
  for (int s = 0; s <= 10; ++s)
    if ((1 << s) == c->page_size) o.page_shift = s;
  o.h_kv = c->h_kv;
  o.d = c->d;
  return SSA_OK;
}

ssa_status check_rows(const SsaPagedCache* c, int64_t rows, const int32_t* q_starts) {
  if (rows < 0 || rows >= (1ll << 31)) return fail(SSA_ERR_INVALID_ARG, "rows %lld: need 0..2^31 - 1",
                                                   static_cast<long long>(rows));
  if (c->batch > 0 && !q_starts) return fail(SSA_ERR_INVALID_ARG, "q_starts is NULL");
  return SSA_OK;
}

ssa_status attn_params(const SsaPagedCache* c, const SsaPagedAttnArgs* a, ssa::PagedAttnParams& p) {
  ssa_status s = check_cache(c, p.c);
  if (s != SSA_OK) return s;
  if (!a) return fail(SSA_ERR_INVALID_ARG, "args is NULL");
  s = check_rows(c, a->rows, a->q_starts);
  if (s != SSA_OK) return s;
  if (a->h_q < 1 || a->h_q % c->h_kv != 0)
    return fail(SSA_ERR_INVALID_ARG, "num_q_heads (%d) must be a multiple of num_kv_heads (%d)", a->h_q, c->h_kv);
  if (a->h_q / c->h_kv > 16)
    return fail(SSA_ERR_UNSUPPORTED, "%d query heads per KV head: at most 16", a->h_q / c->h_kv);
  if (!(std::isfinite(a->scale) && a->scale != 0.f && std::isfinite(1.f / a->scale)))
    return fail(SSA_ERR_INVALID_ARG, "scale must be finite and not 0, and so must its reciprocal");
  if (a->rows > 0 && (!a->q || !a->out)) return fail(SSA_ERR_INVALID_ARG, "q / out is NULL");
  if (!aligned_rows(a->q, a->q_stride_n, a->q_stride_h, c->dtype) ||
      !aligned_rows(a->out, a->out_stride_n, a->out_stride_h, c->dtype))
    return fail(SSA_ERR_ALIGNMENT, "q and out must be 16-byte aligned with 16-byte strides");
  p.q_starts = a->q_starts;
  p.q = a->q; p.q_sn = a->q_stride_n; p.q_sh = a->q_stride_h;
  p.out = a->out; p.o_sn = a->out_stride_n; p.o_sh = a->out_stride_h;
  p.lse = a->lse;
  p.rows = a->rows;
  p.group = a->h_q / c->h_kv;
  p.causal = a->causal ? 1 : 0;
  p.inv_scale = 1.f / a->scale;
  return SSA_OK;
}

}  // namespace

extern "C" {

ssa_status ssa_paged_append(const SsaPagedCache* cache, const SsaPagedAppendArgs* args, void* stream) {
  ssa::PagedAppendParams p{};
  ssa_status s = check_cache(cache, p.c);
  if (s != SSA_OK) return s;
  if (!args) return fail(SSA_ERR_INVALID_ARG, "args is NULL");
  s = check_rows(cache, args->rows, args->q_starts);
  if (s != SSA_OK) return s;
  if (args->rows == 0 || cache->batch == 0) return SSA_OK;
  if (!args->k_new || !args->v_new) return fail(SSA_ERR_INVALID_ARG, "k_new / v_new is NULL");
  if (!aligned_rows(args->k_new, args->k_new_stride_n, args->k_new_stride_h, cache->dtype) ||
      !aligned_rows(args->v_new, args->v_new_stride_n, args->v_new_stride_h, cache->dtype))
    return fail(SSA_ERR_ALIGNMENT, "k_new and v_new must be 16-byte aligned with 16-byte strides");
  p.q_starts = args->q_starts;
  p.k_new = args->k_new; p.kn_sn = args->k_new_stride_n; p.kn_sh = args->k_new_stride_h;
  p.v_new = args->v_new; p.vn_sn = args->v_new_stride_n; p.vn_sh = args->v_new_stride_h;
  p.rows = args->rows;
  return cuda_status(ssa::launch_paged_append(p, cache->dtype, static_cast<cudaStream_t>(stream)), "paged_append");
}

size_t ssa_paged_attn_workspace_size(const SsaPagedCache* cache, const SsaPagedAttnArgs* args) {
  ssa::PagedAttnParams p{};
  if (attn_params(cache, args, p) != SSA_OK) return 0;
  return ssa::paged_attn_workspace(p, cache->dtype);
}

ssa_status ssa_paged_attn(const SsaPagedCache* cache, const SsaPagedAttnArgs* args, void* workspace,
                          size_t workspace_bytes, void* stream) {
  ssa::PagedAttnParams p{};
  const ssa_status s = attn_params(cache, args, p);
  if (s != SSA_OK) return s;
  if (args->rows == 0 || cache->batch == 0) return SSA_OK;
  const size_t need = ssa::paged_attn_workspace(p, cache->dtype);
  if (!workspace || workspace_bytes < need)
    return fail(SSA_ERR_WORKSPACE, "workspace needs %zu bytes, got %zu", need, workspace_bytes);
  if (!aligned16(workspace)) return fail(SSA_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  return cuda_status(ssa::launch_paged_attn(p, cache->dtype, workspace, static_cast<cudaStream_t>(stream)),
                     "paged_attn");
}

ssa_status ssa_paged_evict(const SsaPagedCache* cache, const SsaPagedEvictArgs* args, void* stream) {
  ssa::PagedEvictParams p{};
  const ssa_status s = check_cache(cache, p.c);
  if (s != SSA_OK) return s;
  if (!args) return fail(SSA_ERR_INVALID_ARG, "args is NULL");
  if (args->budget < 1 || args->recent < 0 || args->recent > args->budget)
    return fail(SSA_ERR_INVALID_ARG, "budget %d, recent %d: need budget >= 1 and 0 <= recent <= budget", args->budget,
                args->recent);
  if (args->new_max_pages < 0) return fail(SSA_ERR_INVALID_ARG, "new_max_pages %d < 0", args->new_max_pages);
  if (cache->batch == 0) return SSA_OK;
  if (!cache->weights) return fail(SSA_ERR_INVALID_ARG, "weights is NULL: eviction ranks slots by them");
  if (!args->kept || !args->new_lens || (args->new_max_pages > 0 && !args->new_table))
    return fail(SSA_ERR_INVALID_ARG, "kept / new_lens / new_table is NULL");
  p.new_table = args->new_table;
  p.new_table_stride = args->new_table_stride;
  p.kept = args->kept;
  p.new_lens = args->new_lens;
  p.new_max_pages = args->new_max_pages;
  p.budget = args->budget;
  p.recent = args->recent;
  return cuda_status(ssa::launch_paged_evict(p, cache->dtype, static_cast<cudaStream_t>(stream)), "paged_evict");
}

}  // extern "C"
