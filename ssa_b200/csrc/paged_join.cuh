// What a row's attention ends with: its log-sum-exp, and the join of an item
// that several CTAs hold parts of.
//
// A CTA that does not hold all key tiles of an item leaves, for every row, the
// unnormalised output, the running maximum (base 2) and the sum.  Items of many
// rows are joined by a kernel of their own (combine_kernel, paged_attn.cu), which
// spreads the rows over the GPU.  The few rows of a token's item are joined by the
// last of its CTAs, which saves a launch: each counts itself in, nobody waits.
// The counters are zero before a launch and after it: the joining CTA resets its
// item's.  Either way parts are taken in CTA order.
#pragma once

#include "common.cuh"
#include "mma_utils.cuh"
#include "paged.cuh"

namespace ssa {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// lse of a row from its maximum (base 2) and sum; -inf for a row that saw nothing.
__device__ __forceinline__ void store_lse(const PagedAttnParams& p, int64_t tok, int head, float m, float l) {
  const int64_t at = tok * (static_cast<int64_t>(p.c.h_kv) * p.group) + head;
  const float z = l == 0.f ? -INFINITY : m + log2f(l);
  if (p.lse) p.lse[at] = z * kLn2;
  if (p.lse2) p.lse2[at] = z;
}

template <typename T>
__device__ __forceinline__ void store4(T* dst, const float4& v, float f) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(dst) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  } else {
    uint2 u;
    u.x = pack2<T>(v.x * f, v.y * f);
    u.y = pack2<T>(v.z * f, v.w * f);
    *reinterpret_cast<uint2*>(dst) = u;
  }
}

// Output, maximum and sum of a row over `count` parts, PB of them in flight.
// part(i): the row in part i.  The warp's lanes have four columns each from c0 on.
template <int PB, typename Part>
__device__ __forceinline__ void join_row(const Part& part, int count, int d, int c0, float4& o, float& m, float& l) {
  const int x = c0 + 4 * (threadIdx.x & 31);
  const bool mine = x < d;
  m = -INFINITY;
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < count; i0 += PB) {
    float2 ml[PB];
    float4 a[PB];
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + i < count) {
        // past L1: another SM wrote these, perhaps during this launch
        const float* src = part(i0 + i);
        ml[i] = __ldcg(reinterpret_cast<const float2*>(src + d));
        if (mine) a[i] = __ldcg(reinterpret_cast<const float4*>(src + x));
      }
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < PB; ++i) mn = fmaxf(mn, ml[i].x);
    const float base = mn == -INFINITY ? 0.f : mn, f = exp2f(m - base);
    m = mn;
    l *= f;
    o.x *= f;
    o.y *= f;
    o.z *= f;
    o.w *= f;
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const float g = exp2f(ml[i].x - base);
      l = fmaf(g, ml[i].y, l);
      o.x = fmaf(g, a[i].x, o.x);
      o.y = fmaf(g, a[i].y, o.y);
      o.z = fmaf(g, a[i].z, o.z);
      o.w = fmaf(g, a[i].w, o.w);
    }
  }
}

// A warp writes row r of the tile at row tok0 of q, KV head `kv_head`, joined.
template <typename T, int PB, typename Part>
__device__ __forceinline__ void write_joined(const PagedAttnParams& p, const Part& part, int count, int64_t tok0,
                                             int kv_head, int r) {
  const int lane = threadIdx.x & 31, d = p.c.d;
  const int64_t tok = tok0 + r / p.group;
  const int head = kv_head * p.group + r % p.group;
  T* dst = static_cast<T*>(p.out) + tok * p.o_sn + static_cast<int64_t>(head) * p.o_sh;
  for (int c0 = 0; c0 < d; c0 += 128) {
    float4 o;
    float m, l;
    join_row<PB>(part, count, d, c0, o, m, l);
    if (c0 + 4 * lane < d) store4(dst + c0 + 4 * lane, o, l == 0.f ? 0.f : 1.f / l);
    if (lane == 0 && c0 == 0) store_lse(p, tok, head, m, l);
  }
}

}  // namespace ssa
