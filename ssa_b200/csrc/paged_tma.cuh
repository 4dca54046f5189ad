// Page tiles by TMA, shared by the paged attention kernels: the tensor map over
// the pages, and the boxes of one key tile.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "tc_utils.cuh"

namespace ssa {

// Coordinates of a page box in its 4-D tensor map (d, two of {slot, head}, page).
struct MapOrder {
  int head_first;                  // 1: the head dimension has the smaller stride
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// Where slot j of a sequence lies, for a box that starts there.  Slots from
// `lim` on, and bad pages, get a page coordinate out of range: the copy reads
// zeros.
struct PageSpot {
  int page, row;
};
__device__ __forceinline__ PageSpot page_spot(const PagedCacheParams& c, int seq, int j, int lim) {
  PageSpot s{-1, 0};
  if (j < lim) {
    int lp;
    page_of(c, j, lp, s.row);
    s.page = static_cast<int>(physical_page(c, c.table, c.table_stride, seq, lp));
  }
  return s;
}

// Non-finite 16-bit values: all exponent bits set.  (x & kExp) + kOne carries
// into a half's top bit exactly then.
template <typename T>
struct Half16;
template <> struct Half16<__nv_bfloat16> { static constexpr uint32_t kExp = 0x7f807f80u, kOne = 0x00800080u; };
template <> struct Half16<__half> { static constexpr uint32_t kExp = 0x7c007c00u, kOne = 0x04000400u; };
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  return ((w & Half16<T>::kExp) + Half16<T>::kOne) & 0x80008000u;
}

// x * 0 + acc of both halves: from acc = 0, NaN in a half that met a non-finite
// value and 0 elsewhere.
template <typename T>
__device__ __forceinline__ uint32_t times_zero(uint32_t x, uint32_t acc) {
  uint32_t d;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0u), "r"(acc));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0u), "r"(acc));
  return d;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// The pages as a 4-D tensor of (d, slot and head by ascending stride, page).
// False: the strides are not such a tensor's.
struct PageTensor {
  int64_t s1, s2, sp, n1, n2;
  int head_first;
};
inline bool page_tensor(const PagedCacheParams& c, int64_t sp, int64_t sn, int64_t sh, PageTensor* t) {
  // strides of dimensions with one entry do not matter
  if (c.h_kv == 1) sh = sn * c.page_size;
  t->head_first = sh < sn;
  t->s1 = t->head_first ? sh : sn;
  t->s2 = t->head_first ? sn : sh;
  t->n1 = t->head_first ? c.h_kv : c.page_size;
  t->n2 = t->head_first ? c.page_size : c.h_kv;
  t->sp = c.num_pages == 1 ? t->s2 * t->n2 : sp;
  return t->s1 >= c.d && t->s2 >= t->s1 * t->n1 && t->sp >= t->s2 && t->sp * 2 < (1ll << 40);
}

// Its tensor map, boxes of 64 columns x one page (at most kt slots).
inline bool page_map(const PagedCacheParams& c, const void* base, int64_t sp, int64_t sn, int64_t sh, ssa_dtype dt,
                     int kt, CUtensorMap* map, MapOrder* mo) {
  auto enc = tensor_map_encoder();
  PageTensor t;
  if (!enc || !page_tensor(c, sp, sn, sh, &t)) return false;
  mo->head_first = t.head_first;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.d), static_cast<cuuint64_t>(t.n1),
                              static_cast<cuuint64_t>(t.n2), static_cast<cuuint64_t>(c.num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.s1) * 2, static_cast<cuuint64_t>(t.s2) * 2,
                                 static_cast<cuuint64_t>(t.sp) * 2};
  const cuuint32_t rows = c.page_size < kt ? c.page_size : kt;
  const cuuint32_t box[4] = {64, t.head_first ? 1 : rows, t.head_first ? rows : 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = dt == SSA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, type, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What the kernels on page tiles need of a cache: 16-bit rows of 64 or 128,
// pages of a power of two of at least 8 slots, strides a tensor map takes (K's
// and V's in the same order).
inline bool page_tiles_supported(const PagedAttnParams& p, ssa_dtype dt) {
  if (dt != SSA_BF16 && dt != SSA_F16) return false;
  if (p.c.d != 64 && p.c.d != 128) return false;
  if (p.c.page_shift < 3 || p.c.num_pages < 1 || !(p.inv_scale > 0.f) || !tensor_map_encoder()) return false;
  PageTensor a, b;
  return page_tensor(p.c, p.c.k_sp, p.c.k_sn, p.c.k_sh, &a) && page_tensor(p.c, p.c.v_sp, p.c.v_sn, p.c.v_sh, &b) &&
         a.head_first == b.head_first;
}

}  // namespace ssa
