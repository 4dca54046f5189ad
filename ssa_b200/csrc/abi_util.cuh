// Host helpers of the C-ABI layer: status codes with their text, argument
// predicates, workspace rounding.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "../../include/ssa_b200.h"

namespace ssa {
namespace abi {

inline thread_local std::string g_last_error;

inline ssa_status fail(ssa_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
inline ssa_status fail(ssa_status s, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return s;
}

inline ssa_status cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return SSA_OK;
  return fail(SSA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline size_t elem_size(ssa_dtype t) { return t == SSA_F32 ? 4 : 2; }
inline bool valid_dtype(ssa_dtype t) { return t == SSA_F32 || t == SSA_BF16 || t == SSA_F16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool stride16(int64_t s, ssa_dtype t) { return (s * static_cast<int64_t>(elem_size(t))) % 16 == 0; }

constexpr size_t kAlign = 256;
inline size_t round_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

}  // namespace abi
}  // namespace ssa
