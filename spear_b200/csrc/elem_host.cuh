// Host helpers of the token-major operators: storage types and launch results.
#pragma once

#include "btp_elem.cuh"
#include "btp_host.cuh"

namespace btp_host {

inline int elem_bytes(int dtype) { return dtype == BTP_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == BTP_DTYPE_BF16 || dtype == BTP_DTYPE_F16 || dtype == BTP_DTYPE_F32; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// f(a value of the storage type)
template <class F>
cudaError_t by_type(int dtype, F&& f) {
  if (dtype == BTP_DTYPE_BF16) return f(__nv_bfloat16{});
  if (dtype == BTP_DTYPE_F16) return f(__half{});
  return f(float{});
}

inline int launched(const char* fn, cudaError_t e) {
  if (e != cudaSuccess) return fail(BTP_ERR_CUDA, "%s: launch: %s", fn, cudaGetErrorString(e));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return BTP_OK;
}

}  // namespace btp_host
