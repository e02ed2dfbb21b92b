// ops.cuh — what the serving operators (kv_plan.cu, kv8.cu, kv8_attn.cu,
// sample_rows.cu) share: types of caller tensors, device selection and the
// bounds of their arguments.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace wg {

__host__ __device__ inline int dt_bytes(int dt) { return dt == WG_DT_F32 ? 4 : 2; }
inline bool dt_ok(int dt) { return dt == WG_DT_F32 || dt == WG_DT_F16 || dt == WG_DT_BF16; }

// One element of a caller tensor, as fp32 (exact for every type).
__device__ __forceinline__ float dt_load(const void* p, int64_t i, int dt) {
  if (dt == WG_DT_F32) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (dt == WG_DT_F16) return __half2float(__ldg(reinterpret_cast<const __half*>(p) + i));
  return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p) + i));
}
// One element, rounded to nearest even.
__device__ __forceinline__ void dt_store(void* p, int64_t i, int dt, float v) {
  if (dt == WG_DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == WG_DT_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
// Two fp32 values as a packed 16-bit pair of type dt (first value low).
__device__ __forceinline__ uint32_t dt_pack2(int dt, float a, float b) {
  if (dt == WG_DT_F16) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
// The packed pair as fp32.
__device__ __forceinline__ float2 dt_unpack2(int dt, uint32_t w) {
  if (dt == WG_DT_F16) return __half22float2(*reinterpret_cast<__half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Makes `device` current for a scope and puts the caller's device back.
class OpDevice {
 public:
  int enter(const char* what, int device) {
    static std::atomic<int> known{0};  // devices do not come and go in a process's life
    int n = known.load(std::memory_order_relaxed);
    if (n == 0) {
      if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        cudaGetLastError();
        set_error("no CUDA device is available");
        return WG_ERR_NO_DEVICE;
      }
      known.store(n, std::memory_order_relaxed);
    }
    if (device < 0 || device >= n) {
      set_error("%s: device %d does not exist (%d visible)", what, device, n);
      return WG_ERR_INVALID;
    }
    WG_CHECK_CUDA(cudaGetDevice(&prev_));
    if (prev_ != device) {
      WG_CHECK_CUDA(cudaSetDevice(device));
      moved_ = true;
    }
    return WG_OK;
  }
  ~OpDevice() {
    if (moved_) cudaSetDevice(prev_);
  }

 private:
  int prev_ = -1;
  bool moved_ = false;
};

// Kernel attributes are set once per device; OPS_MAX_DEV bounds the flags.
constexpr int OPS_MAX_DEV = 64;

// The checks of a wg_kv8 descriptor that every cache operator makes.
int kv8_check(const char* what, const wg_kv8* c);
inline bool kv_page_ok(int page) { return page >= 16 && page <= 128 && (page & (page - 1)) == 0; }
inline int log2_of(int pow2) {
  int s = 0;
  while ((1 << s) < pow2) s++;
  return s;
}
// int32 and fp32 tensors: what starts elsewhere would fault the GPU
template <typename... P>
inline bool aligned4(const P*... p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & 3) == 0; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace wg
