// Shared by the decode operators (kv_append.cu, kv_attention.cu, matvec_w4.cu): element types,
// e4m3 conversions, the geometry of the paged cache and the device status of its kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace piton {
namespace decode {

// Device status words beside the bounded waits' (sm100.cuh): an index that a kernel found out of
// range on the device and therefore did not follow.
enum : int {
    STATUS_BAD_PAGE = 16,      // a page-table entry outside [0, num_pages)
    STATUS_BAD_POSITION = 17,  // a position outside the page table or the rotation tables, or bad offsets
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float e4m3_to_float(uint8_t c) {
    __nv_fp8_e4m3 v;
    v.__x = c;
    return (float)v;
}
// Nearest e4m3 value, ties to even; |x| <= 448 here, NaN stays NaN.
__device__ __forceinline__ uint8_t float_to_e4m3(float x) {
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// WORDS words of shared memory in one load.
template <int WORDS> __device__ __forceinline__ void load_words(uint32_t (&w)[WORDS], uint32_t at) {
    if constexpr (WORDS == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    else if constexpr (WORDS == 2)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}

// A copy of N bytes (4, 8 or 16) from global to shared memory that is waited for later.
template <int N> __device__ __forceinline__ void copy_async(uint32_t dst, const void *src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}

// Query (or new) tokens [t0, t0 + n) of sequence b: from the offsets `cu`, clamped to the tensor,
// or `uniform` each.
struct Span {
    int64_t t0, n;
};
__device__ __forceinline__ Span span_of(const int32_t *cu, int64_t b, int64_t uniform, int64_t tokens) {
    if (!cu) return {b * uniform, uniform};
    int64_t lo = cu[b], hi = cu[b + 1];
    lo = lo < 0 ? 0 : (lo > tokens ? tokens : lo);
    hi = hi < lo ? lo : (hi > tokens ? tokens : hi);
    return {lo, hi - lo};
}

// Runs f with a value of the element type that `type` names.
template <typename F> int with_type(int32_t type, F f) {
    switch (type) {
        case PITON_B200_TYPE_F32: return f(float());
        case PITON_B200_TYPE_F16: return f(__half());
        case PITON_B200_TYPE_BF16: return f(__nv_bfloat16());
    }
    return set_error(PITON_B200_EINVAL, "unknown element type %d", type);
}

// The status words of the two cache kernels' files, then reset (read by piton_b200_device_status).
int kv_append_status_read_and_clear(int *status);
int kv_attention_status_read_and_clear(int *status);

}  // namespace decode
}  // namespace piton
