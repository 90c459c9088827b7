// The 8-bit quantization shared by the INT8 KV cache (kv_q8.hip) and the
// INT8 activations (qmm_a8.hip), and the cache's checks.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "vm_device.h"
#include "vm_hip.h"

namespace vmhip {

// 16-bit elements; arithmetic is done in fp32.
struct F16 {
    uint16_t bits;
};
struct BF16 {
    uint16_t bits;
};

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<F16>(F16 v) { return static_cast<float>(__builtin_bit_cast(_Float16, v.bits)); }
template <>
__device__ __forceinline__ float widen<BF16>(BF16 v) { return __uint_as_float(static_cast<uint32_t>(v.bits) << 16); }

// An fp32 value rounded to nearest even.  (The empty statement keeps the
// compiler from folding the product that made v into its conversion to fp16,
// v_fma_mixlo_f16: that skips the product's own rounding to fp32, which
// results are defined with.)
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ F16 narrow<F16>(float v) {
    asm("" : "+v"(v));
    return F16{__builtin_bit_cast(uint16_t, static_cast<_Float16>(v))};
}
template <>
__device__ __forceinline__ BF16 narrow<BF16>(float v) { return BF16{f32_to_bf16_ref(v)}; }

// Checks of the cache that every entry point shares (VM_HIP_EINVAL with a
// message that names `who`).
int check_kv_q8(const vm_hip_kv_q8* c, const char* who);

// The same pointer, by an offset of zero that the compiler does not know: keeps
// the element-wise branch of a guarded vector access apart from the vector
// branch (with the first element in common, it was taken out of both, and what
// was left of 16 bytes became a 4- and a 12-byte access).
template <typename T>
__device__ __forceinline__ T* apart(T* p) {
    int zero = 0;
    asm("" : "+v"(zero));
    return p + zero;
}

struct Q8Scale {
    float scale;   // what a code stands for
    float inv;     // what a value is multiplied by before it is rounded
};

// The scale of a row whose largest magnitude has these bits.  Below 2^-119
// the reciprocal would leave fp32's range: such a row is stored as zeros.  An
// infinity or NaN in the row: zeros with scale NaN.
__device__ __forceinline__ Q8Scale q8_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return {NAN, 0.0f};
    if (amax_bits < 0x04000000u) return {1.0f, 0.0f};   // 2^-119
    const float s = __uint_as_float(amax_bits) / 127.0f;
    return {s, 1.0f / s};
}

// round(x * inv) half away from zero, clamped to +-127.  (inv 0: code 0, also
// for an infinity or NaN.)
__device__ __forceinline__ int8_t q8_code(float x, float inv) {
    const float v = roundf(x * inv);
    if (!(inv > 0.0f)) return 0;
    return static_cast<int8_t>(v < -127.0f ? -127.0f : v > 127.0f ? 127.0f : v);
}

}  // namespace vmhip
