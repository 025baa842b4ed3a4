// yk_kvcache.cuh -- the e4m3 cells of a paged KV cache: their scale bytes,
// conversions, and the launchers of the operators on such a cache.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "yk_common.cuh"
#include "yk_internal.h"

namespace yk {

// A cell stands for code * 2^(byte - 127).  The exponent stays in -60..60, so
// that two blocks' scales differ by at most 2^120: the attention can carry
// weights relative to the largest scale in fp32 without losing any.
constexpr int KV8_BIAS = 127, KV8_EMIN = -60, KV8_EMAX = 60;

__host__ __device__ __forceinline__ int kv8_exponent(uint32_t byte) {
    const int e = (int)byte - KV8_BIAS;
    return e < KV8_EMIN ? KV8_EMIN : (e > KV8_EMAX ? KV8_EMAX : e);
}
// Smallest exponent e with amax <= 448 * 2^e: 448 = 1.75 * 2^8, so for amax =
// m * 2^E (1 <= m < 2) e = E - 8, one more when m > 1.75 (exact, from the bits).
__device__ __forceinline__ int kv8_cover(float amax) {
    const uint32_t u = __float_as_uint(amax) & 0x7fffffffu;
    if (u == 0) return KV8_EMIN;
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(KV8_EMIN, min(KV8_EMAX, e));
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// Two values to two codes, round to nearest even, saturating; NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2_from(float lo, float hi) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// The low (or high) two codes of w as f16x2: exact.
__device__ __forceinline__ uint32_t f16x2_lo(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_hi(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ float2 f32x2(uint32_t f16x2) {
    return __half22float2(*reinterpret_cast<const __half2*>(&f16x2));
}

// A launch on `stream`; pdl: it may start while the previous kernel of the
// stream finishes (every kernel here waits before it touches memory that
// earlier kernels write).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_on(cudaStream_t stream, bool pdl, void (*kernel)(KArgs...), dim3 grid, dim3 block,
                             size_t smem, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Argument checks shared by the operators' entries, and the launches (on the
// current device).
yk_status kv_pages_check(const yk_kv_pages& p, int32_t layer);
yk_status kv_append_check(const yk_kv_append_args& a);
yk_status kv_append_launch(cudaStream_t stream, bool pdl, int num_sms, const yk_kv_append_args& a);
yk_status attention_e4m3_check(const yk_attention_e4m3_args& a);  // (all but the workspace's size)
yk_status attention_e4m3_launch(cudaStream_t stream, bool pdl, int num_sms, const yk_attention_e4m3_args& a);
size_t attention_e4m3_ws_bytes(int num_sms, int head_dim);

}  // namespace yk
