// kv8.cuh -- the 8-bit key / value pool: format, exponents and conversions shared by its kernels.
//
// kv8 [num_pages, Hkv, 4096] bytes of e4m3 codes and scales [num_pages, Hkv, 2] stored exponents (keys,
// values): value = code * 2^(scale - 127). Of a page and kv head,
//   keys    byte  (d / 64) * 1024 + t * 64 + d % 64                     of token t, dimension d;
//   values  byte  2048 + (d / 4) * 64 + (t % 8) / 2 * 16 + (d % 4) * 4 + (t / 8) * 2 + t % 2.
// That is the order in which an m16n8k16 MMA wants its fragments: lane 4 g + c takes 16 bytes of key g
// (or 8 + g) at dimension 16 c of a half, and 4 dimensions x the tokens 2 c, 2 c + 1, 8 + 2 c, 9 + 2 c of the
// values, so a warp reads 512 consecutive bytes at a time, from global or shared memory, and neither
// ldmatrix nor a swizzle is needed. A page and head is one copy of 4 KB.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "kv8_args.h"

namespace msgl {
// Attention of chunks (kv8_chunk.cu): more than 64 rows x heads of a group.
int launch_attend_chunk(const Kv8AttnArgs& a, msgl_stream_t stream);

constexpr int kKv8Page = 16;
constexpr int kKv8Head = 128;
constexpr int kKv8Bytes = 4096;   // of a page and kv head
constexpr int kKv8Values = 2048;  // where the values begin
// Smallest stored exponent, 2^-96: the weights' sum of the attention, which counts a page in units of
// its values' scale, stays within fp32 then.
constexpr int kKv8Floor = 31;

// Stored exponent of the smallest power of two s with amax <= 448 s (448: the largest e4m3 value).
__device__ __forceinline__ int kv8_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    return max(kKv8Floor, static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u));
}
__device__ __forceinline__ float kv8_power(int stored) { return __uint_as_float(static_cast<uint32_t>(stored) << 23); }
// 2^-(stored - 127), stored in [1, 253]
__device__ __forceinline__ float kv8_inverse(int stored) { return __uint_as_float(static_cast<uint32_t>(254 - stored) << 23); }

// Two e4m3 codes (the low 16 bits) as two halves, exactly.
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t codes) {
    uint32_t h;
    asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(codes));
    return h;
}
// Four codes of a word: halves of bytes 0, 1 and of bytes 2, 3.
__device__ __forceinline__ void e4m3x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
// Codes of x0 (low byte) and x1, rounded to nearest even; |x| <= 448 or NaN.
__device__ __forceinline__ uint32_t e4m3_codes2(float x0, float x1) {
    return __nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3);
}

}  // namespace msgl
