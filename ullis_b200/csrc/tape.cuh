// The 8-bit tape: what one block of 32 channels of a row is kept as.
//
// e = the smallest integer of -126 .. 121 with 127 * 2^e >= max |x| of the block (121 where none has), codes round(x * 2^-e)
// (ties to even, int8, kept within +/-127: beyond them lie only the last values of f32, whose next step would be 2^128), the
// exponent as the byte e + 127; a code stands for code * 2^e.  A step of a block is at most 2 / 127 of its largest value, and the
// steps are powers of two: packing divides exactly, a code is exact in bf16 and f32, and scaling by 2^e rounds nothing, so an
// 8-bit operand goes through the tensor cores as the number it stands for.  A block with a value that is not finite has the
// byte 255 and stands for NaN throughout.
//
// Kernels take a row in chunks of eight channels, one per thread, four threads to a block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ullis {
namespace tape {

constexpr uint32_t BLOCK = 32, CHUNK = 8;
constexpr uint32_t NOT_FINITE = 255;

__host__ __device__ inline size_t blocks_of(size_t channels) { return (channels + BLOCK - 1) / BLOCK; }

// the exponent byte of a block by the bits of its largest |x|
__host__ __device__ inline uint32_t exponent_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return NOT_FINITE;
    // 127 = 1.984375 * 2^6: the mantissa's last 2^17 steps need the next exponent
    const uint32_t field = (amax_bits + 0x1FFFFu) >> 23;   // biased exponent of amax, one more there
    return field < 7u ? 1u : field > 254u ? 248u : field - 6u;   // e + 127 = field - 127 - 6 + 127
}

#if defined(__CUDACC__)
__device__ __forceinline__ float power(uint32_t byte) {          // 2^e
    return byte == NOT_FINITE ? __int_as_float(0x7FFFFFFF) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ float inverse_power(uint32_t byte) {  // 2^-e
    return byte == NOT_FINITE ? 0.0f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight channels from c on of a row of `C`; past its end zeros.  VEC: rows start on 16 bytes and C is a multiple of 8, so a
// chunk is whole or absent.
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* row, uint32_t c, uint32_t C, float (&v)[8]) {
    if constexpr (VEC) {
        if (c < C) {
            if constexpr (sizeof(T) == 4) {
                const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            } else {
                const uint4 w = *reinterpret_cast<const uint4*>(row + c);
                const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = to_float(t[i]);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < C ? to_float(row[c + i]) : 0.0f;
    }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* row, uint32_t c, uint32_t C, const float (&v)[8]) {
    if constexpr (VEC) {
        if (c >= C) return;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint4 w;
            T* t = reinterpret_cast<T*>(&w);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = from_float<T>(v[i]);
            *reinterpret_cast<uint4*>(row + c) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < C) row[c + i] = from_float<T>(v[i]);
    }
}
// The exponent byte of the block whose four chunks the four lanes of a quad hold.
__device__ __forceinline__ uint32_t quad_exponent(const float (&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);   // of NaN too: above infinity
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    return exponent_byte(top);
}
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* codes, uint32_t c, uint32_t C, const float (&v)[8], float inverse) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i >> 2] |= (uint32_t)(min(max(__float2int_rn(v[i] * inverse), -127), 127) & 0xFF) << (8 * (i & 3));   // (0 for NaN)
    if constexpr (VEC) {
        if (c < C) *reinterpret_cast<uint2*>(codes + c) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < C) codes[c + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}
// Eight codes times `step`; past the row's end zeros (whatever the step).
template <bool VEC>
__device__ __forceinline__ void load_codes(const uint8_t* codes, float step, uint32_t c, uint32_t C, float (&v)[8]) {
    uint32_t w[2] = {0u, 0u};
    if (c < C) {
        if constexpr (VEC) {
            const uint2 t = *reinterpret_cast<const uint2*>(codes + c);
            w[0] = t.x; w[1] = t.y;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < C) w[i >> 2] |= (uint32_t)codes[c + i] << (8 * (i & 3));
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * step;
        v[i] = (VEC ? c : c + i) < C ? x : 0.0f;
    }
}
// What they stand for.
template <bool VEC>
__device__ __forceinline__ void load_codes(const uint8_t* codes, const uint8_t* exponents, uint32_t c, uint32_t C, float (&v)[8]) {
    load_codes<VEC>(codes, c < C ? power(exponents[c / BLOCK]) : 0.0f, c, C, v);
}
#endif

}  // namespace tape
}  // namespace ullis
