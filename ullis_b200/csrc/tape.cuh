// The 8-bit tape: what one block of 32 channels of a row is kept as.
//
// e = the smallest integer of -126 .. 121 with 127 * 2^e >= max |x| of the block (121 where none has), codes round(x * 2^-e)
// (ties to even, int8, kept within +/-127: beyond them lie only the last values of f32, whose next step would be 2^128), the
// exponent as the byte e + 127; a code stands for code * 2^e.  A step of a block is at most 2 / 127 of its largest value, and the
// steps are powers of two: packing divides exactly, a code is exact in bf16 and f32, and scaling by 2^e rounds nothing, so an
// 8-bit operand goes through the tensor cores as the number it stands for.  A block with a value that is not finite has the
// byte 255 and stands for NaN throughout.
//
// Kernels take a row in chunks of 16 bytes, one per thread: four channels in f32, eight in 16 bits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ullis {
namespace tape {

constexpr uint32_t BLOCK = 32;
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

// The channels of a chunk as they lie in memory: 16 bytes, so that neighbouring threads read and write neighbouring pieces.
template <typename T>
constexpr int CHUNK = 16 / (int)sizeof(T);
template <typename T>
struct Raw {
    uint4 q;
    __device__ __forceinline__ void unpack(float (&v)[CHUNK<T>]) const {
        const T* t = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int i = 0; i < CHUNK<T>; ++i) v[i] = to_float(t[i]);
    }
};
// From channel c on of a row of `C`; past its end zeros.  VEC: rows start on 16 bytes and C is a multiple of 8, so a chunk is whole or
// absent.
template <bool VEC, typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* row, uint32_t c, uint32_t C) {
    Raw<T> r;
    r.q = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (VEC) {
        if (c < C) r.q = *reinterpret_cast<const uint4*>(row + c);
    } else {
        T* t = reinterpret_cast<T*>(&r.q);
#pragma unroll
        for (int i = 0; i < CHUNK<T>; ++i)
            if (c + i < C) t[i] = row[c + i];
    }
    return r;
}
// N FP16 numbers (weights), N = 4 or 8
template <bool VEC, int N>
__device__ __forceinline__ void load_halves(const uint16_t* row, uint32_t c, uint32_t C, float (&v)[N]) {
    uint32_t w[N / 2] = {};
    if constexpr (VEC) {
        if (c < C) {
            if constexpr (N == 8) {
                const uint4 t = *reinterpret_cast<const uint4*>(row + c);
                w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
            } else {
                const uint2 t = *reinterpret_cast<const uint2*>(row + c);
                w[0] = t.x; w[1] = t.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < C) w[i >> 1] |= (uint32_t)row[c + i] << (16 * (i & 1));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __half2float(__ushort_as_half((uint16_t)(w[i >> 1] >> (16 * (i & 1)))));
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_chunk(T* row, uint32_t c, uint32_t C, const float (&v)[CHUNK<T>]) {
    if constexpr (VEC) {
        if (c >= C) return;
        uint4 w;
        T* t = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < CHUNK<T>; ++i) t[i] = from_float<T>(v[i]);
        *reinterpret_cast<uint4*>(row + c) = w;
    } else {
#pragma unroll
        for (int i = 0; i < CHUNK<T>; ++i)
            if (c + i < C) row[c + i] = from_float<T>(v[i]);
    }
}
// The exponent byte of the block whose chunks of N channels lie in 32 / N neighbouring lanes.
__device__ __forceinline__ float larger(float a, float b) {   // of a and |b|, NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}
template <int N>
__device__ __forceinline__ uint32_t block_exponent(const float (&v)[N]) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = larger(top, v[i]);
    uint32_t bits = __float_as_uint(top) & 0x7FFFFFFFu;   // (of NaN: above infinity)
#pragma unroll
    for (int o = 1; o < (int)BLOCK / N; o <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    return exponent_byte(bits);
}
// Codes of a block with this exponent byte.  x * 2^-e + 1.5 * 2^23 is rounded to whole numbers by the addition (ties to even; the
// product is exact), and its lowest byte is the code: an FMA instead of a multiplication and a conversion, which goes at a quarter
// of its rate and, with the two bounds, made LayerNorm with the tape issue-bound (131072 x 512 bf16 78 us, so 60).
template <int N>
__device__ __forceinline__ void codes_of(const float (&v)[N], uint32_t byte, uint32_t (&w)[N / 4]) {
    const float inverse = inverse_power(byte);
    uint32_t r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = __float_as_uint(fmaf(v[i], inverse, 12582912.0f));
    if (byte >= 248u) {   // the last exponent, above which lies what no code reaches, or not finite: hardly ever
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = byte == NOT_FINITE ? 0u : (uint32_t)min(max(__float2int_rn(v[i] * inverse), -127), 127);
    }
#pragma unroll
    for (int k = 0; k < N / 4; ++k)
        w[k] = __byte_perm(__byte_perm(r[k * 4], r[k * 4 + 1], 0x0040), __byte_perm(r[k * 4 + 2], r[k * 4 + 3], 0x0040), 0x5410);
}
template <bool VEC, int N>
__device__ __forceinline__ void store_codes(uint8_t* codes, uint32_t c, uint32_t C, const float (&v)[N], uint32_t byte) {
    uint32_t w[N / 4];
    codes_of(v, byte, w);
    if constexpr (VEC) {
        if (c >= C) return;
        if constexpr (N == 8) *reinterpret_cast<uint2*>(codes + c) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(codes + c) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < C) codes[c + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}
// N codes times `step`; past the row's end zeros (whatever the step).
template <int N>
__device__ __forceinline__ void values_of(const uint32_t (&w)[N / 4], float step, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * step;
}
template <bool VEC, int N>
__device__ __forceinline__ void raw_codes(const uint8_t* codes, uint32_t c, uint32_t C, uint32_t (&w)[N / 4]) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) w[k] = 0;
    if constexpr (VEC) {
        if (c < C) {
            if constexpr (N == 8) {
                const uint2 t = *reinterpret_cast<const uint2*>(codes + c);
                w[0] = t.x; w[1] = t.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t*>(codes + c);
            }
        }
    } else {
        uint32_t t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = c + i < C ? codes[c + i] : 0u;
#pragma unroll
        for (int i = 0; i < N; ++i) w[i >> 2] |= t[i] << (8 * (i & 3));
    }
}
template <bool VEC, int N>
__device__ __forceinline__ void load_codes(const uint8_t* codes, float step, uint32_t c, uint32_t C, float (&v)[N]) {
    uint32_t w[N / 4];
    raw_codes<VEC, N>(codes, c, C, w);
    if constexpr (VEC) {
        values_of(w, c < C ? step : 0.0f, v);
    } else {
        values_of(w, step, v);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i >= C) v[i] = 0.0f;
    }
}
#endif

}  // namespace tape
}  // namespace ullis
