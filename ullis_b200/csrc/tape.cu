// Activations kept in 8 bits and LayerNorm over them.  All of these kernels are bound by memory: each reads its inputs once,
// keeps a row in registers and writes its outputs once.
//
// LayerNorm (reference src/model.rs:259-276): y = (x - mean) * inv * w + b, inv = 1 / sqrt(var + 1e-5).  Its backward pass
// (src/model.rs:270-315) from the tape, with xh = (x^ - mean^) * inv^ of what the codes stand for and dx = gy * w:
//   gx = residual + inv^ * (dx - mean(dx) - xh * mean(dx * xh)),  g_weight = sum over rows of gy * xh,  g_bias = sum of gy.
#include "tape.cuh"

#include <algorithm>

#include "device_ops.hpp"

namespace ullis {
namespace dev {
namespace {

using namespace tape;

constexpr float LN_EPS = 1e-5f;   // src/model.rs:22
constexpr int THREADS = 256;

// ------------------------------------------------------------------------------------------------ pack, unpack
// A chunk of eight channels per thread; `per_row` chunks, a multiple of four.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS)
tape_pack_kernel(const T* __restrict__ x, size_t stride, uint32_t rows, uint32_t C, uint32_t per_row, uint8_t* __restrict__ codes,
                 uint8_t* __restrict__ exponents) {
    chain_entry();
    const size_t item = (size_t)blockIdx.x * THREADS + threadIdx.x;
    const size_t row = item >> 32 ? item / per_row : (uint32_t)item / per_row;
    const uint32_t c = (uint32_t)(item - row * per_row) * CHUNK;
    float v[8] = {};
    if (row < rows) load8<VEC>(x + row * stride, c, C, v);
    const uint32_t byte = quad_exponent(v);
    if (row >= rows) return;
    store_codes<VEC>(codes + row * C, c, C, v, inverse_power(byte));
    if ((threadIdx.x & 3) == 0) exponents[row * (per_row / 4) + c / BLOCK] = (uint8_t)byte;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS)
tape_unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, uint32_t rows, uint32_t C, uint32_t per_row,
                   T* __restrict__ x, size_t stride) {
    chain_entry();
    const size_t item = (size_t)blockIdx.x * THREADS + threadIdx.x;
    const size_t row = item >> 32 ? item / per_row : (uint32_t)item / per_row;
    if (row >= rows) return;
    const uint32_t c = (uint32_t)(item - row * per_row) * CHUNK;
    float v[8];
    load_codes<VEC>(codes + row * C, exponents + row * (per_row / 4), c, C, v);
    store8<VEC>(x + row * stride, c, C, v);
}

// ------------------------------------------------------------------------------------------------ LayerNorm
// G warps have a row, N chunks of eight channels to a lane; a CTA of max(8, G) warps has as many rows as fit.
template <int G>
constexpr int cta_warps() { return G > 8 ? G : 8; }

// Sums of K values over the G warps of a row; every thread of the CTA takes part.
template <int G, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*shared)[K], int warp, int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if constexpr (G > 1) {
        __syncthreads();   // what an earlier sum left there has been read
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) shared[warp][k] = v[k];
        __syncthreads();
        const int first = warp / G * G;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[k] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) v[k] += shared[first + g][k];
        }
    }
}

template <typename T, bool VEC, int G, int N>
__global__ void __launch_bounds__(32 * cta_warps<G>())
tape_layer_norm_kernel(const T* __restrict__ x, size_t stride, const uint16_t* __restrict__ weight, const uint16_t* __restrict__ bias,
                       uint32_t rows, uint32_t C, T* __restrict__ y, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents) {
    chain_entry();
    __shared__ float shared[cta_warps<G>()][1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t row = (size_t)blockIdx.x * (cta_warps<G>() / G) + warp / G;
    const bool here = row < rows;
    const uint32_t c0 = (uint32_t)(warp % G * 32 + lane) * CHUNK;
    float v[N][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) load8<VEC>(x + row * stride, c0 + i * (G * 32 * CHUNK), here ? C : 0u, v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t c = c0 + i * (G * 32 * CHUNK), byte = quad_exponent(v[i]);
        if (here) {
            store_codes<VEC>(codes + row * C, c, C, v[i], inverse_power(byte));
            if ((lane & 3) == 0 && c < C) exponents[row * ((C + BLOCK - 1) / BLOCK) + c / BLOCK] = (uint8_t)byte;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[0] += v[i][e];
    }
    row_sums<G, 1>(sum, shared, warp, lane);
    const float mean = sum[0] / (float)C;
    float square[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t c = c0 + i * (G * 32 * CHUNK);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[i][e] -= mean;
            if (c + e < C) square[0] += v[i][e] * v[i][e];
        }
    }
    row_sums<G, 1>(square, shared, warp, lane);
    if (!here) return;
    const float inv = 1.0f / sqrtf(square[0] / (float)C + LN_EPS);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t c = c0 + i * (G * 32 * CHUNK);
        float w[8], b[8];
        load8<VEC>(reinterpret_cast<const __half*>(weight), c, C, w);
        load8<VEC>(reinterpret_cast<const __half*>(bias), c, C, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * inv * w[e] + b[e];
        store8<VEC>(y + row * C, c, C, v[i]);
    }
}

// A CTA walks over the rows and keeps the columns' sums in registers; what its rows leave goes to part [CTA][2][C].
template <typename T, bool VEC, int G, int N>
__global__ void __launch_bounds__(32 * cta_warps<G>())
tape_layer_norm_backward_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, const T* __restrict__ gy,
                                size_t gy_stride, const uint16_t* __restrict__ weight, const T* __restrict__ residual,
                                size_t residual_stride, uint32_t rows, uint32_t C, T* __restrict__ gx, float* __restrict__ part) {
    chain_entry();
    constexpr int WARPS = cta_warps<G>(), ROWS = WARPS / G;
    __shared__ float shared[WARPS][3];
    __shared__ float columns[N * 8][WARPS * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c0 = (uint32_t)(warp % G * 32 + lane) * CHUNK, blocks = (C + BLOCK - 1) / BLOCK;
    float gw[N][8] = {}, gb[N][8] = {};
    const float each = 1.0f / (float)C;
    for (size_t r0 = (size_t)blockIdx.x * ROWS; r0 < rows; r0 += (size_t)gridDim.x * ROWS) {
        const size_t row = r0 + warp / G;
        const bool here = row < rows;
        const uint32_t end = here ? C : 0u;
        float x[N][8], g[N][8], old[N][8];
        float sum[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * (G * 32 * CHUNK);
            load_codes<VEC>(codes + row * C, exponents + row * blocks, c, end, x[i]);
            load8<VEC>(gy + row * gy_stride, c, end, g[i]);
            if (residual) load8<VEC>(residual + row * residual_stride, c, end, old[i]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) old[i][e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[0] += x[i][e];
        row_sums<G, 1>(sum, reinterpret_cast<float(*)[1]>(shared), warp, lane);
        const float mean = sum[0] * each;
        float s[3] = {0.0f, 0.0f, 0.0f};   // (x - mean)^2, dx, dx * (x - mean)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * (G * 32 * CHUNK);
            float w[8];
            load8<VEC>(reinterpret_cast<const __half*>(weight), c, C, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[i][e] = c + e < C ? x[i][e] - mean : 0.0f;
                const float dx = g[i][e] * w[e];
                s[0] += x[i][e] * x[i][e];
                s[1] += dx;
                s[2] += dx * x[i][e];
            }
        }
        row_sums<G, 3>(s, shared, warp, lane);
        const float inv = 1.0f / sqrtf(s[0] * each + LN_EPS);
        const float mean_dx = s[1] * each, mean_dxh = s[2] * inv * each;
        if (!here) continue;   // (the whole CTA leaves the loop after the same round)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * (G * 32 * CHUNK);
            float w[8];
            load8<VEC>(reinterpret_cast<const __half*>(weight), c, C, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float xh = x[i][e] * inv;
                gw[i][e] += g[i][e] * xh;
                gb[i][e] += g[i][e];
                old[i][e] += inv * (g[i][e] * w[e] - mean_dx - xh * mean_dxh);
            }
            store8<VEC>(gx + row * C, c, C, old[i]);
        }
    }
    // the CTA's rows side by side, then one sum per column: thread -> (chunk lane of the row, chunk, element)
    float* out = part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) columns[i * 8 + e][threadIdx.x] = which ? gb[i][e] : gw[i][e];
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < C; c += WARPS * 32) {
            const uint32_t chunk = c / CHUNK, i = chunk / (G * 32), at = chunk % (G * 32);
            float all = 0.0f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) all += columns[i * 8 + c % CHUNK][r * G * 32 + at];
            out[(size_t)which * C + c] = all;
        }
    }
}

// out[c] = sum over p of part[p][c], c < 2 C: first the weights' gradient, then the biases'.  32 columns to a CTA, 32 threads to a
// column, their loads in flight together (eight threads one after the other: 10.8 us for 296 parts of 1024, a third of the pass).
__global__ void __launch_bounds__(1024)
tape_columns_kernel(const float* __restrict__ part, uint32_t parts, uint32_t C, float* __restrict__ g_weight, float* __restrict__ g_bias) {
    chain_entry();
    __shared__ float sums[32][33];
    const uint32_t lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float acc = 0.0f;
    if (c < 2 * C) {
#pragma unroll 10
        for (uint32_t p = slice; p < parts; p += 32) acc += part[(size_t)p * 2 * C + c];
    }
    sums[slice][lane] = acc;
    __syncthreads();
    acc = sums[lane][slice];   // a warp per column
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    const uint32_t own = blockIdx.x * 32 + slice;
    if (lane == 0 && own < 2 * C) (own < C ? g_weight : g_bias)[own < C ? own : own - C] = acc;
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool rows_aligned(Rows x, int dtype) { return aligned(x.data, 16) && x.stride * size_of(dtype) % 16 == 0; }

template <typename F>
void by_type(int dtype, F&& f) {
    if (dtype == F32) f(float{});
    else if (dtype == F16) f(__half{});
    else f(__nv_bfloat16{});
}
template <typename F>
void by_flag(bool flag, F&& f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}
// f(warps per row, chunks per lane): as few warps as hold the row, two chunks of eight to a lane from 257 channels on
template <typename F>
void by_width(size_t channels, F&& f) {
    using std::integral_constant;
    if (channels <= 256) f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (channels <= 512) f(integral_constant<int, 1>{}, integral_constant<int, 2>{});
    else if (channels <= 1024) f(integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (channels <= 2048) f(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (channels <= 4096) f(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
}
size_t rows_per_cta(size_t channels) {
    size_t rows = 0;
    by_width(channels, [&](auto g, auto) { rows = cta_warps<decltype(g)::value>() / decltype(g)::value; });
    return rows;
}
// CTAs that walk over the rows in the backward pass: two per SM
size_t backward_ctas(const ullis_cuda_runtime* rt, size_t rows, size_t channels) {
    return std::min<size_t>((rows + rows_per_cta(channels) - 1) / rows_per_cta(channels), 2 * (size_t)rt->sm_count);
}

}  // namespace

void tape_pack(const Stream& s, int dtype, Rows x, size_t rows, size_t channels, uint8_t* codes, uint8_t* exponents) {
    const uint32_t per_row = (uint32_t)blocks_of(channels) * 4;
    const unsigned grid = (unsigned)((rows * per_row + THREADS - 1) / THREADS);
    const bool vec = rows_aligned(x, dtype) && channels % 8 == 0 && aligned(codes, 8);
    by_type(dtype, [&](auto t) {
        by_flag(vec, [&](auto v) {
            using T = decltype(t);
            s.chain("tape_pack", tape_pack_kernel<T, decltype(v)::value>, grid, THREADS, 0, static_cast<const T*>(x.data), x.stride,
                    (uint32_t)rows, (uint32_t)channels, per_row, codes, exponents);
        });
    });
}

void tape_unpack(const Stream& s, int dtype, const uint8_t* codes, const uint8_t* exponents, size_t rows, size_t channels, void* x,
                 size_t x_stride) {
    const uint32_t per_row = (uint32_t)blocks_of(channels) * 4;
    const unsigned grid = (unsigned)((rows * per_row + THREADS - 1) / THREADS);
    const bool vec = rows_aligned(Rows{x, x_stride}, dtype) && channels % 8 == 0 && aligned(codes, 8);
    by_type(dtype, [&](auto t) {
        by_flag(vec, [&](auto v) {
            using T = decltype(t);
            s.chain("tape_unpack", tape_unpack_kernel<T, decltype(v)::value>, grid, THREADS, 0, codes, exponents, (uint32_t)rows,
                    (uint32_t)channels, per_row, static_cast<T*>(x), x_stride);
        });
    });
}

void tape_layer_norm(const Stream& s, int dtype, Rows x, const uint16_t* weight, const uint16_t* bias, size_t rows, size_t channels,
                     void* y, uint8_t* codes, uint8_t* exponents) {
    const unsigned grid = (unsigned)((rows + rows_per_cta(channels) - 1) / rows_per_cta(channels));
    const bool vec = rows_aligned(x, dtype) && channels % 8 == 0 && aligned(codes, 8) && aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16);
    by_type(dtype, [&](auto t) {
        by_flag(vec, [&](auto v) {
            by_width(channels, [&](auto g, auto n) {
                using T = decltype(t);
                s.chain("tape_layer_norm", tape_layer_norm_kernel<T, decltype(v)::value, decltype(g)::value, decltype(n)::value>, grid,
                        32 * cta_warps<decltype(g)::value>(), 0, static_cast<const T*>(x.data), x.stride, weight, bias, (uint32_t)rows,
                        (uint32_t)channels, static_cast<T*>(y), codes, exponents);
            });
        });
    });
}

size_t tape_layer_norm_backward_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels) {
    return backward_ctas(rt, rows, channels) * 2 * channels * 4;
}

void tape_layer_norm_backward(const Stream& s, int dtype, const uint8_t* codes, const uint8_t* exponents, Rows gy, const uint16_t* weight,
                              Rows residual, size_t rows, size_t channels, void* gx, float* g_weight, float* g_bias, void* workspace) {
    const size_t ctas = backward_ctas(s.rt, rows, channels);
    float* part = static_cast<float*>(workspace);
    const bool vec = rows_aligned(gy, dtype) && (!residual.data || rows_aligned(residual, dtype)) && channels % 8 == 0 &&
                     aligned(codes, 8) && aligned(gx, 16) && aligned(weight, 16);
    by_type(dtype, [&](auto t) {
        by_flag(vec, [&](auto v) {
            by_width(channels, [&](auto g, auto n) {
                using T = decltype(t);
                s.chain("tape_layer_norm_backward",
                        tape_layer_norm_backward_kernel<T, decltype(v)::value, decltype(g)::value, decltype(n)::value>, (unsigned)ctas,
                        32 * cta_warps<decltype(g)::value>(), 0, codes, exponents, static_cast<const T*>(gy.data), gy.stride, weight,
                        static_cast<const T*>(residual.data), residual.stride, (uint32_t)rows, (uint32_t)channels, static_cast<T*>(gx),
                        part);
            });
        });
    });
    s.chain("tape_columns", tape_columns_kernel, (unsigned)((2 * channels + 31) / 32), 1024, 0, part, (uint32_t)ctas, (uint32_t)channels,
            g_weight, g_bias);
}

}  // namespace dev
}  // namespace ullis
