// Activations kept in 8 bits and LayerNorm over them.  All of these kernels are bound by memory: each reads its inputs once,
// keeps a row in registers and writes its outputs once.  131072 x 512 in bf16: LayerNorm 59 us (337 MB, 5.7 TB/s), its backward pass
// 92 (471 MB, 5.1 TB/s; 72 % of the issue slots); 16384 x 512 in f32: 14.4 and 19.6 us, 4.5 for the columns' sums.
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
// PER_THREAD chunks per thread, their loads in flight together; `per_row` chunks, whole blocks of them.  us for pack and unpack with
// one / two / four: 16384 x 512 f32 10.7, 9.9 / 9.5, 8.5 / 9.7, 9.6; 131072 x 512 f32 76, 94 / 64, 76 / 65, 79; 7655 x 1000 bf16
// 5.9, 5.5 / 5.9, 5.5 / 7.3, 6.3.
constexpr int PER_THREAD = 2;
struct Place {
    size_t row;
    uint32_t c;
};
template <typename T>
__device__ __forceinline__ Place place_of(int k, uint32_t per_row) {
    const size_t item = ((size_t)blockIdx.x * PER_THREAD + k) * THREADS + threadIdx.x;
    const size_t row = item >> 32 ? item / per_row : (uint32_t)item / per_row;
    return Place{row, (uint32_t)(item - row * per_row) * CHUNK<T>};
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS)
tape_pack_kernel(const T* __restrict__ x, size_t stride, uint32_t rows, uint32_t C, uint32_t per_row, uint8_t* __restrict__ codes,
                 uint8_t* __restrict__ exponents) {
    chain_entry();
    Place p[PER_THREAD];
    Raw<T> raw[PER_THREAD];
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) {
        p[k] = place_of<T>(k, per_row);
        raw[k] = load_raw<VEC>(x + p[k].row * stride, p[k].c, p[k].row < rows ? C : 0u);
    }
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) {
        float v[CHUNK<T>];
        raw[k].unpack(v);
        const uint32_t byte = block_exponent(v);
        if (p[k].row >= rows) continue;
        store_codes<VEC>(codes + p[k].row * C, p[k].c, C, v, byte);
        if (p[k].c % BLOCK == 0) exponents[p[k].row * ((C + BLOCK - 1) / BLOCK) + p[k].c / BLOCK] = (uint8_t)byte;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS)
tape_unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, uint32_t rows, uint32_t C, uint32_t per_row,
                   T* __restrict__ x, size_t stride) {
    chain_entry();
    Place p[PER_THREAD];
    float v[PER_THREAD][CHUNK<T>];
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) {
        p[k] = place_of<T>(k, per_row);
        const bool in = p[k].row < rows && p[k].c < C;
        load_codes<VEC>(codes + p[k].row * C, in ? power(exponents[p[k].row * ((C + BLOCK - 1) / BLOCK) + p[k].c / BLOCK]) : 0.0f, p[k].c, in ? C : 0u,
                        v[k]);
    }
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k)
        if (p[k].row < rows) store_chunk<VEC>(x + p[k].row * stride, p[k].c, C, v[k]);
}

// ------------------------------------------------------------------------------------------------ LayerNorm
// G warps have a row, N chunks to a lane; a CTA of max(8, G) warps has as many rows as fit.
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

// Warps walk over the rows with weight and bias in registers and the next row on its way.
template <typename T, bool VEC, int G, int N>
__global__ void __launch_bounds__(32 * cta_warps<G>(), G > 8 ? 1 : 3)
tape_layer_norm_kernel(const T* __restrict__ x, size_t stride, const uint16_t* __restrict__ weight, const uint16_t* __restrict__ bias,
                       uint32_t rows, uint32_t C, T* __restrict__ y, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents) {
    chain_entry();
    constexpr uint32_t ROWS = cta_warps<G>() / G;
    __shared__ float shared[cta_warps<G>()][1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int CH = CHUNK<T>;
    constexpr uint32_t NEXT = G * 32 * CH;   // channels from a lane's chunk to its next
    const uint32_t c0 = (uint32_t)(warp % G * 32 + lane) * CH, blocks = (C + BLOCK - 1) / BLOCK;
    const float each = 1.0f / (float)C;
    size_t row = (size_t)blockIdx.x * ROWS + warp / G;
    Raw<T> ahead[N];
    const auto fetch = [&]() {
#pragma unroll
        for (int i = 0; i < N; ++i) ahead[i] = load_raw<VEC>(x + row * stride, c0 + i * NEXT, row < rows ? C : 0u);
    };
    fetch();
    float w[N][CH], b[N][CH];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        load_halves<VEC>(weight, c0 + i * NEXT, C, w[i]);
        load_halves<VEC>(bias, c0 + i * NEXT, C, b[i]);
    }
    for (size_t r0 = (size_t)blockIdx.x * ROWS; r0 < rows; r0 += (size_t)gridDim.x * ROWS) {   // (the same rounds for the whole CTA)
        const size_t now = row;
        const bool here = now < rows;
        float v[N][CH];
        float sum[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < N; ++i) ahead[i].unpack(v[i]);
        row += (size_t)gridDim.x * ROWS;
        fetch();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * NEXT, byte = block_exponent(v[i]);
            if (here) {
                store_codes<VEC>(codes + now * C, c, C, v[i], byte);
                if (c % BLOCK == 0 && c < C) exponents[now * blocks + c / BLOCK] = (uint8_t)byte;
            }
#pragma unroll
            for (int e = 0; e < CH; ++e) sum[0] += v[i][e];
        }
        row_sums<G, 1>(sum, shared, warp, lane);
        const float mean = sum[0] * each;
        float square[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * NEXT;
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                v[i][e] = (VEC ? c : c + e) < C ? v[i][e] - mean : 0.0f;
                square[0] += v[i][e] * v[i][e];
            }
        }
        row_sums<G, 1>(square, shared, warp, lane);
        if (!here) continue;
        const float inv = 1.0f / sqrtf(square[0] * each + LN_EPS);
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int e = 0; e < CH; ++e) v[i][e] = v[i][e] * inv * w[i][e] + b[i][e];
            store_chunk<VEC>(y + now * C, c0 + i * NEXT, C, v[i]);
        }
    }
}

// What a lane needs of a row in the backward pass is copied to shared memory of its own two rows ahead (STAGES - 1): the row's own
// registers and the columns' sums leave none for loads in flight, and two CTAs to an SM.  Rows that do not start on 16 bytes are
// loaded when they are needed.
constexpr int STAGES = 3;
template <typename T, int N>
constexpr size_t stage_bytes() { return (size_t)N * (CHUNK<T> + 32); }   // per lane: codes, gy, residual
template <typename T, bool VEC, int G, int N>
constexpr size_t backward_smem() {
    const size_t ring = VEC ? STAGES * stage_bytes<T, N>() : 0, sums = (size_t)N * CHUNK<T> * 4;
    return 32 * cta_warps<G>() * (ring > sums ? ring : sums);
}
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}

// A CTA walks over the rows and keeps the columns' sums in registers; what its rows leave goes to part [CTA][2][C].
template <typename T, bool VEC, int G, int N>
__global__ void __launch_bounds__(32 * cta_warps<G>(), G > 8 ? 1 : 2)
tape_layer_norm_backward_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, const T* __restrict__ gy,
                                size_t gy_stride, const uint16_t* __restrict__ weight, const T* __restrict__ residual,
                                size_t residual_stride, uint32_t rows, uint32_t C, T* __restrict__ gx, float* __restrict__ part) {
    chain_entry();
    constexpr int WARPS = cta_warps<G>(), ROWS = WARPS / G, THREADS_ = WARPS * 32;
    constexpr int CH = CHUNK<T>;
    constexpr uint32_t NEXT = G * 32 * CH;
    extern __shared__ __align__(16) uint8_t ring[];   // [stage][gy, residual][chunk][thread] of 16 bytes, [stage][chunk][thread] of codes
    __shared__ float shared[WARPS][3];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c0 = (uint32_t)(warp % G * 32 + lane) * CH, blocks = (C + BLOCK - 1) / BLOCK;
    const size_t step = (size_t)gridDim.x * ROWS, first = (size_t)blockIdx.x * ROWS + warp / G;
    const auto piece = [&](int stage, int which, int i) {   // which: 0 gy, 1 residual
        return reinterpret_cast<uint4*>(ring) + ((stage * 2 + which) * N + i) * THREADS_ + threadIdx.x;
    };
    const auto code_piece = [&](int stage, int i) {   // CH bytes
        return reinterpret_cast<uint32_t*>(ring + (size_t)STAGES * 2 * N * 16 * THREADS_) + ((stage * N + i) * THREADS_ + threadIdx.x) * (CH / 4);
    };
    const auto fetch = [&](size_t row, int stage) {
        if (VEC && row < rows) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t c = c0 + i * NEXT;
                if (c >= C) continue;
                copy_async<16>(piece(stage, 0, i), gy + row * gy_stride + c);
                if (residual) copy_async<16>(piece(stage, 1, i), residual + row * residual_stride + c);
                copy_async<CH>(code_piece(stage, i), codes + row * C + c);
            }
        }
        if (VEC) asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(first + s * step, s);
    const auto exponents_of = [&](size_t row, uint32_t (&e)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * NEXT;
            e[i] = row < rows && c < C ? exponents[row * blocks + c / BLOCK] : 0u;
        }
    };
    uint32_t e_ahead[N];
    exponents_of(first, e_ahead);
    float w[N][CH], gw[N][CH] = {}, gb[N][CH] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) load_halves<VEC>(weight, c0 + i * NEXT, C, w[i]);
    const float each = 1.0f / (float)C;
    int stage = 0;
    size_t row = first;
    for (size_t r0 = (size_t)blockIdx.x * ROWS; r0 < rows; r0 += step, row += step) {
        const bool here = row < rows;
        float x[N][CH], g[N][CH];
        float sum[1] = {0.0f};
        fetch(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
        if (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * NEXT, end = here ? C : 0u;
            const float scale = c < end ? power(e_ahead[i]) : 0.0f;
            if constexpr (VEC) {
                Raw<T> r{};
                uint32_t k[CH / 4] = {};
                if (c < end) {
                    r.q = *piece(stage, 0, i);
#pragma unroll
                    for (int q = 0; q < CH / 4; ++q) k[q] = code_piece(stage, i)[q];
                }
                r.unpack(g[i]);
                values_of(k, scale, x[i]);
            } else {
                load_raw<false>(gy + row * gy_stride, c, end).unpack(g[i]);
                load_codes<false>(codes + row * C, scale, c, end, x[i]);
            }
        }
        exponents_of(row + step, e_ahead);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < CH; ++e) sum[0] += x[i][e];
        row_sums<G, 1>(sum, reinterpret_cast<float(*)[1]>(shared), warp, lane);
        const float mean = sum[0] * each;
        float s[3] = {0.0f, 0.0f, 0.0f};   // (x - mean)^2, dx, dx * (x - mean)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = c0 + i * NEXT;
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                x[i][e] = (VEC ? c : c + e) < C ? x[i][e] - mean : 0.0f;
                const float dx = g[i][e] * w[i][e];
                s[0] += x[i][e] * x[i][e];
                s[1] += dx;
                s[2] += dx * x[i][e];
            }
        }
        row_sums<G, 3>(s, shared, warp, lane);
        if (here) {
            const float inv = 1.0f / sqrtf(s[0] * each + LN_EPS);
            const float mean_dx = s[1] * each, mean_dxh = s[2] * inv * each;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t c = c0 + i * NEXT;
                float old[CH] = {};
                if (residual && c < C) {
                    Raw<T> r;
                    if constexpr (VEC) r.q = *piece(stage, 1, i);
                    else r = load_raw<false>(residual + row * residual_stride, c, C);
                    r.unpack(old);
                }
#pragma unroll
                for (int e = 0; e < CH; ++e) {
                    const float xh = x[i][e] * inv;
                    gw[i][e] += g[i][e] * xh;
                    gb[i][e] += g[i][e];
                    old[e] += inv * (g[i][e] * w[i][e] - mean_dx - xh * mean_dxh);
                }
                store_chunk<VEC>(gx + row * C, c, C, old);
            }
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    if (VEC) asm volatile("cp.async.wait_all;" ::: "memory");
    // the CTA's rows side by side, then one sum per column: thread -> (chunk lane of the row, chunk, element)
    float* columns = reinterpret_cast<float*>(ring);   // [N * CH][THREADS_]
    float* out = part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < CH; ++e) columns[(i * CH + e) * THREADS_ + threadIdx.x] = which ? gb[i][e] : gw[i][e];
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < C; c += THREADS_) {
            const uint32_t chunk = c / CH, i = chunk / (G * 32), at = chunk % (G * 32);
            float all = 0.0f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) all += columns[(i * CH + c % CH) * THREADS_ + r * G * 32 + at];
            out[(size_t)which * C + c] = all;
        }
    }
}

// out[c] = sum over p of part[p][c], c < 2 C: first the weights' gradient, then the biases'.  Eight columns to a CTA, 128 threads to a
// column, their loads in flight together (eight threads one after the other: 10.8 us for 296 parts of 1024, a third of the pass).
__global__ void __launch_bounds__(1024)
tape_columns_kernel(const float* __restrict__ part, uint32_t parts, uint32_t C, float* __restrict__ g_weight, float* __restrict__ g_bias) {
    chain_entry();
    __shared__ float sums[32][8];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 8 + (lane & 7);
    float acc = 0.0f;
    if (c < 2 * C) {
#pragma unroll 4
        for (uint32_t p = warp * 4 + (lane >> 3); p < parts; p += 128) acc += part[(size_t)p * 2 * C + c];
    }
    acc += __shfl_xor_sync(0xffffffffu, acc, 8);
    acc += __shfl_xor_sync(0xffffffffu, acc, 16);
    if (lane < 8) sums[warp][lane] = acc;
    __syncthreads();
    if (warp >= 8) return;
    acc = sums[lane][warp];   // a warp per column
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    const uint32_t own = blockIdx.x * 8 + warp;
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
// f(warps per row, chunks per lane): as few warps as hold the row, 16 channels to a lane from 257 on (8 below)
template <typename T, typename F>
void by_width(size_t channels, F&& f) {
    using std::integral_constant;
    constexpr int HALF = 8 / CHUNK<T>, FULL = 16 / CHUNK<T>;
    if (channels <= 256) f(integral_constant<int, 1>{}, integral_constant<int, HALF>{});
    else if (channels <= 512) f(integral_constant<int, 1>{}, integral_constant<int, FULL>{});
    else if (channels <= 1024) f(integral_constant<int, 2>{}, integral_constant<int, FULL>{});
    else if (channels <= 2048) f(integral_constant<int, 4>{}, integral_constant<int, FULL>{});
    else if (channels <= 4096) f(integral_constant<int, 8>{}, integral_constant<int, FULL>{});
    else f(integral_constant<int, 16>{}, integral_constant<int, FULL>{});
}
size_t rows_per_cta(size_t channels) {
    size_t rows = 0;
    by_width<float>(channels, [&](auto g, auto) { rows = cta_warps<decltype(g)::value>() / decltype(g)::value; });
    return rows;
}
// CTAs that walk over the rows in the backward pass: two per SM
size_t backward_ctas(const ullis_cuda_runtime* rt, size_t rows, size_t channels) {
    return std::min<size_t>((rows + rows_per_cta(channels) - 1) / rows_per_cta(channels), 2 * (size_t)rt->sm_count);
}

}  // namespace

void tape_pack(const Stream& s, int dtype, Rows x, size_t rows, size_t channels, uint8_t* codes, uint8_t* exponents) {
    const uint32_t per_row = (uint32_t)(blocks_of(channels) * BLOCK * size_of(dtype) / 16);
    const unsigned grid = (unsigned)((rows * per_row + THREADS * PER_THREAD - 1) / (THREADS * PER_THREAD));
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
    const uint32_t per_row = (uint32_t)(blocks_of(channels) * BLOCK * size_of(dtype) / 16);
    const unsigned grid = (unsigned)((rows * per_row + THREADS * PER_THREAD - 1) / (THREADS * PER_THREAD));
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
    // three CTAs to an SM walk over the rows
    const unsigned grid = (unsigned)std::min<size_t>((rows + rows_per_cta(channels) - 1) / rows_per_cta(channels), 3 * (size_t)s.rt->sm_count);
    const bool vec = rows_aligned(x, dtype) && channels % 8 == 0 && aligned(codes, 8) && aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16);
    by_type(dtype, [&](auto t) {
        by_flag(vec, [&](auto v) {
            using T = decltype(t);
            by_width<T>(channels, [&](auto g, auto n) {
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
            using T = decltype(t);
            by_width<T>(channels, [&](auto g, auto n) {
                constexpr bool VEC = decltype(v)::value;
                constexpr int G = decltype(g)::value, N = decltype(n)::value;
                constexpr size_t smem = backward_smem<T, VEC, G, N>();
                const auto kernel = tape_layer_norm_backward_kernel<T, VEC, G, N>;
                if (smem > 48 * 1024) ULLIS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
                s.chain("tape_layer_norm_backward", kernel, (unsigned)ctas, 32 * cta_warps<G>(), smem, codes, exponents, static_cast<const T*>(gy.data), gy.stride, weight,
                        static_cast<const T*>(residual.data), residual.stride, (uint32_t)rows, (uint32_t)channels, static_cast<T*>(gx),
                        part);
            });
        });
    });
    s.chain("tape_columns", tape_columns_kernel, (unsigned)((2 * channels + 7) / 8), 1024, 0, part, (uint32_t)ctas, (uint32_t)channels,
            g_weight, g_bias);
}

}  // namespace dev
}  // namespace ullis
