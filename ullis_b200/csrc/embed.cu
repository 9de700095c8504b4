// Embedding lookup and the gradient of its table, on a caller's device memory.
//
//   y[r] = scale * table[token[r]]          G[v] = scale * sum of gy[r] over the rows r with token[r] = v
//
// Both are bound by memory: the lookup reads a table row and writes a row, the gradient reads gy once and writes the table once.
// The gradient's sums have a fixed order, with no atomics: the rows of a token in rising order, in pieces where there are many.
#include <algorithm>
#include <type_traits>

#include "block_sort.cuh"
#include "device_ops.hpp"
#include "tape.cuh"

namespace ullis {
namespace dev {
namespace {

constexpr int THREADS = 256;

size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }
size_t ceil_div(size_t n, size_t by) { return (n + by - 1) / by; }
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A lane's N channels of a row: side by side from c on, read and written at once where they lie on their own size (WIDE), else
// GAP apart, so that neighbouring threads have neighbouring channels; past the row's end zeros.
template <bool WIDE, int N, int GAP, typename T>
struct Channels {
    __align__(WIDE ? sizeof(T) * N : sizeof(T)) T t[N];
    __device__ __forceinline__ void load(const T* row, uint32_t c, uint32_t C) {
        if constexpr (WIDE) {
            using Word = std::conditional_t<sizeof(T) * N == 16, uint4, uint2>;
            *reinterpret_cast<Word*>(t) = c < C ? *reinterpret_cast<const Word*>(row + c) : Word{};
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) t[i] = c + i * GAP < C ? row[c + i * GAP] : tape::from_float<T>(0.0f);
        }
    }
};
template <bool WIDE, int N, int GAP, typename T>
__device__ __forceinline__ void load_channels(const T* row, uint32_t c, uint32_t C, float (&v)[N]) {
    Channels<WIDE, N, GAP, T> r;
    r.load(row, c, C);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = tape::to_float(r.t[i]);
}
template <bool WIDE, int N, int GAP, typename T>
__device__ __forceinline__ void store_channels(T* row, uint32_t c, uint32_t C, const float (&v)[N]) {
    if constexpr (WIDE) {
        __align__(16) T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = tape::from_float<T>(v[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) * N / 16; ++i) reinterpret_cast<uint4*>(row + c)[i] = reinterpret_cast<const uint4*>(t)[i];
        if constexpr (sizeof(T) * N == 8) *reinterpret_cast<uint2*>(row + c) = *reinterpret_cast<const uint2*>(t);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i * GAP < C) row[c + i * GAP] = tape::from_float<T>(v[i]);
    }
}

// ------------------------------------------------------------------------------------------------ lookup
constexpr int PER_THREAD = 2;   // chunks, their loads in flight together
// A thread has chunks of N channels.
template <typename T, typename Y, int N>
__global__ void __launch_bounds__(THREADS)
embed_kernel(const T* __restrict__ table, size_t stride, const uint32_t* __restrict__ tokens, uint32_t ignore_id, float scale, uint32_t rows,
             uint32_t C, uint32_t vocab, uint32_t per_row, Y* __restrict__ y) {
    chain_entry();
    constexpr bool WIDE = N > 1;
    size_t row[PER_THREAD];
    uint32_t c[PER_THREAD], token[PER_THREAD];
    float v[PER_THREAD][N];
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) {
        const size_t item = ((size_t)blockIdx.x * PER_THREAD + k) * THREADS + threadIdx.x;
        row[k] = item >> 32 ? item / per_row : (uint32_t)item / per_row;
        c[k] = (uint32_t)(item - row[k] * per_row) * N;
        token[k] = row[k] < rows ? tokens[row[k]] : ignore_id;
    }
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) {
        const float other = token[k] == ignore_id ? 0.0f : NAN;
        if (token[k] != ignore_id && token[k] < vocab) {
            load_channels<WIDE, N, 1>(table + token[k] * stride, c[k], C, v[k]);
#pragma unroll
            for (int i = 0; i < N; ++i) v[k][i] *= scale;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[k][i] = other;
        }
    }
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k)
        if (row[k] < rows) store_channels<WIDE, N, 1>(y + row[k] * C, c[k], C, v[k]);
}

template <typename T, typename Y, int N>
bool embed_by(const Stream& s, Rows table, const uint32_t* tokens, uint32_t ignore_id, float scale, size_t rows, size_t C, size_t vocab, void* y) {
    if (C % N || table.stride % N || !aligned(table.data, N * sizeof(T)) || !aligned(y, N * sizeof(Y))) return false;
    const uint32_t per_row = (uint32_t)(C / N);
    s.chain("embed", embed_kernel<T, Y, N>, (unsigned)ceil_div(rows * per_row, PER_THREAD * THREADS), THREADS, 0, static_cast<const T*>(table.data),
            table.stride, tokens, ignore_id, scale, (uint32_t)rows, (uint32_t)C, (uint32_t)vocab, per_row, static_cast<Y*>(y));
    return true;
}
// As many channels to a chunk as the wider type has in 16 bytes; 16-bit rows on 8 bytes half of them; others one.
template <typename T, typename Y>
void embed_as(const Stream& s, Rows table, const uint32_t* tokens, uint32_t ignore_id, float scale, size_t rows, size_t C, size_t vocab, void* y) {
    constexpr int N = 16 / (int)(sizeof(T) > sizeof(Y) ? sizeof(T) : sizeof(Y));
    if (embed_by<T, Y, N>(s, table, tokens, ignore_id, scale, rows, C, vocab, y)) return;
    if constexpr (N == 8)
        if (embed_by<T, Y, 4>(s, table, tokens, ignore_id, scale, rows, C, vocab, y)) return;
    embed_by<T, Y, 1>(s, table, tokens, ignore_id, scale, rows, C, vocab, y);
}
template <typename T>
void embed_from(const Stream& s, int dtype, Rows table, const uint32_t* tokens, uint32_t ignore_id, float scale, size_t rows, size_t C,
                size_t vocab, void* y) {
    if (dtype == F32) embed_as<T, float>(s, table, tokens, ignore_id, scale, rows, C, vocab, y);
    else if (dtype == F16) embed_as<T, __half>(s, table, tokens, ignore_id, scale, rows, C, vocab, y);
    else embed_as<T, __nv_bfloat16>(s, table, tokens, ignore_id, scale, rows, C, vocab, y);
}

// The number of elements of a rising list below `token` (or_equal: not above it).
__device__ __forceinline__ uint32_t below(const uint32_t* list, uint32_t n, uint32_t token, bool or_equal) {
    const uint32_t limit = token + or_equal;   // (tokens are below 2^31)
    uint32_t at = 0;
    while (n > 0) {
        const uint32_t half = n >> 1;
        const bool right = list[at + half] < limit;
        at += right ? half + 1 : 0u;
        n = right ? n - half - 1 : half;
    }
    return at;
}

// ------------------------------------------------------------------------------------------------ gradient of few rows
// One launch.  CTA b has the table rows v with v % CTAs == b: it writes zeros, lists the rows whose token is one of them, sorts
// the list (a handful: a rank per entry by comparison with all others), and sums run by run with all of its threads: a group of
// threads per row of gy, the groups' sums added in their order.
constexpr uint32_t FEW = 1024;

template <typename T, int N>
__global__ void __launch_bounds__(THREADS)
embed_grad_few_kernel(const uint32_t* __restrict__ tokens, uint32_t ignore_id, const T* __restrict__ gy, size_t stride, uint32_t rows, uint32_t C,
                      uint32_t vocab, float scale, float* __restrict__ g) {
    chain_entry();
    constexpr bool WIDE = N > 1;
    __shared__ uint32_t found_token[FEW], found_row[FEW], token_at[FEW], row_at[FEW], warp_counts[THREADS / 32];
    __shared__ float sums[THREADS][N + 1];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t first = (size_t)blockIdx.x * C, step = (size_t)gridDim.x * C;
    if (C % 4 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0) {
        for (size_t at = first; at < (size_t)vocab * C; at += step)
            for (uint32_t c = threadIdx.x * 4; c < C; c += THREADS * 4) *reinterpret_cast<float4*>(g + at + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    } else {
        for (size_t at = first; at < (size_t)vocab * C; at += step)
            for (uint32_t c = threadIdx.x; c < C; c += THREADS) g[at + c] = 0.0f;
    }
    uint32_t count = 0;
    for (uint32_t base = 0; base < rows; base += THREADS) {   // (in the order of the rows)
        const uint32_t r = base + threadIdx.x, token = r < rows ? tokens[r] : ignore_id;
        const bool mine = token != ignore_id && token < vocab && token % gridDim.x == blockIdx.x;
        const uint32_t mask = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) warp_counts[warp] = __popc(mask);
        __syncthreads();
        uint32_t at = count + __popc(mask & ((1u << lane) - 1u));
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 32; ++w) {
            at += w < warp ? warp_counts[w] : 0u;
            count += warp_counts[w];
        }
        if (mine) {
            found_token[at] = token;
            found_row[at] = r;
        }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
        const uint32_t token = found_token[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < count; ++j) rank += found_token[j] < token || (found_token[j] == token && j < i);
        token_at[rank] = token;
        row_at[rank] = found_row[i];
    }
    __syncthreads();   // (the zeros too, of which some are written over)
    const uint32_t chunks = (C + N - 1) / N, width = min(chunks, (uint32_t)THREADS), groups = THREADS / width;
    const uint32_t group = threadIdx.x / width, chunk = threadIdx.x - group * width;
    for (uint32_t i = 0; i < count;) {
        const uint32_t token = token_at[i];
        const uint32_t end = i + below(token_at + i, count - i, token, true);
        for (uint32_t base = 0; base < chunks; base += width) {
            const uint32_t c = (base + chunk) * N;
            const bool in = group < groups && c < C;
            float sum[N] = {};
            if (in) {
                uint32_t k = i + group;
                for (; k + 3 * groups < end; k += 4 * groups) {
                    float v[4][N];
#pragma unroll
                    for (int u = 0; u < 4; ++u) load_channels<WIDE, N, 1>(gy + row_at[k + u * groups] * stride, c, C, v[u]);
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int e = 0; e < N; ++e) sum[e] += v[u][e];
                }
                for (; k < end; k += groups) {
                    float v[N];
                    load_channels<WIDE, N, 1>(gy + row_at[k] * stride, c, C, v);
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] += v[e];
                }
            }
            const uint32_t parts = min(groups, end - i);   // of the groups, those that had a row
            if (parts > 1) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < N; ++e) sums[threadIdx.x][e] = sum[e];
                __syncthreads();
                if (group == 0)
                    for (uint32_t k = 1; k < parts; ++k)
#pragma unroll
                        for (int e = 0; e < N; ++e) sum[e] += sums[k * width + chunk][e];
            }
            if (group == 0 && c < C) {
                float* to = g + (size_t)token * C;
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (c + e < C) to[c + e] = sum[e] * scale;
            }
        }
        i = end;
    }
}

// ------------------------------------------------------------------------------------------------ gradient of many rows
// Tokens are sorted by chunks in shared memory (beside which other CTAs write the table's zeros), an element's place among all is its
// place in its chunk and what searches in the others give, and warps sum runs of rows in that order, a fixed number of
// places each whatever the tokens are: a run that ends in another warp's places leaves a part of its sum, and a last launch adds those.
constexpr uint32_t SORT_EACH = 8;   // keys to a thread
constexpr uint32_t WINDOW = 8;      // of sorted tokens, the last of which are kept apart

// Keys token << BITS | place, padded with the largest.
template <typename K, uint32_t BITS>
__global__ void __launch_bounds__((1u << BITS) / SORT_EACH)
embed_sort_kernel(const uint32_t* __restrict__ tokens, uint32_t ignore_id, uint32_t rows, uint32_t vocab, uint32_t chunks,
                  uint32_t* __restrict__ sorted_token, uint32_t* __restrict__ sorted_row, uint32_t* __restrict__ samples,
                  float* __restrict__ g, size_t elements) {
    chain_entry();
    constexpr uint32_t SIZE = 1u << BITS, SORT_THREADS = SIZE / SORT_EACH;
    if (blockIdx.x >= chunks) {
        const size_t at = (size_t)(blockIdx.x - chunks) * SORT_THREADS + threadIdx.x, step = (size_t)(gridDim.x - chunks) * SORT_THREADS;
        size_t quads = 0;
        if (reinterpret_cast<uintptr_t>(g) % 16 == 0) {
            quads = elements / 4;
#pragma unroll 4
            for (size_t i = at; i < quads; i += step) reinterpret_cast<float4*>(g)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        for (size_t i = quads * 4 + at; i < elements; i += step) g[i] = 0.0f;
        return;
    }
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t base = blockIdx.x * SIZE, first = threadIdx.x * SORT_EACH;
    K keys[SORT_EACH];
#pragma unroll
    for (uint32_t i = 0; i < SORT_EACH; ++i) {
        keys[i] = ~(K)0;
        if (base + first + i < rows) {
            uint32_t token = tokens[base + first + i];
            if (token == ignore_id || token > vocab) token = vocab;   // behind all others
            keys[i] = (K)token << BITS | (first + i);
        }
    }
    block_sort<K, SORT_EACH, SORT_THREADS>(keys, reinterpret_cast<K*>(smem_raw), threadIdx.x);
#pragma unroll
    for (uint32_t i = 0; i < SORT_EACH; ++i) {
        if (i % WINDOW == WINDOW - 1) samples[(base + first + i) / WINDOW] = (uint32_t)(keys[i] >> BITS);
        sorted_token[base + first + i] = (uint32_t)(keys[i] >> BITS);
        sorted_row[base + first + i] = base + (uint32_t)(keys[i] & (SIZE - 1));
    }
}

// An element's place: how many elements of every other chunk come before it.  The last token of every eight of a chunk lies in shared
// memory, where the eight are found; they are a sector of memory, read at once.  Four chunks are searched side by side, so that
// their reads wait for memory together.  (Steps of a search in memory are a sector each: 33 us for 38 chunks of 2048, so 8.)
constexpr uint32_t SAMPLES_HELD = 16384;
__global__ void __launch_bounds__(THREADS)
embed_rank_kernel(const uint32_t* __restrict__ chunk_token, const uint32_t* __restrict__ chunk_row, const uint32_t* __restrict__ samples,
                  uint32_t rows, uint32_t size, uint32_t chunks, uint32_t* __restrict__ sorted_token, uint32_t* __restrict__ sorted_row) {
    chain_entry();
    constexpr uint32_t TOGETHER = 4;
    extern __shared__ __align__(16) uint32_t held[];
    const uint32_t i = blockIdx.x * THREADS + threadIdx.x, per_chunk = size / WINDOW, chunks_held = SAMPLES_HELD / per_chunk;
    const uint32_t own = i / size, token = chunk_token[i], row = chunk_row[i];   // (whole chunks are there)
    uint32_t rank = i - own * size;
    for (uint32_t c0 = 0; c0 < chunks; c0 += chunks_held) {
        const uint32_t n = min(chunks_held, chunks - c0);
        if (c0) __syncthreads();
        for (uint32_t k = threadIdx.x * 4; k < n * per_chunk; k += THREADS * 4)
            *reinterpret_cast<uint4*>(held + k) = *reinterpret_cast<const uint4*>(samples + (size_t)c0 * per_chunk + k);
        __syncthreads();
        for (uint32_t k0 = 0; k0 < n; k0 += TOGETHER) {
            uint32_t at[TOGETHER], limit[TOGETHER];
            uint4 eight[TOGETHER][2];
#pragma unroll
            for (uint32_t u = 0; u < TOGETHER; ++u) {
                const uint32_t c = c0 + k0 + u;
                // (tokens that are the same come first in earlier chunks; of the own one and of those behind the last nothing counts)
                limit[u] = c == own || k0 + u >= n ? 0u : token + (c < own);
                at[u] = min(k0 + u, n - 1) * per_chunk;
            }
            for (uint32_t step = per_chunk / 2; step > 0; step >>= 1)
#pragma unroll
                for (uint32_t u = 0; u < TOGETHER; ++u)
                    if (held[at[u] + step - 1] < limit[u]) at[u] += step;
#pragma unroll
            for (uint32_t u = 0; u < TOGETHER; ++u) {   // (a chunk's last eight, where all eights end below the limit)
                const uint4* from = reinterpret_cast<const uint4*>(chunk_token + ((size_t)c0 * per_chunk + at[u]) * WINDOW);
                eight[u][0] = from[0];
                eight[u][1] = from[1];
            }
#pragma unroll
            for (uint32_t u = 0; u < TOGETHER; ++u) {
                if (limit[u] == 0) continue;
                rank += (at[u] - (k0 + u) * per_chunk) * WINDOW;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    rank += (eight[u][h].x < limit[u]) + (eight[u][h].y < limit[u]) + (eight[u][h].z < limit[u]) + (eight[u][h].w < limit[u]);
            }
        }
    }
    if (i < rows) {
        sorted_token[rank] = token;
        sorted_row[rank] = row;
    }
}

struct GradSums {
    const uint32_t *token, *row;   // sorted
    const void* gy;
    size_t stride;
    uint32_t rows, C, vocab, places, blocks;   // places and blocks of channels to a warp
    float scale;
    float *g, *head, *tail;        // parts of sums that began before a warp's places, and that go on behind them: [warp][C]
};
// A warp has `places` (a power of two, at most 32) places of the sorted order and 32 chunks of channels.
template <typename T, int N, bool WIDE>
__global__ void __launch_bounds__(THREADS)
embed_sums_kernel(const GradSums o) {
    chain_entry();
    const uint32_t lane = threadIdx.x & 31;
    const size_t warp = (size_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    const uint32_t tile = (uint32_t)(warp / o.blocks), block = (uint32_t)(warp - (size_t)tile * o.blocks);
    const uint32_t first = tile * o.places;
    if (first >= o.rows) return;
    const uint32_t n = min(o.places, o.rows - first), at = first + min(lane, n - 1);
    const uint32_t my_token = o.token[at], my_row = o.row[at];
    const uint32_t before = first > 0 ? o.token[first - 1] : 0xFFFFFFFFu, after = first + n < o.rows ? o.token[first + n] : 0xFFFFFFFFu;
    const uint32_t c = block * 32 * N + lane * (WIDE ? N : 1);
    const bool in = c < o.C;
    const T* gy = static_cast<const T*>(o.gy);
    float sum[N] = {};
    bool began_here = __shfl_sync(0xffffffffu, my_token, 0) != before;
    constexpr int AHEAD = 8;   // rows on their way (16 of 8 bytes: 121 registers, and 82 us instead of 42 for 76550 x 500 bf16)
    for (uint32_t k0 = 0; k0 < n; k0 += AHEAD) {
        Channels<WIDE, N, 32, T> v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t k = min(k0 + u, n - 1);
            const uint32_t token = __shfl_sync(0xffffffffu, my_token, k), row = __shfl_sync(0xffffffffu, my_row, k);
            v[u].load(gy + row * o.stride, c, in && token < o.vocab && k0 + u < n ? o.C : 0u);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t k = k0 + u;
            if (k >= n) break;
            const uint32_t token = __shfl_sync(0xffffffffu, my_token, k), next_lane = __shfl_sync(0xffffffffu, my_token, min(k + 1, n - 1));
            const uint32_t next = k + 1 < n ? next_lane : after;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += tape::to_float(v[u].t[e]);
            if (token == next && k + 1 < n) continue;
            if (in && token < o.vocab) {
                const bool whole = began_here && token != next;
                float* to = whole ? o.g + (size_t)token * o.C : (began_here ? o.tail : o.head) + (size_t)tile * o.C;
                const float times = whole ? o.scale : 1.0f;
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] *= times;
                store_channels<WIDE, N, 32>(to, c, o.C, sum);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = 0.0f;
            began_here = true;
        }
    }
}

// The sums that several warps have parts of: the tail of the warp they began in and the heads of those after it, in their order.  A CTA
// has 128 channels of what began in the places of eight warps: sums of few parts a warp each, then those of many one after the other, by
// eight warps a stretch of the parts each.
constexpr uint32_t FEW_PARTS = 4;
__global__ void __launch_bounds__(THREADS)
embed_join_kernel(const GradSums o, uint32_t tiles) {
    chain_entry();
    constexpr uint32_t WARPS = THREADS / 32;
    __shared__ uint32_t all_parts[WARPS];
    __shared__ float sums[WARPS][128];
    const uint32_t per_tile = (o.C + 127) / 128, block = blockIdx.x % per_tile, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t first_tile = blockIdx.x / per_tile * WARPS, tile = first_tile + warp, c = block * 128 + lane;
    uint32_t parts = 0;   // heads
    if (tile + 1 < tiles) {   // (the last warp's sums go on nowhere)
        const uint32_t first = tile * o.places, next = first + o.places, token = o.token[next - 1];
        if (token < o.vocab && o.token[next] == token && !(first > 0 && o.token[first - 1] == token)) {
            // warps whose first place has the token: 32 of them at a time
            for (uint32_t t = tile + 1;; t += 32) {
                const bool more = t + lane < tiles && o.token[(t + lane) * o.places] == token;
                const uint32_t mask = __ballot_sync(0xffffffffu, more);
                parts += __popc(mask);
                if (mask != 0xffffffffu) break;
            }
        }
    }
    const auto add = [&](float (&sum)[4], uint32_t of, uint32_t from, uint32_t to) {   // heads [from, to) of the sum that began in warp `of`
#pragma unroll 4
        for (uint32_t k = from; k < to; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + 32 * e < o.C) sum[e] += o.head[(size_t)(of + 1 + k) * o.C + c + 32 * e];
    };
    const auto tail = [&](float (&sum)[4], uint32_t of, bool wanted) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = wanted && c + 32 * e < o.C ? o.tail[(size_t)of * o.C + c + 32 * e] : 0.0f;
    };
    float sum[4];
    if (parts > 0 && parts <= FEW_PARTS) {
        tail(sum, tile, true);
        add(sum, tile, 0, parts);
        float* to = o.g + (size_t)o.token[tile * o.places + o.places - 1] * o.C;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + 32 * e < o.C) to[c + 32 * e] = sum[e] * o.scale;
    }
    if (lane == 0) all_parts[warp] = parts;
    __syncthreads();
    for (uint32_t w = 0; w < WARPS; ++w) {
        const uint32_t n = all_parts[w], of = first_tile + w;
        if (n <= FEW_PARTS) continue;
        tail(sum, of, warp == 0);
        add(sum, of, (uint32_t)((uint64_t)warp * n / WARPS), (uint32_t)((uint64_t)(warp + 1) * n / WARPS));
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[warp][lane + 32 * e] = sum[e];
        __syncthreads();
        if (threadIdx.x < 128 && block * 128 + threadIdx.x < o.C) {
            float all = sums[0][threadIdx.x];
#pragma unroll
            for (uint32_t k = 1; k < WARPS; ++k) all += sums[k][threadIdx.x];
            o.g[(size_t)o.token[of * o.places + o.places - 1] * o.C + block * 128 + threadIdx.x] = all * o.scale;
        }
        __syncthreads();
    }
}

struct GradPlan {
    bool few;
    uint32_t bits, chunks, places, blocks;
    size_t tiles, samples, chunk_token, chunk_row, token, row, head, tail, bytes;
};
GradPlan grad_plan(const ullis_cuda_runtime* rt, size_t rows, size_t C) {
    GradPlan p{};
    p.few = rows <= FEW;
    if (p.few) return p;
    // Chunks of 2048 are sorted faster than those of 8192 by more than the search in four times as many takes, up to 64 of them.
    p.bits = rows <= 131072 ? 11 : 13;
    p.chunks = (uint32_t)ceil_div(rows, (size_t)1 << p.bits);
    // Places of a warp: as many as leave sixteen warps to an SM, each with 128 channels.
    p.blocks = (uint32_t)ceil_div(C, 128);
    p.places = 32;
    while (p.places > 4 && ceil_div(rows, p.places) * p.blocks < (size_t)rt->sm_count * 16) p.places /= 2;
    p.tiles = ceil_div(rows, p.places);
    size_t at = 0;
    const auto add = [&](size_t n) {
        const size_t here = at;
        at += up(n, 256);
        return here;
    };
    const size_t whole = (size_t)p.chunks << p.bits;   // the padding of the last chunk with it
    p.samples = add(whole / WINDOW * 4);
    p.chunk_token = add(p.chunks > 1 ? whole * 4 : 0);
    p.chunk_row = add(p.chunks > 1 ? whole * 4 : 0);
    p.token = add(whole * 4);
    p.row = add(whole * 4);
    p.head = add(p.tiles * C * 4);
    p.tail = add(p.tiles * C * 4);
    p.bytes = at;
    return p;
}

template <typename K, uint32_t BITS>
void launch_sort(const Stream& s, unsigned zeros, const uint32_t* tokens, uint32_t ignore_id, size_t rows, size_t vocab, uint32_t chunks,
                 uint32_t* token, uint32_t* row, uint32_t* samples, float* g, size_t elements) {
    const auto kernel = embed_sort_kernel<K, BITS>;
    constexpr size_t SMEM = sizeof(K) << BITS;
    if (SMEM > 48 * 1024) ULLIS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    s.chain("embed_sort", kernel, chunks + zeros, (1u << BITS) / SORT_EACH, SMEM, tokens, ignore_id, (uint32_t)rows, (uint32_t)vocab, chunks, token,
            row, samples, g, elements);
}

template <typename T>
void embed_grad_as(const Stream& s, const uint32_t* tokens, uint32_t ignore_id, Rows gy, size_t rows, size_t C, size_t vocab, float scale, float* g,
                   void* workspace) {
    const GradPlan p = grad_plan(s.rt, rows, C);
    constexpr int N = 16 / (int)sizeof(T);
    const auto on = [&](size_t n) { return C % n == 0 && gy.stride % n == 0 && aligned(gy.data, n * sizeof(T)) && aligned(g, 16); };
    const bool wide = on(N);
    if (p.few) {
        const unsigned grid = (unsigned)std::min<size_t>(vocab, (size_t)s.rt->sm_count * 8);
        s.chain("embed_grad_few", wide ? embed_grad_few_kernel<T, N> : embed_grad_few_kernel<T, 1>, grid, THREADS, 0, tokens, ignore_id,
                static_cast<const T*>(gy.data), gy.stride, (uint32_t)rows, (uint32_t)C, (uint32_t)vocab, scale, g);
        return;
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    uint32_t *token = reinterpret_cast<uint32_t*>(ws + p.token), *row = reinterpret_cast<uint32_t*>(ws + p.row);
    uint32_t *chunk_token = p.chunks > 1 ? reinterpret_cast<uint32_t*>(ws + p.chunk_token) : token;
    uint32_t *chunk_row = p.chunks > 1 ? reinterpret_cast<uint32_t*>(ws + p.chunk_row) : row;
    uint32_t* samples = reinterpret_cast<uint32_t*>(ws + p.samples);
    const size_t elements = vocab * C;
    const unsigned zeros = (unsigned)std::min<size_t>((size_t)s.rt->sm_count * 8, ceil_div(elements, 4096));
    const bool narrow = (vocab + 1) >> (32 - p.bits) == 0;   // the largest key is that of the padding
    const auto sort = p.bits == 11 ? (narrow ? launch_sort<uint32_t, 11> : launch_sort<uint64_t, 11>)
                                   : (narrow ? launch_sort<uint32_t, 13> : launch_sort<uint64_t, 13>);
    sort(s, zeros, tokens, ignore_id, rows, vocab, p.chunks, chunk_token, chunk_row, samples, g, elements);
    if (p.chunks > 1) {
        const size_t held = std::min<size_t>(SAMPLES_HELD, ((size_t)p.chunks << p.bits) / WINDOW) * 4;
        if (held > 48 * 1024) ULLIS_CUDA_CHECK(cudaFuncSetAttribute(embed_rank_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)held));
        s.chain("embed_rank", embed_rank_kernel, (unsigned)ceil_div(rows, THREADS), THREADS, held, static_cast<const uint32_t*>(chunk_token),
                static_cast<const uint32_t*>(chunk_row), static_cast<const uint32_t*>(samples), (uint32_t)rows, 1u << p.bits, p.chunks, token, row);
    }
    GradSums o{};
    o.token = token;
    o.row = row;
    o.gy = gy.data;
    o.stride = gy.stride;
    o.rows = (uint32_t)rows;
    o.C = (uint32_t)C;
    o.vocab = (uint32_t)vocab;
    o.places = p.places;
    o.scale = scale;
    o.g = g;
    o.head = reinterpret_cast<float*>(ws + p.head);
    o.tail = reinterpret_cast<float*>(ws + p.tail);
    const auto sums = [&](auto kernel, int each) {
        o.blocks = (uint32_t)ceil_div(C, 32 * each);
        s.chain("embed_sums", kernel, (unsigned)ceil_div(p.tiles * o.blocks, THREADS / 32), THREADS, 0, o);
    };
    if (wide) sums(embed_sums_kernel<T, N, true>, N);
    else if (N == 8 && on(4)) sums(embed_sums_kernel<T, N == 8 ? 4 : N, true>, 4);
    else sums(embed_sums_kernel<T, 4, false>, 4);
    if (p.tiles > 1)
        s.chain("embed_join", embed_join_kernel, (unsigned)(ceil_div(p.tiles - 1, THREADS / 32) * ceil_div(C, 128)), THREADS, 0, o, (uint32_t)p.tiles);
}

}  // namespace

void embed(const Stream& s, int table_dtype, Rows table, const uint32_t* tokens, uint32_t ignore_id, float scale, size_t rows, size_t channels,
           size_t vocab, int dtype, void* y) {
    if (table_dtype == F32) embed_from<float>(s, dtype, table, tokens, ignore_id, scale, rows, channels, vocab, y);
    else if (table_dtype == F16) embed_from<__half>(s, dtype, table, tokens, ignore_id, scale, rows, channels, vocab, y);
    else embed_from<__nv_bfloat16>(s, dtype, table, tokens, ignore_id, scale, rows, channels, vocab, y);
}

size_t embed_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels) {
    return rows ? grad_plan(rt, rows, channels).bytes : 0;
}

void embed_grad(const Stream& s, int dtype, const uint32_t* tokens, uint32_t ignore_id, Rows gy, size_t rows, size_t channels, size_t vocab,
                float scale, float* g, void* workspace) {
    if (dtype == F32) embed_grad_as<float>(s, tokens, ignore_id, gy, rows, channels, vocab, scale, g, workspace);
    else if (dtype == F16) embed_grad_as<__half>(s, tokens, ignore_id, gy, rows, channels, vocab, scale, g, workspace);
    else embed_grad_as<__nv_bfloat16>(s, tokens, ignore_id, gy, rows, channels, vocab, scale, g, workspace);
}

}  // namespace dev
}  // namespace ullis
