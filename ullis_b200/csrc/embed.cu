// Embedding lookup and the gradient of its table, on a caller's device memory.
//
//   y[r] = scale * table[token[r]]          G[v] = scale * sum of gy[r] over the rows r with token[r] = v
//
// Both read and write what they name once: the lookup is bound by memory, the gradient of many rows by memory and the steps of its sort.
// The gradient's sums have a fixed order, with no atomics: the rows of a token in rising order, in pieces where there are many.
// In a graph, us: lookup of 16384 x 512 from FP16 into f32 9.5 where the outputs leave L2 (42 MB, 4.4 TB/s; call by call 8.5, the host's, as
// a lookup of 512 x 256 whose kernel takes 2), of 131072 rows 56 (277 MB, 4.9 TB/s).  Gradient of 512 x 256 into 8192 rows 7 to 8.5,
// 16384 x 512 f32 27 (sort 15, sums 8, parts 7 with their launches; 50 MB), 76550 x 500 bf16 into 50021 rows 66 (sort 14, searches 17,
// sums 27, parts 9; 177 MB), 131072 x 512 bf16 73.
#include <algorithm>
#include <type_traits>
#include <utility>

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
// One launch, bound by its latency.  CTA b has the table rows v with v % CTAs == b, so that frequent tokens, which lie close together, go to
// different SMs: it writes zeros, lists the rows whose token is one of them, sorts
// the list (a handful: a rank per entry by comparison with all others), and sums run by run with all of its threads: a group of
// threads per row of gy, the groups' sums added in their order.
// us in a graph, into 8192 rows of 256 FP16 channels, so / by the sort below: 512 rows 7.0 / 10.9, 1024 8.8 / 11.6, 1536 10.8 / 12.5, 2048
// 13.0 / 12.7.  Where one token has all rows one CTA ranks and sums them: 256 rows 11 / 11, 512 23 / 13, 1024 62 / 15 (512 f32 channels
// 115 / 16).
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
    uint32_t tokens_here[FEW / THREADS];   // on their way beside the zeros
#pragma unroll
    for (uint32_t k = 0; k < FEW / THREADS; ++k) tokens_here[k] = k * THREADS + threadIdx.x < rows ? tokens[k * THREADS + threadIdx.x] : ignore_id;
    const size_t first = (size_t)blockIdx.x * C, step = (size_t)gridDim.x * C;
    if (C % 4 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0) {
        for (size_t at = first; at < (size_t)vocab * C; at += step)
            for (uint32_t c = threadIdx.x * 4; c < C; c += THREADS * 4) *reinterpret_cast<float4*>(g + at + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    } else {
        for (size_t at = first; at < (size_t)vocab * C; at += step)
            for (uint32_t c = threadIdx.x; c < C; c += THREADS) g[at + c] = 0.0f;
    }
    uint32_t count = 0;
#pragma unroll
    for (uint32_t k = 0; k < FEW / THREADS; ++k) {   // (in the order of the rows)
        const uint32_t r = k * THREADS + threadIdx.x, token = tokens_here[k];
        if (k * THREADS >= rows) break;
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
// Tokens are sorted by chunks, each by a cluster; with more chunks than one an element's place among all is its place in its chunk and
// what searches in the others give.  Beside the last of these launches other CTAs write the table's zeros, which costs little there
// (zeros for the rows alone that no chunk has, found by the same searches: 76550 x 500 into 50021 rows 108 us instead of 82).  Then warps
// sum runs of rows in that order, a fixed number of places each whatever the tokens are: a run that ends in another warp's places leaves a
// part of its sum, and a last launch adds those.
constexpr uint32_t SORT_EACH = 8, SORT_THREADS = 256, SORT_CTA = SORT_EACH * SORT_THREADS;   // keys to a thread, of a CTA
constexpr uint32_t MOST_CTAS = 8;   // of a cluster
constexpr uint32_t WINDOW = 8;      // of sorted tokens, the last of which are kept apart

// Zeros for `elements` of g, by threads `at`, `at` + `step` ...; the first to leave L2.
__device__ __forceinline__ void write_zeros(float* g, size_t elements, size_t at, size_t step) {
    size_t quads = 0;
    if (reinterpret_cast<uintptr_t>(g) % 16 == 0) {
        quads = elements / 4;
#pragma unroll 4
        for (size_t i = at; i < quads; i += step) __stcs(reinterpret_cast<float4*>(g) + i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    }
    for (size_t i = quads * 4 + at; i < elements; i += step) g[i] = 0.0f;
}

// Keys token * size of the chunk + place, padded with the largest.  A chunk is what a cluster's CTAs hold: a network over 2048 keys keeps one SM
// busy with its shuffles (64 warp instructions a step), and eight SMs sort 16384 in the time of one and 39 more steps, 14 us; chunks of
// 2048, and the searches that they need, took 9 more at 16384 rows, 16 at 76550.
template <typename K>
__global__ void __launch_bounds__(SORT_THREADS)
embed_sort_kernel(const uint32_t* __restrict__ tokens, uint32_t ignore_id, uint32_t rows, uint32_t vocab, uint32_t bits, uint32_t sort_ctas,
                  uint32_t* __restrict__ sorted_token, uint32_t* __restrict__ sorted_row, uint32_t* __restrict__ samples,
                  float* __restrict__ g, size_t zeros) {
    chain_entry();
    if (blockIdx.x >= sort_ctas) {   // (whole clusters)
        write_zeros(g, zeros, (size_t)(blockIdx.x - sort_ctas) * SORT_THREADS + threadIdx.x, (size_t)(gridDim.x - sort_ctas) * SORT_THREADS);
        return;
    }
    __shared__ __align__(16) K buffers[3 * SORT_CTA];
    uint32_t rank, ctas;
    asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %cluster_nctaid.x;" : "=r"(ctas));
    const uint32_t first = blockIdx.x * SORT_CTA + threadIdx.x * SORT_EACH, in_chunk = first & ((1u << bits) - 1);
    K keys[SORT_EACH];
#pragma unroll
    for (uint32_t i = 0; i < SORT_EACH; ++i) {
        keys[i] = ~(K)0;
        if (first + i < rows) {
            uint32_t token = tokens[first + i];
            if (token == ignore_id || token > vocab) token = vocab;   // behind all others
            keys[i] = (K)token << bits | (in_chunk + i);
        }
    }
    cluster_sort<K, SORT_EACH, SORT_THREADS>(keys, buffers, buffers + SORT_CTA, rank, ctas);
    uint32_t token[SORT_EACH], row[SORT_EACH];
#pragma unroll
    for (uint32_t i = 0; i < SORT_EACH; ++i) {
        token[i] = (uint32_t)(keys[i] >> bits);
        row[i] = (first - in_chunk) + (uint32_t)(keys[i] & ((K)1 << bits) - 1);
    }
#pragma unroll
    for (uint32_t i = 0; i < SORT_EACH; i += 4) {
        *reinterpret_cast<uint4*>(sorted_token + first + i) = make_uint4(token[i], token[i + 1], token[i + 2], token[i + 3]);
        *reinterpret_cast<uint4*>(sorted_row + first + i) = make_uint4(row[i], row[i + 1], row[i + 2], row[i + 3]);
    }
    static_assert(SORT_EACH == WINDOW, "");
    samples[first / WINDOW] = token[WINDOW - 1];
}

// An element's place: how many elements of every other chunk come before it.  The last token of every eight of a chunk lies in shared
// memory, where the eight are found; they are a sector of memory, read at once.  Four chunks are searched side by side, so that
// their reads wait for memory together.  (Steps of a search in memory are a sector each: 38 chunks of 2048 took 33 us so, 18 this way.)
constexpr uint32_t CHUNK_BITS = 14, SAMPLES_HELD = 16384;
static_assert(1u << CHUNK_BITS == MOST_CTAS * SORT_CTA, "");
__global__ void __launch_bounds__(THREADS, 3)
embed_rank_kernel(const uint32_t* __restrict__ chunk_token, const uint32_t* __restrict__ chunk_row, const uint32_t* __restrict__ samples,
                  uint32_t rows, uint32_t chunks, uint32_t* __restrict__ sorted_token, uint32_t* __restrict__ sorted_row, float* __restrict__ g,
                  size_t zeros) {
    chain_entry();
    constexpr uint32_t TOGETHER = 4, size = 1u << CHUNK_BITS, per_chunk = size / WINDOW, chunks_held = SAMPLES_HELD / per_chunk;
    extern __shared__ __align__(16) uint32_t held[];
    const uint32_t rank_ctas = (rows + THREADS - 1) / THREADS;
    const auto hold = [&](uint32_t c0, uint32_t n) {
        __syncthreads();
#pragma unroll 8
        for (uint32_t k = threadIdx.x * 4; k < n * per_chunk; k += THREADS * 4)
            *reinterpret_cast<uint4*>(held + k) = *reinterpret_cast<const uint4*>(samples + (size_t)c0 * per_chunk + k);
        __syncthreads();
    };
    if (blockIdx.x >= rank_ctas) {
        write_zeros(g, zeros, (size_t)(blockIdx.x - rank_ctas) * THREADS + threadIdx.x, (size_t)(gridDim.x - rank_ctas) * THREADS);
        return;
    }
    const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
    const uint32_t own = i / size, token = chunk_token[i], row = chunk_row[i];   // (whole chunks are there)
    uint32_t rank = i - own * size;
    for (uint32_t c0 = 0; c0 < chunks; c0 += chunks_held) {
        const uint32_t n = min(chunks_held, chunks - c0);
        hold(c0, n);
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
#pragma unroll
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

// Many chunks, whose searches in one another would grow with the square of the rows, are merged instead: runs of `run` sorted elements,
// two and two, an element's place being its own in its run and what a search in the other gives (of tokens that are the same those of
// the first run come first).  Neighbours search in neighbouring places.
__global__ void __launch_bounds__(THREADS)
embed_merge_kernel(const uint32_t* __restrict__ from_token, const uint32_t* __restrict__ from_row, uint32_t rows, uint32_t run,
                   uint32_t* __restrict__ to_token, uint32_t* __restrict__ to_row, float* __restrict__ g, size_t zeros) {
    chain_entry();
    const uint32_t merge_ctas = (rows + THREADS - 1) / THREADS;
    if (blockIdx.x >= merge_ctas) {
        write_zeros(g, zeros, (size_t)(blockIdx.x - merge_ctas) * THREADS + threadIdx.x, (size_t)(gridDim.x - merge_ctas) * THREADS);
        return;
    }
    const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
    if (i >= rows) return;
    const uint32_t token = from_token[i], row = from_row[i];
    const uint32_t own = i / run * run, other = own ^ run;   // (run: a power of two)
    uint32_t at = i;
    if (other < rows) {
        const uint32_t n = min(run, rows - other), before = below(from_token + other, n, token, other < own);
        at = min(own, other) + (i - own) + before;
    }
    to_token[at] = token;
    to_row[at] = row;
}

struct GradSums {
    const uint32_t *token, *row;   // sorted
    const void* gy;
    size_t stride;
    uint32_t rows, C, vocab, places, blocks;   // places and blocks of channels to a warp
    float scale;
    float *g, *head, *tail;        // parts of sums that began before a warp's places, and that go on behind them: [warp][C]
};
// A warp has `places` (a power of two, at most 32) places of the sorted order and 256 channels, a lane BLOCKS times N of them.  Bound by
// memory's latency and by instructions (45 to a row): rows are read without tests, the runs' ends are bits of a word, eight rows are on
// their way at once (16384 x 512 f32 8 us, 76550 x 500 bf16 27).
template <typename T, int N, int BLOCKS, bool WIDE>
__global__ void __launch_bounds__(THREADS)
embed_sums_kernel(const GradSums o) {
    chain_entry();
    constexpr uint32_t ALL = 0xffffffffu;
    const uint32_t lane = threadIdx.x & 31;
    const size_t warp = (size_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    const uint32_t tile = (uint32_t)(warp / o.blocks), block = (uint32_t)(warp - (size_t)tile * o.blocks);
    const uint32_t first = tile * o.places;
    if (first >= o.rows) return;
    const uint32_t there = min(o.places, o.rows - first), at = first + min(lane, there - 1);
    const uint32_t my_token = o.token[at], my_row = o.row[at];
    const uint32_t before = first > 0 ? o.token[first - 1] : 0xFFFFFFFFu, after = first + there < o.rows ? o.token[first + there] : 0xFFFFFFFFu;
    const uint32_t right = __shfl_down_sync(ALL, my_token, 1);
    const uint32_t ends = __ballot_sync(ALL, lane < there && my_token != (lane + 1 < there ? right : after));   // places that a run ends at
    const uint32_t n = __popc(__ballot_sync(ALL, lane < there && my_token < o.vocab));   // (those that do not count come last)
    // What a lane reads of a row; past the row's end something of it that is not kept.
    const uint32_t c = block * (32 * N * BLOCKS) + lane * (WIDE ? N : 1);
    uint32_t from[BLOCKS][WIDE ? 1 : N];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int e = 0; e < (WIDE ? 1 : N); ++e) {
            const uint32_t channel = c + b * 32 * N + e * 32;
            from[b][e] = channel < o.C ? channel : 0u;
        }
    const T* gy = static_cast<const T*>(o.gy);
    float sum[BLOCKS][N] = {};
    bool began_here = __shfl_sync(ALL, my_token, 0) != before;
    constexpr int AHEAD = WIDE ? 32 / (BLOCKS * N * (int)sizeof(T) / 4) : 4;   // rows on their way: 32 registers of them
    for (uint32_t k0 = 0; k0 < n; k0 += AHEAD) {
        Channels<WIDE, N, 32, T> v[AHEAD][BLOCKS];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {   // (behind the last: that row again)
            const T* row = gy + __shfl_sync(ALL, my_row, k0 + u) * o.stride;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                if constexpr (WIDE) {
                    v[u][b].load(row, from[b][0], 0xFFFFFFFFu);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) v[u][b].t[e] = row[from[b][e]];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t k = k0 + u;
            if (k >= n) break;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[b][e] += tape::to_float(v[u][b].t[e]);
            const bool end = ends >> k & 1u;
            if (!end && k + 1 < n) continue;
            const bool whole = began_here && end;
            float* to = whole ? o.g + (size_t)__shfl_sync(ALL, my_token, k) * o.C : (began_here ? o.tail : o.head) + (size_t)tile * o.C;
            const float times = whole ? o.scale : 1.0f;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
                for (int e = 0; e < N; ++e) sum[b][e] *= times;
                if (c + b * 32 * N < o.C) store_channels<WIDE, N, 32>(to, c + b * 32 * N, o.C, sum[b]);
#pragma unroll
                for (int e = 0; e < N; ++e) sum[b][e] = 0.0f;
            }
            began_here = true;
        }
    }
}

// The sums that several warps have parts of: the tail of the warp they began in and the heads of those after it, in their order.  A CTA
// has 128 channels of what began in the places of eight warps: sums of few parts a warp each, then those of many one after the other, by
// eight warps a stretch of the parts each.
constexpr uint32_t FEW_PARTS = 4;
template <bool WIDE>
__global__ void __launch_bounds__(THREADS)
embed_join_kernel(const GradSums o, uint32_t tiles) {
    chain_entry();
    constexpr uint32_t WARPS = THREADS / 32;
    __shared__ uint32_t all_parts[WARPS];
    __shared__ float sums[WARPS][4][32];
    const uint32_t per_tile = (o.C + 127) / 128, block = blockIdx.x % per_tile, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t first_tile = blockIdx.x / per_tile * WARPS, tile = first_tile + warp, c = block * 128 + lane * (WIDE ? 4 : 1);
    const auto first_token = [&](uint32_t t) { return o.token[(size_t)t * o.places]; };
    uint32_t parts = 0;   // heads
    if (tile + 1 < tiles) {   // (the last warp's sums go on nowhere)
        const uint32_t first = tile * o.places, token = o.token[first + o.places - 1], next = o.token[first + o.places];
        const uint32_t before = first > 0 ? o.token[first - 1] : 0xFFFFFFFFu;
        if (token < o.vocab && next == token && before != token) {
            // one behind the last warp whose first place has the token: 32 looks at once
            uint32_t low = tile + 1, high = tiles;   // low has it, high has not or is none
            while (high - low > 1) {
                const uint32_t step = (high - low + 31) / 32, at = low + lane * step;
                const uint32_t mask = __ballot_sync(0xffffffffu, at < high && first_token(min(at, high - 1)) == token);   // (lanes from 0 on)
                const uint32_t last = 31 - __clz(mask);
                high = min(high, low + (last + 1) * step);
                low += last * step;
            }
            parts = high - tile - 1;
        }
    }
    using Part = Channels<WIDE, 4, 32, float>;
    const auto add = [&](float (&sum)[4], uint32_t of, uint32_t from, uint32_t to) {   // heads [from, to) of the sum that began in warp `of`
        constexpr uint32_t AHEAD = 8;
        for (uint32_t k = from; k < to; k += AHEAD) {
            Part part[AHEAD];
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u) part[u].load(o.head + (size_t)(of + 1 + k + u) * o.C, c, k + u < to ? o.C : 0u);
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += part[u].t[e];
        }
    };
    const auto tail = [&](float (&sum)[4], uint32_t of, bool wanted) {
        load_channels<WIDE, 4, 32>(o.tail + (size_t)of * o.C, c, wanted ? o.C : 0u, sum);
    };
    const auto leave = [&](float (&sum)[4], uint32_t of) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] *= o.scale;
        if (c < o.C) store_channels<WIDE, 4, 32>(o.g + (size_t)o.token[(size_t)of * o.places + o.places - 1] * o.C, c, o.C, sum);
    };
    float sum[4];
    if (parts > 0 && parts <= FEW_PARTS) {
        tail(sum, tile, true);
        add(sum, tile, 0, parts);
        leave(sum, tile);
    }
    if (lane == 0) all_parts[warp] = parts;
    __syncthreads();
    for (uint32_t w = 0; w < WARPS; ++w) {
        const uint32_t n = all_parts[w], of = first_tile + w;
        if (n <= FEW_PARTS) continue;
        tail(sum, of, warp == 0);
        add(sum, of, (uint32_t)((uint64_t)warp * n / WARPS), (uint32_t)((uint64_t)(warp + 1) * n / WARPS));
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[warp][e][lane] = sum[e];
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (uint32_t k = 1; k < WARPS; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += sums[k][e][lane];
            leave(sum, of);
        }
        __syncthreads();
    }
}

// Chunks that are ranked by searches in all others, not merged.  us of a call, 64 channels and 50021 tokens, ranked / merged: 8 chunks 47 / 52,
// 12 61 / 65, 16 82 / 75, 32 183 / 129, 64 557 / 265, 256 6664 / 1046.
constexpr uint32_t MOST_RANKED = 12;
struct GradPlan {
    bool few, merged;   // merged: run by run
    uint32_t bits, chunks, places, blocks;
    size_t tiles, samples, chunk_token, chunk_row, token, row, head, tail, bytes;
};
GradPlan grad_plan(const ullis_cuda_runtime* rt, size_t rows, size_t C) {
    GradPlan p{};
    p.few = rows <= FEW;
    if (p.few) return p;
    // One chunk of as many CTAs as hold the rows, or several of eight CTAs.
    p.bits = 11;
    while (p.bits < CHUNK_BITS && (size_t)1 << p.bits < rows) ++p.bits;
    p.chunks = (uint32_t)ceil_div(rows, (size_t)1 << p.bits);
    // Places of a warp: as many as leave sixteen warps to an SM.
    p.blocks = (uint32_t)ceil_div(C, 256);
    p.places = 32;
    while (p.places > 4 && ceil_div(rows, p.places) * p.blocks < (size_t)rt->sm_count * 16) p.places /= 2;
    p.tiles = ceil_div(rows, p.places);
    p.merged = p.chunks > MOST_RANKED;
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
    uint32_t merges = 0;   // to and fro
    while (p.merged && (size_t)1 << (p.bits + merges) < rows) ++merges;
    uint32_t* samples = reinterpret_cast<uint32_t*>(ws + p.samples);
    const size_t elements = vocab * C;
    const size_t zeros = p.chunks > 1 ? 0 : elements;   // beside the sort if it is the only launch before the sums
    const auto zero_ctas = [&](size_t n) { return std::min<size_t>((size_t)s.rt->sm_count * 8, ceil_div(n, 4096)); };
    const bool narrow = (vocab + 1) >> (32 - p.bits) == 0;   // the largest key is that of the padding
    const uint32_t ctas = (1u << p.bits) / SORT_CTA, sort_ctas = p.chunks * ctas;
    const auto sort = narrow ? embed_sort_kernel<uint32_t> : embed_sort_kernel<uint64_t>;
    s.chain_cluster("embed_sort", sort, sort_ctas + (unsigned)ceil_div(zero_ctas(zeros), ctas) * ctas, SORT_THREADS, 0, ctas, tokens, ignore_id,
                    (uint32_t)rows, (uint32_t)vocab, p.bits, sort_ctas, chunk_token, chunk_row, samples, g, zeros);
    for (uint32_t k = 0; k < merges; ++k) {
        if (k > 0) {
            std::swap(token, chunk_token);
            std::swap(row, chunk_row);
        }
        const size_t now = k + 1 == merges ? elements : 0;
        s.chain("embed_merge", embed_merge_kernel, (unsigned)(ceil_div(rows, THREADS) + zero_ctas(now)), THREADS, 0,
                static_cast<const uint32_t*>(chunk_token), static_cast<const uint32_t*>(chunk_row), (uint32_t)rows, 1u << (p.bits + k), token, row, g, now);
    }
    if (p.chunks > 1 && !p.merged) {
        const size_t held = std::min<size_t>(SAMPLES_HELD, ((size_t)p.chunks << p.bits) / WINDOW) * 4;
        if (held > 48 * 1024) s.allow_shared(embed_rank_kernel, SAMPLES_HELD * 4);
        s.chain("embed_rank", embed_rank_kernel, (unsigned)(ceil_div(rows, THREADS) + zero_ctas(elements - zeros)), THREADS, held,
                static_cast<const uint32_t*>(chunk_token), static_cast<const uint32_t*>(chunk_row), static_cast<const uint32_t*>(samples),
                (uint32_t)rows, p.chunks, token, row, g + zeros, elements - zeros);
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
    o.blocks = p.blocks;
    const auto sums = [&](auto kernel) { s.chain("embed_sums", kernel, (unsigned)ceil_div(p.tiles * p.blocks, THREADS / 32), THREADS, 0, o); };
    if (wide) sums(embed_sums_kernel<T, N, 8 / N, true>);
    else if (N == 8 && on(4)) sums(embed_sums_kernel<T, 4, 2, true>);
    else sums(embed_sums_kernel<T, 4, 2, false>);
    if (p.tiles > 1) {
        const auto join = C % 4 == 0 && aligned(g, 16) ? embed_join_kernel<true> : embed_join_kernel<false>;
        s.chain("embed_join", join, (unsigned)(ceil_div(p.tiles - 1, THREADS / 32) * ceil_div(C, 128)), THREADS, 0, o, (uint32_t)p.tiles);
    }
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
