// The largest k of every row of logits, in falling order, equal ones by rising column; what a teacher hands to a student.
//
// Values and columns become keys of 64 bits whose order is the wanted one (the value's bits turned so that they rise with it, NaN
// above all, and below them the column's complement), so the k largest keys are one set, found in whatever order.  A warp goes
// through a row once, in tiles of eight 16-byte chunks per lane, and keeps the keys that are not below its bound in shared memory.
// The bound begins as the k-th largest of the first tile's chunk maxima (k chunks hold something as large) and rises whenever
// the buffer is full: bits of the new bound are found from the top by counting.  Where there are few rows several warps share one and
// the first of them goes through what the others have kept.
#include <algorithm>

#include "device_ops.hpp"
#include "tape.cuh"

namespace ullis {
namespace dev {
namespace {

constexpr uint32_t CTA_WARPS = 8, TILE = 8;   // chunks per lane
constexpr uint32_t FULL = 0xffffffffu;

size_t ceil_div(size_t n, size_t by) { return (n + by - 1) / by; }

// 32 bits that rise with the value: -0 is 0, NaN above infinity.  0: below every value.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return v != v ? 0xFFFFFFFFu : bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
}
// The value; a NaN for the bits of none, which no comparison holds for.
__device__ __forceinline__ float of_order(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

// Keys of one warp.
template <uint32_t CAP>
struct Best {
    uint64_t* keys;
    uint32_t k, lane, count = 0;
    uint64_t bound = 0;      // keys below it are not among the k largest
    float least = NAN;       // a value below it is not either

    __device__ void set_bound(uint64_t b) {
        bound = b;
        least = of_order((uint32_t)(b >> 32));
    }
    // The warp's keys, where they are not below the bound, behind those that are there.
    __device__ void add(uint64_t key) {
        const bool in = key != 0 && key >= bound;
        const uint32_t mask = __ballot_sync(FULL, in);
        if (in) keys[count + __popc(mask & ((1u << lane) - 1u))] = key;
        count += __popc(mask);
        if (count > CAP - 32) keep(k + k / 2);
    }
    // Raises the bound until at most `most` >= k keys are left (where there are more than k), and drops the others.
    __device__ __noinline__ void keep(uint32_t most) {
        __syncwarp();
        if (count <= most) return;
        uint32_t high[CAP / 32];
#pragma unroll
        for (uint32_t r = 0; r < CAP / 32; ++r) high[r] = r * 32 + lane < count ? (uint32_t)(keys[r * 32 + lane] >> 32) : 0u;
        uint32_t t = 0, left = count;
        for (uint32_t bit = 0x80000000u; bit && left > most; bit >>= 1) {
            uint32_t n = 0;
#pragma unroll
            for (uint32_t r = 0; r < CAP / 32; ++r) n += high[r] >= (t | bit);
            n = __reduce_add_sync(FULL, n);
            if (n >= k) {
                t |= bit;
                left = n;
            }
        }
        uint32_t low = 0;
        if (left > most) {   // equal values: by their columns
            uint32_t above = 0;
#pragma unroll
            for (uint32_t r = 0; r < CAP / 32; ++r) above += high[r] > t;
            above = __reduce_add_sync(FULL, above);
            for (uint32_t bit = 0x80000000u; bit && left > most; bit >>= 1) {
                uint32_t n = 0;
#pragma unroll
                for (uint32_t r = 0; r < CAP / 32; ++r)
                    if (high[r] == t) n += (uint32_t)keys[r * 32 + lane] >= (low | bit);
                n = __reduce_add_sync(FULL, n);
                if (above + n >= k) {
                    low |= bit;
                    left = above + n;
                }
            }
        }
        set_bound((uint64_t)t << 32 | low);
        uint32_t n = 0;
        for (uint32_t r = 0; r * 32 < count; ++r) {
            const uint64_t key = r * 32 + lane < count ? keys[r * 32 + lane] : 0u;
            const bool in = key != 0 && key >= bound;
            const uint32_t mask = __ballot_sync(FULL, in);
            __syncwarp();
            if (in) keys[n + __popc(mask & ((1u << lane) - 1u))] = key;
            n += __popc(mask);
            __syncwarp();
        }
        count = n;
    }
    __device__ void sort() {   // falling
        __syncwarp();
        for (uint32_t run = 2; run < 2 * count; run <<= 1) {
            for (uint32_t half = run >> 1; half > 0; half >>= 1) {
                for (uint32_t i = lane;; i += 32) {
                    const uint32_t a = (i & ~(half - 1)) * 2 + (i & (half - 1));
                    if (a >= count) break;
                    const uint32_t b = half == run >> 1 ? a ^ (run - 1) : a + half;   // (the first step of a run mirrors: all runs fall)
                    if (b < count) {
                        const uint64_t x = keys[a], y = keys[b];
                        if (x < y) {
                            keys[a] = y;
                            keys[b] = x;
                        }
                    }
                }
                __syncwarp();
            }
        }
    }
};

struct Top {
    const void* logits;
    size_t stride;
    uint32_t rows, vocab, k, warps;   // warps to a row: 1, 2, 4 or 8
    int32_t* ids;
    void* out;
};

template <typename T, uint32_t CAP>
__global__ void __launch_bounds__(CTA_WARPS * 32)
top_kernel(const Top o) {
    chain_entry();
    constexpr int N = tape::CHUNK<T>;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint64_t* all_keys = reinterpret_cast<uint64_t*>(smem_raw);   // [warp][CAP]
    __shared__ uint32_t counts[CTA_WARPS];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % o.warps;
    const size_t row = (size_t)blockIdx.x * (CTA_WARPS / o.warps) + warp / o.warps;
    const bool live = row < o.rows;
    Best<CAP> best{all_keys + warp * CAP, o.k, lane};
    if (live) {
        const T* from = static_cast<const T*>(o.logits) + row * o.stride;
        // chunks on 16 bytes; the first and the last may reach out of the row
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(from) % 16) / sizeof(T), chunks = (o.vocab + off + N - 1) / N;
        const uint32_t begin = (uint32_t)((uint64_t)chunks * part / o.warps), end = (uint32_t)((uint64_t)chunks * (part + 1) / o.warps);
        for (uint32_t tile = begin; tile < end; tile += TILE * 32) {
            tape::Raw<T> raw[TILE];
#pragma unroll
            for (uint32_t u = 0; u < TILE; ++u) {
                const uint32_t chunk = tile + u * 32 + lane;
                const int64_t first = (int64_t)chunk * N - off;
                if (chunk < end && first >= 0 && first + N <= o.vocab) {
                    raw[u].q = *reinterpret_cast<const uint4*>(from + first);
                } else {
                    T* t = reinterpret_cast<T*>(&raw[u].q);
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        t[e] = chunk < end && first + e >= 0 && first + e < o.vocab ? from[first + e] : tape::from_float<T>(-INFINITY);
                }
            }
            float most[TILE];   // of a chunk, NaN if it holds one
#pragma unroll
            for (uint32_t u = 0; u < TILE; ++u) {
                float v[N];
                raw[u].unpack(v);
                most[u] = v[0];
#pragma unroll
                for (int e = 1; e < N; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most[u]) : "f"(v[e]));
            }
            if (tile == begin && end - begin > o.k) {
                // a first bound: bits from the top while k chunk maxima are not below it
                uint32_t high[TILE], t = 0;
#pragma unroll
                for (uint32_t u = 0; u < TILE; ++u) high[u] = tile + u * 32 + lane < end ? order_of(most[u]) : 0u;
                for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1) {   // (20 bits: 2^-11 of the value)
                    uint32_t n = 0;
#pragma unroll
                    for (uint32_t u = 0; u < TILE; ++u) n += high[u] >= (t | bit);
                    if (__reduce_add_sync(FULL, n) >= o.k) t |= bit;
                }
                best.set_bound((uint64_t)t << 32);
            }
            // which elements of the tile are not below the bound, a bit each
            uint32_t pass[TILE * N / 32] = {};
#pragma unroll
            for (uint32_t u = 0; u < TILE; ++u) {
                if (__any_sync(FULL, !(most[u] < best.least))) {
                    float v[N];
                    raw[u].unpack(v);
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (!(v[e] < best.least)) pass[(u * N + e) / 32] |= 1u << (u * N + e) % 32;
                }
            }
#pragma unroll
            for (uint32_t w = 0; w < TILE * N / 32; ++w) {
                while (__any_sync(FULL, pass[w] != 0)) {
                    uint64_t key = 0;
                    if (pass[w]) {
                        const uint32_t at = w * 32 + __ffs(pass[w]) - 1, chunk = tile + at / N * 32 + lane;
                        pass[w] &= pass[w] - 1;
                        const int64_t column = (int64_t)chunk * N - off + at % N;
                        if (chunk < end && column >= 0 && column < o.vocab)
                            key = (uint64_t)order_of(tape::to_float(from[column])) << 32 | (0xFFFFFFFFu - (uint32_t)column);
                    }
                    best.add(key);
                }
            }
        }
        best.keep(o.k);
    }
    if (o.warps > 1) {
        if (lane == 0) counts[warp] = best.count;
        __syncthreads();
        if (part) return;
        if (live) {
            for (uint32_t w = 1; w < o.warps; ++w) {
                const uint32_t n = counts[warp + w];
                for (uint32_t i = 0; i < n; i += 32) best.add(i + lane < n ? all_keys[(warp + w) * CAP + i + lane] : 0u);
            }
            best.keep(o.k);
        }
    }
    if (!live) return;
    best.sort();
    T* out = static_cast<T*>(o.out);
    for (uint32_t i = lane; i < o.k; i += 32) {
        const uint64_t key = best.keys[i];
        o.ids[row * o.k + i] = (int32_t)(0xFFFFFFFFu - (uint32_t)key);
        out[row * o.k + i] = tape::from_float<T>(of_order((uint32_t)(key >> 32)));
    }
}

template <typename T, uint32_t CAP>
void launch(const Stream& s, const Top& o) {
    constexpr size_t SMEM = CTA_WARPS * CAP * 8;
    if (SMEM > 48 * 1024) ULLIS_CUDA_CHECK(cudaFuncSetAttribute(top_kernel<T, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    s.chain("top_logits", top_kernel<T, CAP>, (unsigned)ceil_div(o.rows, CTA_WARPS / o.warps), CTA_WARPS * 32, SMEM, o);
}
template <typename T>
void launch_by_k(const Stream& s, const Top& o) {
    if (o.k <= 64) launch<T, 256>(s, o);
    else if (o.k <= 128) launch<T, 512>(s, o);
    else launch<T, 1024>(s, o);
}

}  // namespace

void top_logits(const Stream& s, int dtype, Rows logits, size_t rows, size_t vocab, size_t k, int32_t* ids, void* out) {
    Top o{};
    o.logits = logits.data;
    o.stride = logits.stride;
    o.rows = (uint32_t)rows;
    o.vocab = (uint32_t)vocab;
    o.k = (uint32_t)k;
    o.ids = ids;
    o.out = out;
    // warps enough for every SM, of whole tiles each
    const size_t tiles = ceil_div(vocab * size_of(dtype), TILE * 32 * 16);
    o.warps = 1;
    while (o.warps < CTA_WARPS && rows * o.warps < (size_t)s.rt->sm_count * 16 && tiles >= 2 * o.warps) o.warps *= 2;
    if (dtype == F32) launch_by_k<float>(s, o);
    else if (dtype == F16) launch_by_k<__half>(s, o);
    else launch_by_k<__nv_bfloat16>(s, o);
}

}  // namespace dev
}  // namespace ullis
