// The largest k of every row of logits, in falling order, equal ones by rising column; what a teacher hands to a student.
//
// Values and columns become keys of 64 bits whose order is the wanted one (the value's bits turned so that they rise with it, NaN
// above all, and below them the column's complement), so the k largest keys are one set, found in whatever order.  A warp goes
// through a row once, in tiles of four 16-byte chunks per lane, and compares each chunk's largest value with its bound.  The numbers of
// the chunks that hold something as large go into a queue, and 32 of them at a time are looked at element by element, a lane each, so that
// the rare ones cost a warp no more than they are.  Keys that are not below the bound are kept in shared memory.
// The bound begins as the k-th largest maximum of the first 512 chunks (k of them hold something as large) and rises whenever
// the buffer is full: bits of the new bound are found from the top by counting.  Where there are few rows several warps share one; the least
// of the bounds that each finds for its share of the k holds for all of them, and the first goes through what the others have kept.
//
// Bound by memory on long rows and by instructions on short ones: 4096 x 131072 bf16, k = 64 195 us (1.07 GB, 5.5 TB/s); 16384 x 8192 f32 132 us
// (537 MB, 4.1 TB/s; some 5000 warp instructions to a row, a fifth of them for reading it by count, the others for what is kept).
// Tried and slower there: tiles of 2 or 8 chunks (155, 127 but 220 on the long rows), a sample of 8 or 32 (139), a buffer of 384 keys
// (149), the next tiles prefetched into L2 (127, long rows 214).  k = 128 and 256 take 250 and 476 us there: they keep two and four times
// as much, and the bound begins at the k-th of 512 chunk maxima whatever k is.
#include <algorithm>

#include "block_sort.cuh"
#include "device_ops.hpp"
#include "tape.cuh"

namespace ullis {
namespace dev {
namespace {

constexpr uint32_t MOST_WARPS = 16, TILE = 4, SAMPLE = 16;   // chunks per lane: of a tile; looked at for the first bound
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

// The bits that all of a warp's numbers have in common from the top, and the first that they have not (0: none).
__device__ __forceinline__ uint32_t common(uint32_t largest, uint32_t smallest, uint32_t* bit) {
    largest = __reduce_max_sync(FULL, largest);
    smallest = __reduce_min_sync(FULL, smallest);
    const uint32_t differ = largest ^ smallest;
    *bit = differ ? 0x80000000u >> __clz(differ) : 0u;
    return differ ? largest & ~(2 * *bit - 1) : largest;
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
        uint32_t high[CAP / 32], largest = 0, smallest = FULL;
#pragma unroll
        for (uint32_t r = 0; r < CAP / 32; ++r) {
            const bool in = r * 32 + lane < count;
            high[r] = in ? (uint32_t)(keys[r * 32 + lane] >> 32) : 0u;
            largest = max(largest, high[r]);
            smallest = min(smallest, in ? high[r] : FULL);
        }
        uint32_t bit, t = common(largest, smallest, &bit), left = count;
        for (; bit && left > most; bit >>= 1) {
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
            for (bit = 0x80000000u; bit && left > most; bit >>= 1) {
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
};

struct Top {
    const void* logits;
    size_t stride;
    uint32_t rows, vocab, k, warps;   // warps to a row: 1, 2, 4, 8 or 16
    int32_t* ids;
    void* out;
};

// The largest value of a chunk, NaN if it holds one, as one of two halves of a word for 16-bit types.
__device__ __forceinline__ float larger(float a, float b) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
}
template <typename T>
struct Most;
template <>
struct Most<float> {
    float v;
    __device__ __forceinline__ explicit Most(const uint4& q) {
        v = larger(larger(__uint_as_float(q.x), __uint_as_float(q.y)), larger(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
    using Bound = float;
    static __device__ __forceinline__ Bound bound(float least) { return least; }
    __device__ __forceinline__ bool reaches(Bound b) const { return !(v < b); }
    __device__ __forceinline__ float value() const { return v; }
};
template <>
struct Most<__half> {
    __half2 v;
    __device__ __forceinline__ explicit Most(const uint4& q) {
        const __half2* h = reinterpret_cast<const __half2*>(&q);
        v = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    }
    using Bound = __half2;
    static __device__ __forceinline__ Bound bound(float least) { return __half2half2(__float2half_rd(least)); }
    __device__ __forceinline__ bool reaches(Bound b) const { return __hgeu2_mask(v, b) != 0u; }
    __device__ __forceinline__ float value() const { return larger(__low2float(v), __high2float(v)); }
};
template <>
struct Most<__nv_bfloat16> {
    __nv_bfloat162 v;
    __device__ __forceinline__ explicit Most(const uint4& q) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
        v = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    }
    using Bound = __nv_bfloat162;
    static __device__ __forceinline__ Bound bound(float least) { return __bfloat162bfloat162(__float2bfloat16_rd(least)); }
    __device__ __forceinline__ bool reaches(Bound b) const { return __hgeu2_mask(v, b) != 0u; }
    __device__ __forceinline__ float value() const { return larger(__low2float(v), __high2float(v)); }
};

constexpr uint32_t QUEUE = 64;   // chunk numbers of a warp

template <typename T, uint32_t CAP>
__global__ void __launch_bounds__(MOST_WARPS * 32, CAP <= 256 ? 2 : 1)
top_kernel(const Top o) {
    chain_entry();
    constexpr int N = tape::CHUNK<T>, E = CAP / 128;   // E: keys to a lane when they are sorted
    constexpr uint32_t LEFT = 32 * E;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint64_t* all_keys = reinterpret_cast<uint64_t*>(smem_raw);   // [warp][CAP]
    __shared__ uint32_t counts[MOST_WARPS], queues[MOST_WARPS][QUEUE];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % o.warps;
    const size_t mine = (size_t)blockIdx.x * (blockDim.x / 32 / o.warps) + warp / o.warps, row = min(mine, (size_t)o.rows - 1);   // (the last again)
    Best<CAP> best{all_keys + warp * CAP, o.k, lane};
    const T* from = static_cast<const T*>(o.logits) + row * o.stride;
    // chunks on 16 bytes; the first and the last may reach out of the row
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(from) % 16) / sizeof(T), chunks = (o.vocab + off + N - 1) / N;
    const uint32_t begin = (uint32_t)((uint64_t)chunks * part / o.warps), end = (uint32_t)((uint64_t)chunks * (part + 1) / o.warps);
    const uint32_t first_whole = off ? 1 : 0, behind_whole = (o.vocab + off) / N;   // [..): chunks that lie in the row
    const T* aligned = from - off;
    const auto load = [&](uint32_t chunk) {
        tape::Raw<T> raw;
        if (chunk >= first_whole && chunk < behind_whole && chunk < end) {
            raw.q = *reinterpret_cast<const uint4*>(aligned + (size_t)chunk * N);
        } else {
            T* t = reinterpret_cast<T*>(&raw.q);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const uint32_t column = chunk * N + e - off;   // (above the row's length where it lies before the row)
                t[e] = chunk < end && column < o.vocab ? from[column] : tape::from_float<T>(-INFINITY);
            }
        }
        return raw;
    };
    uint32_t* queue = queues[warp];
    uint32_t queued = 0;
    auto bound = Most<T>::bound(best.least);
    // The first of the queue, up to 32, element by element.
    const auto look = [&]() {
        __syncwarp();
        const uint32_t n = min(queued, 32u), chunk = lane < n ? queue[lane] : 0u;
        const uint32_t left = lane + 32 < queued ? queue[lane + 32] : 0u;
        const tape::Raw<T> raw = load(chunk);
        float v[N];
        raw.unpack(v);
        uint32_t pass = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) pass |= (uint32_t)(lane < n && chunk * N + e - off < o.vocab && !(v[e] < best.least)) << e;
        while (__any_sync(FULL, pass != 0)) {
            const uint32_t e = __ffs(pass) - 1;   // (of none: no element)
            float value = v[0];
#pragma unroll
            for (uint32_t i = 1; i < N; ++i) value = e == i ? v[i] : value;
            best.add(pass ? (uint64_t)order_of(value) << 32 | (0xFFFFFFFFu - (chunk * N + e - off)) : 0u);
            pass &= pass - 1;
        }
        if (lane + 32 < queued) queue[lane] = left;
        queued -= n;
        bound = Most<T>::bound(best.least);
    };
    const uint32_t whole_end = min(end, behind_whole);
    // A first bound: bits from the top while `need` chunk maxima are not below it, until not many more are.  Of several warps each looks
    // for its share of the k, and no bound is above the least of theirs.
    const uint32_t need = (o.k + o.warps - 1) / o.warps;
    uint32_t t = 0;
    if (end - begin > need) {
        uint32_t high[SAMPLE], largest = 0, smallest = FULL;
#pragma unroll
        for (uint32_t u = 0; u < SAMPLE; ++u) {
            const uint32_t chunk = begin + u * 32 + lane;
            const bool whole = chunk >= first_whole && chunk < whole_end;
            high[u] = whole ? order_of(Most<T>(*reinterpret_cast<const uint4*>(aligned + (size_t)chunk * N)).value()) : 0u;
            largest = max(largest, high[u]);
            smallest = min(smallest, high[u]);
        }
        uint32_t bit;
        t = common(largest, smallest, &bit);
        for (uint32_t left = FULL; bit >= 0x1000u && left > need + need / 8; bit >>= 1) {
            uint32_t n = 0;
#pragma unroll
            for (uint32_t u = 0; u < SAMPLE; ++u) n += high[u] >= (t | bit);
            n = __reduce_add_sync(FULL, n);
            if (n >= need) {
                t |= bit;
                left = n;
            }
        }
    }
    if (o.warps > 1) {
        if (lane == 0) counts[warp] = t;
        __syncthreads();
        for (uint32_t w = 0; w < o.warps; ++w) t = min(t, counts[warp - part + w]);
        __syncthreads();
    }
    if (t) {
        best.set_bound((uint64_t)t << 32);
        bound = Most<T>::bound(best.least);
    }
    for (uint32_t tile = begin; tile < end; tile += TILE * 32) {
        tape::Raw<T> raw[TILE];
        if (tile >= first_whole && tile + TILE * 32 <= whole_end) {
            const T* at = aligned + (size_t)(tile + lane) * N;
#pragma unroll
            for (uint32_t u = 0; u < TILE; ++u) raw[u].q = *reinterpret_cast<const uint4*>(at + u * 32 * N);
        } else {
#pragma unroll
            for (uint32_t u = 0; u < TILE; ++u) raw[u] = load(tile + u * 32 + lane);
        }
        uint32_t pass = 0;   // a bit per chunk
#pragma unroll
        for (uint32_t u = 0; u < TILE; ++u) pass |= (uint32_t)Most<T>(raw[u].q).reaches(bound) << u;
        for (;;) {   // (a round for each of the most that a lane has: in the middle of a long row none or one)
            const uint32_t mask = __ballot_sync(FULL, pass != 0);
            if (!mask) break;
            if (pass) queue[queued + __popc(mask & ((1u << lane) - 1u))] = tile + (__ffs(pass) - 1) * 32 + lane;
            pass &= pass - 1;
            queued += __popc(mask);
            if (queued >= 32) look();
        }
    }
    while (queued) look();
    best.keep(max(o.k, LEFT));
    if (o.warps > 1) {
        if (lane == 0) counts[warp] = best.count;
        __syncthreads();
        if (part) return;
        for (uint32_t w = 1; w < o.warps; ++w) {
            const uint32_t n = counts[warp + w];
            for (uint32_t i = 0; i < n; i += 32) best.add(i + lane < n ? all_keys[(warp + w) * CAP + i + lane] : 0u);
        }
        best.keep(max(o.k, LEFT));
    }
    if (mine >= o.rows) return;
    // in falling order: the complements in rising order
    uint64_t v[E];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = lane * E + i < best.count ? ~best.keys[lane * E + i] : ~0ull;
    block_sort<uint64_t, E, 32>(v, nullptr, lane);
    T* out = static_cast<T*>(o.out) + row * o.k;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (lane * E + i >= o.k) break;
        o.ids[row * o.k + lane * E + i] = (int32_t)(uint32_t)v[i];   // (the complement of the column's)
        out[lane * E + i] = tape::from_float<T>(of_order(~(uint32_t)(v[i] >> 32)));
    }
}

template <typename T, uint32_t CAP>
void launch(const Stream& s, const Top& o) {
    const uint32_t warps = std::max(4u, o.warps);   // of a CTA: few, since they end together
    const size_t smem = warps * CAP * 8;
    if (smem > 48 * 1024) s.allow_shared(top_kernel<T, CAP>, MOST_WARPS * CAP * 8);
    s.chain("top_logits", top_kernel<T, CAP>, (unsigned)ceil_div(o.rows, warps / o.warps), warps * 32, smem, o);
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
    // Warps enough for every SM, of two tiles each at least.  us with up to 8 / 16: 1 x 131072 f32, k = 64 28.6 / 22.0, k = 256 51 / 38;
    // 32 x 131072 bf16 32 / 26.
    const size_t tiles = ceil_div(vocab * size_of(dtype), TILE * 32 * 16);
    o.warps = 1;
    while (o.warps < MOST_WARPS && rows * o.warps < (size_t)s.rt->sm_count * 16 && tiles >= 4 * o.warps) o.warps *= 2;
    if (dtype == F32) launch_by_k<float>(s, o);
    else if (dtype == F16) launch_by_k<__half>(s, o);
    else launch_by_k<__nv_bfloat16>(s, o);
}

}  // namespace dev
}  // namespace ullis
