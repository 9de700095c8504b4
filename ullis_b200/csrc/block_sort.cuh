// Keys of a CTA in rising order: a bitonic network over E keys per thread in registers.  Steps over fewer than E keys stay in a
// thread, those over fewer than 32 E go by shuffles, the few others through shared memory: 2048 keys of 32 bits by 256 threads take six
// such exchanges where a network in shared memory takes 66 barriers.
#pragma once
#include <stdint.h>

namespace ullis {
namespace dev {

// Thread t of THREADS has keys t * E .. of them; `shared` has room for E * THREADS keys and is free before and after (32 threads, a
// warp: none is needed, and nobody waits).
template <typename K, int E, int THREADS>
__device__ __forceinline__ void block_sort(K (&v)[E], K* shared, uint32_t t) {
    constexpr uint32_t N = (uint32_t)E * THREADS;
    const uint32_t first = t * E;
    const auto within = [&](uint32_t run) {   // the steps over fewer than E keys; runs of at most E keys have no others
#pragma unroll
        for (int step = E / 2; step > 0; step >>= 1) {
            if ((uint32_t)step >= run) continue;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if (i & step) continue;
                const bool rising = ((first + i) & run) == 0;
                const K a = v[i], b = v[i | step];
                const bool keep = (a < b) == rising;
                v[i] = keep ? a : b;
                v[i | step] = keep ? b : a;
            }
        }
    };
#pragma unroll
    for (uint32_t run = 2; run <= (uint32_t)E && run <= N; run <<= 1) within(run);
#pragma unroll 1
    for (uint32_t run = 2 * E; run <= N; run <<= 1) {
        const bool rising = (first & run) == 0;
#pragma unroll 1
        for (uint32_t step = run >> 1; step >= (uint32_t)E; step >>= 1) {
            const uint32_t apart = step / E;
            const bool smaller = ((t & apart) == 0) == rising;
            if (THREADS == 32 || apart < 32) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const K other = __shfl_xor_sync(0xffffffffu, v[i], apart);
                    v[i] = (v[i] < other) == smaller ? v[i] : other;
                }
            } else if constexpr (THREADS > 32) {
#pragma unroll
                for (int i = 0; i < E; ++i) shared[i * THREADS + t] = v[i];
                __syncthreads();
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const K other = shared[i * THREADS + (t ^ apart)];
                    v[i] = (v[i] < other) == smaller ? v[i] : other;
                }
                __syncthreads();
            }
        }
        within(run);
    }
}

}  // namespace dev
}  // namespace ullis
