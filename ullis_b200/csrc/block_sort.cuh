// Keys of a CTA in rising order: a bitonic network over E keys per thread in registers.  Steps over fewer than E keys stay in a
// thread, those over fewer than 32 E go by shuffles, the few others through shared memory: 2048 keys of 32 bits by 256 threads take six
// such exchanges where a network in shared memory takes 66 barriers.  cluster_sort goes on from there over the CTAs of a cluster.
#pragma once
#include <stdint.h>

namespace ullis {
namespace dev {

// Steps of one run, from `step` down to 1, over E keys of each of THREADS threads: thread t has keys t * E .. of them, which lie at `base`
// among all that are sorted (a multiple of E * THREADS).  `shared`: room for E * THREADS keys, free before and after (32 threads, a warp:
// none is needed, and nobody waits).
template <typename K, int E, int THREADS>
__device__ __forceinline__ void sort_steps(K (&v)[E], K* shared, uint32_t t, uint32_t base, uint32_t run, uint32_t step) {
    const uint32_t first = base + t * E;
    const bool rising = (first & run) == 0;   // (of runs of more than E keys: the same for all of a thread's)
    if constexpr (THREADS > 32) {
#pragma unroll 1
        for (; step >= 32u * E; step >>= 1) {
            const uint32_t apart = step / E;
            const bool smaller = ((t & apart) == 0) == rising;
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
#pragma unroll
    for (uint32_t apart = 16; apart > 0; apart >>= 1) {
        if (step < apart * E) continue;
        const bool smaller = ((t & apart) == 0) == rising;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const K other = __shfl_xor_sync(0xffffffffu, v[i], apart);
            v[i] = (v[i] < other) == smaller ? v[i] : other;
        }
    }
#pragma unroll
    for (int within = E / 2; within > 0; within >>= 1) {
        if ((uint32_t)within >= run) continue;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (i & within) continue;
            const K a = v[i], b = v[i | within];
            const bool keep = (a < b) == (((first + i) & run) == 0);
            v[i] = keep ? a : b;
            v[i | within] = keep ? b : a;
        }
    }
}
// Of a CTA's keys alone; rising where `base` has the bit E * THREADS not set.
template <typename K, int E, int THREADS>
__device__ __forceinline__ void block_sort(K (&v)[E], K* shared, uint32_t t, uint32_t base = 0) {
    constexpr uint32_t N = (uint32_t)E * THREADS;
#pragma unroll
    for (uint32_t run = 2; run <= (uint32_t)E && run <= N; run <<= 1) sort_steps<K, E, THREADS>(v, shared, t, base, run, 0);
#pragma unroll 1
    for (uint32_t run = 2 * E; run <= N; run <<= 1) sort_steps<K, E, THREADS>(v, shared, t, base, run, run >> 1);
}
// Of the keys of all `ctas` (a power of two) CTAs of a cluster: CTA r has those from r * E * THREADS on.  Steps between CTAs go through
// `outbox`, room for 2 E * THREADS keys in the same place of each CTA's shared memory, in two halves that take turns.
template <typename K, int E, int THREADS>
__device__ __forceinline__ void cluster_sort(K (&v)[E], K* shared, K* outbox, uint32_t rank, uint32_t ctas) {
    constexpr uint32_t N = (uint32_t)E * THREADS;
    const uint32_t t = threadIdx.x, base = rank * N;
    block_sort<K, E, THREADS>(v, shared, t, base);
    uint32_t turn = 0;
    for (uint32_t run = 2 * N; run <= ctas * N; run <<= 1) {
        const bool rising = (base & run) == 0;
        for (uint32_t apart = run / N / 2; apart > 0; apart >>= 1) {
            K* box = outbox + turn * N;
            turn ^= 1;
#pragma unroll
            for (int i = 0; i < E; ++i) box[i * THREADS + t] = v[i];
            // (before a half is written again all have met once more, and have read it before)
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            const bool smaller = ((rank & apart) == 0) == rising;
            uint32_t from;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"((uint32_t)__cvta_generic_to_shared(box + t)), "r"(rank ^ apart));
#pragma unroll
            for (int i = 0; i < E; ++i) {
                K other;
                if constexpr (sizeof(K) == 4)
                    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(from + (uint32_t)(i * THREADS * sizeof(K))) : "memory");
                else
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(other) : "r"(from + (uint32_t)(i * THREADS * sizeof(K))) : "memory");
                v[i] = (v[i] < other) == smaller ? v[i] : other;
            }
        }
        sort_steps<K, E, THREADS>(v, shared, t, base, run, N >> 1);
    }
    // (no CTA leaves while another may still read its box)
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace dev
}  // namespace ullis
