// Matrix products D[M,N] = A . B^T on CTA pairs (tcgen05.mma.cta_group::2, M = 256), 16-bit operands, f32 accumulators in TMEM,
// for the gradient of the head and of linears.  Either operand may lie in memory with its K elements side by side (row-major [M,K])
// or with its M (N) elements side by side ([K,M] row-major): the tensor cores read both from 128-byte-swizzled tiles, so a
// gradient product takes an activation as the forward pass left it and nothing is transposed in memory.
//
//  * A pair has 256 rows and 256 * ACCS columns of the output.  CTA r of it brings rows 128 r .. of A and of each 256 columns'
//    B into its own ring of shared memory; the even CTA issues the products, each CTA finds its 128 rows in its own TMEM.
//    ACCS = 1: two accumulators take turns, the epilogue drains one while the other fills.  ACCS = 2: one of 512 columns, every
//    element of A is fetched once for 512 columns; for products whose K is long beside the epilogue.
//  * Warp 0 fetches, warp 1 multiplies, 16 warps are the epilogue: four to a TMEM lane quarter, 64 columns each, with 96 registers
//    to a thread.
//  * The grid is persistent; which tiles a pair has follows from its number alone (Work below), so all sums have a fixed order.
//
// Epilogues:
//   LSE    z = scale * acc + bias: running maximum and sum of exp over the columns but the target's, per row and quarter of the
//          columns.  (The target's logit, whose terms have one sign where a model has learnt anything, is computed with rounding
//          elsewhere: the loss is the difference of two large numbers, and what the tensor cores cut off would stay in it.)
//   GRAD   g = softmax(z) - onehot, by rows as the 16-bit operand g * scale * 2^k of the products that follow, and by columns the
//          f32 sums of g and g * acc
//   STORE  alpha * acc in 16 bits, or into an f32 accumulator, or as one of several partial sums
//   SUM    acc in f32: the tensor cores cut off what falls below the accumulator's last bit (measured: K = 16384 1.9e-5 off in
//          norm, 1.1e-4 where all terms have one sign; K = 512 6e-7), so every 512 terms the accumulator moves to registers
//          and is added there with rounding, in FP16 with a factor per 32 columns.  A stretch of 512 terms whose B does not fit into
//          FP16 comes in bf16, and goes through the accumulator twice, for the two bf16 parts of A
// Measured at 16384 x 512 x 8192 in FP16 (137 GFLOP each, cold caches): LSE 106 us, GRAD 125, STORE 105 (one accumulator at a time)
// and 95 (two); SUM at 2048 x 16384 -> 512 in bf16 35 us for 34 GFLOP.  The tensor pipe is busy 65, 54, 69, 70 and 48 % of the
// time.  The products of such a call take the pipe 113 thousand cycles, a loop without an epilogue 148 (the same without the loads of
// A: neither L2 nor the ring bounds it), LSE 177, GRAD 211: there it is the exp and the sums of the 16 epilogue warps, 36 and 45 %
// of the issue slots; a STORE has 64 tiles for 74 pairs.
// Every wait is bounded and reports through the status words, as in tc_gemm_ws2.cuh.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.hpp"
#include "tc_ptx.cuh"

namespace ullis {
namespace pg {

enum { LSE = 0, GRAD = 1, STORE = 2, SUM = 3 };

constexpr uint32_t BM = 256, BN = 256, BK = 64;         // of a pair, per accumulator
constexpr uint32_t OPERAND_BYTES = 128 * BK * 2;        // one CTA's 128 rows of A, or of one accumulator's B
constexpr uint32_t EPI_WARPS = 16;
constexpr int THREADS = 64 + 32 * (int)EPI_WARPS;
constexpr uint32_t MAX_STAGES = 6, SMEM_LIMIT = 227 * 1024;
// per epilogue warp
constexpr uint32_t STAGING_BYTES = 16 * 128;            // 16 rows of 64 16-bit outputs; GRAD has two of them
constexpr uint32_t COLUMN_BYTES = 2 * 64 * 4;           // constants of its columns
constexpr uint32_t ROW_BYTES = 2 * 4 * 32 * 4;          // GRAD: what its rows need, of this tile and of the next
constexpr uint32_t SUM_BLOCKS = 8;                      // k-blocks of a stretch of K, after which SUM adds with rounding

struct Maps {
    CUtensorMap a, b;
    CUtensorMap out;           // GRAD: [M, pitch] in boxes of 64 columns x 16 rows; SUM: A in two bf16 parts (Params::parts)
};

struct Params {
    uint32_t M, N, K;
    uint32_t a_mn, b_mn;       // operand with M (N) side by side
    uint32_t stages;
    uint32_t* status;
    // How many of the rows of a batch count is known on the device only: M (count_k: K) is *counted and at most what it says above,
    // which the arrays are laid out for.  null: it is what it says.
    const uint32_t* counted;
    uint32_t count_k;
    // LSE, GRAD: columns [n_first, n_first + N) of the vocabulary
    const uint16_t *scale, *bias;   // FP16 or null, of the first column
    const int32_t* target;          // [M] column of the vocabulary, or negative
    uint32_t n_first;
    uint32_t piece_tiles;      // LSE: column tiles that all pairs go through before the next ones
    float2* row_part;          // LSE: [piece] of [slot][4][rows that count, whole tiles]
    size_t row_part_piece;     // elements of a piece
    const float* lse2;         // GRAD: [M] log2 of the sum of exp, +inf for a row that does not count
    const float* target_acc;   // GRAD: [M] the target's product, added with rounding
    const float* target_g;     // GRAD: [M] its probability - 1
    const float* factor;       // GRAD: 2^k ; STORE: alpha
    uint32_t pitch;            // GRAD: of col_part, whole tiles
    float* col_part;           // GRAD: [slot][8][2][pitch]
    // STORE, SUM
    uint32_t splits;           // of K
    uint32_t beside;           // STORE: nothing of the kernel before this one is read or written, only of those before that
    void* out;                 // 16 bits [M][N] (STORE) or f32 [M][N] (SUM, STORE with out_f32), where nothing follows
    uint32_t out_f32;
    const int32_t* out_rows;   // STORE: the row of `out` that row m goes to, or null
    float* accum;              // f32 [M][N]; STORE: read first if `accum_read`, written unless `out` is
    uint32_t accum_read;
    float* partial;            // splits > 1: [split][M][N]
    uint32_t pairs_ok;         // two columns of every row of its f32 arrays lie on 8 bytes (`out` is aligned to its elements only)
    // SUM, FP16: for each stretch of K and 32 columns what its sums are multiplied by, [stretch][ceil(N / 32)], and for each tile of
    // columns and stretch, [n_tiles][parts_pitch, a multiple of 8], a byte that is not 0 where B lies there in bf16 instead of FP16: A is
    // then the sum of two bf16 matrices, columns [0, M) and [parts_at, parts_at + M) of maps.out, and the product goes through the
    // stretch once with each
    const float* col_factor;
    const uint8_t* parts;
    uint32_t parts_pitch, parts_at;
};

inline uint32_t stage_bytes(int accs) { return OPERAND_BYTES * (1 + accs); }
// Barriers first, then (on 1024 bytes) the ring, then what the epilogue warps have.
constexpr uint32_t epi_bytes(int epi) {
    return epi == GRAD ? 2 * STAGING_BYTES + COLUMN_BYTES + ROW_BYTES : epi == STORE ? STAGING_BYTES : epi == LSE ? COLUMN_BYTES : 0u;
}
inline uint32_t fixed_bytes(int epi) { return 2 * 1024 /*barriers, alignment*/ + EPI_WARPS * epi_bytes(epi); }
inline uint32_t stages_for(int epi, int accs) {
    const uint32_t fit = (SMEM_LIMIT - fixed_bytes(epi)) / stage_bytes(accs);
    return fit < MAX_STAGES ? fit : MAX_STAGES;
}
inline uint32_t smem_bytes(int epi, int accs) { return fixed_bytes(epi) + stages_for(epi, accs) * stage_bytes(accs); }

// `total` tiles in a row are shared out to `pairs` (at most `total`) pairs without gaps: pair c has [first(c), first(c + 1)).
struct Share {
    uint32_t total, pairs;
    __host__ __device__ uint32_t first(uint32_t c) const { return (uint32_t)((uint64_t)c * total / pairs); }
    __host__ __device__ uint32_t owner(uint32_t tile) const { return (uint32_t)((((uint64_t)tile + 1) * pairs - 1) / total); }
};
__host__ __device__ inline Share share_of(uint32_t total, uint32_t pairs) { return Share{total, total < pairs ? total : pairs}; }

// What a pair computes, tile by tile; every warp of the pair goes through the same list.
//  LSE   piece after piece of the columns (whose B stays in L2); in a piece the tiles of 256 rows follow one another
//  GRAD  tiles of 256 columns follow one another
//  STORE, SUM  jobs of one tile and one range of K, dealt out in turn
template <int EPI, int ACCS>
struct Work {
    const Params& p;
    uint32_t pair, pairs, M, m_tiles, n_tiles, blocks;
    uint32_t piece = 0, left = 0, outer = 0, inner = 0, width = 0;   // LSE, GRAD: tiles left in the piece, (outer, inner < width) of the next
    uint32_t job = 0;                                                // STORE, SUM
    // the tile; of K the k-blocks [k0, k1), none where there are fewer than ranges (its sum is 0 and nobody waits for it)
    uint32_t m = 0, n = 0, k0 = 0, k1 = 0, split = 0, in_piece = 0;

    __device__ Work(const Params& p_, uint32_t pair_, uint32_t pairs_) : p(p_), pair(pair_), pairs(pairs_) {
        const uint32_t counted = p.counted ? *p.counted : 0xFFFFFFFFu;
        M = p.count_k ? p.M : min(p.M, counted);
        m_tiles = (M + BM - 1) / BM;
        n_tiles = (p.N + BN * ACCS - 1) / (BN * ACCS);
        blocks = ((p.count_k ? min(p.K, counted) : p.K) + BK - 1) / BK;
        k1 = blocks;
        job = pair;
        if (EPI == LSE) open(m_tiles, min(p.piece_tiles, n_tiles));
        if (EPI == GRAD) open(n_tiles, m_tiles);
    }
    // where the stretch from k-block kb on ends (STORE: the range)
    __device__ uint32_t stretch_end(uint32_t kb) const { return EPI == SUM ? min(k1, kb + SUM_BLOCKS) : k1; }
    __device__ void open(uint32_t outers, uint32_t inners) {
        const Share s = share_of(outers * inners, pairs);
        width = inners;
        left = 0;
        if (pair < s.pairs) {   // (no pair has a share of nothing)
            const uint32_t first = s.first(pair);
            left = s.first(pair + 1) - first;
            outer = first / inners;
            inner = first - outer * inners;
        }
    }
    __device__ bool next() {
        if (EPI == LSE || EPI == GRAD) {
            while (left == 0) {
                if (EPI == GRAD || ++piece * p.piece_tiles >= n_tiles) return false;
                open(m_tiles, min(p.piece_tiles, n_tiles - piece * p.piece_tiles));
            }
            m = EPI == LSE ? outer : inner;
            n = EPI == LSE ? piece * p.piece_tiles + inner : outer;
            in_piece = piece;
            --left;
            if (++inner == width) { inner = 0; ++outer; }
            return true;
        }
        if (job >= m_tiles * n_tiles * p.splits) return false;
        const uint32_t tile = job / p.splits;
        split = job % p.splits;
        m = tile / n_tiles;
        n = tile % n_tiles;
        const uint32_t step = EPI == SUM ? SUM_BLOCKS : 1u, steps = (blocks + step - 1) / step;   // SUM: whole stretches
        k0 = (uint32_t)((uint64_t)split * steps / p.splits) * step;
        k1 = min(blocks, (uint32_t)((uint64_t)(split + 1) * steps / p.splits) * step);
        job += pairs;
        return true;
    }
};

// Whether A comes in two parts in the stretch of k-block kb of a tile: eight stretches to a load (one each took 6 of 113 us at 16384 x
// 2048 -> 2048, whatever the distance between the load and its use).
struct InParts {
    uint64_t eight = 0;
    uint32_t held = 0xFFFFFFFFu;
    __device__ bool operator()(const Params& p, uint32_t n, uint32_t kb) {
        const uint32_t stretch = kb / SUM_BLOCKS;
        if (stretch / 8 != held) {
            held = stretch / 8;
            eight = *reinterpret_cast<const uint64_t*>(p.parts + (size_t)n * p.parts_pitch + held * 8);
        }
        return (eight >> 8 * (stretch % 8) & 0xFFu) != 0;
    }
};

// 16 lanes x 64 columns: register 4 j + i of thread t has row t / 4 + 8 (i / 2), column 8 j + 2 (t % 4) + i % 2
__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// the same, 32 and 16 columns
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_16x16(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
// 32 lanes x 16 columns, a row per thread
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// All loads so far have landed; the registers that the last one wrote are named, so that nothing is read from them before.
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// Four 8 x 8 blocks of 16-bit pairs as the loads above leave them (a register each) to rows of 16 bytes; lane 8 b + i gives the
// address of row i of block b.
__device__ __forceinline__ void store_blocks(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t smem, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem),
                 "r"(x), "r"(y)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int LEFT>
__device__ __forceinline__ void tma_store_read() {   // all but LEFT of this thread's stores have read their shared memory
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void copy_word(const void* to, const void* from, bool in) {   // global -> shared, or a zero
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(ptx::smem_u32(to)), "l"(from), "r"(in ? 4 : 0) : "memory");
}

// Descriptor of a tile with the M (N) elements side by side: atoms of 64 of them (128 bytes, swizzled) x 8 k, 1024 bytes apart
// along k; the next 64 elements 64 k-rows, 8192 bytes, on.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two f32 operations per instruction
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 of_two(uint64_t r) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float half_at(const uint16_t* p, uint32_t i, float missing) {
    return p ? __half2float(__ushort_as_half(p[i])) : missing;
}

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile uint32_t* s_error) {
    for (uint32_t spin = 0; spin < ptx::WAIT_POLLS; ++spin) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        if (spin > 64) {
            __nanosleep(spin > 4096 ? 256 : 32);
            if ((spin & 1023u) == 0 && *s_error) return false;
        }
    }
    return false;
}

// A wait at `site` has run out.  On a caller's stream `status` is pinned host memory.
__device__ __forceinline__ void report_wait(volatile uint32_t* status, uint32_t site) {
    status[1] = site;
    __threadfence_system();
    status[0] = ULLIS_DEV_WAIT_TIMEOUT;
}

constexpr float LOG2E = 1.4426950408889634f;

// Scale and bias (FP16, two lanes' worth: columns lane and 32 + lane) of 64 columns from n0 on, on their way while the tile before
// is worked on; and as the constants that the epilogue reads: both times log2 e.  Columns past N have a probability of 0.
struct Columns {
    float scale[2], bias[2];
    __device__ void fetch(const Params& p, uint32_t n0, int lane) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t n = n0 + i * 32 + lane;
            scale[i] = n < p.N ? half_at(p.scale, n, 1.0f) : 0.0f;
            bias[i] = n < p.N ? half_at(p.bias, n, 0.0f) : -INFINITY;
        }
    }
    __device__ void keep(float* to, int lane) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            to[i * 32 + lane] = scale[i] * LOG2E;
            to[64 + i * 32 + lane] = bias[i] * LOG2E;
        }
    }
};
// The accumulator has been read: one arrival on the even CTA's barrier.  (With release at the scope of the cluster the arrival
// waits for the warp's stores to memory, which this barrier says nothing of.)
__device__ __forceinline__ void arrive_even(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

template <int EPI, int ACCS, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
pair_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr uint32_t STAGE = OPERAND_BYTES * (1 + ACCS);
    const uint32_t STAGES = p.stages;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem);   // [STAGES] even CTA: both CTAs' bytes have landed
    uint64_t* empty = full + MAX_STAGES;                  // [STAGES] the products that read the stage are done
    uint64_t* tmem_full = empty + MAX_STAGES;             // [2] accumulator complete
    uint64_t* tmem_empty = tmem_full + 2;                 // [2] even CTA: drained in both CTAs
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
    uint32_t* s_error = tmem_slot + 1;
    smem += 1024;
    uint8_t* epi_smem = smem + STAGES * STAGE;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            ptx::mbar_init(&tmem_full[b], 1);
            ptx::mbar_init(&tmem_empty[b], 2 * EPI_WARPS);
        }
        *s_error = 0;
        ptx::fence_mbar_init();
        ptx::tma_prefetch_desc(&maps.a);
        ptx::tma_prefetch_desc(&maps.b);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(tmem_slot, 512);
        ptx::tmem_relinquish_pair();
    }
    // A kernel with `beside` runs beside the one before: that one has waited for those before it, or this one would not have been
    // launched, and it is waited for at the end, so that whoever waits for this kernel has waited for both.
    if (EPI == STORE && p.beside) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    else chain_entry();
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    constexpr uint32_t BUFFERS = ACCS == 1 ? 2 : 1;
    constexpr bool BY_STRETCH = EPI == SUM && !BF16;   // stretches of K with a type and a factor of their own
    Work<EPI, ACCS> work(p, pair, pairs);

    if (warp == 0) {
        // ------------------------------------------------------ fetching (both CTAs, own rows)
        if (ptx::elect_one()) {
            const uint32_t full_even = ptx::cluster_map(full, 0);
            uint32_t it = 0;
            bool ok = true;
            while (ok && work.next()) {
                const int32_t m0 = (int32_t)(work.m * BM + rank * 128), n0 = (int32_t)(work.n * BN * ACCS + rank * 128);
                const auto fetch = [&](uint32_t kb, const CUtensorMap* map_a, int32_t ma) {
                    const uint32_t s = it % STAGES;
                    if (it >= STAGES && !wait(&empty[s], ((it / STAGES) & 1u) ^ 1u, s_error)) {
                        atomicCAS(s_error, 0u, 1u);
                        ok = false;
                        return;
                    }
                    uint8_t* st = smem + s * STAGE;
                    const int32_t k = (int32_t)(kb * BK);
                    const uint32_t bar = full_even + 8 * s;
                    if (rank == 0) ptx::mbar_arrive_expect_tx(&full[s], 2 * STAGE);
                    if (p.a_mn) {
                        ptx::tma_load_2d_pair(st, map_a, bar, ma, k);
                        ptx::tma_load_2d_pair(st + 8192, map_a, bar, ma + 64, k);
                    } else {
                        ptx::tma_load_2d_pair(st, map_a, bar, k, ma);
                    }
#pragma unroll
                    for (int i = 0; i < ACCS; ++i) {
                        uint8_t* bt = st + (1 + i) * OPERAND_BYTES;
                        const int32_t nb = n0 + i * (int32_t)BN;
                        if (p.b_mn) {
                            ptx::tma_load_2d_pair(bt, &maps.b, bar, nb, k);
                            ptx::tma_load_2d_pair(bt + 8192, &maps.b, bar, nb + 64, k);
                        } else {
                            ptx::tma_load_2d_pair(bt, &maps.b, bar, k, nb);
                        }
                    }
                    ++it;
                };
                if constexpr (BY_STRETCH) {
                    InParts in_parts;
                    for (uint32_t from = work.k0; from < work.k1 && ok;) {
                        const uint32_t last = work.stretch_end(from);
                        const bool parts = in_parts(p, work.n, from);
                        for (uint32_t kb = from; kb < last && ok; ++kb) fetch(kb, parts ? &maps.out : &maps.a, m0);
                        if (parts)
                            for (uint32_t kb = from; kb < last && ok; ++kb) fetch(kb, &maps.out, m0 + (int32_t)p.parts_at);
                        from = last;
                    }
                } else {
                    for (uint32_t kb = work.k0; kb < work.k1; ++kb) {
                        fetch(kb, &maps.a, m0);
                        if (!ok) break;
                    }
                }
            }
            // On the way out after a failed wait, leave no copy in flight (as in tc_gemm_ws2.cuh: the even CTA waits for every
            // stage filled last, the odd one, which cannot poll those barriers, far longer than a copy takes).
            if (!ok && rank == 0) {
                const uint32_t first = it > STAGES ? it - STAGES : 0;
                for (uint32_t k = first; k < it; ++k) ptx::mbar_wait(&full[k % STAGES], (k / STAGES) & 1u, 1u << 12);
            }
            if (!ok && rank == 1)
                for (int i = 0; i < 64; ++i) __nanosleep(1000);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------ products (even CTA)
        if (rank == 0 && ptx::elect_one()) {
            const uint32_t idesc_own = ptx::idesc_f16(BF16, BF16, BM, BN) | p.a_mn << 15 | p.b_mn << 16;
            const uint32_t idesc_bf16 = ptx::idesc_f16(true, true, BM, BN) | p.a_mn << 15 | p.b_mn << 16;
            const uint32_t a_step = p.a_mn ? 2048u : 32u, b_step = p.b_mn ? 2048u : 32u;   // 16 k
            const uint32_t ring = ptx::smem_u32(smem);
            uint32_t it = 0, done = 0;   // k-blocks, accumulators
            bool ok = true;
            while (ok && work.next()) {
                InParts in_parts;
                for (uint32_t kb = work.k0; kb < work.k1 && ok;) {
                    const bool parts = BY_STRETCH && in_parts(p, work.n, kb);   // this stretch's products in bf16, and twice as many
                    const uint32_t last = EPI == SUM ? work.stretch_end(kb) : work.k1, idesc = BY_STRETCH && parts ? idesc_bf16 : idesc_own;
                    const uint32_t end = BY_STRETCH && parts ? 2 * last - kb : last;
                    const uint32_t buf = done % BUFFERS;
                    if (done >= BUFFERS && !wait(&tmem_empty[buf], ((done / BUFFERS) & 1u) ^ 1u, s_error)) {
                        atomicCAS(s_error, 0u, 2u);
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    bool add = false;
                    for (; kb < end; ++kb, ++it) {
                        const uint32_t s = it % STAGES;
                        if (!wait(&full[s], (it / STAGES) & 1u, s_error)) {
                            atomicCAS(s_error, 0u, 3u);
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after_sync();
                        const uint32_t a = ring + s * STAGE, b = a + OPERAND_BYTES;
#pragma unroll
                        for (uint32_t k4 = 0; k4 < BK / 16; ++k4) {
                            const uint64_t da = p.a_mn ? smem_desc_mn(a + k4 * a_step) : ptx::smem_desc_sw128(a + k4 * a_step);
#pragma unroll
                            for (int i = 0; i < ACCS; ++i) {
                                const uint32_t bi = b + i * OPERAND_BYTES + k4 * b_step;
                                const uint64_t db = p.b_mn ? smem_desc_mn(bi) : ptx::smem_desc_sw128(bi);
                                ptx::mma_f16_ss_pair(tmem_base + (ACCS == 1 ? buf : i) * BN, da, db, idesc, add || k4);
                            }
                        }
                        add = true;
                        ptx::mma_commit_pair(&empty[s]);
                    }
                    ptx::mma_commit_pair(&tmem_full[buf]);   // on the way out too: the epilogues do not wait in vain
                    ++done;
                    if (BY_STRETCH) kb = last;
                }
            }
        }
    } else {
        // ------------------------------------------------------ epilogue (both CTAs, own rows)
        const uint32_t quarter = warp & 3, group = (uint32_t)(warp - 2) >> 2, mine = warp - 2;
        const uint32_t empty_even = ptx::cluster_map(tmem_empty, 0);
        constexpr uint32_t STAGINGS = EPI == GRAD ? 2 : EPI == STORE ? 1 : 0;
        uint8_t* staging = epi_smem + mine * STAGINGS * STAGING_BYTES;   // on 1024 bytes
        float* columns = reinterpret_cast<float*>(epi_smem + EPI_WARPS * STAGINGS * STAGING_BYTES + mine * COLUMN_BYTES);
        uint32_t done = 0;
        // Waits for the next accumulator; false: leave.  The loads are warp-collective: the whole warp decides.
        const auto filled = [&](uint32_t* taddr) {
            const uint32_t buf = done % BUFFERS;
            if (!__all_sync(0xffffffffu, wait(&tmem_full[buf], (done / BUFFERS) & 1u, s_error))) {
                atomicCAS(s_error, 0u, 4u);
                return false;
            }
            ptx::tc_fence_after_sync();
            if (__any_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(s_error) != 0u)) return false;
            *taddr = tmem_base + buf * BN + ((quarter * 32) << 16);
            return true;
        };
        const auto drained = [&]() {
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_even(empty_even + 8 * (done % BUFFERS));
            ++done;
        };
        const uint32_t M = work.M;
        const uint32_t q2 = (lane & 3) * 2, r0 = lane >> 2;   // of the 16 x 64 form: first column of a pair, first row

        if constexpr (EPI == LSE) {
            const uint32_t rows = work.m_tiles * BM;
            uint32_t m_now = 0xFFFFFFFFu, piece_now = 0;
            float top = -INFINITY, sum = 0.0f;
            int32_t target = -1;
            const auto leave = [&]() {
                if (m_now == 0xFFFFFFFFu) return;
                const uint32_t width = min(p.piece_tiles, work.n_tiles - piece_now * p.piece_tiles);
                const uint32_t slot = pair - share_of(work.m_tiles * width, pairs).owner(m_now * width);
                const size_t row = m_now * BM + rank * 128 + quarter * 32 + lane;
                p.row_part[piece_now * p.row_part_piece + (size_t)(slot * 4 + group) * rows + row] = make_float2(top, sum);
            };
            Columns ahead;
            bool more = work.next();
            if (more) ahead.fetch(p, work.n * BN + group * 64, lane);
            while (more) {
                const uint32_t n0 = work.n * BN + group * 64;
                if (work.m != m_now || work.in_piece != piece_now) {
                    leave();
                    m_now = work.m;
                    piece_now = work.in_piece;
                    top = -INFINITY;
                    sum = 0.0f;
                    const uint32_t row = m_now * BM + rank * 128 + quarter * 32 + lane;
                    target = row < M ? p.target[row] : -1;
                }
                __syncwarp();
                ahead.keep(columns, lane);
                __syncwarp();
                more = work.next();
                if (more) ahead.fetch(p, work.n * BN + group * 64, lane);
                uint32_t taddr;
                if (!filled(&taddr)) break;
                // 16 columns are on their way while 16 are worked on
                taddr += group * 64;
                uint32_t r[2][16];
                tmem_ld_32x16(taddr, r[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t(&now)[16] = r[c & 1];
                    tmem_landed(now);
                    if (c < 3) tmem_ld_32x16(taddr + (c + 1) * 16, r[(c + 1) & 1]);
                    else drained();
                    const int32_t hit = target - (int32_t)(n0 + c * 16);
                    const bool hits = __any_sync(0xffffffffu, hit >= 0 && hit < 16);   // of the warp's rows
                    uint64_t z[8];
                    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(columns + c * 16 + i * 2);
                        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(columns + 64 + c * 16 + i * 2);
                        z[i] = fma2((uint64_t)now[i * 2 + 1] << 32 | now[i * 2], s.x, b.x);
                        z[i + 1] = fma2((uint64_t)now[i * 2 + 3] << 32 | now[i * 2 + 2], s.y, b.y);
                    }
                    if (hits) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            z[i] = add2(z[i], two(hit == i * 2 ? -INFINITY : 0.0f, hit == i * 2 + 1 ? -INFINITY : 0.0f));
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 v = of_two(z[i]);
                        best[i & 1] = fmaxf(best[i & 1], fmaxf(v.x, v.y));
                    }
                    best[0] = fmaxf(best[0], best[1]);
                    if (best[0] > top) {
                        sum *= exp2_fast(top - best[0]);   // top = -inf: 0 * 0
                        top = best[0];
                    }
                    const float base = top == -INFINITY ? 0.0f : -top;   // (a NaN among z makes the sum one)
                    const uint64_t base2 = two(base, base);
                    uint64_t here[2] = {0, 0};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 v = of_two(add2(z[i], base2));
                        here[i & 1] = add2(here[i & 1], two(exp2_fast(v.x), exp2_fast(v.y)));
                    }
                    const float2 all = of_two(add2(here[0], here[1]));
                    sum += all.x + all.y;
                }
            }
            leave();
        } else if constexpr (EPI == GRAD) {
            const float from_log2 = *p.factor / LOG2E;   // scale * log2 e -> scale * 2^k
            const Share all = share_of(work.m_tiles * work.n_tiles, pairs);
            uint32_t n_now = 0xFFFFFFFFu;
            uint64_t g_sum[8], ga_sum[8];   // of column pairs 8 j + q2
#pragma unroll
            for (int j = 0; j < 8; ++j) g_sum[j] = ga_sum[j] = 0;
            const auto leave = [&]() {   // the sums of 32 rows: over the lanes that share columns, then out
                if (n_now == 0xFFFFFFFFu) return;
                const uint32_t slot = pair - all.owner(n_now * work.m_tiles);
                float* to = p.col_part + (((size_t)slot * 8 + rank * 4 + quarter) * 2) * p.pitch + n_now * BN + group * 64 + q2;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        g_sum[j] = add2(g_sum[j], __shfl_xor_sync(0xffffffffu, g_sum[j], o));
                        ga_sum[j] = add2(ga_sum[j], __shfl_xor_sync(0xffffffffu, ga_sum[j], o));
                    }
                    if (lane < 4) {
                        *reinterpret_cast<uint64_t*>(to + j * 8) = g_sum[j];
                        *reinterpret_cast<uint64_t*>(to + p.pitch + j * 8) = ga_sum[j];
                    }
                    g_sum[j] = ga_sum[j] = 0;
                }
            };
            // What the rows need lies in shared memory, two tiles in turn; the next tile's is on its way while one is worked on: a
            // word each of lse2, the target's product, its g and the target per lane.
            float* row_smem = reinterpret_cast<float*>(epi_smem + EPI_WARPS * (2 * STAGING_BYTES + COLUMN_BYTES) + mine * ROW_BYTES);
            const auto fetch = [&](uint32_t turn) {
                const uint32_t row = work.m * BM + rank * 128 + quarter * 32 + lane;
                const bool in = row < M;
                float* to = row_smem + turn * 128 + lane;
                copy_word(to, p.lse2 + (in ? row : 0), in);
                copy_word(to + 32, p.target_acc + (in ? row : 0), in);
                copy_word(to + 64, p.target_g + (in ? row : 0), in);
                copy_word(to + 96, p.target + (in ? row : 0), in);
            };
            const uint32_t blocks_at = ptx::smem_u32(staging) + ((lane >> 3) & 1) * 1024 + (lane & 7) * 128;   // of store_blocks: block b has
            const uint32_t block_piece = lane >> 4;                                                           // rows 8 (b % 2) .., piece b / 2
            uint32_t turn = 0;
            bool more = work.next();
            if (more) fetch(0);
            while (more) {
                const uint32_t n0 = work.n * BN + group * 64, m0 = work.m * BM + rank * 128 + quarter * 32;
                if (work.n != n_now) {
                    leave();
                    n_now = work.n;
                    __syncwarp();
                    Columns c;
                    c.fetch(p, n0, lane);
                    c.keep(columns, lane);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
                const float* rows = row_smem + turn * 128;
                turn ^= 1;
                const uint32_t first = p.n_first + n0;
                const bool any = __any_sync(0xffffffffu, m0 + lane < M && reinterpret_cast<const uint32_t*>(rows)[96 + lane] - first < 64u);
                more = work.next();
                if (more) fetch(turn);
                uint32_t taddr;
                if (!filled(&taddr)) break;
                taddr += group * 64;
                // 16 rows at a time, one copy of the code for both: with two the registers ran out.  TARGETS: the target of one of the
                // warp's rows lies in its columns.  Its product and its g are the row's: lse2 is a number of the size of the logits, off
                // by 2e-6 where those are 36, and a model that is sure leaves a g of that size.
                const auto half = [&](int h, auto targets) {
                    uint32_t r[2][8];   // 16 columns are on their way while 16 are worked on
                    tmem_ld_16x16(taddr + ((h * 16) << 16), r[0]);
                    uint64_t l[2];
                    uint32_t at[2];   // the target's column less q2
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t row = h * 16 + i * 8 + r0;
                        const float lse = m0 + row < M ? -rows[row] : -INFINITY;
                        l[i] = two(lse, lse);
                        if (decltype(targets)::value)
                            at[i] = m0 + row < M ? reinterpret_cast<const uint32_t*>(rows)[96 + row] - first - q2 : 0x80000000u;
                    }
                    const uint32_t to = blocks_at + h * STAGING_BYTES;
                    if (lane == 0) tma_store_read<1>();   // the store before the last has read this half
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        uint32_t(&now)[8] = r[j / 2 & 1];
                        tmem_landed(now);
                        if (j < 6) tmem_ld_16x16(taddr + (j + 2) * 8 + ((h * 16) << 16), r[(j / 2 + 1) & 1]);
                        else if (h == 1) drained();
                        uint32_t w[4];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint64_t s = *reinterpret_cast<const uint64_t*>(columns + (j + u) * 8 + q2);
                            const uint64_t b = *reinterpret_cast<const uint64_t*>(columns + 64 + (j + u) * 8 + q2);
                            const uint64_t k = mul2(s, two(from_log2, from_log2));
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint64_t a = (uint64_t)now[u * 4 + i * 2 + 1] << 32 | now[u * 4 + i * 2];
                                const float2 e = of_two(add2(fma2(a, s, b), l[i]));
                                uint64_t g = two(exp2_fast(e.x), exp2_fast(e.y));
                                if (decltype(targets)::value) {
                                    const uint32_t row = h * 16 + i * 8 + r0;
                                    const bool x = at[i] == (uint32_t)(j + u) * 8, y = at[i] == (uint32_t)(j + u) * 8 + 1;
                                    const float2 av = of_two(a), gv = of_two(g);
                                    a = two(x ? rows[32 + row] : av.x, y ? rows[32 + row] : av.y);
                                    g = two(x ? rows[64 + row] : gv.x, y ? rows[64 + row] : gv.y);
                                }
                                g_sum[j + u] = add2(g_sum[j + u], g);
                                ga_sum[j + u] = fma2(g, a, ga_sum[j + u]);
                                const float2 o = of_two(mul2(g, k));
                                w[u * 2 + i] = pack16<BF16>(o.x, o.y);
                            }
                        }
                        // 16-byte piece c of row r at c ^ (r % 8), as the copy below reads it; no bank conflicts
                        store_blocks(to + (((j + block_piece) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (m0 + h * 16 < p.M) tma_store_2d(&maps.out, ptx::smem_u32(staging) + h * STAGING_BYTES, (int32_t)n0, (int32_t)(m0 + h * 16));
                        else asm volatile("cp.async.bulk.commit_group;" ::: "memory");   // (the groups stay in turn)
                    }
                };
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    if (any) half(h, std::true_type{});
                    else half(h, std::false_type{});
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (lane == 0) tma_store_done();
            __syncwarp();
            leave();
        } else if constexpr (EPI == STORE) {
            const float alpha = p.factor ? *p.factor : 1.0f;
            const bool wide = (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
            uint16_t* out = static_cast<uint16_t*>(p.out);
            while (work.next()) {
                uint32_t taddr = 0;
                const bool none = work.k0 == work.k1;
                if (!none && !filled(&taddr)) break;
                const uint32_t m0 = work.m * BM + rank * 128 + quarter * 32;
                float* partial = p.splits > 1 ? p.partial + (size_t)work.split * p.M * p.N : nullptr;
                const bool to16 = !partial && p.out && !p.out_f32;
#pragma unroll 1
                for (uint32_t part = 0; part < 2 * ACCS; ++part) {
                    const uint32_t h = part & 1, c0 = (group * ACCS + (part >> 1)) * 64, n0 = work.n * BN * ACCS + c0;
                    uint32_t r[32] = {};
                    if (!none) {
                        tmem_ld_16x64(taddr + c0 + ((h * 16) << 16), r);
                        ptx::tmem_ld_wait();
                        if (part == 2 * ACCS - 1) drained();
                    }
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                    const auto f32_rows = [&](float* at, const int32_t* rows, bool read, bool write, float times) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t row = m0 + h * 16 + r0 + i * 8;
                            if (row >= M) continue;
                            float* line = at + (size_t)(rows ? rows[row] : row) * p.N;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint32_t c = n0 + j * 8 + q2;
                                float &x = v[j * 4 + i * 2], &y = v[j * 4 + i * 2 + 1];
                                if (p.pairs_ok) {
                                    if (c < p.N) {
                                        float2* both = reinterpret_cast<float2*>(line + c);
                                        if (read) { const float2 old = *both; x += old.x; y += old.y; }
                                        if (write) *both = make_float2(x * times, y * times);
                                    }
                                } else {
                                    if (c < p.N) { if (read) x += line[c]; if (write) line[c] = x * times; }
                                    if (c + 1 < p.N) { if (read) y += line[c + 1]; if (write) line[c + 1] = y * times; }
                                }
                            }
                        }
                    };
                    if (partial) { f32_rows(partial, nullptr, false, true, 1.0f); continue; }
                    if (p.accum) f32_rows(p.accum, nullptr, p.accum_read, !p.out, 1.0f);
                    if (p.out && p.out_f32) f32_rows(static_cast<float*>(p.out), p.out_rows, false, true, alpha);
                    if (!to16) continue;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            *reinterpret_cast<uint32_t*>(staging + (r0 + i * 8) * 128 + ((j ^ r0) << 4) + (lane & 3) * 4) =
                                pack16<BF16>(v[j * 4 + i * 2] * alpha, v[j * 4 + i * 2 + 1] * alpha);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t row = i * 4 + (lane >> 3), piece = lane & 7, gm = m0 + h * 16 + row, c = n0 + piece * 8;
                        const uint4 w = *reinterpret_cast<const uint4*>(staging + row * 128 + ((piece ^ (row & 7)) << 4));
                        if (gm >= M || c >= p.N) continue;
                        uint16_t* to = out + (size_t)(p.out_rows ? p.out_rows[gm] : gm) * p.N + c;
                        if (wide) {
                            *reinterpret_cast<uint4*>(to) = w;
                        } else {
                            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (c + e < p.N) to[e] = (uint16_t)(words[e >> 1] >> (16 * (e & 1)));
                        }
                    }
                    __syncwarp();
                }
            }
        } else {
            static_assert(EPI != SUM || ACCS == 1, "");
            bool ok = true;
            while (ok && work.next()) {
                float v[64];
#pragma unroll
                for (int i = 0; i < 64; ++i) v[i] = 0.0f;
                const uint32_t m0 = work.m * BM + rank * 128 + quarter * 32, n0 = work.n * BN + group * 64, blocks32 = (p.N + 31) / 32;
                for (uint32_t kb = work.k0; kb < work.k1; kb = work.stretch_end(kb)) {
                    uint32_t taddr;
                    float f[2];
                    if constexpr (BY_STRETCH) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            f[i] = n0 + i * 32 < p.N ? p.col_factor[(size_t)(kb / SUM_BLOCKS) * blocks32 + n0 / 32 + i] : 0.0f;
                    }
                    ok = filled(&taddr);
                    if (!ok) break;
#pragma unroll
                    for (int part = 0; part < 4; ++part) {   // 16 rows of 32 columns: with 64 at a time registers spill (47.5 us, so 45.8)
                        uint32_t r[16];
                        tmem_ld_16x32(taddr + group * 64 + (part & 1) * 32 + ((part >> 1) * 16 << 16), r);
                        tmem_landed(r);
                        if (part == 3) drained();
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float& sum = v[part * 16 + i];
                            sum = BY_STRETCH ? fmaf(__uint_as_float(r[i]), f[part & 1], sum) : sum + __uint_as_float(r[i]);   // (f: powers of two)
                        }
                    }
                }
                if (!ok) break;
                float* out = p.splits > 1 ? p.partial + (size_t)work.split * p.M * p.N : static_cast<float*>(p.out);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t row = m0 + r0 + i * 8;
                    if (row >= M) continue;
                    float* line = out + (size_t)row * p.N;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t c = n0 + j * 8 + q2;
                        const int at = (i >> 1) * 32 + j * 4 + (i & 1) * 2;
                        const float x = v[at], y = v[at + 1];
                        if (p.pairs_ok) {
                            if (c < p.N) *reinterpret_cast<float2*>(line + c) = make_float2(x, y);
                        } else {
                            if (c < p.N) line[c] = x;
                            if (c + 1 < p.N) line[c + 1] = y;
                        }
                    }
                }
            }
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();   // neither CTA leaves while the other may still read its tiles or ring its barriers
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
    if (EPI == STORE && p.beside) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (threadIdx.x == 0 && *s_error) report_wait(p.status, 64u + *s_error);
}

}  // namespace pg
}  // namespace ullis
