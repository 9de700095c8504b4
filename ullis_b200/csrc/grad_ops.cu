// Cross-entropy of the head with its gradient, and weight gradients from the 8-bit tape, on the products of pair_gemm.cuh.
//
// Head (reference src/model.rs:3132-3275): a = h . s^T, z = scale * a + bias, loss = log sum exp z - z[target], and with
// g = loss_scale * (softmax(z) - onehot), 0 on the rows that do not count (src/model.rs:27-39),
//   g_hidden = (g * scale) . s,  g_weight = (g * scale)^T . h,  g_scale = sum over rows of g * a,  g_bias = sum of g.
// The logits are never kept: one product gives log sum exp of every row, and piece by piece of the vocabulary a second one gives
// g * scale in 16 bits, which the two gradient products read where it lies, by rows and by columns.  8 R V D operations instead of
// the 6 R V D of a step that keeps R x V logits in 32 bits; a logit costs 2 D operations (0.7 ns at D = 512 and 1.5 PFLOP/s per
// 1000) and would cost 8 bytes to write and read (1.2 ns).
//
// g is at most 1, the row scales are FP16 of any size: 2^k with max |scale| * 2^k in [2^14, 2^15) brings g * scale where 16 bits
// hold most of it (FP16 from 2^-24 to 65504), and the products are multiplied by 2^-k * loss_scale at the end.  The rounding of
// g * scale to 16 bits is the same that the training step's operands have (half a step: 2^-11 in FP16, 2^-8 in bf16, independent
// from term to term); g_scale and g_bias are sums of what was not rounded.
//
// Beside the products a call of 16384 x 512 x 8192 takes 7.6 us to list the rows that count, 11.4 to bring both operands into 16
// bits, 5.6 for the rows' sums and 4.7 for the columns': reads and writes of what they name, bound by their latency.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include <cudaTypedefs.h>

#include "device_ops.hpp"
#include "head_entries.cuh"
#include "pair_gemm.cuh"
#include "tape.cuh"

namespace ullis {
namespace dev {
namespace {

constexpr int THREADS = 256;

size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }
size_t ceil_div(size_t n, size_t by) { return (n + by - 1) / by; }
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// The parts of a workspace, one behind the other on 256 bytes.
struct Parts {
    size_t bytes = 0;
    size_t add(size_t n) {
        const size_t at = bytes;
        bytes += up(n, 256);
        return at;
    }
};

// ------------------------------------------------------------------------------------------------ products
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        ULLIS_CUDA_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
        if (!p || q != cudaDriverEntryPointSuccess) fail(ULLIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}
// A 16-bit row-major matrix as an operand: boxes of 64 columns and 128 rows, or (mn: the columns are the operand's M or N) 64 rows.
// The first column is 16-byte aligned and the stride a multiple of 8 elements.
struct Operand {
    const void* data;
    size_t rows, columns, stride;
    bool mn;
};
CUtensorMap map_of(const void* data, size_t rows, size_t columns, size_t stride, uint32_t box_rows, bool bf16) {
    CUtensorMap m;
    const cuuint64_t dims[2] = {columns, rows}, strides[1] = {stride * 2};
    const cuuint32_t box[2] = {64, box_rows}, steps[2] = {1, 1};
    const CUresult r = encode_fn()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(data),
                                   dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail(ULLIS_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
    return m;
}
CUtensorMap operand_map(const Operand& o, bool bf16) { return map_of(o.data, o.rows, o.columns, o.stride, o.mn ? 64 : 128, bf16); }

uint32_t pairs_of(const ullis_cuda_runtime* rt) { return std::max(1, rt->sm_count / 2); }

template <int EPI, int ACCS, bool BF16>
void launch_form(const Stream& s, const char* what, const pg::Maps& maps, const pg::Params& p, uint32_t pairs) {
    const auto kernel = pg::pair_gemm_kernel<EPI, ACCS, BF16>;
    const size_t smem = pg::smem_bytes(EPI, ACCS);
    constexpr int form = (ACCS - 1) * 2 * pg::FORMS + EPI * 2 + BF16;
    static_assert(form < 64, "");
    const uint64_t flag = 1ull << form;
    if (!(s.rt->pair_gemms_ready & flag)) {
        ULLIS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        s.rt->pair_gemms_ready |= flag;
    }
    s.chain(what, kernel, 2 * pairs, pg::THREADS, smem, maps, p);
}
template <int EPI, int ACCS>
void launch(const Stream& s, const char* what, const Operand& a, const Operand& b, bool bf16, pg::Params p, uint32_t pairs,
            const CUtensorMap* out = nullptr) {
    p.a_mn = a.mn;
    p.b_mn = b.mn;
    p.stages = pg::stages_for(EPI, ACCS);
    p.pairs_ok = p.N % 2 == 0 && (!(EPI == pg::SUM || p.out_f32) || aligned(p.out, 8));   // (all others are parts of the workspace)
    p.status = s.status;
    const pg::Maps maps{operand_map(a, bf16), operand_map(b, bf16), out ? *out : CUtensorMap{}};
    if (bf16) launch_form<EPI, ACCS, true>(s, what, maps, p, pairs);
    else launch_form<EPI, ACCS, false>(s, what, maps, p, pairs);
}

// How a product [M, N] over K is cut for `pairs` pairs: accumulators of 256 columns per pair (one or two) and ranges of K.
// Estimated in k-blocks (256 x 256 x 64 on a pair, 0.3 us): rounds * (k-blocks + an epilogue nothing overlaps) and, with several
// ranges, their sums written and read once more: at 8 TB/s for a product that runs alone, whose sums stay in L2 (2048 x 512 x 2048
// takes 1.5 % less in four ranges than in one, which 4 TB/s would choose), at 4 TB/s for the head's two beside one another (at 8 a
// ragged batch of 7655 x 256 x 10007, half of its rows not counted, takes 148 us instead of 117).
// Two accumulators fetch A half as often, which counts where the power limit sets the clock: a head of 16384 x 512 x 8192 takes
// 487 us instead of 494 over seconds, 430 instead of 437 before the limit acts.
// (two: a product of the head, else a SUM, whose ranges are whole stretches of K)
// A product of the head has no more than LONGEST k-blocks in one accumulator, whose additions the tensor cores cut off: sums of 16 384
// terms of one sign are 1.0e-4 too small, of 65 536 4.3e-4, and half a step of FP16 is 2.4e-4 to 4.9e-4.  (4096 x 512 x 131072, whose hidden
// gradient has four ranges for it instead of two: 2.08 ms, with two 2.07.)
struct Cut {
    uint32_t accs, splits;
};
constexpr size_t LONGEST = 16384 / pg::BK;
Cut cut_of(size_t M, size_t N, size_t K, uint32_t pairs, bool two) {
    const size_t blocks = std::max<size_t>(1, ceil_div(K, pg::BK));
    const size_t fewest = two ? ceil_div(blocks, LONGEST) : 1;
    Cut best{1, 1};
    double least = 1e300;
    for (uint32_t accs = 1; accs <= (two && N > 256 ? 2u : 1u); ++accs) {
        const size_t tiles = ceil_div(M, 256) * ceil_div(N, 256 * accs);
        for (uint32_t splits = (uint32_t)fewest; splits <= std::max(fewest, std::min<size_t>(16, std::max<size_t>(1, blocks / 4))); ++splits) {
            const double rounds = (double)ceil_div(tiles * splits, pairs);
            const double epilogue = accs == 2 ? 10.0 : 1.0;
            const size_t most = two ? ceil_div(blocks, splits) : std::min(blocks, ceil_div(ceil_div(blocks, pg::SUM_BLOCKS), splits) * pg::SUM_BLOCKS);
            const double k_blocks = (double)most * (accs == 2 ? 1.9 : 1.0);
            double cost = rounds * (k_blocks + epilogue) + 4.0;
            if (splits > 1) cost += (2.0 * splits + 1.0) * M * N * 4.0 / (two ? 4e6 : 8e6) / 0.3 + 8.0;
            if (cost < least) {
                least = cost;
                best = Cut{accs, splits};
            }
        }
    }
    return best;
}
size_t partial_bytes(size_t M, size_t N, const Cut& c) { return c.splits > 1 ? c.splits * M * N * 4 : 0; }

// The sum of `splits` arrays [M][N], in their order, times alpha as 16 bits or f32; with `accum` added to it, or left there where
// `out` is null.  Of the M rows the first *counted, if given, and row m goes to row out_rows[m] of `out`.  TWICE: of `out` a row is the sum of
// two that follow on one another.  (A form of its own: as an argument it took 1 us of the 19 of a weight gradient of 2048 x 512 x 2048.)
template <typename T, bool TWICE>
__global__ void __launch_bounds__(THREADS)
combine_kernel(const float* __restrict__ partial, uint32_t splits, uint32_t M, uint32_t N, const float* __restrict__ factor, float* __restrict__ accum,
               uint32_t accum_read, T* __restrict__ out, const uint32_t* __restrict__ counted, const int32_t* __restrict__ out_rows) {
    chain_entry();
    const size_t n = (size_t)M * N, i = ((size_t)blockIdx.x * THREADS + threadIdx.x) * 4;
    const size_t end = (counted ? min((size_t)*counted, (size_t)M) * N : n) >> TWICE;
    if (i >= end) return;
    const float alpha = factor ? *factor : 1.0f;
    const bool whole = N % 4 == 0;   // four elements of one row, each of the arrays on 16 bytes
    float v[4] = {};
    if (whole) {
        const size_t at = TWICE ? i + i / N * N : i;   // TWICE: rows 2 m and 2 m + 1
#pragma unroll 8
        for (uint32_t k = 0; k < splits + (accum && accum_read); ++k) {
            const float* from = (k < splits ? partial + k * n : accum) + at;
            float4 t = *reinterpret_cast<const float4*>(from);
            if (TWICE) {
                const float4 u = *reinterpret_cast<const float4*>(from + N);
                t.x += u.x; t.y += u.y; t.z += u.z; t.w += u.w;
            }
            v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
        }
    } else {
        for (uint32_t k = 0; k < splits + (accum && accum_read); ++k)
            for (int e = 0; e < 4; ++e)
                for (uint32_t t = 0; t <= TWICE && i + e < end; ++t)
                    v[e] += (k < splits ? partial + k * n : accum)[i + e + (TWICE ? ((i + e) / N + t) * N : 0)];
    }
    uint32_t row = (uint32_t)(i / N), c = (uint32_t)(i - (size_t)row * N);
    for (int e = 0; e < 4; ++e) {
        if (i + e >= end) break;
        if (out) out[(size_t)(out_rows ? out_rows[row << TWICE] : (int32_t)row) * N + c] = tape::from_float<T>(v[e] * alpha);
        else accum[i + e] = v[e];
        if (++c == N) { c = 0; ++row; }
    }
}

struct Output {
    void* out;             // 16 bits or (f32) f32; null: `accum` is left
    bool f32;
    float* accum;
    bool accum_read;
    const float* factor;
    float* partial;
    const uint32_t* counted;   // pair_gemm.cuh: rows of the product, or (count_k) terms of its sums
    bool count_k;
    const int32_t* rows;       // where its rows go
    bool beside;               // pair_gemm.cuh
    bool twice;                // combine_kernel's TWICE, where `out` is written
};
// A product, alpha * (a . b + accum) ...
void product(const Stream& s, const char* what, const Operand& a, const Operand& b, bool bf16, size_t M, size_t N, size_t K, const Cut& cut,
             const Output& o) {
    pg::Params p{};
    p.M = (uint32_t)M;
    p.N = (uint32_t)N;
    p.K = (uint32_t)K;
    p.splits = cut.splits;
    p.out = o.out;
    p.out_f32 = o.f32;
    p.accum = o.accum;
    p.accum_read = o.accum_read;
    p.factor = o.factor;
    p.partial = o.partial;
    p.counted = o.counted;
    p.count_k = o.count_k;
    p.out_rows = o.rows;
    p.beside = o.beside;
    const uint32_t pairs = (uint32_t)std::min<size_t>(pairs_of(s.rt), ceil_div(M, 256) * ceil_div(N, 256 * cut.accs) * cut.splits);
    if (cut.accs == 2) launch<pg::STORE, 2>(s, what, a, b, bf16, p, pairs);
    else launch<pg::STORE, 1>(s, what, a, b, bf16, p, pairs);
}
// ... and the sum of its ranges of K, if there are several
void combine(const Stream& s, bool bf16, size_t M, size_t N, const Cut& cut, const Output& o) {
    if (cut.splits == 1) return;
    const unsigned grid = (unsigned)ceil_div(M * N, 4 * THREADS);
    const auto launch = [&](auto kernel, auto* out) {
        s.chain("combine", kernel, grid, THREADS, 0, static_cast<const float*>(o.partial), cut.splits, (uint32_t)M, (uint32_t)N, o.factor, o.accum,
                (uint32_t)o.accum_read, out, o.count_k ? nullptr : o.counted, o.rows);
    };
    const bool twice = o.twice && o.out;
    if (o.f32) launch(combine_kernel<float, false>, static_cast<float*>(o.out));
    else if (bf16) launch(twice ? combine_kernel<__nv_bfloat16, true> : combine_kernel<__nv_bfloat16, false>, static_cast<__nv_bfloat16*>(o.out));
    else launch(twice ? combine_kernel<__half, true> : combine_kernel<__half, false>, static_cast<__half*>(o.out));
}

// ------------------------------------------------------------------------------------------------ operands of the head
// Which rows count: place[row] = the row's place among those that do, or -1 - its place among those that do not; list[place] = row
// and how many there are.  A CTA has 1024 rows and counts those before them by itself (all labels are a few KB that lie in L2; one
// CTA with a run of rows per warp took 18 us for 16 384).  HeadLabels: head_entries.cuh.
__global__ void __launch_bounds__(1024)
head_list_kernel(const HeadLabels l, int32_t* __restrict__ place, int32_t* __restrict__ list, uint32_t* __restrict__ counted) {
    chain_entry();
    __shared__ uint32_t counts[2][32];   // per warp: of the rows before, of its own
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = blockIdx.x * 1024, row = first + threadIdx.x;
    uint32_t n = 0;
#pragma unroll 8
    for (uint32_t r = threadIdx.x; r < first; r += 1024) n += l.target(r) >= 0;
    const bool mine = row < l.rows && l.target(row) >= 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, mine);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) {
        counts[0][warp] = n;
        counts[1][warp] = __popc(mask);
    }
    __syncthreads();
    uint32_t at = counts[0][lane] + (lane < warp ? counts[1][lane] : 0u);   // counted before this warp's rows
    uint32_t all = counts[0][lane] + counts[1][lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        at += __shfl_xor_sync(0xffffffffu, at, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    at += __popc(mask & ((1u << lane) - 1u));
    if (mine) list[at] = (int32_t)row;
    if (row < l.rows) place[row] = mine ? (int32_t)at : -1 - (int32_t)(row - at);
    if (threadIdx.x == 0 && blockIdx.x + 1 == gridDim.x) *counted = all;
}

// The rows of hidden that count, one behind the other, as the operand [., Dp] (columns from D on 0, and rows up to a whole tile: what
// other rows hold, an infinity say, stays out of the products), their targets, their targets' products and logits in f32, zeros (or
// a NaN) for the others' losses and gradients; the weights [vocab, Dp] (+/-1, or a copy of dense rows that no tensor map takes) and
// the largest |scale| per CTA of that part.  A warp has a row of hidden, a thread a chunk of eight weights.
struct HeadOperands {
    const void* hidden;
    size_t stride;
    uint32_t rows, D, Dp, vocab;
    HeadLabels labels;
    const int32_t* place;       // null: each CTA finds its rows' places itself (few rows), and leaves `list` and `counted`
    int32_t* list;
    uint32_t* counted;
    float* row_loss;
    void* g_hidden;             // [rows, D]
    uint32_t g_bytes;           // of a row of it
    uint16_t* h16;
    int32_t* target;
    float *target_acc, *logit2; // the target's product; its logit times log2 e (or what the first softmax takes)
    float log2e;
    const uint32_t* bits;
    const uint16_t *dense, *scale, *bias;
    uint16_t* w16;              // null: the dense weights are taken as they are
    float* scale_max;
    uint32_t hidden_ctas;
    uint32_t bf16;
    uint32_t fold;              // weights +/-scale instead of +/-1 (FP16 has both)
    uint32_t twice;             // 1: every row that counts has two places, one behind the other (few rows; `place` is null)
    uint32_t* status;           // hidden in f32: a finite value beyond FP16 is reported
};
constexpr uint32_t WEIGHT_CTAS = 1024;

__device__ __forceinline__ float from16(uint32_t bits, bool bf16) {
    return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((uint16_t)bits));
}
// signs of eight weights from bit `bit` of `words` words on, the first in the lowest bit
__device__ __forceinline__ uint32_t signs8(const uint32_t* bits, size_t bit, size_t words) {
    const uint32_t shift = (uint32_t)bit & 31u;
    uint32_t v = bits[bit >> 5] >> shift;
    if (shift > 24 && (bit >> 5) + 1 < words) v |= bits[(bit >> 5) + 1] << (32 - shift);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
head_operands_kernel(const HeadOperands o) {
    chain_entry();
    const uint32_t chunks = o.Dp / 8;
    const size_t words = ((size_t)o.vocab * o.D + 31) / 32;
    if (blockIdx.x < o.hidden_ctas) {
        constexpr uint32_t ROWS = THREADS / 32;
        const uint32_t first_row = blockIdx.x * ROWS, warp = threadIdx.x >> 5, row = first_row + warp, lane = threadIdx.x & 31;
        const int32_t target = row < o.rows ? o.labels.target(row) : -1;
        int32_t place = 0;
        uint32_t counted = 0;
        if (o.place) {
            if (row >= o.rows) return;
            place = o.place[row];
            counted = *o.counted;
        } else {
            __shared__ uint32_t before[ROWS], all[ROWS], own[ROWS];
            uint32_t n = 0, total = 0;
#pragma unroll 4
            for (uint32_t r = threadIdx.x; r < o.rows; r += THREADS) {
                const uint32_t counts = o.labels.target(r) >= 0;
                total += counts;
                n += r < first_row ? counts : 0u;
            }
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) {
                n += __shfl_xor_sync(0xffffffffu, n, k);
                total += __shfl_xor_sync(0xffffffffu, total, k);
            }
            if (lane == 0) {
                before[warp] = n;
                all[warp] = total;
                own[warp] = target >= 0;
            }
            __syncthreads();
            uint32_t at = 0;
#pragma unroll
            for (uint32_t w = 0; w < ROWS; ++w) {
                at += before[w] + (w < warp ? own[w] : 0u);
                counted += all[w];
            }
            if (blockIdx.x == 0 && threadIdx.x == 0) *o.counted = counted << o.twice;
            if (row >= o.rows) return;
            place = target >= 0 ? (int32_t)at : -1 - (int32_t)(row - at);
            if (target >= 0 && lane <= o.twice) o.list[(at << o.twice) + lane] = (int32_t)row;
        }
        if (place < 0) {
            if (lane == 0) o.row_loss[row] = target == -1 ? 0.0f : NAN;
            uint8_t* g = static_cast<uint8_t*>(o.g_hidden) + (size_t)row * o.g_bytes;
            if (o.g_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(o.g_hidden) % 16 == 0) {
                for (uint32_t i = lane * 16; i < o.g_bytes; i += 512) *reinterpret_cast<uint4*>(g + i) = make_uint4(0u, 0u, 0u, 0u);
            } else {
                for (uint32_t i = lane * 2; i < o.g_bytes; i += 64) *reinterpret_cast<uint16_t*>(g + i) = 0;
            }
            for (uint32_t t = 0; t <= o.twice; ++t) {
                const uint32_t pad = ((counted + (uint32_t)(-1 - place)) << o.twice) + t;   // a row behind the last, for each such row
                if (pad < ((counted << o.twice) + pg::BM - 1) / pg::BM * pg::BM)
                    for (uint32_t chunk = lane; chunk < chunks; chunk += 32)
                        *reinterpret_cast<uint4*>(o.h16 + (size_t)pad * o.Dp + chunk * 8) = make_uint4(0u, 0u, 0u, 0u);
            }
            return;
        }
        float dot = 0.0f;
        const size_t first = (size_t)target * o.D;   // of the target's weights
        for (uint32_t chunk = lane; chunk < chunks; chunk += 32) {
            const uint32_t c = chunk * 8;
            uint32_t w[4] = {};
            const T* from = static_cast<const T*>(o.hidden) + row * o.stride + c;
            if (sizeof(T) == 2 && c + 8 <= o.D && reinterpret_cast<uintptr_t>(from) % 16 == 0) {
                const uint4 t = *reinterpret_cast<const uint4*>(from);
                w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < o.D) {
                        uint16_t h;
                        if constexpr (sizeof(T) == 4) {
                            const float v = from[e];
                            if (fabsf(v) > 65504.0f && fabsf(v) <= 3.4028234e38f &&
                                atomicCAS(o.status, ULLIS_DEV_OK, ULLIS_DEV_FP16_RANGE) == ULLIS_DEV_OK) o.status[1] = row;
                            h = __half_as_ushort(__float2half_rn(v));
                        } else h = *reinterpret_cast<const uint16_t*>(from + e);
                        w[e >> 1] |= (uint32_t)h << (16 * (e & 1));
                    }
            }
            if (o.bits) {
                const uint32_t signs = signs8(o.bits, first + c, words);
#pragma unroll
                for (int e = 0; e < 8; ++e)   // (0 past the row's end)
                    dot += from16(((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu) ^ ((signs >> e) & 1u ? 0u : 0x8000u), o.bf16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < o.D) dot = fmaf(from16((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu, o.bf16), from16(o.dense[first + c + e], o.bf16), dot);
            }
            for (uint32_t t = 0; t <= o.twice; ++t)
                *reinterpret_cast<uint4*>(o.h16 + (((size_t)place << o.twice) + t) * o.Dp + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        for (int k = 16; k > 0; k >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, k);
        if (lane <= o.twice) o.target[(place << o.twice) + lane] = target;
        if (lane <= o.twice) {
            const uint32_t at = (place << o.twice) + lane;
            if (o.fold) dot *= __half2float(__ushort_as_half(o.scale[target]));
            o.target_acc[at] = dot;
            // rounded as the epilogues round theirs: the difference of two logits is then what it is
            const float scale = o.scale && !o.fold ? __half2float(__ushort_as_half(o.scale[target])) : 1.0f;
            const float bias = o.bias ? __half2float(__ushort_as_half(o.bias[target])) : 0.0f;
            o.logit2[at] = fmaf(dot, scale * o.log2e, bias * o.log2e);
        }
        return;
    }
    const uint32_t cta = blockIdx.x - o.hidden_ctas;
    const uint32_t plus = o.bf16 ? 0x3F80u : 0x3C00u;
    const size_t items = (size_t)o.vocab * chunks;
    float top = 0.0f;
    for (size_t item = (size_t)cta * THREADS + threadIdx.x; item < items; item += (size_t)WEIGHT_CTAS * THREADS) {
        const size_t v = item >> 32 ? item / chunks : (uint32_t)item / chunks;
        const uint32_t c = (uint32_t)(item - v * chunks) * 8;
        uint32_t w[4] = {};
        if (o.bits) {
            const uint32_t signs = signs8(o.bits, v * o.D + c, words);
            const uint32_t one = o.fold ? o.scale[v] : plus;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < o.D) w[e >> 1] |= (one ^ ((signs >> e) & 1u ? 0u : 0x8000u)) << (16 * (e & 1));
            if (c == 0 && !o.fold) top = fmaxf(top, fabsf(__half2float(__ushort_as_half(o.scale[v]))));
        } else {
            const uint16_t* from = o.dense + v * o.D + c;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < o.D) w[e >> 1] |= (uint32_t)from[e] << (16 * (e & 1));
        }
        *reinterpret_cast<uint4*>(o.w16 + v * o.Dp + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (!o.bits || o.fold) return;
    __shared__ float tops[THREADS / 32];
    for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 32; ++w) top = fmaxf(top, tops[w]);
        o.scale_max[cta] = top;
    }
}

// log2 sum exp of every row out of its parts, the row's loss, and (first CTA) the powers of two of g * scale.
struct HeadRows {
    const float2* part;
    size_t part_piece;
    const uint32_t* counted;
    const int32_t* list;
    uint32_t n_tiles, piece_tiles, pairs;
    const float* logit2;
    float *lse2, *target_g, *row_loss;
    const float* scale_max;   // null: no row scales
    float* factors;           // 2^k, 2^-k * loss_scale
    float loss_scale;
};
__global__ void __launch_bounds__(128)
head_rows_kernel(const HeadRows o) {
    chain_entry();
    if (blockIdx.x == 0) {
        __shared__ float tops[4];
        float top = o.scale_max ? 0.0f : 1.0f;
        if (o.scale_max) {
#pragma unroll
            for (uint32_t i = 0; i < WEIGHT_CTAS; i += 128) top = fmaxf(top, o.scale_max[i + threadIdx.x]);
        }
        for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
        __syncthreads();
        if (threadIdx.x == 0) {
            top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            const int exponent = (int)(__float_as_uint(top) >> 23) - 127;
            const int k = top > 0.0f && exponent < 128 ? 14 - exponent : 0;
            o.factors[0] = exp2f((float)k);
            o.factors[1] = exp2f((float)-k) * o.loss_scale;
        }
    }
    // two rows to a warp; a row's sixteen lanes: a quarter of the columns, every fourth slot
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5) * 2 + (threadIdx.x & 1), lane = (threadIdx.x >> 1) & 15, quarter = lane & 3;
    const uint32_t rows = *o.counted, m = row / pg::BM, m_tiles = (rows + pg::BM - 1) / pg::BM, whole_rows = m_tiles * pg::BM;
    if (m >= m_tiles) return;   // (a CTA's rows are all of one tile)
    float top = -INFINITY, sum = 0.0f;
    const auto add = [&](float t, float s) {
        if (t > top) {
            sum = sum * exp2f(top - t) + s;
            top = t;
        } else if (s != 0.0f) {   // (NaN too)
            sum += s * exp2f(t - top);
        }
    };
    for (uint32_t first = 0, piece = 0; first < o.n_tiles; first += o.piece_tiles, ++piece) {
        const uint32_t width = min(o.piece_tiles, o.n_tiles - first);
        const pg::Share share = pg::share_of(m_tiles * width, o.pairs);
        const uint32_t slots = share.owner(m * width + width - 1) - share.owner(m * width) + 1;
        const float2* part = o.part + piece * o.part_piece + row;
        for (uint32_t i = lane >> 2; i < slots; i += 16) {
            float2 t[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) t[u] = i + 4 * u < slots ? part[(size_t)((i + 4 * u) * 4 + quarter) * whole_rows] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int u = 0; u < 4; ++u) add(t[u].x, t[u].y);
        }
    }
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) {   // (within a row's lanes, in a fixed order)
        const float t = __shfl_xor_sync(0xffffffffu, top, 2 * k), s = __shfl_xor_sync(0xffffffffu, sum, 2 * k);
        const float a = top, b = sum;
        const bool mine_first = !(lane & k);
        top = mine_first ? a : t;
        sum = mine_first ? b : s;
        add(mine_first ? t : a, mine_first ? s : b);
    }
    if (lane || row >= rows) return;
    const float logit2 = o.logit2[row];
    // The loss and the target's 1 - p from the sum of the other columns, which a sum with the target in it has lost where a row is sure
    float more, loss, g;   // (more: lse2 over the larger of logit2 and top)
    if (top <= logit2) {
        const float others = sum * exp2f(top - logit2);
        loss = log1pf(others) + (logit2 - logit2);   // (NaN where that is infinite)
        g = -others / (1.0f + others);
        more = loss * pg::LOG2E;
        top = logit2;
    } else {
        const float all = sum + exp2f(logit2 - top);
        more = log2f(all);
        loss = ((top - logit2) + more) * LN2;
        g = -sum / all;
    }
    o.lse2[row] = top + more;
    o.target_g[row] = g;
    o.row_loss[o.list[row]] = loss;
}

// The columns' sums of a piece out of their parts, and of `stretches` that the entries add, times loss_scale.  32 columns to a CTA, a warp
// to each of a slot's eight parts.
__global__ void __launch_bounds__(256)
head_columns_kernel(const float* __restrict__ part, uint32_t pitch, const uint32_t* __restrict__ counted, uint32_t n_tiles, uint32_t pairs,
                    uint32_t columns, float loss_scale, const float* __restrict__ more, size_t more_pitch, uint32_t stretches,
                    float* __restrict__ g_scale, float* __restrict__ g_bias) {
    chain_entry();
    __shared__ float sums[2][8][32];
    const uint32_t lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;   // c < pitch, whole tiles
    const uint32_t m_tiles = (*counted + pg::BM - 1) / pg::BM, n = blockIdx.x * 32 / pg::BN;
    uint32_t slots = 0;
    if (m_tiles) {
        const pg::Share share = pg::share_of(m_tiles * n_tiles, pairs);
        slots = share.owner(n * m_tiles + m_tiles - 1) - share.owner(n * m_tiles) + 1;
    }
    float g = 0.0f, ga = 0.0f;
#pragma unroll 4
    for (uint32_t i = 0; i < slots; ++i) {
        const float* from = part + (size_t)(i * 8 + slice) * 2 * pitch + c;
        g += from[0];
        ga += from[pitch];
    }
    sums[0][slice][lane] = g;
    sums[1][slice][lane] = ga;
    __syncthreads();
    if (slice > 1 || c >= columns) return;
    float all = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) all += sums[slice][k][lane];
    float entries = 0.0f;
#pragma unroll 4
    for (uint32_t i = 0; i < stretches; ++i) entries += more[((size_t)i * 2 + slice) * more_pitch + c];
    float* out = slice ? g_scale : g_bias;
    if (out) out[c] = (all + entries) * loss_scale;
}

// ------------------------------------------------------------------------------------------------ the head's plan
struct HeadPlan {
    size_t Dp, m_tiles, n_tiles;
    uint32_t pairs;
    uint32_t lse_tiles, lse_pieces;              // column tiles of a piece, pieces
    size_t row_part_piece;                       // parts of the rows' sums in a piece
    size_t piece, pieces;                        // columns of a piece of g (a multiple of 256), pieces
    uint32_t col_slots;
    Cut hidden, weight;
    // with entries: K1 to a row that counts, sorted by blocks of 32 rows and groups of 64 columns
    size_t K1, blocks, groups, stretch, stretches;
    size_t state, entry_bits, entry_column, entry_weight, entry_logits, entry_place, offsets, constant, entry_target, second_lse2, row_part2, column_sums;
    size_t h16, w16, counted, place, list, target, target_acc, target_g, lse2, logit, factors, scale_max, row_part, grad, col_part, accum, hidden_partial, weight_partial, bytes;
};
constexpr size_t GRAD_ELEMENTS = (size_t)1 << 28;   // of a piece of g: 512 MiB

// How many pairs at most have a part of `inner` tiles in a row, where outer * inner tiles are shared out (pg::Share): with x = tiles per
// pair they begin at floor(c x), of which inner / x + 1 lie in a run of `inner`, and one begins before it.
size_t most_slots(size_t outer, uint32_t pairs) { return pairs / outer + 2; }

HeadPlan head_plan(const ullis_cuda_runtime* rt, size_t rows, size_t D, size_t V, bool copies_weight, size_t K1 = 0, bool twice = false) {
    HeadPlan p{};
    p.K1 = K1;
    p.pairs = pairs_of(rt);
    p.Dp = up(D, 8);
    p.m_tiles = ceil_div(rows, pg::BM);
    p.n_tiles = ceil_div(V, pg::BN);
    // weights of a piece: up to 32 MiB, a quarter of L2
    p.lse_tiles = (uint32_t)std::min(p.n_tiles, std::max<size_t>(8, ((size_t)32 << 20) / (pg::BN * p.Dp * 2)));
    p.lse_pieces = (uint32_t)ceil_div(p.n_tiles, p.lse_tiles);
    // [slot][4][rows] for any number of row tiles m that turns out to count: most_slots(m) * m <= pairs + 2 m
    p.row_part_piece = (p.pairs + 2 * p.m_tiles) * 4 * pg::BM;
    const size_t most = std::max<size_t>(1, GRAD_ELEMENTS / (p.m_tiles * pg::BM) / pg::BN);   // column tiles of a piece
    p.pieces = ceil_div(p.n_tiles, most);
    const size_t tiles = ceil_div(p.n_tiles, p.pieces);
    p.pieces = ceil_div(p.n_tiles, tiles);
    p.piece = tiles * pg::BN;
    const size_t last = p.n_tiles - (p.pieces - 1) * tiles;
    p.col_slots = (uint32_t)std::min(p.m_tiles, most_slots(last, p.pairs));   // (of one tile at least)
    const size_t width = std::min(p.piece, V);
    p.hidden = cut_of(rows, D, width, p.pairs, true);
    if (twice) p.hidden.splits = std::max(2u, p.hidden.splits);   // (combine_kernel adds the two rows)
    p.weight = cut_of(width, D, rows, p.pairs, true);
    Parts at;
    p.h16 = at.add(rows * p.Dp * 2);
    p.w16 = at.add(copies_weight ? V * p.Dp * 2 : 0);
    p.counted = at.add(4);
    p.place = at.add(rows * 4);
    p.list = at.add(rows * 4);
    p.target = at.add(rows * 4);
    p.target_acc = at.add(rows * 4);
    p.target_g = at.add(rows * 4);
    p.lse2 = at.add(rows * 4);
    p.logit = at.add(rows * 4);
    p.factors = at.add(8);
    p.scale_max = at.add(WEIGHT_CTAS * 4);
    p.row_part = at.add(p.lse_pieces * p.row_part_piece * 8);
    p.grad = at.add(rows * p.piece * 2);
    p.col_part = at.add((size_t)p.col_slots * 16 * p.piece * 4);
    p.accum = at.add(p.pieces > 1 ? rows * D * 4 : 0);
    p.hidden_partial = at.add(partial_bytes(rows, D, p.hidden));
    p.weight_partial = at.add(partial_bytes(width, D, p.weight));
    if (K1) {
        p.blocks = ceil_div(rows, BLOCK_ROWS);
        p.groups = p.n_tiles * (pg::BN / GROUP_COLUMNS);
        // Blocks of rows whose entries' column sums a CTA takes: 32, and at most 64 such parts.
        p.stretch = std::max<size_t>(32, ceil_div(p.blocks, 64));
        p.stretches = ceil_div(p.blocks, p.stretch);
        const size_t entries = p.blocks * BLOCK_ROWS * K1;
        p.state = at.add(rows * 4);
        p.entry_bits = at.add(entries * 4);
        p.entry_column = at.add(entries * 4);
        p.entry_weight = at.add(entries * 4);
        p.entry_logits = at.add(entries * 8);
        p.entry_place = at.add(entries * 2);
        p.offsets = at.add(p.blocks * (2 * p.groups + 1) * 2);
        p.constant = at.add(rows * 4);
        p.entry_target = at.add(rows * 2);
        p.second_lse2 = at.add(rows * 4);
        p.row_part2 = at.add(p.lse_pieces * p.row_part_piece * 4);
        p.column_sums = at.add(p.stretches * 2 * p.n_tiles * pg::BN * 4);
    }
    p.bytes = at.bytes;
    return p;
}

}  // namespace

size_t head_ce_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels, size_t vocab, bool copies_weight) {
    return rows ? head_plan(rt, rows, channels, vocab, copies_weight).bytes : 0;
}

// Dense weights that a tensor map takes are read where they are.
bool head_copies_weight(const void* dense, size_t channels) { return !dense || channels % 8 != 0 || !aligned(dense, 16); }

// A distilled row's gradient is a handful of terms, whose roundings to 16 bits do not average out over few rows.  Up to 128 rows, which
// with two places each are one tile of the products all the same, g * scale goes in as the sum of two 16-bit numbers (pair_gemm.cuh, TWICE):
// its rounding is then far below that of what leaves.  (32 x 256 x 8192, FP16, 16 entries: g_hidden off by 2.1e-4 in norm instead of 3.2e-4;
// 57 us so 60.)  From 129 rows on g * scale is rounded once, as head_ce_grad's: gradients are off by 3.0e-4 in norm in FP16 and 2.4e-3 in
// bf16, of which the rounding of what leaves is 2.1e-4 and 1.7e-3.  Two places would cost 5 % of a call of 192 rows, 12 to 25 % of one of
// 512; in large calls every product has twice the rows.
constexpr size_t RESIDUAL_ROWS = 128;
size_t head_distill_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels, size_t vocab, size_t top, bool labels,
                                   bool copies_weight) {
    return rows ? head_plan(rt, rows << (rows <= RESIDUAL_ROWS), channels, vocab, copies_weight, top + labels, rows <= RESIDUAL_ROWS).bytes : 0;
}

namespace {

template <typename T, typename Key, int E>
void launch_entries_list_of(const Stream& s, const Teacher& t, size_t blocks, const int32_t* target, const int32_t* list, const uint32_t* counted,
                            const EntryLists& lists) {
    const auto kernel = entries_list_kernel<T, Key, E>;
    const size_t smem = E * LIST_THREADS * sizeof(Key) + BLOCK_ROWS * t.K * 4;
    if (smem > 48 * 1024) s.allow_shared(kernel, E * LIST_THREADS * sizeof(Key) + BLOCK_ROWS * DISTILL_MOST * 4);
    s.chain("entries_list", kernel, (unsigned)blocks, LIST_THREADS, smem, t, target, list, counted, lists);
}
template <typename T>
void launch_entries_list(const Stream& s, const Teacher& t, size_t blocks, const int32_t* target, const int32_t* list, const uint32_t* counted,
                         const EntryLists& lists) {
    const uint32_t each = BLOCK_ROWS * t.K;   // keys of a block
    // keys: 8 bits for an entry's number, 11 for its place in a group, the others for the group
    const auto launch = lists.groups1 / 2 >= 1u << 13  ? launch_entries_list_of<T, uint64_t, 16>
                        : each <= LIST_THREADS       ? launch_entries_list_of<T, uint32_t, 1>
                        : each <= 2 * LIST_THREADS ? launch_entries_list_of<T, uint32_t, 2>
                        : each <= 4 * LIST_THREADS ? launch_entries_list_of<T, uint32_t, 4>
                        : each <= 8 * LIST_THREADS ? launch_entries_list_of<T, uint32_t, 8>
                                                   : launch_entries_list_of<T, uint32_t, 16>;
    static_assert(BLOCK_ROWS * DISTILL_MOST <= 16 * LIST_THREADS && DISTILL_MOST <= 256, "");
    launch(s, t, blocks, target, list, counted, lists);
}

// `d`: null, or what the target is spread over.
void head_grad(const Stream& s, const HeadGrad& h, const Distill* d, void* workspace) {
    const bool as_is = !head_copies_weight(h.weight, h.channels);
    const uint32_t twice = d && h.rows <= RESIDUAL_ROWS;
    const HeadPlan p = head_plan(s.rt, h.rows << twice, h.channels, h.vocab, !as_is, d ? d->top + (h.labels != nullptr) : 0, twice);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const bool bf16 = h.dtype == BF16;
    const size_t D = h.channels, V = h.vocab;
    size_t rows = h.rows;   // (later: of the operands)
    const void* w16 = as_is ? h.weight : static_cast<const void*>(ws + p.w16);

    uint32_t* counted = reinterpret_cast<uint32_t*>(ws + p.counted);
    int32_t *place = reinterpret_cast<int32_t*>(ws + p.place), *list = reinterpret_cast<int32_t*>(ws + p.list);
    HeadLabels labels{h.labels, h.ignore_id, (uint32_t)rows, (uint32_t)h.time, (uint32_t)V, nullptr};
    Teacher teacher{};
    EntryLists lists{};
    bool two = false;
    int squarings = 0;
    if (d) {
        teacher.ids = d->ids;
        teacher.logits = d->logits;
        teacher.K = (uint32_t)d->top;
        teacher.K1 = (uint32_t)p.K1;
        teacher.alpha = d->alpha;
        teacher.hard = h.labels ? (float)(1.0 - (double)d->alpha) : 0.0f;
        teacher.temperature = d->alpha > 0.0f ? d->temperature : 1.0f;
        two = teacher.hard > 0.0f && teacher.temperature != 1.0f;
        squarings = !two ? 0 : teacher.temperature == 2.0f ? 1 : teacher.temperature == 4.0f ? 2 : 0;
        teacher.first = two ? 1.0f : 1.0f / teacher.temperature;
        teacher.second = two ? 1.0f / teacher.temperature : 0.0f;
        lists.bits = reinterpret_cast<uint32_t*>(ws + p.entry_bits);
        lists.column = reinterpret_cast<uint32_t*>(ws + p.entry_column);
        lists.weight = reinterpret_cast<float*>(ws + p.entry_weight);
        lists.offsets = reinterpret_cast<uint16_t*>(ws + p.offsets);
        lists.groups1 = 2 * (uint32_t)p.groups + 1;
        lists.place = reinterpret_cast<uint16_t*>(ws + p.entry_place);
        lists.constant = reinterpret_cast<float*>(ws + p.constant);
        lists.target = reinterpret_cast<uint16_t*>(ws + p.entry_target);
        int32_t* state = reinterpret_cast<int32_t*>(ws + p.state);
        const auto kernel = d->dtype == F32 ? entries_state_kernel<float> : d->dtype == F16 ? entries_state_kernel<__half> : entries_state_kernel<__nv_bfloat16>;
        s.chain("entries_state", kernel, (unsigned)ceil_div(rows, 8), 256, 0, labels, teacher, (uint32_t)rows, (uint32_t)V, state);
        labels.ready = state;
    }
    // Few rows find their places where they are gathered, each CTA of eight from all labels.  us of a call in a graph, 256 channels
    // and a vocabulary of 1024, so / with the list by a launch of its own: 32 rows 31.6 / 32.4, 512 35.3 / 36.0, 2048 42.4 / 42.0,
    // 8192 62.0 / 55.0, 16 384 115 / 86.
    const bool listed = rows > 1024;
    if (listed) s.chain("head_list", head_list_kernel, (unsigned)ceil_div(rows, 1024), 1024, 0, labels, place, list, counted);

    HeadOperands o{};
    o.hidden = h.hidden.data;
    o.stride = h.hidden.stride;
    o.rows = (uint32_t)rows;
    o.D = (uint32_t)D;
    o.Dp = (uint32_t)p.Dp;
    o.vocab = (uint32_t)V;
    o.target_acc = reinterpret_cast<float*>(ws + p.target_acc);
    o.logit2 = reinterpret_cast<float*>(ws + p.logit);
    o.log2e = d ? pg::LOG2E * teacher.first : pg::LOG2E;
    o.labels = labels;
    o.place = listed ? place : nullptr;
    o.list = list;
    o.counted = counted;
    o.row_loss = h.row_loss;
    o.g_hidden = h.g_hidden;
    o.g_bytes = (uint32_t)(D * (h.out_f32 ? 4 : 2));
    o.h16 = reinterpret_cast<uint16_t*>(ws + p.h16);
    o.target = reinterpret_cast<int32_t*>(ws + p.target);
    o.bits = h.bits;
    o.dense = static_cast<const uint16_t*>(h.weight);
    o.scale = h.scale;
    o.bias = h.bias;
    o.w16 = as_is ? nullptr : reinterpret_cast<uint16_t*>(ws + p.w16);
    o.scale_max = reinterpret_cast<float*>(ws + p.scale_max);
    o.hidden_ctas = (uint32_t)ceil_div(rows, THREADS / 32);
    o.bf16 = bf16;
    o.fold = h.fold_scale;
    o.twice = twice;
    o.status = s.status;
    const unsigned grid = o.hidden_ctas + (as_is ? 0 : WEIGHT_CTAS);
    if (h.hidden_f32) s.chain("head_operands", head_operands_kernel<float>, grid, THREADS, 0, o);
    else s.chain("head_operands", head_operands_kernel<__half>, grid, THREADS, 0, o);   // (moved, not read: bf16 too)

    rows <<= twice;
    const Operand hidden{o.h16, rows, D, p.Dp, false}, weight{w16, V, D, as_is ? D : p.Dp, false};
    pg::Params q{};
    q.M = (uint32_t)rows;
    q.N = (uint32_t)V;
    q.K = (uint32_t)D;
    q.scale = h.bits && !h.fold_scale ? h.scale : nullptr;
    q.bias = h.bias;
    q.target = o.target;
    q.piece_tiles = p.lse_tiles;
    q.counted = counted;
    q.row_part_piece = p.row_part_piece;
    q.row_part = reinterpret_cast<float2*>(ws + p.row_part);
    q.target_acc = o.target_acc;
    q.target_g = reinterpret_cast<float*>(ws + p.target_g);
    q.lse2 = reinterpret_cast<float*>(ws + p.lse2);
    float* factors = reinterpret_cast<float*>(ws + p.factors);
    if (d) {
        q.offsets = lists.offsets;
        q.groups1 = lists.groups1;
        q.block_entries = (uint32_t)(BLOCK_ROWS * p.K1);
        q.entries = lists.bits;
        q.entry_logits = reinterpret_cast<float2*>(ws + p.entry_logits);
        q.column_factor = squarings ? teacher.second : teacher.first;
        q.second_factor = teacher.second;
        q.row_part2 = reinterpret_cast<float*>(ws + p.row_part2);
        q.second_lse2 = reinterpret_cast<float*>(ws + p.second_lse2);
        const auto list_kernel = d->dtype == F32 ? launch_entries_list<float> : d->dtype == F16 ? launch_entries_list<__half> : launch_entries_list<__nv_bfloat16>;
        list_kernel(s, teacher, p.blocks, o.target, list, counted, lists);
        if (squarings == 1) launch<pg::LSE_ENTRIES_SQUARE, 1>(s, "head_lse", hidden, weight, bf16, q, p.pairs);
        else if (squarings == 2) launch<pg::LSE_ENTRIES_FOURTH, 1>(s, "head_lse", hidden, weight, bf16, q, p.pairs);
        else if (two) launch<pg::LSE_ENTRIES_2, 1>(s, "head_lse", hidden, weight, bf16, q, p.pairs);
        else launch<pg::LSE_ENTRIES, 1>(s, "head_lse", hidden, weight, bf16, q, p.pairs);
    } else {
        launch<pg::LSE, 1>(s, "head_lse", hidden, weight, bf16, q, p.pairs);
    }

    HeadRows r{};
    r.part = q.row_part;
    r.part_piece = p.row_part_piece;
    r.counted = counted;
    r.list = list;
    r.n_tiles = (uint32_t)p.n_tiles;
    r.piece_tiles = p.lse_tiles;
    r.pairs = p.pairs;
    r.logit2 = o.logit2;
    r.lse2 = reinterpret_cast<float*>(ws + p.lse2);
    r.target_g = reinterpret_cast<float*>(ws + p.target_g);
    r.row_loss = h.row_loss;
    r.scale_max = q.scale ? o.scale_max : nullptr;
    r.factors = factors;
    r.loss_scale = h.loss_scale;
    const bool columns = h.g_bias || h.g_scale;
    EntryRows e{};
    if (d) {
        e.teacher = teacher;
        e.lists = lists;
        e.part = r.part;
        e.part2 = q.row_part2;
        e.part_piece = r.part_piece;
        e.counted = counted;
        e.list = list;
        e.n_tiles = r.n_tiles;
        e.piece_tiles = r.piece_tiles;
        e.pairs = r.pairs;
        e.logits = q.entry_logits;
        e.target_acc = o.target_acc;
        e.target_logit = o.logit2;
        e.scale = q.scale;
        e.scale_max = r.scale_max;
        e.n_scale_max = WEIGHT_CTAS;
        e.bf16 = bf16;
        e.residual = twice;
        // |g| is at most both shares: up to 2^7, and far below 1 for a small alpha or temperature, which FP16 would lose bits of
        e.headroom = std::max(-14, (int)std::ceil(std::log2(std::max(1e-30f, teacher.hard + teacher.alpha * teacher.temperature))));
        e.lse2 = r.lse2;
        e.second_lse2 = reinterpret_cast<float*>(ws + p.second_lse2);
        e.row_loss = r.row_loss;
        e.factors = factors;
        e.loss_scale = r.loss_scale;
        e.stretch = (uint32_t)p.stretch;
        e.stretches = (uint32_t)p.stretches;
        e.column_sums = reinterpret_cast<float*>(ws + p.column_sums);
        e.column_pitch = p.n_tiles * pg::BN;
        s.chain("entries_rows", entries_rows_kernel, (unsigned)p.blocks, ROWS_THREADS, 0, e);
        q.entries = lists.column;
    } else {
        s.chain("head_rows", head_rows_kernel, (unsigned)ceil_div(rows, 8), 128, 0, r);
    }

    uint16_t* grad = reinterpret_cast<uint16_t*>(ws + p.grad);
    for (size_t piece = 0; piece < p.pieces; ++piece) {
        const size_t v0 = piece * p.piece, width = std::min(p.piece, V - v0);
        const uint32_t n_tiles = (uint32_t)ceil_div(width, pg::BN);
        pg::Params g = q;
        g.N = (uint32_t)width;
        g.n_first = (uint32_t)v0;
        g.scale = q.scale ? q.scale + v0 : nullptr;
        g.bias = q.bias ? q.bias + v0 : nullptr;
        g.factor = factors;
        g.pitch = (uint32_t)p.piece;
        g.col_part = reinterpret_cast<float*>(ws + p.col_part);
        Operand wp = weight;
        wp.data = static_cast<const uint16_t*>(w16) + v0 * weight.stride;
        wp.rows = width;
        const CUtensorMap grad_map = map_of(grad, rows, p.piece, p.piece, 16, bf16);
        const auto launch_grad = [&](auto form) { launch<decltype(form)::value, 1>(s, "head_grad", hidden, wp, bf16, g, p.pairs, &grad_map); };
        const auto launch_entries = [&](auto more) {
            constexpr int TWICE = decltype(more)::value;
            if (squarings == 1) launch_grad(std::integral_constant<int, pg::GRAD_ENTRIES_SQUARE + TWICE>{});
            else if (squarings == 2) launch_grad(std::integral_constant<int, pg::GRAD_ENTRIES_FOURTH + TWICE>{});
            else if (two) launch_grad(std::integral_constant<int, pg::GRAD_ENTRIES_2 + TWICE>{});
            else launch_grad(std::integral_constant<int, pg::GRAD_ENTRIES + TWICE>{});
        };
        if (!d) launch_grad(std::integral_constant<int, pg::GRAD>{});
        else if (twice) launch_entries(std::integral_constant<int, pg::TWICE>{});
        else launch_entries(std::integral_constant<int, 0>{});
        if (d && columns && piece == 0)
            s.chain("entries_columns", entries_columns_kernel, (unsigned)(p.groups * p.stretches), COLUMNS_THREADS, 0, e);
        // What follows reads g and nothing of one another: few rows leave room for all three at once.
        if (columns)
            s.chain("head_columns", head_columns_kernel, (unsigned)ceil_div(width, 32), 256, 0, static_cast<const float*>(g.col_part), g.pitch,
                    counted, n_tiles, p.pairs, (uint32_t)width, h.loss_scale,
                    d ? reinterpret_cast<const float*>(ws + p.column_sums) + v0 : nullptr, p.n_tiles * pg::BN, (uint32_t)p.stretches,
                    h.g_scale ? h.g_scale + v0 : nullptr, h.g_bias ? h.g_bias + v0 : nullptr);
        const Operand by_columns{grad, rows, width, p.piece, true};
        Operand hc = hidden;
        hc.mn = true;
        Output w{};
        w.out = static_cast<uint8_t*>(h.g_weight) + v0 * D * (h.out_f32 ? 4 : 2);
        w.f32 = h.out_f32;
        w.factor = factors + 1;
        w.partial = reinterpret_cast<float*>(ws + p.weight_partial);
        w.counted = counted;
        w.count_k = true;
        w.beside = columns;
        product(s, "head_g_weight", by_columns, hc, bf16, width, D, rows, p.weight, w);
        // g_hidden: over the pieces in f32
        const Operand by_rows{grad, rows, width, p.piece, false};
        wp.mn = true;
        Output x{};
        x.out = piece + 1 == p.pieces ? h.g_hidden : nullptr;
        x.f32 = h.out_f32;
        x.accum = p.pieces > 1 ? reinterpret_cast<float*>(ws + p.accum) : nullptr;
        x.accum_read = piece > 0;
        x.factor = factors + 1;
        x.partial = reinterpret_cast<float*>(ws + p.hidden_partial);
        x.counted = counted;
        x.rows = list;
        x.beside = true;
        x.twice = twice;
        product(s, "head_g_hidden", by_rows, wp, bf16, rows, D, width, p.hidden, x);
        combine(s, bf16, width, D, p.weight, w);
        combine(s, bf16, rows, D, p.hidden, x);
    }
}

}  // namespace

void head_ce_grad(const Stream& s, const HeadGrad& h, void* workspace) { head_grad(s, h, nullptr, workspace); }
void head_distill_grad(const Stream& s, const HeadGrad& h, const Distill& d, void* workspace) { head_grad(s, h, &d, workspace); }

// ------------------------------------------------------------------------------------------------ a wait that runs out
namespace {
__global__ void wait_selftest_kernel(uint32_t polls, uint32_t* status) {
    __shared__ __align__(8) uint64_t bar;
    if (threadIdx.x == 0) {
        ptx::mbar_init(&bar, 1);
        ptx::fence_mbar_init();
    }
    __syncthreads();
    if (threadIdx.x == 0 && !ptx::mbar_wait(&bar, 0, polls)) pg::report_wait(status, 99u);   // site: self-test
}
}  // namespace

void wait_selftest(const Stream& s, uint32_t polls) {
    wait_selftest_kernel<<<1, 32, 0, s.stream>>>(polls, s.status);
    s.launched("wait_selftest");
}

// ------------------------------------------------------------------------------------------------ weight gradient from the tape
namespace {

// What the codes stand for as a 16-bit operand [rows, Cp].  A thread has a chunk of eight columns and OPERAND_ROWS rows.  VEC: as in
// tape.cuh.
constexpr int OPERAND_ROWS = 8;
template <bool VEC>
struct OperandRows {
    uint32_t codes[OPERAND_ROWS][2], bytes[OPERAND_ROWS];
    __device__ __forceinline__ void load(const uint8_t* __restrict__ from, const uint8_t* __restrict__ exponents, size_t row0, uint32_t rows,
                                         uint32_t c, uint32_t C) {
        const uint32_t blocks = (C + 31) / 32, b = c / 32;
#pragma unroll
        for (int k = 0; k < OPERAND_ROWS; ++k) {
            const size_t row = min(row0 + k, (size_t)rows - 1);   // (no branch between the loads)
            bytes[k] = exponents[row * blocks + b];
            tape::raw_codes<VEC, 8>(from + row * C, c, C, codes[k]);
        }
    }
};
template <bool BF>
__device__ __forceinline__ void store_operand(uint16_t* to, const uint32_t (&codes)[2], uint32_t byte) {
    float v[8];
    tape::values_of(codes, tape::power(byte), v);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pg::pack16<BF>(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

// bf16 holds every value: 8 significant bits, the range of f32.  16384 x 512: 5.8 us (25 MB).
template <bool VEC>
__global__ void __launch_bounds__(THREADS)
tape_operand_bf16_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, uint32_t rows, uint32_t C, uint32_t Cp,
                         uint16_t* __restrict__ out) {
    chain_entry();
    const uint32_t chunks = Cp / 8;
    const size_t item = (size_t)blockIdx.x * THREADS + threadIdx.x;
    const size_t group = item >> 32 ? item / chunks : (uint32_t)item / chunks, row0 = group * OPERAND_ROWS;
    if (row0 >= rows) return;
    const uint32_t c = (uint32_t)(item - group * chunks) * 8;
    OperandRows<VEC> o;
    o.load(codes, exponents, row0, rows, c, C);
#pragma unroll
    for (int k = 0; k < OPERAND_ROWS; ++k)
        if (row0 + k < rows) store_operand<true>(out + (row0 + k) * Cp + c, o.codes[k], o.bytes[k]);
}

// FP16 does not: there the codes of 32 channels and a stretch of 512 rows, whose sums SUM adds up with rounding anyway, are shifted by a
// power of two in common, so that their largest exponent comes to 8 (127 * 2^8 = 32 512), and the sums are shifted back.  FP16's last
// bit, 2^-24, is then that of a code whose exponent lies 32 below the largest.  Where a smaller one turns up (a row of very large values is
// enough, a padded one whose gy is 0 too), the 256 columns that a product's tile has of the stretch go to bf16 after all, and gy's rows
// into the sum of two bf16 matrices, which 11 bits always are: the same products, exact again, with twice the operations.
// A CTA has 64 rows of 256 columns and looks at the exponents of the whole stretch (4 KB, in L2).  BYTES8: a row's eight start on 8 bytes.
// 7655 x 2048: 12.2 us (47 MB); the largest exponents of all rows by a kernel before it took 6.5 and 9.4, and held 32 binades.
constexpr uint32_t STRETCH = pg::SUM_BLOCKS * pg::BK, F16_ROWS = THREADS / 32 * OPERAND_ROWS;
static_assert(STRETCH % F16_ROWS == 0 && STRETCH / 32 <= 32 && THREADS == 8 * 32 && pg::BN == 256, "");

struct GyRows {   // gy [rows, O] as two bf16 matrices side by side, [rows, 2 Op]
    const uint16_t* gy;
    size_t stride;
    uint32_t O, Op;
    uint16_t* out;
    // the nearest bf16 number, and what is left (at most 3 bits; 0 where that is not finite)
    __device__ __noinline__ void in_parts(size_t first, size_t last) const {
        const uint32_t chunks = Op / 8;
        const size_t items = (last - first) * chunks;
        for (size_t i = threadIdx.x; i < items; i += THREADS) {
            const size_t row = first + i / chunks;
            const uint32_t c = (uint32_t)(i % chunks) * 8;
            uint32_t w[2][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float high[2], low[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float v = c + 2 * e + k < O ? __half2float(__ushort_as_half(gy[row * stride + c + 2 * e + k])) : 0.0f;
                    high[k] = __bfloat162float(__float2bfloat16_rn(v));
                    low[k] = isfinite(v) ? v - high[k] : 0.0f;
                }
                w[0][e] = pg::pack16<true>(high[0], high[1]);
                w[1][e] = pg::pack16<true>(low[0], low[1]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
                *reinterpret_cast<uint4*>(out + (row * 2 + k) * Op + c) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
        }
    }
};
template <bool VEC, bool BYTES8>
__global__ void __launch_bounds__(THREADS)
tape_operand_f16_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, uint32_t rows, uint32_t C, uint32_t Cp,
                        uint16_t* __restrict__ out, float* __restrict__ col_factor, uint8_t* __restrict__ parts, uint32_t parts_pitch,
                        const GyRows gy) {
    chain_entry();
    const uint32_t tiles = (C + pg::BN - 1) / pg::BN, blocks = (C + 31) / 32;
    const uint32_t tile = blockIdx.x % tiles, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b0 = tile * 8;
    const size_t first = (size_t)(blockIdx.x / tiles) * F16_ROWS, row0 = first + warp * OPERAND_ROWS;
    const size_t stretch = first / STRETCH, end = min((stretch + 1) * STRETCH, (size_t)rows);
    const uint32_t c = tile * pg::BN + lane * 8;
    const bool mine = row0 < rows && c < Cp;
    OperandRows<VEC> o;
    if (mine) o.load(codes, exponents, row0, rows, c, C);
    // A warp for each of the tile's eight blocks: the largest exponent byte of the stretch, and the smallest of those whose codes are not
    // all 0 (255: none).  A block of zeros has the lowest byte there is, 1: only where that turns up are codes read.
    __shared__ __align__(8) uint8_t bytes[STRETCH][8];   // 0: no row or no block there
    __shared__ uint32_t range[2][8];
#pragma unroll
    for (uint32_t r = threadIdx.x; r < STRETCH; r += THREADS) {
        const size_t row = stretch * STRETCH + r;
        const uint8_t* at = exponents + row * blocks + b0;
        uint2 e = make_uint2(0u, 0u);
        if (BYTES8) {
            if (row < end) e = *reinterpret_cast<const uint2*>(at);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (row < end && b0 + k < blocks) (k < 4 ? e.x : e.y) |= (uint32_t)at[k] << 8 * (k & 3);
        }
        *reinterpret_cast<uint2*>(bytes[r]) = e;
    }
    __syncthreads();
    uint32_t largest = 0, smallest = 255, ones = 0;
#pragma unroll
    for (uint32_t i = 0; i < STRETCH / 32; ++i) {
        const uint32_t e = bytes[i * 32 + lane][warp];
        largest = max(largest, e);
        smallest = min(smallest, e > 1 ? e : 255u);
        ones |= (uint32_t)(e == 1) << i;
    }
    while (ones) {
        const size_t row = stretch * STRETCH + (__ffs(ones) - 1) * 32 + lane;
        ones &= ones - 1;
        uint32_t any = 0;
        for (uint32_t i = 0; i < 4; ++i) {
            uint32_t w[2];
            tape::raw_codes<VEC, 8>(codes + row * C, (b0 + warp) * 32 + i * 8, C, w);
            any |= w[0] | w[1];
        }
        if (any) smallest = 1;
    }
    largest = __reduce_max_sync(0xffffffffu, largest);
    smallest = __reduce_min_sync(0xffffffffu, smallest);
    if (lane == 0) {
        range[0][warp] = largest;
        range[1][warp] = smallest;
    }
    __syncthreads();
    largest = range[0][lane & 7];   // of block b0 + lane % 8
    smallest = range[1][lane & 7];
    const bool exact = __any_sync(0xffffffffu, largest != tape::NOT_FINITE && smallest + 32 < largest);   // (the same for all warps)
    if (first % STRETCH == 0 && threadIdx.x < 8) {
        if (b0 + lane < blocks)
            col_factor[stretch * blocks + b0 + lane] = exact || largest == tape::NOT_FINITE ? 1.0f : exp2f((float)((int)largest - 127 - 8));
        if (lane == 0) parts[(size_t)tile * parts_pitch + stretch] = exact;
    }
    if (exact) gy.in_parts(first, min(first + F16_ROWS, (size_t)rows));
    const uint32_t own = __shfl_sync(0xffffffffu, largest, lane >> 2);   // the largest of this thread's block
    if (!mine) return;
#pragma unroll
    for (int k = 0; k < OPERAND_ROWS; ++k) {
        if (row0 + k >= rows) break;
        uint16_t* to = out + (row0 + k) * Cp + c;
        uint32_t byte = o.bytes[k];
        if (exact) {
            store_operand<true>(to, o.codes[k], byte);
        } else {
            if (byte != tape::NOT_FINITE)   // 2^(e - largest + 8)
                byte = own == tape::NOT_FINITE ? 127u : (uint32_t)max((int)byte - (int)own + 8 + 127, 1);
            store_operand<false>(to, o.codes[k], byte);
        }
    }
}

// 16-bit rows that no tensor map takes, with a stride of whole 16 bytes
__global__ void __launch_bounds__(THREADS)
rows16_kernel(const uint16_t* __restrict__ x, size_t stride, uint32_t rows, uint32_t C, uint32_t Cp, uint16_t* __restrict__ out) {
    chain_entry();
    const uint32_t chunks = Cp / 8;
    const size_t item = (size_t)blockIdx.x * THREADS + threadIdx.x;
    const size_t row = item >> 32 ? item / chunks : (uint32_t)item / chunks;
    if (row >= rows) return;
    const uint32_t c = (uint32_t)(item - row * chunks) * 8;
    uint32_t w[4] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (c + e < C) w[e >> 1] |= (uint32_t)x[row * stride + c + e] << (16 * (e & 1));
    *reinterpret_cast<uint4*>(out + row * Cp + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct WeightPlan {
    size_t ip, op;
    Cut cut;
    size_t x16, gy16, gy_parts, col_factor, parts_pitch, parts, partial, bytes;
};
WeightPlan weight_plan(const ullis_cuda_runtime* rt, size_t rows, size_t in, size_t out) {
    WeightPlan p{};
    p.ip = up(in, 8);
    p.op = up(out, 8);
    p.cut = cut_of(out, in, rows, pairs_of(rt), false);
    Parts at;
    p.x16 = at.add(rows * p.ip * 2);
    p.gy16 = at.add(rows * p.op * 2);
    p.gy_parts = at.add(rows * 2 * p.op * 2);
    p.col_factor = at.add(ceil_div(rows, STRETCH) * tape::blocks_of(in) * 4);
    p.parts_pitch = up(ceil_div(rows, STRETCH), 8);
    p.parts = at.add(p.parts_pitch * ceil_div(in, pg::BN));
    p.partial = at.add(partial_bytes(out, in, p.cut));
    p.bytes = at.bytes;
    return p;
}

}  // namespace

size_t tape_weight_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t in_features, size_t out_features) {
    return rows ? weight_plan(rt, rows, in_features, out_features).bytes : 0;
}

void tape_weight_grad(const Stream& s, int dtype, const uint8_t* codes, const uint8_t* exponents, Rows gy, size_t rows, size_t in,
                      size_t out, float* g, void* workspace) {
    const WeightPlan p = weight_plan(s.rt, rows, in, out);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const bool bf16 = dtype == BF16;
    uint16_t* x16 = reinterpret_cast<uint16_t*>(ws + p.x16);
    uint16_t* gy16 = reinterpret_cast<uint16_t*>(ws + p.gy16);
    float* col_factor = reinterpret_cast<float*>(ws + p.col_factor);
    uint8_t* parts = ws + p.parts;
    Operand a{gy.data, rows, out, gy.stride, true};
    uint16_t* gy_parts = reinterpret_cast<uint16_t*>(ws + p.gy_parts);
    if (!aligned(gy.data, 16) || gy.stride % 8) {
        s.chain("rows16", rows16_kernel, (unsigned)ceil_div(rows * (p.op / 8), THREADS), THREADS, 0, static_cast<const uint16_t*>(gy.data),
                gy.stride, (uint32_t)rows, (uint32_t)out, (uint32_t)p.op, gy16);
        a = Operand{gy16, rows, out, p.op, true};
    }
    const bool vec = in % 8 == 0 && aligned(codes, 8);
    if (bf16) {
        s.chain("tape_operand", vec ? tape_operand_bf16_kernel<true> : tape_operand_bf16_kernel<false>,
                (unsigned)ceil_div(ceil_div(rows, OPERAND_ROWS) * (p.ip / 8), THREADS), THREADS, 0, codes, exponents, (uint32_t)rows, (uint32_t)in,
                (uint32_t)p.ip, x16);
    } else {
        const bool bytes8 = tape::blocks_of(in) % 8 == 0 && aligned(exponents, 8);
        const auto operand = vec ? (bytes8 ? tape_operand_f16_kernel<true, true> : tape_operand_f16_kernel<true, false>)
                                 : (bytes8 ? tape_operand_f16_kernel<false, true> : tape_operand_f16_kernel<false, false>);
        s.chain("tape_operand", operand, (unsigned)(ceil_div(rows, F16_ROWS) * ceil_div(in, pg::BN)), THREADS, 0, codes, exponents, (uint32_t)rows,
                (uint32_t)in, (uint32_t)p.ip, x16, col_factor, parts, (uint32_t)p.parts_pitch,
                GyRows{static_cast<const uint16_t*>(gy.data), gy.stride, (uint32_t)out, (uint32_t)p.op, gy_parts});
    }
    const Operand b{x16, rows, in, p.ip, true};
    pg::Params q{};
    q.M = (uint32_t)out;
    q.N = (uint32_t)in;
    q.K = (uint32_t)rows;
    q.splits = p.cut.splits;
    q.out = g;
    q.partial = reinterpret_cast<float*>(ws + p.partial);
    if (!bf16) {
        q.col_factor = col_factor;
        q.parts = parts;
        q.parts_pitch = (uint32_t)p.parts_pitch;
        q.parts_at = (uint32_t)p.op;
    }
    const CUtensorMap in_parts = operand_map(Operand{gy_parts, rows, 2 * p.op, 2 * p.op, true}, true);
    const uint32_t pairs = (uint32_t)std::min<size_t>(pairs_of(s.rt), ceil_div(out, 256) * ceil_div(in, 256) * p.cut.splits);
    launch<pg::SUM, 1>(s, "tape_weight_grad", a, b, bf16, q, pairs, &in_parts);
    if (p.cut.splits > 1)
        s.chain("combine", combine_kernel<float, false>, (unsigned)ceil_div(out * in, 4 * THREADS), THREADS, 0, static_cast<const float*>(q.partial), p.cut.splits,
                (uint32_t)out, (uint32_t)in, nullptr, nullptr, 0u, g, nullptr, nullptr);
}

}  // namespace dev
}  // namespace ullis
