// Which rows of a head's batch count, and, for distillation, the teacher's entries: their probabilities, their order for the epilogues of
// pair_gemm.cuh, and what comes of them between the two products.
//
// Of a row that counts, with z the student's logits, T the temperature, p = softmax(t / T) over its entries (a negative id is none,
// t = -infinity has p = 0), y its label and alpha the teacher's share,
//   loss = (1 - alpha) * (lse(z) - z[y]) + alpha * T^2 * sum p * (log p - z / T + lse(z / T)),
//   g = (1 - alpha) * softmax(z) + alpha * T * softmax(z / T) - w,  w = alpha * T * p at the entries, 1 - alpha more at y:
// a label is one more entry, and an id that comes twice in a row is one entry with both weights.  With top the largest logit,
//   loss = (1 - alpha) * (lse(z) - top) + alpha * T^2 * (lse(z / T) - top / T) + sum w * (top - z) + alpha * T^2 * sum p * log p,
// none of whose terms but the last is negative.  Without labels the first parts are left out; where only one of the softmaxes has a
// share, or T = 1, one is computed, and z and top below are those at its temperature.
//
// A label that is an entry already adds its weight there (so every id of a row has one live entry), else it is one more.
//
// The rows that count are taken 32 at a time, and their entries sorted by groups of 64 columns and within them by entry_bits: what an
// epilogue warp has of a tile then lies in a row, and entries of one column beside one another.  Sums go by that order: a call gives the
// same result every time.  What this costs, us with 64 entries in each of 16384 rows: states 7, lists 39, entries_rows 22 and
// entries_columns 24 warm and one after the other, 80 of a call, where entries_columns begins behind GRAD; and 15 more in GRAD, whose
// pairs with the first columns have hundreds of entries to a tile (a teacher's favourites).  All four kernels are bound by instructions
// (40 to 70 % of the slots) and the latency between them.
#pragma once
#include "block_sort.cuh"
#include "pair_gemm.cuh"
#include "tape.cuh"

namespace ullis {
namespace dev {
namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr uint32_t BLOCK_ROWS = 32, GROUP_COLUMNS = 64;
constexpr uint32_t NO_PLACE = 0xFFFFu;   // of an entry that is none, among those of its block

struct HeadLabels {
    const uint32_t* labels;
    uint32_t ignore_id, rows, time, vocab;
    const int32_t* ready;   // the answers (distillation: entries_state_kernel), or null
    // the target of a row, -1 where it does not count (the last of its sequence, an ignored label), -2 for a label outside the vocabulary
    __device__ int32_t target(uint32_t row) const {
        if (ready) return ready[min(row, rows - 1u)];
        const uint32_t label = labels[min(row + 1u, rows - 1u)];   // (always read, so that several are on their way)
        if (row % time + 1u >= time || label == ignore_id) return -1;
        return label < vocab ? (int32_t)label : -2;
    }
};

struct Teacher {
    const int32_t* ids;       // [rows, K]
    const void* logits;       // [rows, K]
    uint32_t K, K1;           // K1: with the label's entry
    float alpha, hard;        // the teacher's share and, with labels, 1 - alpha (else 0)
    float temperature;
    // what is computed: 1 / the temperature of the first softmax, and of the second over the first's (0: none)
    float first, second;
};

// The state of every row: HeadLabels::target's numbers; without labels its target is the entry that the teacher holds for the likeliest.  The
// target is the column whose logit is computed with rounding beside the products: its terms have one sign where a student has learnt
// anything, and what the tensor cores cut off would stay in the loss and the sums over the columns.  A warp has a row.
template <typename T>
__global__ void __launch_bounds__(256)
entries_state_kernel(const HeadLabels labels, const Teacher t, uint32_t rows, uint32_t vocab, int32_t* __restrict__ state) {
    chain_entry();
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= rows) return;
    bool bad = false;
    uint32_t best = 0, best_id = 0;   // of what lies above -infinity: a number that rises with the logit
    const size_t at = (size_t)row * t.K;
#pragma unroll 4
    for (uint32_t k = lane; k < t.K; k += 32) {
        const int32_t id = t.ids[at + k];
        const float v = tape::to_float(static_cast<const T*>(t.logits)[at + k]);
        if (id < 0) continue;
        bad |= (uint32_t)id >= vocab || !(v < INFINITY);
        const uint32_t raw = __float_as_uint(v), order = v > -INFINITY ? raw ^ ((uint32_t)((int32_t)raw >> 31) | 0x80000000u) : 0u;
        if (order > best) {
            best = order;
            best_id = (uint32_t)id;
        }
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    best_id = __reduce_min_sync(0xffffffffu, best == top ? best_id : 0xFFFFFFFFu);
    bad = __any_sync(0xffffffffu, bad);
    if (lane) return;
    int32_t s = labels.labels ? labels.target(row) : top ? (int32_t)best_id : -1;
    if (bad && (s >= 0 || !labels.labels)) s = -2;
    state[row] = s;
}

struct EntryLists {
    // by block of 32 rows that count: 32 * K1 places, and groups1 = 2 groups + 1 offsets among them, for each group that of its first
    // sixteen rows and of the others
    uint32_t* bits;            // entry_bits (and ENTRY_DEAD, ENTRY_TARGET)
    uint32_t* column;          // of the vocabulary; later what GRAD takes: bits and above them the 16-bit g * scale * 2^k
    float* weight;             // w, of a dead one 0
    uint16_t* offsets;
    uint32_t groups1;
    // by row that counts
    uint16_t* place;           // [row][K1], in the block's list, of those that have a weight there
    float* constant;           // alpha * T^2 * sum p * log p; without entries NAN, which marks that
    uint16_t* target;          // the place of the target's entry
};
constexpr uint32_t LIST_THREADS = 512;

// How many of a rising list are below `limit`.
template <typename Key>
__device__ __forceinline__ uint32_t keys_below(const Key* list, uint32_t n, Key limit) {
    uint32_t at = 0;
    while (n > 0) {
        const uint32_t half = n >> 1;
        const bool right = list[at + half] < limit;
        at += right ? half + 1 : 0u;
        n = right ? n - half - 1 : half;
    }
    return at;
}

// A CTA has a block of rows.  Of its time a third goes to the sort, a fifth each to the probabilities and the places.  The teacher's entries are
// sorted by spot (group of columns and entry_bits) and the entry's number in its row
// below it, in 32 bits up to 524 032 columns; the labels that are no entries, at most a warp's width, are merged into them.  E: keys to
// a thread, 32 K <= 512 E.
template <typename T, typename Key, int E>
__global__ void __launch_bounds__(LIST_THREADS)
entries_list_kernel(const Teacher t, const int32_t* __restrict__ target, const int32_t* __restrict__ list, const uint32_t* __restrict__ counted,
                    const EntryLists o) {
    chain_entry();
    constexpr uint32_t N = E * LIST_THREADS, WARPS = LIST_THREADS / 32, NUMBER_BITS = 8, NO_SPOT = 0xFFFFFFFFu;
    constexpr Key NO_KEY = ~(Key)0;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ uint32_t row_target[BLOCK_ROWS], row_label[BLOCK_ROWS], more[BLOCK_ROWS];   // spots; more: of labels that are no entries, rising
    const uint32_t first = blockIdx.x * BLOCK_ROWS, rows = *counted, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (first >= rows) return;
    const uint32_t n_rows = min(BLOCK_ROWS, rows - first), n = n_rows * t.K;
    const bool labels = t.K1 > t.K;
    Key* sorted = reinterpret_cast<Key*>(smem_raw);                  // [N]
    float* weight = reinterpret_cast<float*>(sorted + N);            // [row][K]
    const auto spot_of = [](uint32_t row, uint32_t column) { return column / GROUP_COLUMNS * pg::ENTRY_PLACES | pg::entry_bits(row, column); };
    const float times = 1.0f / t.temperature, share = t.alpha * t.temperature;
    for (uint32_t r = warp; r < n_rows; r += WARPS) {
        const size_t at = (size_t)list[first + r] * t.K;
        const T* logits = static_cast<const T*>(t.logits) + at;
        uint16_t* place = o.place + (size_t)(first + r) * t.K1;
        float top = -INFINITY;
#pragma unroll 2
        for (uint32_t k = lane; k < t.K; k += 32) {
            const float v = tape::to_float(logits[k]);
            top = fmaxf(top, t.ids[at + k] < 0 ? -INFINITY : v);
        }
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const bool has = top != -INFINITY;
        float sum = 0.0f, sum_x = 0.0f;
#pragma unroll 2
        for (uint32_t k = lane; k < t.K; k += 32) {
            const int32_t id = t.ids[at + k];
            const bool is = has && id >= 0;
            const float x = (tape::to_float(logits[k]) - top) * times, e = is ? expf(x) : 0.0f;
            sum += e;
            if (e > 0.0f) sum_x += e * x;
            sorted[r * t.K + k] = is ? (Key)spot_of(r, (uint32_t)id) << NUMBER_BITS | k : NO_KEY;
            if (!is) place[k] = (uint16_t)NO_PLACE;
            weight[r * t.K + k] = e;
        }
        for (int d = 16; d > 0; d >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, d);
            sum_x += __shfl_xor_sync(0xffffffffu, sum_x, d);
        }
        const float each = share / sum;
        if (has)
            for (uint32_t k = lane; k < t.K; k += 32) weight[r * t.K + k] *= each;
        if (lane == 0) {
            // sum of p * log p, with log p = x - log sum
            o.constant[first + r] = has ? share * t.temperature * (sum_x / sum - logf(sum)) : NAN;
            row_target[r] = spot_of(r, (uint32_t)target[first + r]);
            row_label[r] = labels ? row_target[r] : NO_SPOT;
        }
    }
    __syncthreads();
    Key v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = threadIdx.x * E + i < n ? sorted[threadIdx.x * E + i] : NO_KEY;
    __syncthreads();
    block_sort<Key, E, LIST_THREADS>(v, sorted, threadIdx.x);
#pragma unroll
    for (int i = 0; i < E; ++i) sorted[threadIdx.x * E + i] = v[i];
    __syncthreads();
    const uint32_t valid = keys_below(sorted, N, NO_KEY);
    const auto find = [&](uint32_t spot) { return keys_below(sorted, valid, (Key)spot << NUMBER_BITS); };
    const auto is_at = [&](uint32_t i, uint32_t spot) { return i < valid && (uint32_t)(sorted[i] >> NUMBER_BITS) == spot; };
    if (warp == 0) {
        uint32_t spot = labels && lane < n_rows ? row_label[lane] : NO_SPOT;
        if (spot != NO_SPOT && is_at(find(spot), spot)) spot = NO_SPOT;
#pragma unroll
        for (uint32_t run = 2; run <= 32; run <<= 1)
#pragma unroll
            for (uint32_t step = run >> 1; step > 0; step >>= 1) {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, spot, step);
                spot = ((lane & step) == 0) == ((lane & run) == 0) ? min(spot, other) : max(spot, other);
            }
        more[lane] = spot;
    }
    __syncthreads();
    const size_t base = (size_t)blockIdx.x * BLOCK_ROWS * t.K1;
    const auto labels_below = [&](uint32_t spot) { return labels ? keys_below(more, BLOCK_ROWS, spot) : 0u; };
    const auto leave = [&](uint32_t place, uint32_t spot, bool dead, float w) {
        const uint32_t r = pg::entry_row(spot);
        const bool is_target = !dead && row_target[r] == spot;
        o.bits[base + place] = (spot & (pg::ENTRY_PLACES - 1)) | (dead ? pg::ENTRY_DEAD : 0u) | (is_target ? pg::ENTRY_TARGET : 0u);
        if (is_target) o.target[first + r] = (uint16_t)place;
        o.column[base + place] = spot / pg::ENTRY_PLACES * GROUP_COLUMNS + pg::entry_column(spot);
        o.weight[base + place] = w;
    };
    for (uint32_t i = threadIdx.x; i < valid; i += LIST_THREADS) {
        const Key key = sorted[i];
        const uint32_t spot = (uint32_t)(key >> NUMBER_BITS), r = pg::entry_row(spot), k = (uint32_t)key & ((1u << NUMBER_BITS) - 1);
        const uint32_t place = i + labels_below(spot);
        const bool dead = i > 0 && is_at(i - 1, spot);   // the first of its spot has the sum
        float w = 0.0f;
        if (!dead) {
            w = weight[r * t.K + k];
            for (uint32_t j = i + 1; is_at(j, spot); ++j) w += weight[r * t.K + ((uint32_t)sorted[j] & ((1u << NUMBER_BITS) - 1))];
            if (row_label[r] == spot) w += t.hard;
        }
        leave(place, spot, dead, w);
        o.place[(size_t)(first + r) * t.K1 + k] = (uint16_t)(dead ? NO_PLACE : place);
    }
    if (labels && threadIdx.x < n_rows) {
        const uint32_t spot = row_label[threadIdx.x], at = find(spot), place = at + labels_below(spot);
        const bool entry = is_at(at, spot);
        o.place[(size_t)(first + threadIdx.x) * t.K1 + t.K] = (uint16_t)(entry ? NO_PLACE : place);
        if (!entry) leave(place, spot, false, t.hard);
    }
    for (uint32_t g = threadIdx.x; g < o.groups1; g += LIST_THREADS) {
        const uint32_t spot = g * (pg::ENTRY_PLACES / 2);
        o.offsets[(size_t)blockIdx.x * o.groups1 + g] = (uint16_t)(find(spot) + labels_below(spot));
    }
}

// Between the products.  A CTA has a block of 32 rows: log2 sum exp of its rows out of their parts (sixteen lanes to a row) and their
// targets' logits, less the logarithm of the softmax's share so that GRAD's exp has it as a factor; the losses; and of every entry the
// 16-bit g * scale * 2^k that GRAD puts in its place, and what it adds to GRAD's sums over its column: -w and -w * product, and at the
// target g less the probability that GRAD has there, and the same of the product.  Where a student is sure of its target, its g is the
// small difference of what it and the teacher leave to other columns, which a sum with a probability of 1 in it would lose: from 63 / 64 of
// the softmaxes' share on GRAD leaves it out of its sums (32 rows and a group of columns at a time), and the entry adds its whole g.
// (16384 x 512 x 8192, 64 entries: GRAD at two temperatures 152 us, with half of the rows sure 163, at one 146 and 150; without any of this
// 151 and 140.  With every target left out it took 17 to 33 % more, in five forms.)
struct EntryRows {
    Teacher teacher;
    EntryLists lists;
    const float2* part;
    const float* part2;
    size_t part_piece;
    const uint32_t* counted;
    const int32_t* list;
    uint32_t n_tiles, piece_tiles, pairs;
    float2* logits;            // of entries: product, logit; after it what the entry adds to GRAD's sums over its column
    const float *target_acc, *target_logit;   // by row: the same of its target, with rounding
    const uint16_t* scale;     // or null
    const float* scale_max;    // null: no row scales
    uint32_t n_scale_max;
    uint32_t bf16, residual;   // residual: of two places that follow on one another the second has what rounding takes from the first's g
    int headroom;              // 2^headroom: bound of the softmaxes' shares
    float *lse2, *second_lse2, *row_loss, *factors;
    float loss_scale;
    // entries_columns
    uint32_t stretch, stretches;   // blocks of a CTA
    float* column_sums;        // [stretches][2][groups of 64]
    size_t column_pitch;
};
constexpr uint32_t ROWS_THREADS = 512, ROWS_WARPS = ROWS_THREADS / 32;
constexpr uint32_t COLUMNS_THREADS = 256, COLUMNS_WARPS = COLUMNS_THREADS / 32, WORDS = 4;

// Sums of exp over a row's columns: the parts that one of sixteen lanes has, then the target's.
struct RowSums {
    float top = -INFINITY, sum = 0.0f, sum2 = 0.0f;
    __device__ void add(const EntryRows& o, float u, float s, float s2) {
        const float second = o.teacher.second;
        if (u > top) {
            sum = sum * exp2f(top - u) + s;
            if (second != 0.0f) sum2 = sum2 * exp2f((top - u) * second) + s2;
            top = u;
        } else if (s != 0.0f) {   // (NaN too)
            sum += s * exp2f(u - top);
            if (second != 0.0f) sum2 += s2 * exp2f((u - top) * second);
        }
    }
    __device__ void parts(const EntryRows& o, uint32_t rows, uint32_t row, uint32_t lane) {
        const uint32_t m = row / pg::BM, m_tiles = (rows + pg::BM - 1) / pg::BM, whole_rows = m_tiles * pg::BM;
        for (uint32_t begin = 0, piece = 0; begin < o.n_tiles; begin += o.piece_tiles, ++piece) {
            const uint32_t width = min(o.piece_tiles, o.n_tiles - begin);
            const pg::Share share = pg::share_of(m_tiles * width, o.pairs);
            const uint32_t slots = share.owner(m * width + width - 1) - share.owner(m * width) + 1;
            const size_t at = piece * o.part_piece + row;
#pragma unroll 4
            for (uint32_t i = lane; i < slots * 4; i += 16) {   // a slot's quarters of the columns
                const size_t from = at + (size_t)i * whole_rows;
                const float2 p = o.part[from];
                add(o, p.x, p.y, o.teacher.second != 0.0f ? o.part2[from] : 0.0f);
            }
        }
    }
    // log2 of both sums over all columns, less `top` (times the second's factor), and `p`, the target's probabilities: each as itself, or
    // where it is above a half less 1 (with the sign set, of 0 too).  Where the target is the largest, from what the others add to its 1,
    // which a sum with it has lost where a row is sure.
    __device__ float2 logs(const EntryRows& o, float target, float2* p) {
        const float second = o.teacher.second;
        float hit = 1.0f, hit2 = 1.0f, log, log2 = 0.0f;   // (target's and others' parts of a sum)
        if (target >= top) {
            sum = sum * exp2f(top - target) + (target - target);   // (NaN where that is infinite)
            sum2 *= exp2f((top - target) * second);
            top = target;
            log = log1pf(sum) * pg::LOG2E;
            if (second != 0.0f) log2 = log1pf(sum2) * pg::LOG2E;
        } else {
            hit = exp2f(target - top);
            hit2 = exp2f((target - top) * second);
            log = log2f(sum + hit);
            if (second != 0.0f) log2 = log2f(sum2 + hit2);
        }
        const auto share = [](float hit, float others) { return (hit > others ? -others : hit) / (hit + others); };
        p->x = share(hit, sum);
        p->y = second != 0.0f ? share(hit2, sum2) : p->x;
        return make_float2(log, log2);
    }
    // The target's g.  p: of `logs`; w: its weight, hard and the teacher's; others: the weights of the row's other entries, which add up to what
    // the teacher's is short of its share.  A sure row's is the difference of what student and teacher leave to other columns.
    static __device__ float target_g(const Teacher& t, float2 p, bool has, float w, float others) {
        const float soft = has ? t.alpha * t.temperature : 0.0f;
        const float of_label = t.hard * (signbit(p.x) ? p.x : p.x - 1.0f);
        const float of_teacher = fmaf(soft, p.y, signbit(p.y) ? others : t.hard - w);
        return t.hard > 0.0f ? of_label + of_teacher : of_teacher;
    }
    static __device__ bool sure(const Teacher& t, float2 p, bool has) {
        const float soft = has ? t.alpha * t.temperature : 0.0f;
        return signbit(p.x) && signbit(p.y) && -fmaf(t.hard, p.x, soft * p.y) < (t.hard + soft) * (1.0f / 64.0f);
    }
    // ... and with the shares taken off, what GRAD takes from a logit (times the second's factor) before its exp
    struct Lse {
        float first, second;
        __device__ float probability(const EntryRows& o, float z) const {   // (both shares times theirs)
            float g = pg::exp2_fast(z - first);
            if (o.teacher.second != 0.0f) g += pg::exp2_fast(fmaf(z, o.teacher.second, -second));
            return g;
        }
    };
    __device__ Lse lse(const EntryRows& o, float2 logs, bool has) const {
        const Teacher& t = o.teacher;
        const float soft = has ? t.alpha * t.temperature : 0.0f;
        if (t.second != 0.0f)   // (no entries: infinity, whose exp is 0)
            return Lse{top + logs.x - log2f(t.hard), top * t.second + logs.y - log2f(soft)};
        return Lse{top + logs.x - log2f(t.hard + soft), 0.0f};
    }
};
__global__ void __launch_bounds__(ROWS_THREADS, 2)
entries_rows_kernel(const EntryRows o) {
    chain_entry();
    const Teacher& t = o.teacher;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = *o.counted;
    const size_t block_entries = (size_t)BLOCK_ROWS * t.K1;
    __shared__ float tops[ROWS_WARPS];
    // Of a row's target: g, and times the product; GRAD's probability, and times its product; where it lies among the offsets, and SURE.
    constexpr uint32_t SURE = 0x80000000u;
    __shared__ float2 row_target[BLOCK_ROWS], row_cut[BLOCK_ROWS];
    __shared__ uint32_t row_at[BLOCK_ROWS];
    __shared__ RowSums::Lse row_lse[BLOCK_ROWS];
    // the power of two of g * scale
    float largest = o.scale_max ? 0.0f : 1.0f;
    if (o.scale_max)
        for (uint32_t i = threadIdx.x; i < o.n_scale_max; i += ROWS_THREADS) largest = fmaxf(largest, o.scale_max[i]);
    for (int d = 16; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, d));
    if (lane == 0) tops[warp] = largest;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < ROWS_WARPS; ++w) largest = fmaxf(largest, tops[w]);
    const int exponent = (int)(__float_as_uint(largest) >> 23) - 127;
    const int power = largest > 0.0f && exponent < 128 ? 14 - exponent - o.headroom : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        o.factors[0] = exp2f((float)power);
        o.factors[1] = exp2f((float)-power) * o.loss_scale;
    }
    const uint32_t first = blockIdx.x * BLOCK_ROWS;
    if (first >= rows) return;
    // two rows to a warp, sixteen lanes to a row
    const uint32_t r = warp * 2 + (lane & 1), row = first + r, part_lane = lane >> 1;   // (32 rows: of one tile)
    RowSums sums_of;
    sums_of.parts(o, rows, row, part_lane);
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) {   // (within a row's lanes, in a fixed order)
        const RowSums mine = sums_of;
        RowSums other;
        other.top = __shfl_xor_sync(0xffffffffu, mine.top, 2 * k);
        other.sum = __shfl_xor_sync(0xffffffffu, mine.sum, 2 * k);
        other.sum2 = __shfl_xor_sync(0xffffffffu, mine.sum2, 2 * k);
        const bool mine_first = !(part_lane & k);
        sums_of = mine_first ? mine : other;
        if (mine_first) sums_of.add(o, other.top, other.sum, other.sum2);
        else sums_of.add(o, mine.top, mine.sum, mine.sum2);
    }
    const bool in = row < rows;
    const float target = in ? o.target_logit[row] : 0.0f;
    float2 p_target;
    const float2 logs = sums_of.logs(o, target, &p_target);
    float off = 0.0f, others = 0.0f;   // sums of w * (top - z), and of w without the target's
    if (in) {
        const uint32_t target_place = o.lists.target[row];
#pragma unroll 4
        for (uint32_t k = part_lane; k < t.K1; k += 16) {
            const uint32_t i = o.lists.place[(size_t)row * t.K1 + k];
            if (i == NO_PLACE) continue;
            const float w = o.lists.weight[blockIdx.x * block_entries + i];
            const float z = i == target_place ? target : o.logits[blockIdx.x * block_entries + i].y;
            if (w != 0.0f) off += w * (sums_of.top - z);
            if (i != target_place) others += w;
        }
    }
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) {
        off += __shfl_xor_sync(0xffffffffu, off, 2 * k);
        others += __shfl_xor_sync(0xffffffffu, others, 2 * k);
    }
    if (in && part_lane == 0) {
        const float constant = o.lists.constant[row];
        const bool has = constant == constant;
        const float soft = has ? t.alpha * t.temperature * t.temperature : 0.0f;   // of the loss
        const RowSums::Lse lse = sums_of.lse(o, logs, has);
        float loss;
        if (t.second != 0.0f) {
            loss = t.hard * logs.x + soft * logs.y;
        } else {
            loss = t.hard + soft != 0.0f ? (t.hard + soft) * logs.x : 0.0f;
            off /= t.first;
        }
        if (!(o.residual & row)) o.row_loss[o.list[row]] = (loss + off) * LN2 + (has ? constant : 0.0f);
        o.lse2[row] = lse.first;
        if (t.second != 0.0f) o.second_lse2[row] = lse.second;
        row_lse[r] = lse;
        const size_t i = blockIdx.x * block_entries + o.lists.target[row];
        const float g = RowSums::target_g(t, p_target, has, o.lists.weight[i], others);
        const float2 cut = o.logits[i];
        const float p_cut = lse.probability(o, cut.y);
        row_target[r] = make_float2(g, g * o.target_acc[row]);
        row_cut[r] = make_float2(p_cut, p_cut * cut.x);
        row_at[r] = o.lists.column[i] / GROUP_COLUMNS * 2 | (RowSums::sure(t, p_target, has) ? SURE : 0u);
    }
    __syncthreads();
    const uint32_t n = o.lists.offsets[(size_t)blockIdx.x * o.lists.groups1 + o.lists.groups1 - 1];
    // the rows whose targets GRAD leaves out: with a sure one in the same group of columns
    const uint32_t row_there = first + lane < rows ? row_at[lane] : 0u, all_sure = __ballot_sync(0xffffffffu, row_there & SURE);
    uint32_t left_out = 0;
    if (all_sure) {
        const uint32_t place = row_there & ~SURE, same = __match_any_sync(0xffffffffu, first + lane < rows ? place : SURE | lane), sure = all_sure & same;
        left_out = __ballot_sync(0xffffffffu, sure != 0);
        if (warp == 0 && sure && (uint32_t)__ffs(same) - 1 == lane) o.lists.offsets[(size_t)blockIdx.x * o.lists.groups1 + place] |= pg::OFFSET_SURE;
    }
    const float times = exp2f((float)power);
    const auto to_bits = [&](float v) {
        return o.bf16 ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)) : (uint32_t)__half_as_ushort(__float2half_rn(v));
    };
#pragma unroll 2
    for (uint32_t j = threadIdx.x; j < n; j += ROWS_THREADS) {
        const size_t i = blockIdx.x * block_entries + j;
        const uint32_t bits = o.lists.bits[i], column = o.lists.column[i], of = pg::entry_row(bits);
        const float w = o.lists.weight[i];
        const float2 logit = o.logits[i];
        const bool is_target = bits & pg::ENTRY_TARGET;
        o.logits[i] = (w == 0.0f && !is_target) || (o.residual & bits) ? make_float2(0.0f, 0.0f)
                      : !is_target                                 ? make_float2(-w, -w * logit.x)
                      : left_out >> of & 1u                        ? row_target[of]
                                   : make_float2(row_target[of].x - row_cut[of].x, row_target[of].y - row_cut[of].y);
        const float g = (is_target ? row_target[of].x : row_lse[of].probability(o, logit.y) - w) * times * pg::half_at(o.scale, column, 1.0f);
        uint32_t g16 = to_bits(g);
        if (o.residual & bits) g16 = to_bits(g - (o.bf16 ? __uint_as_float(g16 << 16) : __half2float(__ushort_as_half((uint16_t)g16))));
        o.lists.column[i] = bits | g16 << 16;
    }
}

// The sums over the columns of what their entries add, four words of entries on their way (one, whose
// targets' parts are looked up by row: 42 us instead of 24): a CTA has 64 columns and a stretch of blocks, and sums over runs of one column in a
// word of 32 entries, then over the words and blocks of a warp, then over the warps.  It needs nothing of GRAD, which has waited for
// entries_rows, or this would not have been launched: it begins on the SMs that GRAD leaves first, and waits for GRAD at its end, so that
// whoever waits for this kernel has waited for both.
__global__ void __launch_bounds__(COLUMNS_THREADS)
entries_columns_kernel(const EntryRows o) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = *o.counted;
    const size_t block_entries = (size_t)BLOCK_ROWS * o.teacher.K1;
    __shared__ float sums[COLUMNS_WARPS][2][GROUP_COLUMNS];
    const uint32_t group = blockIdx.x / o.stretches, stretch = blockIdx.x % o.stretches;
    for (uint32_t i = lane; i < 2 * GROUP_COLUMNS; i += 32) sums[warp][0][i] = 0.0f;
    __syncwarp();
    const uint32_t end = min((stretch + 1) * o.stretch, (rows + BLOCK_ROWS - 1) / BLOCK_ROWS);
    // block by block, words of 32 entries, the next four of them on their way
    uint32_t block = stretch * o.stretch + warp, at = 0, last = 0;
    struct {
        uint32_t words, bits[WORDS];
        float2 g[WORDS];   // and times the product
    } now, next;
    const auto open = [&]() {   // the next block that has any
        while (at >= last && block < end) {
            const uint16_t* offsets = o.lists.offsets + (size_t)block * o.lists.groups1 + 2 * group;
            at = offsets[0] & (pg::OFFSET_SURE - 1);
            last = offsets[2] & (pg::OFFSET_SURE - 1);
            if (at < last) break;
            block += COLUMNS_WARPS;
        }
    };
    const auto fetch = [&]() {
        next.words = 0;
        if (block >= end) return;
        const size_t i = block * block_entries + at + lane;
#pragma unroll
        for (uint32_t k = 0; k < WORDS; ++k) {
            const bool in = at + k * 32 + lane < last;
            next.bits[k] = in ? o.lists.bits[i + k * 32] : pg::NO_ENTRY;
            next.g[k] = in ? o.logits[i + k * 32] : make_float2(0.0f, 0.0f);
        }
        next.words = min(WORDS, (last - at + 31) / 32);
        at += WORDS * 32;
        if (at >= last) {
            block += COLUMNS_WARPS;
            open();
        }
    };
    open();
    fetch();
    while (next.words) {
        now = next;
        fetch();
#pragma unroll
        for (uint32_t k = 0; k < WORDS; ++k) {
            if (k >= now.words) break;
            const bool in = now.bits[k] != pg::NO_ENTRY;
            const uint32_t run = in ? (now.bits[k] & (pg::ENTRY_PLACES - 1)) >> 4 : pg::NO_ENTRY;   // half, column
            float2 g = now.g[k];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const bool same = __shfl_up_sync(0xffffffffu, run, d) == run && (int)lane >= d;
                if (!__any_sync(0xffffffffu, in && same)) break;   // (nor further apart)
                const float2 u = make_float2(__shfl_up_sync(0xffffffffu, g.x, d), __shfl_up_sync(0xffffffffu, g.y, d));
                if (same) g = make_float2(g.x + u.x, g.y + u.y);
            }
            const uint32_t right = __shfl_down_sync(0xffffffffu, run, 1);
            const bool ends = in && (lane == 31 || right != run);
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {   // (a column may end a run of either)
                if (ends && run >> 6 == half) {
                    sums[warp][0][run & 63u] += g.x;
                    sums[warp][1][run & 63u] += g.y;
                }
                __syncwarp();
            }
        }
    }
    __syncthreads();
    if (threadIdx.x < 2 * GROUP_COLUMNS) {
        const uint32_t which = threadIdx.x / GROUP_COLUMNS, c = threadIdx.x % GROUP_COLUMNS;
        float all = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < COLUMNS_WARPS; ++w) all += sums[w][which][c];
        o.column_sums[((size_t)stretch * 2 + which) * o.column_pitch + group * GROUP_COLUMNS + c] = all;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace
}  // namespace dev
}  // namespace ullis
