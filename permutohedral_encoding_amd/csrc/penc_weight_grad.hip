// The weight gradient of a linear layer from its kept input:
//
//     dW[o][c] = sum over rows of g[row][o] x^[row][c],     db[o] = sum over rows of g[row][o]
//
// A product over the rows, which are the strides of both operands, by v_mfma_f32_16x16x32_bf16.  x^ = q 2^e has at most 7 bits and is exact in
// bfloat16; a gradient is taken whole: bfloat16 as it is, fp16 as a sum of two and fp32 as a sum of three bfloat16 values (8 bits each, the
// rest exactly), so that every product is exact and the sums are those of fp32.  (Of fp32 gradients under 2^-110 the last bits would be under bfloat16's
// least value, 2^-133, and are dropped.)
//
// The matrix instruction wants 8 consecutive rows of one column in a lane.  A lane loads them for kWide neighbouring columns (16 bytes of a row in
// one load; one or two columns where there are few), and v_perm pairs two rows' halves; lane m of 16 then has columns kWide m .. kWide m + kWide - 1,
// one for each of kWide tiles, whose columns are kWide apart.  Which column a lane of a tile stands for is free, so nothing goes through the LDS on the
// way in.
//
// A wave walks over rows 32 at a time, the waves of a workgroup and the workgroups of a tile each over their own, and the partial sums are added in
// a fixed order: the waves' in the LDS, the workgroups' by sum_splits_kernel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "penc_kept.hpp"

namespace penc {
namespace {

constexpr int kStep = 32;  // rows of a matrix instruction
constexpr int kLargeBlock = 256;
constexpr int kLaneRows = 8;

using frag_t = bf16_t __attribute__((ext_vector_type(8)));
using acc_t = float __attribute__((ext_vector_type(4)));

struct Frag {
    uint32_t d[4];
    __device__ __forceinline__ frag_t get() const { return __builtin_bit_cast(frag_t, d); }
};

__device__ __forceinline__ uint32_t low_halves(uint32_t first, uint32_t second) { return __builtin_amdgcn_perm(second, first, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t first, uint32_t second) { return __builtin_amdgcn_perm(second, first, 0x07060302u); }

// Where a lane's 8 rows of a step are.  The last step's lanes that would read behind `last` read the 8 rows before it instead, and `skip` of them count
// for nothing: loads have no conditions.
struct StepRows {
    row_t first;  // of the step, the same in every lane
    uint32_t at;  // the lane's, from there on
    int skip;

    __device__ __forceinline__ StepRows(row_t step, uint32_t row_at, row_t rows) {
        const row_t most = rows - kLaneRows;
        first = min(step, most);
        const row_t row = min(step + row_at, most);
        at = row - first;
        skip = static_cast<int>(step + row_at - row);
    }
};

// Registers of a row.
template <int kWords>
using words_t = uint32_t __attribute__((ext_vector_type(kWords)));

// Rows that count for nothing, after their loads have come.
template <class W>
__device__ __forceinline__ void skip_rows(W (&row)[kLaneRows], int skip) {
    if (skip == 0) return;
#pragma unroll
    for (int j = 0; j < kLaneRows; ++j) row[j] = j < skip ? W{} : row[j];
}

// What a lane has of the gradient, 8 rows of kWide columns as they are in memory, in kWords registers a row.
template <class E, int kWide>
struct GradTile {
    static constexpr int kPieces = std::is_same_v<E, float> ? 3 : std::is_same_v<E, half_t> ? 2 : 1;
    static constexpr int kWords = kWide == 1 ? 1 : kWide * sizeof(E) / 4;
    using Bits = std::conditional_t<sizeof(E) == 4, uint32_t, uint16_t>;
    using Vector = uint32_t __attribute__((ext_vector_type(kWords), aligned(sizeof(E))));

    // The columns from which a lane reads: the last lane of a row, where it has fewer than kWide, takes some that its neighbour has too, and finds the same sums.
    __device__ __forceinline__ static int column_of(int o, int outputs) { return min(o, outputs - kWide); }

    template <class W>
    __device__ __forceinline__ static void load(W (&row)[kLaneRows], const void* grad, int64_t stride, StepRows rows, int column) {
        const char* const first = static_cast<const char*>(grad) + static_cast<int64_t>(rows.first) * stride * static_cast<int64_t>(sizeof(E));
        const uint32_t at = (rows.at * static_cast<uint32_t>(stride) + static_cast<uint32_t>(column)) * static_cast<uint32_t>(sizeof(E));
#pragma unroll
        for (int j = 0; j < kLaneRows; ++j) {
            const char* const p = first + j * stride * static_cast<int64_t>(sizeof(E)) + at;
            if constexpr (kWide == 1) {
                row[j][0] = *reinterpret_cast<const Bits*>(p);
            } else {
                const Vector v = *reinterpret_cast<const Vector*>(p);
#pragma unroll
                for (int w = 0; w < kWords; ++w) row[j][w] = v[w];
            }
        }
    }
    // for fewer rows or columns than a lane takes
    template <class W>
    __device__ __forceinline__ static void load_ragged(W (&row)[kLaneRows], const E* __restrict__ g, int64_t stride, int64_t rows_left, int valid) {
#pragma unroll
        for (int j = 0; j < kLaneRows; ++j) {
            const auto bits = [&](int t) { return j < rows_left && t < valid ? static_cast<uint32_t>(__builtin_bit_cast(Bits, g[j * stride + t])) : 0u; };
#pragma unroll
            for (int w = 0; w < kWords; ++w) row[j][w] = sizeof(E) == 4 ? bits(w) : bits(2 * w) | bits(2 * w + 1) << 16;
        }
    }
    // column t in kPieces parts
    template <class W>
    __device__ __forceinline__ static void column(const W (&row)[kLaneRows], int t, Frag (&f)[kPieces]) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            if constexpr (kPieces == 1) {
                const uint32_t a = row[2 * p][t / 2], b = row[2 * p + 1][t / 2];
                f[0].d[p] = t % 2 == 0 ? low_halves(a, b) : high_halves(a, b);
            } else {
                float a = value(row[2 * p], t), b = value(row[2 * p + 1], t);
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    f[k].d[p] = high_halves(__float_as_uint(a), __float_as_uint(b));
                    a = rest(a), b = rest(b);
                }
            }
        }
    }
    template <class W>
    __device__ __forceinline__ static float value(const W& row, int t) {
        if constexpr (sizeof(E) == 4) return __uint_as_float(row[t]);
        else return static_cast<float>(__builtin_bit_cast(E, static_cast<uint16_t>(row[t / 2] >> 16 * (t % 2))));
    }
    // x without its first 8 bits; nothing is left of an infinity, and a NaN stays one
    __device__ __forceinline__ static float rest(float x) {
        const float first = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
        return fabsf(x) == __builtin_inff() ? 0.0f : x - first;
    }
};

// What a lane has of the checkpoint: 8 rows of kWide columns, all of one block, and behind them the block's exponent.
template <int kWide>
struct KeptTile {
    static constexpr int kWords = kWide / 4 + 1;
    using Vector = uint32_t __attribute__((ext_vector_type(kWide / 4)));

    // (columns behind a row's end are read from within it, for results that are not stored)
    __device__ __forceinline__ static int column_of(int c, const KeptArray& kept) { return min(c, static_cast<int>(kept.pitch) - kWide); }

    template <class W>
    __device__ __forceinline__ static void load(W (&row)[kLaneRows], const KeptArray& kept, StepRows rows, int column) {
        const int8_t* const values = kept.values + offset_of(rows.first, kept.pitch);
        const uint8_t* const exponents = kept.exponents + offset_of(rows.first, kept.blocks);
        const uint32_t at = rows.at * static_cast<uint32_t>(kept.pitch) + static_cast<uint32_t>(column);
        const uint32_t block_at = rows.at * static_cast<uint32_t>(kept.blocks) + static_cast<uint32_t>(column / kKeptBlock);
#pragma unroll
        for (int j = 0; j < kLaneRows; ++j) {
            const Vector v = *reinterpret_cast<const Vector*>(values + j * kept.pitch + at);
#pragma unroll
            for (int w = 0; w < kWide / 4; ++w) row[j][w] = v[w];
            row[j][kWide / 4] = (exponents + j * kept.blocks)[block_at];
        }
    }
    template <class W>
    __device__ __forceinline__ static void load_ragged(W (&row)[kLaneRows], const KeptArray& kept, int64_t first, int64_t rows_left, int column) {
#pragma unroll
        for (int j = 0; j < kLaneRows; ++j) {
            const bool there = j < rows_left;
            const Vector v = there ? *reinterpret_cast<const Vector*>(kept.values + (first + j) * kept.pitch + column) : Vector{};
#pragma unroll
            for (int w = 0; w < kWide / 4; ++w) row[j][w] = v[w];
            row[j][kWide / 4] = there ? kept.exponents[(first + j) * kept.blocks + column / kKeptBlock] : 0;
        }
    }
    // q 2^e, exact
    template <class W>
    __device__ __forceinline__ static uint32_t value(const W& row, int t) {
        return __float_as_uint(static_cast<float>(static_cast<int8_t>(row[t / 4] >> 8 * (t % 4))) * kept_step(row[kWide / 4]));
    }
    template <class W>
    __device__ __forceinline__ static Frag column(const W (&row)[kLaneRows], int t) {
        Frag f;
#pragma unroll
        for (int p = 0; p < 4; ++p) f.d[p] = high_halves(value(row[2 * p], t), value(row[2 * p + 1], t));
        return f;
    }
};

struct WeightGrad {
    row_t rows, split_rows;  // split_rows: of a workgroup, a multiple of its waves' steps
    int64_t grad_stride;
    int channels, outputs, channel_tiles, output_tiles;
    KeptArray kept;
    const void* grad;
    float *sums, *bias_sums;  // [splits][outputs][channels], [splits][outputs] or null
    void *weight, *bias;      // where the rows are not split, the results themselves (else null), of `type`
    int type;
};

// A workgroup's sum of result `at`, of the weight or the bias.
__device__ __forceinline__ void leave(float* sums, void* result, int type, int64_t n, int64_t split, int64_t at, float total) {
    if (result == nullptr) sums[split * n + at] = total;
    else if (type == PENC_FP32) static_cast<float*>(result)[at] = total;
    else if (type == PENC_FP16) static_cast<half_t*>(result)[at] = static_cast<half_t>(total);
    else static_cast<bf16_t*>(result)[at] = static_cast<bf16_t>(total);
}
__device__ __forceinline__ void leave_weight(const WeightGrad& a, int64_t split, int output, int channel, float total) {
    leave(a.sums, a.weight, a.type, static_cast<int64_t>(a.outputs) * a.channels, split, static_cast<int64_t>(output) * a.channels + channel, total);
}
__device__ __forceinline__ void leave_bias(const WeightGrad& a, int64_t split, int output, float total) {
    leave(a.bias_sums, a.bias, a.type, a.outputs, split, output, total);
}

// The work of a workgroup.  Consecutive workgroups go to the 8 dies in turn: each of them gets neighbouring items, tiles of the same rows, which its cache
// then holds.
__device__ __forceinline__ int64_t item_of(const WeightGrad& a) {
    constexpr unsigned kDies = 8;
    const unsigned die = blockIdx.x % kDies, each = gridDim.x / kDies, rest = gridDim.x % kDies;
    return die * each + min(die, rest) + blockIdx.x / kDies;
}

// 16 kWideO outputs by 16 kWideC channels.  Bound by memory: each operand is read once for 64 columns of the other.  1048576 x 48 by 64 outputs fp32 74 us,
// 4.3 TB/s (a wave's next rows are on their way while it multiplies; without that 82).  kWideO is 4, or 1 or 2 for 16 or 32 outputs and fewer (and for few
// rows), which leave the registers and LDS of a second workgroup: 1048576 x 64 by 1 output fp32 64 -> 25 us, by 16 51 -> 28, by 32 52 -> 43; bf16 by 3
// 53 -> 18, by 32 27 -> 28.
template <class E, int kWideO, int kWideC, int kWaves, bool kRagged>
__global__ __launch_bounds__(64 * kWaves) void weight_grad_kernel(WeightGrad a) {
    constexpr int kPieces = GradTile<E, kWideO>::kPieces;
    __shared__ float lds[kWaves][16 * kWideO][16 * kWideC];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, column = lane % 16, rows_at = lane / 16 * kLaneRows;
    const int64_t item = item_of(a);
    const int tile = static_cast<int>(item % (a.channel_tiles * a.output_tiles));
    const int64_t split = item / (a.channel_tiles * a.output_tiles);
    const int c0 = tile % a.channel_tiles * 16 * kWideC, o0 = tile / a.channel_tiles * 16 * kWideO;
    using G = GradTile<E, kWideO>;
    using X = KeptTile<kWideC>;
    const int c = X::column_of(c0 + column * kWideC, a.kept), o = kRagged ? o0 + column * kWideO : G::column_of(o0 + column * kWideO, a.outputs);
    const bool bias = (a.bias_sums != nullptr || a.bias != nullptr) && c0 == 0;
    const row_t first = static_cast<row_t>(split) * a.split_rows, last = min(first + a.split_rows, a.rows);

    acc_t acc[kWideO][kWideC] = {}, bias_acc[kWideO] = {};
    const Frag ones = {{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}};
    words_t<G::kWords> g[kLaneRows], g_ahead[kLaneRows];
    words_t<X::kWords> x[kLaneRows], x_ahead[kLaneRows];
    // (behind the last step: rows that are there)
    const auto load = [&](row_t step) {
        if constexpr (kRagged) {
            const int64_t row = static_cast<int64_t>(step) + rows_at;
            G::load_ragged(g_ahead, static_cast<const E*>(a.grad) + row * a.grad_stride + o, a.grad_stride, static_cast<int64_t>(last) - row, a.outputs - o);
            X::load_ragged(x_ahead, a.kept, row, static_cast<int64_t>(last) - row, c);
        } else {
            const StepRows rows(step, rows_at, a.rows);
            G::load(g_ahead, a.grad, a.grad_stride, rows, o);
            X::load(x_ahead, a.kept, rows, c);
        }
    };
    row_t step = first + wave * kStep;
    if (step < last) load(step);
    for (; step < last; step += kWaves * kStep) {
#pragma unroll
        for (int j = 0; j < kLaneRows; ++j) g[j] = g_ahead[j], x[j] = x_ahead[j];
        load(step + kWaves * kStep);
        if (!kRagged && step + kStep > a.rows) {
            const StepRows rows(step, rows_at, a.rows);
            skip_rows(g, rows.skip);
            skip_rows(x, rows.skip);
        }
        Frag fx[kWideC];
#pragma unroll
        for (int s = 0; s < kWideC; ++s) fx[s] = X::column(x, s);
#pragma unroll
        for (int t = 0; t < kWideO; ++t) {
            Frag fg[kPieces];
            G::column(g, t, fg);
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
#pragma unroll
                for (int s = 0; s < kWideC; ++s) acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fg[k].get(), fx[s].get(), acc[t][s], 0, 0, 0);
                if (bias) bias_acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fg[k].get(), ones.get(), bias_acc[t], 0, 0, 0);
            }
        }
    }
    // Lane (16 i + n) has rows 4 i .. 4 i + 3 of a result's column n.
#pragma unroll
    for (int t = 0; t < kWideO; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int s = 0; s < kWideC; ++s) lds[wave][(lane / 16 * 4 + r) * kWideO + t][column * kWideC + s] = acc[t][s][r];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * kWideO * kWideC; i += 64 * kWaves) {
        const int m = i / (16 * kWideC), n = i % (16 * kWideC), from = o0 + m / kWideO * kWideO;
        if (from >= a.outputs) break;
        const int to = (kRagged ? from : G::column_of(from, a.outputs)) + m % kWideO;
        float total = lds[0][m][n];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) total += lds[w][m][n];
        if (to < a.outputs && c0 + n < a.channels) leave_weight(a, split, to, c0 + n, total);
    }
    if (!bias) return;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kWideO; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (column == 0) lds[wave][0][(lane / 16 * 4 + r) * kWideO + t] = bias_acc[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * kWideO; i += 64 * kWaves) {
        const int from = o0 + i / kWideO * kWideO, to = (kRagged ? from : G::column_of(from, a.outputs)) + i % kWideO;
        float total = lds[0][0][i];
        for (int w = 1; w < kWaves; ++w) total += lds[w][0][i];
        if (from < a.outputs && to < a.outputs) leave_bias(a, split, to, total);
    }
}

// The same for products that the matrix cores bound: 256 outputs by 256 channels to a workgroup of 8 waves, which bring 32 kSteps rows at a time
// into the LDS as the matrix instruction takes them, half of the waves the gradient and half the checkpoint (one of either kind on each SIMD), while all of
// them multiply what was brought before.  Every value is converted once for the workgroup, and a wave's 4 x 8 tiles multiply a fragment 2.7 times.
// Bound by the matrix cores and the LDS, which have as much to do: of bf16, 64 rows take the matrix cores 2060 clocks at their peak, and the 192 KB read and
// 64 KB written 2050 at 128 bytes a clock.  16384 x 1024 by 4096 outputs bf16 145 us with the sum of its splits, 0.95 PFLOP/s (the library's product of bf16
// operands of these sizes 197 us, and of 8192^3, its best, 1.28 PFLOP/s; the 64-column kernel 286).
template <class E, int kSteps>
__global__ __launch_bounds__(512, 2) void weight_grad_lds_kernel(WeightGrad a) {
    constexpr int kBlockO = kLargeBlock, kBlockC = kLargeBlock, kWavesO = 4;
    constexpr int kPieces = GradTile<E, 4>::kPieces, kWavesC = 8 / kWavesO;
    constexpr int kWideO = kBlockO * kSteps / 64, kWideC = kBlockC * kSteps / 64;  // four waves bring each side
    constexpr int kTilesO = kBlockO / 16 / kWavesO, kTilesC = kBlockC / 16 / kWavesC;
    constexpr int kGrad = kSteps * kBlockO / 16 * kPieces, kKept = kSteps * kBlockC / 16;  // fragments of 64 lanes
    __shared__ uint4 fragments[2 * (kGrad + kKept) * 64];                                   // those multiplied, and those brought
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t item = item_of(a);
    const int tiles = a.channel_tiles * a.output_tiles, tile = static_cast<int>(item % tiles);
    const int64_t split = item / tiles;
    const int c0 = tile % a.channel_tiles * kBlockC, o0 = tile / a.channel_tiles * kBlockO;
    const row_t first = static_cast<row_t>(split) * a.split_rows, last = min(first + a.split_rows, a.rows);

    // what this wave brings: 32 rows of 16 kWide columns
    const bool brings_grad = wave < 4;
    const int unit = wave % 4, unit_step = unit % kSteps, unit_column = unit / kSteps;
    const int row_at = unit_step * kStep + lane / 16 * kLaneRows;
    using G = GradTile<E, kWideO>;
    using X = KeptTile<kWideC>;
    const int o = G::column_of(o0 + unit_column * 16 * kWideO + lane % 16 * kWideO, a.outputs);
    const int c = X::column_of(c0 + unit_column * 16 * kWideC + lane % 16 * kWideC, a.kept);
    const auto fragment = [&](const uint4* from, int i) { return __builtin_bit_cast(frag_t, from[i * 64 + lane]); };
    const int first_o = wave % kWavesO * kTilesO, first_c = wave / kWavesO * kTilesC;  // this wave's tiles
    // the bias is one more column, of ones: the waves with the same outputs have some of them each
    constexpr int kBias = (kTilesO + kWavesC - 1) / kWavesC;
    const bool bias = (a.bias_sums != nullptr || a.bias != nullptr) && c0 == 0;
    const int first_bias = wave / kWavesO * kBias;
    const Frag ones = {{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}};
    acc_t acc[kTilesO][kTilesC] = {}, bias_acc[kBias] = {};

    // The loop of a wave that brings the gradient or the checkpoint: conversions and LDS between the products, without branches.  A step's rows are loaded
    // when those before them have been brought, and have half a step to come.  (Behind the last step they are rows that are there, for fragments that
    // nobody reads.)
    const auto walk = [&](auto brings_grad, auto with_bias) {
        constexpr bool kBringsGrad = decltype(brings_grad)::value;
        using Side = std::conditional_t<kBringsGrad, G, X>;
        constexpr int kColumns = kBringsGrad ? kWideO : kWideC, kSlots = kSteps * kPieces * kTilesC, kRows = kSteps * kStep;
        static_assert(kColumns <= kSlots, "every column has its place between the products");
        using Raw = words_t<Side::kWords>;
        const auto load = [&](Raw(&raw)[kLaneRows], row_t step) {
            const StepRows rows(step, row_at, a.rows);
            if constexpr (kBringsGrad) G::load(raw, a.grad, a.grad_stride, rows, o);
            else X::load(raw, a.kept, rows, c);
        };
        const auto skip = [&](Raw(&raw)[kLaneRows], row_t step) {
            if (step + kRows > a.rows) skip_rows(raw, StepRows(step, row_at, a.rows).skip);
        };
        const auto bring = [&](const Raw(&raw)[kLaneRows], uint4* to, int t) {
            if constexpr (kBringsGrad) {
                Frag f[kPieces];
                G::column(raw, t, f);
#pragma unroll
                for (int k = 0; k < kPieces; ++k)
                    to[((unit_step * kPieces + k) * (kBlockO / 16) + unit_column * kWideO + t) * 64 + lane] = make_uint4(f[k].d[0], f[k].d[1], f[k].d[2], f[k].d[3]);
            } else {
                const Frag f = X::column(raw, t);
                to[(kGrad + unit_step * (kBlockC / 16) + unit_column * kWideC + t) * 64 + lane] = make_uint4(f.d[0], f.d[1], f.d[2], f.d[3]);
            }
        };
        Raw raw[kLaneRows];
        load(raw, first);
        skip(raw, first);
#pragma unroll
        for (int t = 0; t < kColumns; ++t) bring(raw, fragments, t);
        load(raw, first + kRows);
        __syncthreads();
        int turn = 0;
        for (row_t step = first; step < last; step += kRows) {
            const uint4* const from = fragments + turn * (kGrad + kKept) * 64;
            uint4* const to = fragments + (turn ^ 1) * (kGrad + kKept) * 64;
            turn ^= 1;
            frag_t fg[kTilesO], fx = fragment(from, kGrad + first_c);
#pragma unroll
            for (int z = 0; z < kSlots; ++z) {
                const int s = z % kTilesC, part = z / kTilesC, more = z + 1;
                if (s == 0) {
#pragma unroll
                    for (int t = 0; t < kTilesO; ++t) fg[t] = fragment(from, part * (kBlockO / 16) + first_o + t);
                }
                const frag_t now = fx;
                if (more < kSlots) fx = fragment(from, kGrad + more / kTilesC / kPieces * (kBlockC / 16) + first_c + more % kTilesC);
#pragma unroll
                for (int t = 0; t < kTilesO; ++t) acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fg[t], now, acc[t][s], 0, 0, 0);
                if (decltype(with_bias)::value && s == kTilesC - 1) {
#pragma unroll
                    for (int t = 0; t < kBias; ++t)
                        bias_acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fragment(from, part * (kBlockO / 16) + first_o + first_bias + t), ones.get(), bias_acc[t], 0, 0, 0);
                }
                const int column = z - (kSlots - kColumns);
                if (column == 0) skip(raw, step + kRows);
                if (column >= 0) bring(raw, to, column);
                __builtin_amdgcn_sched_barrier(0);  // (or all that is converted waits in registers that there are not)
            }
            load(raw, step + 2 * kRows);
            __syncthreads();
        }
    };
    // (a barrier counts waves, wherever in the code they are: all of them pass the same number)
    if (brings_grad) {
        if (bias) walk(std::true_type{}, std::true_type{});
        else walk(std::true_type{}, std::false_type{});
    } else {
        if (bias) walk(std::false_type{}, std::true_type{});
        else walk(std::false_type{}, std::false_type{});
    }
    // Lane (16 i + n) has rows 4 i .. 4 i + 3 of a result's column n; tile T's row m is output (T / kWide * 16 + m) * kWide + T % kWide, and kWideC tiles
    // have neighbouring channels.
    static_assert(kTilesC % kWideC == 0, "a wave has whole groups of neighbouring channels");
    const auto write = [&](auto* to, auto* to_bias) {
        using To = std::remove_pointer_t<decltype(to)>;
        using Wide = To __attribute__((ext_vector_type(kWideC), aligned(sizeof(To))));
#pragma unroll
        for (int t = 0; t < kTilesO; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int big = first_o + t, from = o0 + (big / kWideO * 16 + lane / 16 * 4 + r) * kWideO;
                if (from >= a.outputs) continue;
                To* const row = to + static_cast<int64_t>(G::column_of(from, a.outputs) + big % kWideO) * a.channels;
#pragma unroll
                for (int group = 0; group < kTilesC; group += kWideC) {
                    const int at = c0 + ((first_c + group) / kWideC * 16 + lane % 16) * kWideC;
                    Wide v;
#pragma unroll
                    for (int s = 0; s < kWideC; ++s) v[s] = static_cast<To>(acc[t][group + s][r]);
                    if (at + kWideC <= a.channels) {
                        *reinterpret_cast<Wide*>(row + at) = v;
                    } else {
#pragma unroll
                        for (int s = 0; s < kWideC; ++s)
                            if (at + s < a.channels) row[at + s] = v[s];
                    }
                }
            }
        if (!bias || lane % 16 != 0) return;
#pragma unroll
        for (int t = 0; t < kBias; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int big = first_o + first_bias + t, from = o0 + (big / kWideO * 16 + lane / 16 * 4 + r) * kWideO;
                if (from < a.outputs) to_bias[G::column_of(from, a.outputs) + big % kWideO] = static_cast<To>(bias_acc[t][r]);
            }
    };
    if (a.weight == nullptr) write(a.sums + split * a.outputs * a.channels, a.bias_sums + split * a.outputs);
    else if (a.type == PENC_FP32) write(static_cast<float*>(a.weight), static_cast<float*>(a.bias));
    else if (a.type == PENC_FP16) write(static_cast<half_t*>(a.weight), static_cast<half_t*>(a.bias));
    else write(static_cast<bf16_t*>(a.weight), static_cast<bf16_t*>(a.bias));
}

// The splits of `n` weights and, behind them, `n_bias` of the bias, in a fixed order: 256 / kStrands results to a workgroup, each strand of threads
// with every kStrands-th split.  16 us for the 4 splits of 4096 x 1024, 4.7 TB/s; 5 us for the 256 of 64 x 48.
template <class To, int kStrands>
__global__ __launch_bounds__(256) void sum_splits_kernel(const float* __restrict__ sums, const float* __restrict__ bias_sums, int64_t n, int n_bias,
                                                         int splits, To* __restrict__ weight, To* __restrict__ bias) {
    constexpr int kResults = 256 / kStrands;
    __shared__ float lds[kStrands][kResults];
    const int lane = threadIdx.x % kResults, strand = threadIdx.x / kResults;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kResults + lane;
    float total = 0.0f;
    if (i < n + n_bias) {
        const float* const from = i < n ? sums + i : bias_sums + (i - n);
        const int64_t stride = i < n ? n : n_bias;
#pragma unroll 8
        for (int s = strand; s < splits; s += kStrands) total += from[s * stride];
    }
    if constexpr (kStrands > 1) {
        lds[strand][lane] = total;
        __syncthreads();
        if (strand != 0) return;
        for (int s = 1; s < kStrands; ++s) total += lds[s][lane];
    }
    if (i >= n + n_bias) return;
    if (i < n) weight[i] = static_cast<To>(total);
    else bias[i - n] = static_cast<To>(total);
}

constexpr int64_t kMostStride = 1 << 22;
// Products of as many multiplications (three or two for one of a gradient in parts) go by the larger tiles.  us by 64 columns a side -> by 256:
// 1024 x 1024 bf16, 4096 rows 26 -> 54, 16384 84 -> 75, 131072 643 -> 294; 256 x 1545 bf16, 16384 rows 50 -> 48; 256 x 256 fp32, 131072 rows 90 -> 76,
// 1024 x 1024 fp32, 4096 rows 47 -> 59, 16384 166 -> 115.  Fewer rows do not fill the card with large tiles; 8 rows of 1024 x 1024 7 -> 9.
constexpr int64_t kLargeProduct = int64_t{1} << 34;

// Of few rows the tiles are narrower, until there are as many workgroups.  us, fp32 by 64 outputs: 200 x 1024 8.5 -> 6.8,
// 1000 x 64 11.0 -> 9.4, 16384 x 32 12.1 -> 9.7; bf16 1000 x 32 10.0 -> 9.4.
constexpr int64_t kFewGroups = 128;

// How a product is cut up.
struct WeightPlan {
    int block, splits;  // columns of a workgroup, channels and (but where they are few) outputs; workgroups of a tile
    bool ragged;
    int wide;  // sixteens of outputs of a workgroup that has 64 channels
    int64_t split_rows;
    int output_tiles, channel_tiles;
};
WeightPlan weight_plan(int type, int64_t rows, int64_t channels, int64_t outputs, int64_t grad_stride) {
    WeightPlan p{};
    // (a lane takes 8 rows, at 32-bit offsets from a step's first row)
    p.ragged = rows < kLaneRows || grad_stride > kMostStride;
    const int64_t pieces_of_a_value = type == PENC_FP32 ? 3 : type == PENC_FP16 ? 2 : 1;
    const bool large = !p.ragged && channels > 128 && outputs > 128 && rows * channels * outputs * pieces_of_a_value >= kLargeProduct;
    p.block = large ? kLargeBlock : 64;
    p.channel_tiles = static_cast<int>((channels + p.block - 1) / p.block);
    const int64_t at_a_time = 8 * kStep, pieces = std::max<int64_t>(1, (rows + at_a_time - 1) / at_a_time);
    const auto tiles_of = [&](int outputs_of_tile) { return static_cast<int>((outputs + outputs_of_tile - 1) / outputs_of_tile); };
    p.wide = p.ragged || outputs > 32 ? 4 : outputs > 16 ? 2 : 1;
    while (!p.ragged && !large && p.wide > 1 && tiles_of(16 * p.wide) * p.channel_tiles * pieces < kFewGroups) p.wide /= 2;
    p.output_tiles = tiles_of(large ? kLargeBlock : 16 * p.wide);
    const int64_t tiles = static_cast<int64_t>(p.output_tiles) * p.channel_tiles;
    const int64_t wanted = std::max<int64_t>(1, std::min(pieces, (p.wide < 4 ? 512 : 256) / tiles));
    p.split_rows = (pieces + wanted - 1) / wanted * at_a_time;
    p.splits = static_cast<int>(std::max<int64_t>(1, (rows + p.split_rows - 1) / p.split_rows));
    return p;
}

bool bad_size(int64_t rows, int64_t channels, int64_t outputs) {
    return bad_rows(rows) || channels <= 0 || channels > PENC_MAX_CHANNELS || outputs <= 0 || outputs > PENC_MAX_CHANNELS || channels * outputs >= int64_t{1} << 31;
}

template <class E>
int launch(const WeightGrad& a, const WeightPlan& p, unsigned grid, hipStream_t stream) {
    constexpr int kPieces = GradTile<E, 4>::kPieces, kSteps = kPieces == 1 ? 2 : 1;
    if (p.ragged) hipLaunchKernelGGL((weight_grad_kernel<E, 4, 4, 8, true>), dim3(grid), dim3(512), 0, stream, a);
    else if (p.wide == 1) hipLaunchKernelGGL((weight_grad_kernel<E, 1, 4, 8, false>), dim3(grid), dim3(512), 0, stream, a);
    else if (p.wide == 2) hipLaunchKernelGGL((weight_grad_kernel<E, 2, 4, 8, false>), dim3(grid), dim3(512), 0, stream, a);
    else if (p.block != kLargeBlock) hipLaunchKernelGGL((weight_grad_kernel<E, 4, 4, 8, false>), dim3(grid), dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((weight_grad_lds_kernel<E, kSteps>), dim3(grid), dim3(512), 0, stream, a);
    return launched();
}

}  // namespace
}  // namespace penc

using namespace penc;

extern "C" {

size_t penc_weight_grad_workspace_bytes(int64_t rows, int64_t channels, int64_t outputs) {
    if (bad_size(rows, channels, outputs)) return 0;
    int splits = 1;  // the most of any type and stride
    for (const int type : {PENC_FP32, PENC_FP16, PENC_BF16})
        for (const int64_t stride : {int64_t{0}, kMostStride + 1}) splits = std::max(splits, weight_plan(type, rows, channels, outputs, stride).splits);
    return static_cast<size_t>(splits) * static_cast<size_t>(channels + 1) * static_cast<size_t>(outputs) * 4;
}

int penc_weight_grad(int type, int result_type, int64_t rows, int64_t channels, int64_t outputs, const int8_t* values, const uint8_t* exponents,
                     const void* grad, int64_t grad_row_stride, void* weight_grad, void* bias_grad, void* workspace, size_t workspace_bytes,
                     void* stream) {
    if (bad_size(rows, channels, outputs) || grad_row_stride < 0) return PENC_ERR_BAD_LAYER_SIZE;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        return with_type(result_type, [&](auto r) -> int {
            using To = decltype(r);
            if ((rows > 0 && (!values || !exponents || !grad)) || !weight_grad || !workspace) return PENC_ERR_NULL_POINTER;
            if (!aligned_to(values, kKeptPitch) || !aligned_to(grad, sizeof(E)) || !aligned_to(weight_grad, sizeof(To)) || !aligned_to(bias_grad, sizeof(To)) ||
                !aligned_to(workspace, 16))
                return PENC_ERR_MISALIGNED;
            if (workspace_bytes < penc_weight_grad_workspace_bytes(rows, channels, outputs)) return PENC_ERR_WORKSPACE_TOO_SMALL;
            const WeightPlan p = weight_plan(type, rows, channels, outputs, grad_row_stride);
            float* const sums = static_cast<float*>(workspace);
            const int64_t n = channels * outputs;
            const WeightGrad a{static_cast<row_t>(rows), static_cast<row_t>(p.split_rows), grad_row_stride, static_cast<int>(channels), static_cast<int>(outputs), p.channel_tiles,
                               p.output_tiles, kept_array(values, exponents, channels), grad, sums, bias_grad ? sums + p.splits * n : nullptr,
                               p.splits == 1 ? weight_grad : nullptr, p.splits == 1 ? bias_grad : nullptr, result_type};
            const int64_t grid = static_cast<int64_t>(p.splits) * p.output_tiles * p.channel_tiles;
            const int n_bias = bias_grad ? static_cast<int>(outputs) : 0;
            if (grid > 0x7FFFFFFF) return PENC_ERR_BAD_LAYER_SIZE;
            hipStream_t st = static_cast<hipStream_t>(stream);
            if (const int rc = launch<E>(a, p, static_cast<unsigned>(grid), st)) return rc;
            if (p.splits == 1) return PENC_OK;
            const auto sum = [&](auto kernel, int results) {
                hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n + n_bias + results - 1) / results)), dim3(256), 0, st, sums, a.bias_sums, n, n_bias,
                                   p.splits, static_cast<To*>(weight_grad), static_cast<To*>(bias_grad));
                return launched();
            };
            return p.splits < 16 ? sum(sum_splits_kernel<To, 1>, 256) : sum(sum_splits_kernel<To, 16>, 16);
        });
    });
}

}  // extern "C"
