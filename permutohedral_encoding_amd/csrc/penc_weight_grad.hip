// The weight gradient of a linear layer from its kept input:
//
//     dW[o][c] = sum over rows of g[row][o] x^[row][c],     db[o] = sum over rows of g[row][o]
//
// A product over the rows, which are the strides of both operands, by v_mfma_f32_16x16x32_bf16.  x^ = q 2^e has at most 7 bits and is exact in
// bfloat16; a gradient is taken whole: bfloat16 as it is, fp16 as a sum of two and fp32 as a sum of three bfloat16 values (8 bits each, the
// rest exactly), so that every product is exact and the sums are those of fp32.
//
// The matrix instruction wants 8 consecutive rows of one column in a lane.  A lane loads them for kWide neighbouring columns (16 bytes of a row in
// one load), and v_perm pairs two rows' halves; lane m of 16 then has columns kWide m .. kWide m + kWide - 1, one for each of kWide tiles, whose
// columns are kWide apart.  Which column a lane of a tile stands for is free, so nothing goes through the LDS on the way in.
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
constexpr int kLaneRows = 8;

using frag_t = bf16_t __attribute__((ext_vector_type(8)));
using acc_t = float __attribute__((ext_vector_type(4)));

struct Frag {
    uint32_t d[4];
    __device__ __forceinline__ frag_t get() const { return __builtin_bit_cast(frag_t, d); }
};

__device__ __forceinline__ uint32_t low_halves(uint32_t first, uint32_t second) { return __builtin_amdgcn_perm(second, first, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t first, uint32_t second) { return __builtin_amdgcn_perm(second, first, 0x07060302u); }

// What a lane has of the gradient: 8 rows of kWide columns, as they are in memory.
template <class E, int kWide>
struct GradTile {
    static constexpr int kPieces = std::is_same_v<E, float> ? 3 : std::is_same_v<E, half_t> ? 2 : 1;
    static constexpr int kWords = kWide * sizeof(E) / 4;
    using Bits = std::conditional_t<sizeof(E) == 4, uint32_t, uint16_t>;
    using Vector = uint32_t __attribute__((ext_vector_type(kWords), aligned(sizeof(E))));
    uint32_t row[kLaneRows][kWords];

    __device__ __forceinline__ void load(const E* __restrict__ g, int64_t stride, int64_t rows_left, int valid) {
#pragma unroll
        for (int j = 0; j < kLaneRows; ++j) {
            if (j < rows_left && valid >= kWide) {
                const Vector v = *reinterpret_cast<const Vector*>(g + j * stride);
#pragma unroll
                for (int w = 0; w < kWords; ++w) row[j][w] = v[w];
            } else {
                const auto bits = [&](int t) { return j < rows_left && t < valid ? static_cast<uint32_t>(__builtin_bit_cast(Bits, g[j * stride + t])) : 0u; };
#pragma unroll
                for (int w = 0; w < kWords; ++w) row[j][w] = sizeof(E) == 4 ? bits(w) : bits(2 * w) | bits(2 * w + 1) << 16;
            }
        }
    }
    __device__ __forceinline__ float value(int j, int t) const {
        if constexpr (sizeof(E) == 4) return __uint_as_float(row[j][t]);
        else return static_cast<float>(__builtin_bit_cast(E, static_cast<uint16_t>(row[j][t / 2] >> 16 * (t % 2))));
    }
    // column t in kPieces parts
    __device__ __forceinline__ void column(int t, Frag (&f)[kPieces]) const {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            if constexpr (kPieces == 1) {
                const uint32_t a = row[2 * p][t / 2], b = row[2 * p + 1][t / 2];
                f[0].d[p] = t % 2 == 0 ? low_halves(a, b) : high_halves(a, b);
            } else {
                float a = value(2 * p, t), b = value(2 * p + 1, t);
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    f[k].d[p] = high_halves(__float_as_uint(a), __float_as_uint(b));
                    a = rest(a), b = rest(b);
                }
            }
        }
    }
    // x without its first 8 bits; nothing is left of an infinity, and a NaN stays one
    __device__ __forceinline__ static float rest(float x) {
        const float first = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
        return fabsf(x) == __builtin_inff() ? 0.0f : x - first;
    }
};

// What a lane has of the checkpoint: 8 rows of kWide columns, all of one block.
template <int kWide>
struct KeptTile {
    using Bytes = std::conditional_t<kWide == 8, uint2, uint32_t>;
    Bytes row[kLaneRows];
    uint32_t exponent[kLaneRows];

    __device__ __forceinline__ void load(const KeptArray& kept, int64_t first, int64_t rows_left, int c) {
#pragma unroll
        for (int j = 0; j < kLaneRows; ++j) {
            const bool there = j < rows_left && c < kept.pitch;
            row[j] = there ? *reinterpret_cast<const Bytes*>(kept.values + (first + j) * kept.pitch + c) : Bytes{};
            exponent[j] = there ? kept.exponents[(first + j) * kept.blocks + c / kKeptBlock] : 0;
        }
    }
    __device__ __forceinline__ float value(int j, int t) const {
        uint32_t word;
        if constexpr (kWide == 8) word = t < 4 ? row[j].x : row[j].y;
        else word = row[j];
        return static_cast<float>(static_cast<int8_t>(word >> 8 * (t % 4))) * kept_step(exponent[j]);
    }
    __device__ __forceinline__ Frag column(int t) const {
        Frag f;
#pragma unroll
        for (int p = 0; p < 4; ++p) f.d[p] = high_halves(__float_as_uint(value(2 * p, t)), __float_as_uint(value(2 * p + 1, t)));
        return f;
    }
};

struct WeightGrad {
    int64_t rows, grad_stride, split_rows;  // split_rows: of a workgroup, a multiple of its waves' steps
    int channels, outputs, channel_tiles, output_tiles;
    KeptArray kept;
    const void* grad;
    float *sums, *bias_sums;  // [splits][outputs][channels], [splits][outputs] or null
};

// 16 kWideO outputs by 16 kWideC channels.
template <class E, int kWideO, int kWideC, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void weight_grad_kernel(WeightGrad a) {
    constexpr int kPieces = GradTile<E, kWideO>::kPieces;
    __shared__ float lds[kWaves][16][16 * kWideC];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, column = lane % 16, rows_at = lane / 16 * kLaneRows;
    const int tile = blockIdx.x % (a.channel_tiles * a.output_tiles), split = blockIdx.x / (a.channel_tiles * a.output_tiles);
    const int c0 = tile % a.channel_tiles * 16 * kWideC, o0 = tile / a.channel_tiles * 16 * kWideO;
    const int c = c0 + column * kWideC, o = o0 + column * kWideO;
    const bool bias = a.bias_sums != nullptr && c0 == 0;
    const int64_t first = split * a.split_rows, last = min(first + a.split_rows, a.rows);

    acc_t acc[kWideO][kWideC] = {}, bias_acc[kWideO] = {};
    const Frag ones = {{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}};
    for (int64_t step = first + wave * kStep; step < last; step += kWaves * kStep) {
        GradTile<E, kWideO> g;
        KeptTile<kWideC> x;
        const int64_t row = step + rows_at;
        g.load(static_cast<const E*>(a.grad) + row * a.grad_stride + o, a.grad_stride, last - row, a.outputs - o);
        x.load(a.kept, row, last - row, c);
        Frag fx[kWideC];
#pragma unroll
        for (int s = 0; s < kWideC; ++s) fx[s] = x.column(s);
#pragma unroll
        for (int t = 0; t < kWideO; ++t) {
            Frag fg[kPieces];
            g.column(t, fg);
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
#pragma unroll
                for (int s = 0; s < kWideC; ++s) acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fg[k].get(), fx[s].get(), acc[t][s], 0, 0, 0);
                if (bias) bias_acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fg[k].get(), ones.get(), bias_acc[t], 0, 0, 0);
            }
        }
    }
    // Lane (16 i + n) has rows 4 i .. 4 i + 3 of a result's column n.
    float* const sums = a.sums + static_cast<int64_t>(split) * a.outputs * a.channels;
#pragma unroll
    for (int t = 0; t < kWideO; ++t) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int s = 0; s < kWideC; ++s) lds[wave][lane / 16 * 4 + r][column * kWideC + s] = acc[t][s][r];
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * 16 * kWideC; i += 64 * kWaves) {
            const int m = i / (16 * kWideC), n = i % (16 * kWideC), to = o0 + m * kWideO + t;
            float total = lds[0][m][n];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) total += lds[w][m][n];
            if (to < a.outputs && c0 + n < a.channels) sums[static_cast<int64_t>(to) * a.channels + c0 + n] = total;
        }
    }
    if (!bias) return;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kWideO; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (column == 0) lds[wave][lane / 16 * 4 + r][t] = bias_acc[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * kWideO; i += 64 * kWaves) {
        float total = lds[0][i / kWideO][i % kWideO];
        for (int w = 1; w < kWaves; ++w) total += lds[w][i / kWideO][i % kWideO];
        if (o0 + i < a.outputs) a.bias_sums[static_cast<int64_t>(split) * a.outputs + o0 + i] = total;
    }
}

// The splits of `n` weights and, behind them, `n_bias` of the bias, in a fixed order: 64 results and 16 strands of splits to a workgroup.
template <class To>
__global__ __launch_bounds__(1024) void sum_splits_kernel(const float* __restrict__ sums, const float* __restrict__ bias_sums, int64_t n, int n_bias,
                                                          int splits, To* __restrict__ weight, To* __restrict__ bias) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x % 64, strand = threadIdx.x / 64;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float total = 0.0f;
    if (i < n + n_bias) {
        const float* const from = i < n ? sums + i : bias_sums + (i - n);
        const int64_t stride = i < n ? n : n_bias;
        for (int s = strand; s < splits; s += 16) total += from[s * stride];
    }
    lds[strand][lane] = total;
    __syncthreads();
    if (strand != 0 || i >= n + n_bias) return;
    for (int s = 1; s < 16; ++s) total += lds[s][lane];
    if (i < n) weight[i] = static_cast<To>(total);
    else bias[i - n] = static_cast<To>(total);
}

// How a product is cut up.  Tiles of 128 x 128 read each operand least often; where they would be half empty, or too few for the card even with the
// rows split, 64 columns a side.
struct WeightPlan {
    int wide_o, wide_c, waves, splits;
    int64_t split_rows;
    int output_tiles, channel_tiles;
};
WeightPlan weight_plan(int64_t rows, int64_t channels, int64_t outputs) {
    WeightPlan p{};
    const bool large = channels > 64 && outputs > 64;
    p.wide_o = p.wide_c = large ? 8 : 4;
    p.waves = large ? 4 : 8;
    p.output_tiles = static_cast<int>((outputs + 16 * p.wide_o - 1) / (16 * p.wide_o));
    p.channel_tiles = static_cast<int>((channels + 16 * p.wide_c - 1) / (16 * p.wide_c));
    const int64_t tiles = static_cast<int64_t>(p.output_tiles) * p.channel_tiles, at_a_time = p.waves * kStep;
    const int64_t pieces = std::max<int64_t>(1, (rows + at_a_time - 1) / at_a_time);
    const int64_t wanted = std::max<int64_t>(1, std::min(pieces, 512 / tiles));
    p.split_rows = (pieces + wanted - 1) / wanted * at_a_time;
    p.splits = static_cast<int>(std::max<int64_t>(1, (rows + p.split_rows - 1) / p.split_rows));
    return p;
}

bool bad_size(int64_t rows, int64_t channels, int64_t outputs) {
    return rows < 0 || channels <= 0 || channels > PENC_MAX_CHANNELS || outputs <= 0 || outputs > PENC_MAX_CHANNELS || channels * outputs >= int64_t{1} << 31;
}

template <class E, int kWideO, int kWideC, int kWaves>
void launch(const WeightGrad& a, unsigned grid, hipStream_t stream) {
    hipLaunchKernelGGL((weight_grad_kernel<E, kWideO, kWideC, kWaves>), dim3(grid), dim3(64 * kWaves), 0, stream, a);
}

}  // namespace
}  // namespace penc

using namespace penc;

extern "C" {

size_t penc_weight_grad_workspace_bytes(int64_t rows, int64_t channels, int64_t outputs) {
    if (bad_size(rows, channels, outputs)) return 0;
    return static_cast<size_t>(weight_plan(rows, channels, outputs).splits) * static_cast<size_t>(channels + 1) * static_cast<size_t>(outputs) * 4;
}

int penc_weight_grad(int type, int result_type, int64_t rows, int64_t channels, int64_t outputs, const int8_t* values, const uint8_t* exponents,
                     const void* grad, int64_t grad_row_stride, void* weight_grad, void* bias_grad, void* workspace, size_t workspace_bytes,
                     void* stream) {
    if (bad_size(rows, channels, outputs)) return PENC_ERR_BAD_LAYER_SIZE;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        return with_type(result_type, [&](auto r) -> int {
            using To = decltype(r);
            if ((rows > 0 && (!values || !exponents || !grad)) || !weight_grad || !workspace) return PENC_ERR_NULL_POINTER;
            if (!aligned_to(values, kKeptPitch) || !aligned_to(grad, sizeof(E)) || !aligned_to(weight_grad, sizeof(To)) || !aligned_to(bias_grad, sizeof(To)) ||
                !aligned_to(workspace, 16))
                return PENC_ERR_MISALIGNED;
            if (workspace_bytes < penc_weight_grad_workspace_bytes(rows, channels, outputs)) return PENC_ERR_WORKSPACE_TOO_SMALL;
            const WeightPlan p = weight_plan(rows, channels, outputs);
            float* const sums = static_cast<float*>(workspace);
            const int64_t n = channels * outputs;
            const WeightGrad a{rows, grad_row_stride, p.split_rows, static_cast<int>(channels), static_cast<int>(outputs), p.channel_tiles,
                               p.output_tiles, kept_array(values, exponents, channels), grad, sums, bias_grad ? sums + p.splits * n : nullptr};
            const int64_t grid = static_cast<int64_t>(p.splits) * p.output_tiles * p.channel_tiles;
            const int n_bias = bias_grad ? static_cast<int>(outputs) : 0;
            const int64_t sum_grid = (n + n_bias + 63) / 64;
            if (grid > 0x7FFFFFFF) return PENC_ERR_BAD_LAYER_SIZE;
            hipStream_t st = static_cast<hipStream_t>(stream);
            if (p.wide_o == 8) launch<E, 8, 8, 4>(a, static_cast<unsigned>(grid), st);
            else launch<E, 4, 4, 8>(a, static_cast<unsigned>(grid), st);
            if (const int rc = launched()) return rc;
            hipLaunchKernelGGL(sum_splits_kernel<To>, dim3(static_cast<unsigned>(sum_grid)), dim3(1024), 0, st, sums, a.bias_sums, n, n_bias, p.splits,
                               static_cast<To*>(weight_grad), static_cast<To*>(bias_grad));
            return launched();
        });
    });
}

}  // extern "C"
