// Nearly orthogonal matrices from updates, by Newton-Schulz products (K. Jordan et al., "Muon: an optimizer for hidden layers in neural networks", 2024):
//
//     X = G / (|G|_F + eps);    `steps` times:  S = X X^T (of a tall X: X^T X),  F = b S + c S S,  X = a X + F X (X F)
//
// takes every singular value s in 0 .. 1 through as many times a s + b s^3 + c s^5.  What is small in X is taken up by a factor a in each step, and so is
// what a rounding has added to it.  In 16 bits with 8 of them behind the point (bfloat16) the result would be off by 1e-2 of it, in float16 by 1.4e-3.  So X,
// S and F are kept
//
//     as two float16 values, hi + lo, three products for each: 0.7e-6 to 1.5e-6 of float32 results, which float32 products leave 0.9e-6 to 3.4e-6 off.
//         16-bit results are off by their own rounding and no more, 1.66e-3 in bfloat16
//     for bfloat16 results, where the caller asks for it (`halves`), as float16, one product for each, and F's diagonal, which is most of F, in float32:
//         1.8e-3 to 2.0e-3 (with the diagonal in float16 2.0e-3 to 2.4e-3) in a third of the time: 16 x 4096 x 1024 1517 us, as two values 4796
//
// times 2^12, so that what matters of lo is no subnormal number.  Of the steps above |X| <= 1.2, S <= 1.5 and F <= 3, which is under 2^14.  Coefficients are
// accepted up to |X| <= 3 and F <= 15: S 2^12 <= 36864 and F 2^12 <= 61440, where float16 ends at 65504 and roundings of X (2^-22, in halves 2^-11) add less
// than 2% to F. The matrix cores run float16 8 times as fast as float32, so that three products take 3/8 of the time.
//
// S and S S are symmetric: tiles on one side of the diagonal are computed and stored twice.  Matrices of up to 128 rows (or columns) that fit the LDS go
// through all of their steps there, one to a workgroup; thin ones in 64 bits, by their S alone.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "penc_product.hpp"

namespace penc {
namespace {

constexpr float kScale = 4096.0f, kPerScale = 1.0f / 4096.0f;

struct Coefficients {
    float a, b, c, eps;
};

// Where `column` of a stored row is.
template <class E>
__device__ __forceinline__ int column_at(int column) {
    if constexpr (std::is_same_v<E, split_t>) return column / 32 * 128 + column % 32 * 2;
    else return column * 2;
}
template <int kWide>
using halves = half_t __attribute__((ext_vector_type(kWide)));
template <int kWide>
using floats = float __attribute__((ext_vector_type(kWide)));

// What of v the second half holds.
template <int kWide>
__device__ __forceinline__ halves<kWide> rest_of(floats<kWide> v, halves<kWide> hi) {
    return __builtin_convertvector(v - __builtin_convertvector(hi, floats<kWide>), halves<kWide>);
}
template <class E>
__device__ __forceinline__ floats<8> load_stored(const char* row, int column) {
    const char* const p = row + column_at<E>(column);
    floats<8> v = __builtin_convertvector(*reinterpret_cast<const halves<8>*>(p), floats<8>);
    if constexpr (std::is_same_v<E, split_t>) v += __builtin_convertvector(*reinterpret_cast<const halves<8>*>(p + 64), floats<8>);
    return v;
}
template <class E>
__device__ __forceinline__ void store_stored(char* row, int column, floats<8> v) {
    char* const p = row + column_at<E>(column);
    const halves<8> hi = __builtin_convertvector(v, halves<8>);
    *reinterpret_cast<halves<8>*>(p) = hi;
    if constexpr (std::is_same_v<E, split_t>) *reinterpret_cast<halves<8>*>(p + 64) = rest_of<8>(v, hi);
}

// f v + w, rounded once.
template <class V>
__device__ __forceinline__ V weighted(float f, V v, V w) {
    constexpr int kWide = sizeof(V) / sizeof(float);
#pragma unroll
    for (int i = 0; i < kWide; ++i) w[i] = __builtin_fmaf(f, v[i], w[i]);
    return w;
}

// ------------------------------------------------------------------------------------------
// the norm, and X

constexpr int kThreads = 256;
constexpr int kMostPieces = 256;

// The sum of a workgroup's values; in 64 bits, so that squares of any fp32 values stay finite and above zero.
template <int kSum>
__device__ __forceinline__ double workgroup_sum(double v) {
    __shared__ double of_waves[kSum / 64];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    if (threadIdx.x % 64 == 0) of_waves[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kSum / 64; ++w) v += of_waves[w];
    return v;
}

// 2^12 / (|G|_F + eps): in 64 bits, whatever the norm
__device__ __forceinline__ double per_norm(double squares, float eps) { return static_cast<double>(kScale) / (sqrt(squares) + static_cast<double>(eps)); }
template <class G>
__device__ __forceinline__ float scaled(G g, double factor) { return static_cast<float>(static_cast<double>(static_cast<float>(g)) * factor); }

// 16 x 4096 x 1024 bf16 28 us, 4.8 TB/s.
template <class G>
__global__ __launch_bounds__(kThreads) void squares_kernel(int64_t values, int pieces, const G* __restrict__ g, double* __restrict__ sums) {
    constexpr int kWide = 16 / sizeof(G);
    using Unaligned = G __attribute__((ext_vector_type(kWide), aligned(sizeof(G))));
    const int64_t each = ((values + pieces - 1) / pieces + kWide - 1) / kWide * kWide, piece = blockIdx.x % pieces;
    const int64_t first = piece * each, last = min(first + each, values), whole = max(last - first, int64_t{0}) / kWide;
    const G* const from = g + blockIdx.x / pieces * values + first;
    double sum[kWide] = {};
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < whole; i += kThreads) {
        const Unaligned v = *reinterpret_cast<const Unaligned*>(from + i * kWide);
#pragma unroll
        for (int k = 0; k < kWide; ++k) sum[k] = __builtin_fma(static_cast<double>(static_cast<float>(v[k])), static_cast<double>(static_cast<float>(v[k])), sum[k]);
    }
    for (int64_t i = whole * kWide + threadIdx.x; i < last - first; i += kThreads) {
        const double v = static_cast<double>(static_cast<float>(from[i]));
        sum[0] += v * v;
    }
#pragma unroll
    for (int k = 1; k < kWide; ++k) sum[0] += sum[k];
    sum[0] = workgroup_sum<kThreads>(sum[0]);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum[0];
}

// X 2^12 as it is stored, zeros behind each row's end.  As one float16 (E = half_t) it is rounded to 11 bits, and each of the five steps takes that up again.
// So the first X is the update times a power of two, which of bfloat16 is no rounding, and what the norm has beside, 1 to 2, is left to the first step
// (`rest`, for each matrix): an error of 1.9e-3 to 2.2e-3 became 1.8e-3 to 2.0e-3.
template <class E, class G>
__global__ __launch_bounds__(kThreads) void stage_kernel(int rows, int columns, int padded, int pieces, const G* __restrict__ g, const double* __restrict__ sums,
                                                         float eps, char* __restrict__ x, float* __restrict__ rest, uint32_t blocks) {
    const int64_t matrix = blockIdx.x / blocks;
    const double* const mine = sums + matrix * pieces;
    double squares = 0.0;
    for (int i = static_cast<int>(threadIdx.x); i < pieces; i += kThreads) squares += mine[i];
    double factor = per_norm(workgroup_sum<kThreads>(squares), eps);
    if constexpr (std::is_same_v<E, half_t>) {
        // (of a norm that is not finite the factor is 0 or NaN: all of it is left then)
        const double power = factor > 0.0 ? ldexp(1.0, ilogb(factor)) : 1.0;
        if (blockIdx.x % blocks == 0 && threadIdx.x == 0) rest[matrix] = static_cast<float>(factor / power);
        factor = power;
    }
    const G* const from = g + matrix * rows * columns;
    const int64_t stride = static_cast<int64_t>(padded) * ProductType<E>::kBytes;
    char* const to = x + matrix * rows * stride;
    using Unaligned = G __attribute__((ext_vector_type(8), aligned(sizeof(G))));
    const uint32_t per_row = padded / 8, eights = static_cast<uint32_t>(rows) * per_row;  // (below 2^30: sides are at most 2^16)
    for (uint32_t i = blockIdx.x % blocks * kThreads + threadIdx.x; i < eights; i += blocks * kThreads) {
        const uint32_t row = i / per_row;
        const int column = static_cast<int>(i % per_row) * 8;
        const G* const p = from + static_cast<int64_t>(row) * columns + column;
        floats<8> v{};
        if (column + 8 <= columns) {
            const Unaligned u = *reinterpret_cast<const Unaligned*>(p);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = scaled(u[k], factor);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (column + k < columns) v[k] = scaled(p[k], factor);
        }
        store_stored<E>(to + row * stride, column, v);
    }
}

// ------------------------------------------------------------------------------------------
// a step

enum Stage { kGram, kSquare, kUpdate };

struct StepArgs {
    const char *x, *s, *f;  // as stored: [matrices][rows][padded], [matrices][small][small_padded]
    char* out;
    void* result;           // of the last step: [matrices][rows][columns]
    int rows, columns, padded, small, small_padded;
    Spread spread;
    uint32_t each, tiles_m;  // each: items of a matrix
    int splits;              // kGram: workgroups that share a tile's k, each of which leaves its sums in `partial`
    float* partial;
    float* diagonal;         // F's: [matrices][small_padded]
    const float* rest;       // the first step's, else null: what X is to be multiplied by
    float a, b, c;
};

__device__ __forceinline__ float rest_of_norm(const StepArgs& a, int64_t matrix) { return a.rest != nullptr ? a.rest[matrix] : 1.0f; }

// Pair `t` of tiles on and behind the diagonal: i <= j.
__device__ __forceinline__ void pair_of(uint32_t t, uint32_t& i, uint32_t& j) {
    j = static_cast<uint32_t>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
    while (j * (j + 1) / 2 > t) --j;
    while ((j + 1) * (j + 2) / 2 <= t) ++j;
    i = t - j * (j + 1) / 2;
}

// Where eight halves from m on stand in row n of a tile that is to be turned: neighbouring rows of eight lanes, and four rows of 32 bytes, meet no bank twice.
template <int kWideM>
__device__ __forceinline__ int turned_place(int n, int m) {
    constexpr int kChunks = kWideM / 8;
    return (m / 8 ^ (kChunks >= 8 ? (n & 3) << 1 | (n >> 2 & 1) : n >> 1 & 3)) * 16;
}

template <Stage kStage, bool kTall, class E, class Result, class P>
__global__ __launch_bounds__(P::kThreads) void step_kernel(StepArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    constexpr int kBytes = ProductType<E>::kBytes;
    const uint32_t of_launch = a.spread.item();
    if (of_launch >= a.spread.items) return;
    const uint32_t item = kStage == kGram ? of_launch / a.splits : of_launch, split = kStage == kGram ? of_launch % a.splits : 0, t = item % a.each;
    const int64_t matrix = item / a.each;
    const int64_t stride = static_cast<int64_t>(a.padded) * kBytes, small_stride = static_cast<int64_t>(a.small_padded) * kBytes;
    const char *const x = a.x + matrix * a.rows * stride, *const s = a.s + matrix * a.small * small_stride, *const f = a.f + matrix * a.small * small_stride;
    uint32_t i = t % a.tiles_m, j = t / a.tiles_m;
    if constexpr (kStage != kUpdate) pair_of(t, i, j);
    const int m0 = uniform(static_cast<int>(i)) * P::kM, n0 = uniform(static_cast<int>(j)) * P::kN;
    const auto rows_from = [&](const char* p, int64_t row_bytes, int rows, int first, int most) {
        return Operand{p + first * row_bytes, row_bytes, min(rows - first, most), static_cast<int>(row_bytes)};
    };
    const auto columns_from = [&](int first, int most) { return Operand{x + first * kBytes, stride, a.rows, min(a.padded - first, most) * kBytes}; };
    P p;
    if constexpr (kStage == kGram) {
        const int all = kTall ? a.rows : a.padded, each = ((all + P::kDepth - 1) / P::kDepth + a.splits - 1) / a.splits * P::kDepth;
        const int k0 = min(static_cast<int>(split) * each, all), depth = min(all - k0, each);
        Operand m = kTall ? columns_from(m0, P::kM) : rows_from(x, stride, a.rows, m0, P::kM);
        Operand n = kTall ? columns_from(n0, P::kN) : rows_from(x, stride, a.rows, n0, P::kN);
        m.first += k0 * (kTall ? stride : kBytes), n.first += k0 * (kTall ? stride : kBytes);
        if constexpr (kTall) m.rows = n.rows = depth;
        else m.bytes = n.bytes = depth * kBytes;
        p.run(lds, m, n, depth, P::kZero, P::kNothing);
        if (a.partial != nullptr) {
            float* const to = a.partial + static_cast<int64_t>(of_launch) * (P::kM * P::kN);
            p.each([&](int m, int n, tile_acc v) { *reinterpret_cast<tile_acc*>(to + n * P::kM + m) = v; });
            return;
        }
    }
    if constexpr (kStage == kSquare)
        p.run(lds, rows_from(s, small_stride, a.small, m0, P::kM), rows_from(s, small_stride, a.small, n0, P::kN), a.small_padded, P::kZero, P::kNothing);
    if constexpr (kStage == kUpdate && !kTall) p.run(lds, columns_from(m0, P::kM), rows_from(f, small_stride, a.small, n0, P::kN), a.small, P::kZero, P::kNothing);
    if constexpr (kStage == kUpdate && kTall)
        p.run(lds, rows_from(f, small_stride, a.small, m0, P::kM), rows_from(x, stride, a.rows, n0, P::kN), a.padded, P::kZero, P::kNothing);
    if constexpr (kStage != kUpdate) {
        char* const out = a.out + matrix * a.small * small_stride;
        constexpr int kWideM = P::kM / P::kWavesM, kWideN = P::kN / P::kWavesN, kParts = ProductType<E>::kParts;
        // The other side of the diagonal: a wave's results as halves in the LDS, rows of n, and read back by columns.
        static_assert(kParts * P::kThreads / 64 * kWideM * kWideN * 2 <= P::kLds);
        const float r = kStage == kGram ? rest_of_norm(a, matrix) : 1.0f, per_scale = kPerScale * r * r;
        char* const turned = lds + P::wave() * (kParts * kWideM * kWideN * 2);
        if (m0 != n0) __syncthreads();
        p.each_eight([&](int m, int n, floats<8> v) {
            const int lm = m - P::wave_m(), ln = n - P::wave_n();
            m += m0, n += n0;
            v *= per_scale;
            const bool there = n < a.small && m < a.small_padded;
            if constexpr (kStage == kSquare) v = weighted(a.b, there ? load_stored<E>(s + n * small_stride, m) : floats<8>{}, a.c * v);
            if (kStage == kSquare && m0 == n0) {
                float* const diagonal = a.diagonal + matrix * a.small_padded + n;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (m + k != n) continue;
                    if (n < a.small_padded) *diagonal = n < a.small ? v[k] * kPerScale : 0.0f;  // (zeros behind the end, as in X)
                    v[k] = 0.0f;
                }
            }
            if (there) store_stored<E>(out + n * small_stride, m, v);
            if (m0 == n0) return;
            const halves<8> hi = __builtin_convertvector(v, halves<8>);
            *reinterpret_cast<halves<8>*>(turned + ln * (kWideM * 2) + turned_place<kWideM>(ln, lm)) = hi;
            if constexpr (kParts == 2) *reinterpret_cast<halves<8>*>(turned + (kWideN + ln) * (kWideM * 2) + turned_place<kWideM>(ln, lm)) = rest_of<8>(v, hi);
        });
        if (m0 == n0) return;
        // lane 16 g + i: row m + i of the other side, eight columns from n + 8 g on
        const int lane = threadIdx.x % 64, g = lane / 16, l16 = lane % 16;
        using V = short __attribute__((ext_vector_type(4)));
        using Lds = __attribute__((address_space(3))) V;
#pragma unroll
        for (int m = 0; m < kWideM; m += 16)
#pragma unroll
            for (int n = 0; n < kWideN; n += 32)
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    uint2 w[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int ln = n + g * 8 + h * 4 + l16 / 4, lm = m + l16 % 4 * 4;
                        w[h] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                             (Lds*)(turned + (part * kWideN + ln) * (kWideM * 2) + turned_place<kWideM>(ln, lm & ~7) + lm % 8 * 2)));
                    }
                    const int row = m0 + P::wave_m() + m + l16, column = n0 + P::wave_n() + n + g * 8;
                    if (row < a.small && column < a.small_padded)
                        *reinterpret_cast<uint4*>(out + row * small_stride + column_at<E>(column) + part * 64) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
                }
    } else {
        char* const out = a.out + matrix * a.rows * stride;
        const float r = rest_of_norm(a, matrix), per_scale = kPerScale * r;
        const float* const diagonal = a.diagonal + matrix * a.small_padded;
        Result* const result = static_cast<Result*>(a.result) + matrix * a.rows * a.columns;
        using Eight = Result __attribute__((ext_vector_type(8)));
        p.each_eight([&](int m, int n, floats<8> v) {
            m += m0, n += n0;
            if (n >= a.rows || m >= a.padded) return;
            const floats<8> from = load_stored<E>(x + n * stride, m);
            v *= per_scale;
            if constexpr (kTall) {
                const floats<8> keep = (*reinterpret_cast<const floats<8>*>(diagonal + m) + a.a) * r;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = __builtin_fmaf(keep[k], from[k], v[k]);
            } else {
                v = weighted((diagonal[n] + a.a) * r, from, v);
            }
            if (a.result == nullptr) store_stored<E>(out + n * stride, m, v);
            else if (m < a.columns)
                store_values<Result, 8>(result + static_cast<int64_t>(n) * a.columns + m, __builtin_convertvector(v * kPerScale, Eight), a.columns - m);
        });
    }
}

constexpr int kSumSide = 64, kSumThreads = 512;

// S from the sums of the workgroups that shared its tiles, of 64 x 64, in their order, and the other side of the diagonal.
template <class E>
__global__ __launch_bounds__(kSumThreads) void gram_sum_kernel(StepArgs a) {
    __shared__ float lds[kSumSide][kSumSide + 1];
    const uint32_t t = blockIdx.x % a.each;
    const int64_t matrix = blockIdx.x / a.each, stride = static_cast<int64_t>(a.small_padded) * ProductType<E>::kBytes;
    uint32_t i, j;
    pair_of(t, i, j);
    char* const out = a.out + matrix * a.small * stride;
    const float* const from = a.partial + static_cast<int64_t>(blockIdx.x) * a.splits * (kSumSide * kSumSide);
    const int m0 = static_cast<int>(i) * kSumSide, n0 = static_cast<int>(j) * kSumSide;
    const float r = rest_of_norm(a, matrix), per_scale = kPerScale * r * r;
    for (int at = static_cast<int>(threadIdx.x) * 8; at < kSumSide * kSumSide; at += kSumThreads * 8) {
        floats<8> v{};
#pragma unroll 8
        for (int k = 0; k < a.splits; ++k) v += *reinterpret_cast<const floats<8>*>(from + k * (kSumSide * kSumSide) + at);
        v *= per_scale;
        const int n = at / kSumSide, m = at % kSumSide;
#pragma unroll
        for (int k = 0; k < 8; ++k) lds[m + k][n] = v[k];
        if (n0 + n < a.small && m0 + m < a.small_padded) store_stored<E>(out + (n0 + n) * stride, m0 + m, v);
    }
    if (i == j) return;
    __syncthreads();
    for (int at = static_cast<int>(threadIdx.x) * 8; at < kSumSide * kSumSide; at += kSumThreads * 8) {
        const int m = at / kSumSide, n = at % kSumSide;
        floats<8> v;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = lds[m][n + k];
        if (m0 + m < a.small && n0 + n < a.small_padded) store_stored<E>(out + (m0 + m) * stride, n0 + n, v);
    }
}

// ------------------------------------------------------------------------------------------
// matrices that stay in the LDS

constexpr int kResidentThreads = 512, kResidentWaves = kResidentThreads / 64;
constexpr int kMostSmall = 128;
constexpr int kSliceBytes = 8192;  // for sums of S that waves share (matrices of up to 32 rows)
constexpr int kMostResident = 160 * 1024 - 256;  // bytes of the LDS

// A matrix of Split numbers in the LDS.  Chunks of a row's 128 bytes are permuted by the row, so that neither 8 rows of one chunk nor 4 rows of two chunks
// meet in a bank.
struct Resident {
    char* first;
    int pitch;

    __device__ __forceinline__ char* chunk(int row, int byte) const {
        return first + row * pitch + (byte & ~127) + ((byte >> 4 & 7) ^ ((row & 3) << 1 | (row >> 2 & 1))) * 16 + (byte & 15);
    }
    // 16 rows from `row` on, 32 k from 32 `line` on
    __device__ __forceinline__ chunk16 across(int row, int line, int q) const {
        const int lane = threadIdx.x % 64;
        return *reinterpret_cast<const chunk16*>(chunk(row + lane % 16, line * 128 + q * 64 + lane / 16 * 16));
    }
    // 16 columns from `column` on, 32 k (rows) from `row` on
    __device__ __forceinline__ chunk16 along(int row, int column, int q) const {
        const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
        using V = short __attribute__((ext_vector_type(4)));
        using Lds = __attribute__((address_space(3))) V;
        chunk16 f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const V v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)chunk(row + g * 8 + h * 4 + i / 4, column_at<split_t>(column) + q * 64 + i % 4 * 8));
            const uint2 w = __builtin_bit_cast(uint2, v);
            f[2 * h] = w.x, f[2 * h + 1] = w.y;
        }
        return f;
    }
    template <int kWide>
    __device__ __forceinline__ void store(int row, int column, floats<kWide> v) const {
        const int byte = column_at<split_t>(column);
        const halves<kWide> hi = __builtin_convertvector(v, halves<kWide>);
        *reinterpret_cast<halves<kWide>*>(chunk(row, byte)) = hi;
        *reinterpret_cast<halves<kWide>*>(chunk(row, byte + 64)) = rest_of<kWide>(v, hi);
    }
};

// (the products with a lo have sums of their own: see Product::low.  kAll: with lo lo: of 18 x 1104 fp32 1.4e-6 of error became 1.15e-6
// (float32's own 1.0e-6); of 256 x 64, where it is 1.1e-6 (1.2e-6) without, all of it would take 36 us and not 33)
template <bool kAll>
__device__ __forceinline__ void multiply_split(chunk16 a, chunk16 a_low, chunk16 b, chunk16 b_low, tile_acc& high, tile_acc& low) {
    if constexpr (kAll) low = multiply<half_t>(a_low, b_low, low);
    low = multiply<half_t>(a, b_low, low);
    low = multiply<half_t>(a_low, b, low);
    high = multiply<half_t>(a, b, high);
}

__host__ __device__ constexpr int resident_pitch(int padded) { return padded * 4; }
__host__ __device__ constexpr int round_to_32(int n) { return (n + 31) / 32 * 32; }

// One matrix to a workgroup, X as `small` rows (at most 16 kTiles) of `large` numbers whichever way it lies in memory.  A wave has 16 x 32 results of S and
// of F, and up to kBlocks times 16 columns of X, which are its own: in fp32 in its registers, for a X, and as operands in the LDS, which it overwrites when
// it has read them.
template <class G, int kTiles, int kBlocks>
__global__ __launch_bounds__(kResidentThreads) void resident_kernel(int rows, int columns, int steps, Coefficients k, const G* __restrict__ g, G* __restrict__ result) {
    __shared__ __attribute__((aligned(1024))) char lds[kMostResident];
    constexpr int kPadded = 16 * kTiles, kLines = kPadded / 32, kTogether = kBlocks > 1 && kTiles <= 4 ? 2 : 1;
    constexpr bool kAll = std::is_same_v<G, float> && kTiles <= 2;
    constexpr int kUnroll = kTiles <= 4 ? kLines : 1;  // (more would not fit the registers)
    const bool tall = rows > columns;
    const int small = min(rows, columns), large = max(rows, columns), large_padded = (large + 63) / 64 * 64;
    const Resident x{lds, resident_pitch(large_padded)}, s{lds + kPadded * x.pitch, resident_pitch(kPadded)};
    const int64_t values = static_cast<int64_t>(rows) * columns;
    const G* const from = g + blockIdx.x * values;
    // (where number `column` of row `row` is in memory)
    const int row_step = tall ? 1 : columns, column_step = tall ? columns : 1;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), q4 = lane / 16 * 4, l16 = lane % 16;
    // The matrix from memory: eight numbers of a row to a lane, neighbouring lanes neighbours in memory.  (What a wave has as results is read a second time,
    // below, from the cache.)
    constexpr int kEights = (kMostResident / 4 / 8 + kResidentThreads - 1) / kResidentThreads;
    const int eights = large_padded / 8, all = kPadded * eights;
    floats<8> read[kEights];
#pragma unroll
    for (int e = 0; e < kEights; ++e) {
        read[e] = floats<8>{};
        const int i = e * kResidentThreads + static_cast<int>(threadIdx.x);
        if (e * kResidentThreads >= all) continue;
        const int row = tall ? i % kPadded : i / eights, column = (tall ? i / kPadded : i % eights) * 8;
        const G* const p = from + row * row_step + column * column_step;
        if (row < small && !tall && column + 8 <= large) {
            using Unaligned = G __attribute__((ext_vector_type(8), aligned(sizeof(G))));
            read[e] = __builtin_convertvector(*reinterpret_cast<const Unaligned*>(p), floats<8>);
        } else {
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (row < small && column + n < large) read[e][n] = static_cast<float>(p[n * column_step]);
        }
    }
    double squares = 0.0;
#pragma unroll
    for (int e = 0; e < kEights; ++e)
#pragma unroll
        for (int n = 0; n < 8; ++n) squares = __builtin_fma(static_cast<double>(read[e][n]), static_cast<double>(read[e][n]), squares);
    const double factor = per_norm(workgroup_sum<kResidentThreads>(squares), k.eps);
#pragma unroll
    for (int e = 0; e < kEights; ++e) {
        const int i = e * kResidentThreads + static_cast<int>(threadIdx.x);
        if (i >= all) continue;
        floats<8> v;
#pragma unroll
        for (int n = 0; n < 8; ++n) v[n] = scaled(read[e][n], factor);
        x.store<8>(tall ? i % kPadded : i / eights, (tall ? i / kPadded : i % eights) * 8, v);
    }
    // What this wave has of X as results.
    floats<4> own[kBlocks][kTiles];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const int row = n * 16 + l16, column = (b * kResidentWaves + wave) * 16 + q4;
            own[b][n] = floats<4>{};
            if ((b * kResidentWaves + wave) * 16 >= large) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row < small && column + i < large) own[b][n][i] = scaled(from[row * row_step + (column + i) * column_step], factor);
        }
    __syncthreads();
    constexpr int kUnits = kTiles * kTiles / 2, kMostUnits = (kUnits + kResidentWaves - 1) / kResidentWaves;
    // Of 32 rows there are two units of S: four waves share the k of each, and what three of them have is added by way of the LDS.  Sums of a quarter of the
    // length round less, too.
    constexpr int kSlices = kUnits < kResidentWaves ? kResidentWaves / kUnits : 1;
    static_assert(kSlices == 1 || (kSlices == 4 && kSliceBytes == 2 * kUnits * 2 * 64 * 16));
    for (int step = 0; step < steps; ++step) {
        tile_acc of_s[kMostUnits][2];
        if constexpr (kSlices > 1) {
            const int unit = wave % kUnits, slice = wave / kUnits, m = unit % kTiles * 16, n = unit / kTiles * 32, pairs = large_padded / 64;
            tile_acc high[2] = {}, low[2] = {};
            for (int first = slice * pairs / kSlices * 2; first < (slice + 1) * pairs / kSlices * 2; first += 2) {
#pragma unroll
                for (int line = first; line < first + 2; ++line) {
                    const chunk16 a = x.across(m, line, 0), a_low = x.across(m, line, 1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) multiply_split<kAll>(a, a_low, x.across(n + 16 * h, line, 0), x.across(n + 16 * h, line, 1), high[h], low[h]);
                }
            }
            // slices 2 and 3 to 0 and 1, and 1 to 0
            tile_acc* const left = reinterpret_cast<tile_acc*>(s.first + kPadded * s.pitch) + (slice % 2 * kUnits + unit) * 128 + lane;
#pragma unroll
            for (int h = 0; h < 2; ++h) of_s[0][h] = high[h] + low[h];
#pragma unroll
            for (int most = kSlices; most > 1; most /= 2) {
                if (slice >= most / 2 && slice < most) left[0] = of_s[0][0], left[64] = of_s[0][1];
                __syncthreads();
                const tile_acc* const right = most == 2 ? left + kUnits * 128 : left;
                if (slice < most / 2) of_s[0][0] += right[0], of_s[0][1] += right[64];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                of_s[0][h] *= kPerScale;
                if (slice == 0) s.store<4>(n + 16 * h + l16, m + q4, of_s[0][h]);
            }
        }
#pragma unroll
        for (int u = 0; u < (kSlices > 1 ? 0 : kMostUnits); ++u) {
            const int unit = u * kResidentWaves + wave, m = unit % kTiles * 16, n = unit / kTiles * 32;
            if (unit >= kUnits) continue;
            tile_acc high[2] = {}, low[2] = {};
            for (int first = 0; first < large_padded / 32; first += 2) {
#pragma unroll
                for (int line = first; line < first + 2; ++line) {
                    const chunk16 a = x.across(m, line, 0), a_low = x.across(m, line, 1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) multiply_split<kAll>(a, a_low, x.across(n + 16 * h, line, 0), x.across(n + 16 * h, line, 1), high[h], low[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                of_s[u][h] = (high[h] + low[h]) * kPerScale;
                s.store<4>(n + 16 * h + l16, m + q4, of_s[u][h]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMostUnits; ++u) {
            const int unit = u * kResidentWaves + wave, m = unit % kTiles * 16, n = unit / kTiles * 32;
            if (unit >= kUnits) continue;
            tile_acc high[2] = {}, low[2] = {};
#pragma unroll kUnroll
            for (int line = 0; line < kLines; ++line) {
                const chunk16 a = s.across(m, line, 0), a_low = s.across(m, line, 1);
#pragma unroll
                for (int h = 0; h < 2; ++h) multiply_split<kAll>(a, a_low, s.across(n + 16 * h, line, 0), s.across(n + 16 * h, line, 1), high[h], low[h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) of_s[u][h] = weighted(k.c * kPerScale, high[h], weighted(k.b, of_s[u][h], (k.c * kPerScale) * low[h]));
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMostUnits; ++u) {
            const int unit = u * kResidentWaves + wave, m = unit % kTiles * 16, n = unit / kTiles * 32;
            if (unit >= kUnits) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) s.store<4>(n + 16 * h + l16, m + q4, of_s[u][h]);
        }
        __syncthreads();
        const bool last = step + 1 == steps;
        // (two blocks of columns at a time: each fragment of F is read once for both)
#pragma unroll
        for (int b = 0; b < kBlocks; b += kTogether) {
            if ((b * kResidentWaves + wave) * 16 >= large_padded) continue;
            tile_acc high[kTogether][kTiles] = {}, low[kTogether][kTiles] = {};
#pragma unroll kUnroll
            for (int line = 0; line < kLines; ++line) {
                chunk16 a[kTogether][2];
#pragma unroll
                for (int t = 0; t < kTogether; ++t) {
                    // (where there is no second block: the first one's, for results that are not taken)
                    const int m = ((b + t) * kResidentWaves + wave) * 16, at = m < large_padded ? m : (b * kResidentWaves + wave) * 16;
                    a[t][0] = x.along(line * 32, at, 0), a[t][1] = x.along(line * 32, at, 1);
                }
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    const chunk16 f = s.across(n * 16, line, 0), f_low = s.across(n * 16, line, 1);
#pragma unroll
                    for (int t = 0; t < kTogether; ++t) multiply_split<kAll>(a[t][0], a[t][1], f, f_low, high[t][n], low[t][n]);
                }
            }
#pragma unroll
            for (int t = 0; t < kTogether; ++t) {
                const int m = ((b + t) * kResidentWaves + wave) * 16;
                if (b + t >= kBlocks || m >= large_padded) continue;
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    own[b + t][n] = weighted(k.a, own[b + t][n], (high[t][n] + low[t][n]) * kPerScale);
                    if (!last) x.store<4>(n * 16 + l16, m + q4, own[b + t][n]);
                }
            }
        }
        __syncthreads();
    }
    G* const to = result + blockIdx.x * values;
    using Four = G __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const int row = n * 16 + l16, column = (b * kResidentWaves + wave) * 16 + q4;
            const Four y = __builtin_convertvector(own[b][n] * kPerScale, Four);
            if (row >= small || column >= large) continue;
            if (!tall) {
                store_values<G, 4>(to + row * columns + column, y, large - column);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (column + i < large) to[(column + i) * columns + row] = y[i];
            }
        }
}

// ------------------------------------------------------------------------------------------
// thin matrices

constexpr int kThin = 64, kThinThreads = 256, kThinChunk = 64;  // rows; numbers of the long side at a time
constexpr int kMostThinPieces = 64;
constexpr double kMostThinGrowth = 1 << 27;  // of 2^-53
using four_doubles = double __attribute__((ext_vector_type(4)));

// Matrices of up to 64 rows (or columns) that are long, or too long for the LDS.  X stays what it is multiplied by from the left: X = Q G / (|G| + eps) with
// Q = P P' .., P = a + b S + c S S and S' = P S P, all of them small, so that G is read once for S and once for the result.  S is off by 2^-53 of its largest
// value, and what is small in it is taken up by a^2 in each step: in 64 bits five steps make 2^-35 of it (in 32 it would be 2^-6).

// 64 numbers of the long side from m0 on, for each of the small side's: x[small][64], zeros behind the end.
template <class G, int kRows>
__device__ __forceinline__ void load_thin(float (&x)[kRows][kThinChunk + 1], const G* __restrict__ g, int small, int large, bool tall, int m0) {
    const int there = min(large - m0, kThinChunk);
    if (tall) {
        const G* const from = g + static_cast<int64_t>(m0) * small;
        for (int i = static_cast<int>(threadIdx.x); i < kThinChunk * small; i += kThinThreads)
            x[i % small][i / small] = i < there * small ? static_cast<float>(from[i]) : 0.0f;
    } else {
        for (int i = static_cast<int>(threadIdx.x); i < kThinChunk * small; i += kThinThreads) {
            const int j = i / kThinChunk, m = i % kThinChunk;
            x[j][m] = m < there ? static_cast<float>(g[static_cast<int64_t>(j) * large + m0 + m]) : 0.0f;
        }
    }
}
template <int kRows>
__device__ __forceinline__ void clear_rows_behind(float (&x)[kRows][kThinChunk + 1], int small) {
    for (int i = small * kThinChunk + static_cast<int>(threadIdx.x); i < kRows * kThinChunk; i += kThinThreads) x[i / kThinChunk][i % kThinChunk] = 0.0f;
}

// Where result r of a lane is in a tile of 16 x 16: v_mfma_f64_16x16x4_f64 takes row (column) lane % 16 of k lane / 16.
__device__ __forceinline__ int thin_row(int r) { return 4 * r + static_cast<int>(threadIdx.x) % 64 / 16; }

// The tiles of 16 x 16 on and behind the diagonal, of 16 kTiles rows: waves have every fourth.  All that is multiplied here is symmetric: polynomials of one S.
template <int kTiles>
struct ThinTiles {
    static constexpr int kRows = 16 * kTiles, kUnits = kTiles * (kTiles + 1) / 2, kEach = (kUnits + 3) / 4;
    int i[kEach], j[kEach];
    bool there[kEach];
    __device__ __forceinline__ ThinTiles() {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            int unit = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) + 4 * e, row = 0;
            there[e] = unit < kUnits;
            if (!there[e]) unit = 0;
            while (unit >= kTiles - row) unit -= kTiles - row, ++row;
            i[e] = row * 16, j[e] = (row + unit) * 16;
        }
    }
};

// G G^T of a piece of the long side, each wave's tiles as its registers have them; of one tile each wave has a quarter of the numbers.
template <class G, int kTiles>
__global__ __launch_bounds__(kThinThreads) void thin_gram_kernel(int small, int large, bool tall, int pieces, const G* __restrict__ g, four_doubles* __restrict__ sums) {
    using Tiles = ThinTiles<kTiles>;
    __shared__ float x[16 * kTiles][kThinChunk + 1];
    const int64_t matrix = blockIdx.x / pieces;
    const int l16 = threadIdx.x % 16, q = threadIdx.x % 64 / 16, quarter = kTiles == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * (kThinChunk / 4) : 0;
    const int chunks = (large + kThinChunk - 1) / kThinChunk, piece = static_cast<int>(blockIdx.x % pieces);
    const Tiles tiles;
    g += matrix * small * large;
    clear_rows_behind(x, small);
    four_doubles sum[Tiles::kEach] = {};
    for (int c = piece * chunks / pieces; c < (piece + 1) * chunks / pieces; ++c) {
        load_thin(x, g, small, large, tall, c * kThinChunk);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < (kTiles == 1 ? kThinChunk / 4 : kThinChunk); k += 4) {
#pragma unroll
            for (int e = 0; e < Tiles::kEach; ++e) {
                const int at = quarter + k + q;
                sum[e] = __builtin_amdgcn_mfma_f64_16x16x4f64(static_cast<double>(x[tiles.i[e] + l16][at]),
                    static_cast<double>(x[tiles.j[e] + l16][at]), sum[e], 0, 0, 0);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < Tiles::kEach; ++e) sums[(static_cast<int64_t>(blockIdx.x) * Tiles::kEach + e) * kThinThreads + threadIdx.x] = sum[e];
}

// Q / (|G| + eps) of a matrix.
template <int kTiles>
__global__ __launch_bounds__(kThinThreads) void thin_steps_kernel(int small, int pieces, int steps, Coefficients k,
    const four_doubles* __restrict__ sums, double* __restrict__ result) {
    using Tiles = ThinTiles<kTiles>;
    constexpr int kRows = Tiles::kRows, kEach = Tiles::kEach;
    constexpr int kPitch = kRows + 1;  // (16 rows, or 16 numbers of one, meet no bank twice; kRows + 4, so that 16 rows of 4 do not, is 10 to 20% slower)
    __shared__ double s[kRows][kPitch], p[kRows][kPitch], q[kRows][kPitch], v[kRows][kPitch];
    const int l16 = threadIdx.x % 16, q4 = threadIdx.x % 64 / 16, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const Tiles tiles;
    using Matrix = double[kRows][kPitch];
    const auto product = [&](int e, const Matrix& a, const Matrix& b) {
        four_doubles sum{};
#pragma unroll
        for (int n = 0; n < kRows; n += 4) sum = __builtin_amdgcn_mfma_f64_16x16x4f64(a[tiles.i[e] + l16][n + q4], b[n + q4][tiles.j[e] + l16], sum, 0, 0, 0);
        return sum;
    };
    const auto store = [&](int e, Matrix& to, four_doubles x) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            to[tiles.i[e] + thin_row(r)][tiles.j[e] + l16] = x[r];
            if (tiles.i[e] != tiles.j[e]) to[tiles.j[e] + l16][tiles.i[e] + thin_row(r)] = x[r];
        }
    };
    const auto own = [&](int e, const Matrix& from) {
        four_doubles x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = from[tiles.i[e] + thin_row(r)][tiles.j[e] + l16];
        return x;
    };
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const four_doubles* const from = sums + (static_cast<int64_t>(blockIdx.x) * pieces * kEach + e) * kThinThreads + threadIdx.x;
        four_doubles sum{};
#pragma unroll 8
        for (int n = 0; n < pieces; ++n) sum += from[n * (kEach * kThinThreads)];
        if constexpr (kTiles > 1) {
            if (tiles.there[e]) store(e, s, sum);
        } else {
            // (the four waves' quarters, in order)
            if (wave == 0) store(e, s, sum);
            if (wave == 1) store(e, p, sum);
            if (wave == 2) store(e, q, sum);
            if (wave == 3) store(e, v, sum);
            __syncthreads();
            if (wave == 0) store(e, s, (sum + own(e, p)) + (own(e, q) + own(e, v)));
        }
    }
    __syncthreads();
    double squares = 0.0;
    for (int i = 0; i < small; ++i) squares += s[i][i];
    const double factor = 1.0 / (sqrt(squares) + static_cast<double>(k.eps));
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (tiles.there[e]) store(e, s, own(e, s) * (factor * factor));
    for (int step = 0; step < steps; ++step) {
        const bool last = step + 1 == steps;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (!tiles.there[e]) continue;
            four_doubles x = product(e, s, s) * static_cast<double>(k.c) + own(e, s) * static_cast<double>(k.b);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] += tiles.i[e] + thin_row(r) == tiles.j[e] + l16 ? static_cast<double>(k.a) : 0.0;
            store(e, p, x);
        }
        __syncthreads();
        four_doubles next[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (!tiles.there[e]) continue;
            next[e] = step > 0 ? product(e, q, p) : own(e, p);
            if (!last) store(e, v, product(e, p, s));
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (!tiles.there[e]) continue;
            store(e, q, next[e]);
            if (!last) store(e, s, product(e, v, p));
        }
    }
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < kRows * kRows; i += kThinThreads)
        result[static_cast<int64_t>(blockIdx.x) * kRows * kRows + i] = q[i / kRows][i % kRows] * factor;
}

// Q G: a workgroup takes 64 numbers of the long side at a time.
template <class G, int kTiles>
__global__ __launch_bounds__(kThinThreads) void thin_apply_kernel(int small, int large, bool tall, int blocks, const double* __restrict__ factors,
    const G* __restrict__ g,
                                                                  G* __restrict__ result) {
    constexpr int kRows = 16 * kTiles;
    __shared__ float x[kRows][kThinChunk + 1];
    const int64_t matrix = blockIdx.x / blocks;
    const int lane = threadIdx.x % 64, l16 = lane % 16, q4 = lane / 16, m = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 16 + l16;
    g += matrix * small * large, result += matrix * small * large;
    double q[kTiles][kRows / 4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int n = 0; n < kRows / 4; ++n) q[t][n] = factors[matrix * kRows * kRows + (t * 16 + l16) * kRows + n * 4 + q4];
    clear_rows_behind(x, small);
    for (int m0 = static_cast<int>(blockIdx.x % blocks) * kThinChunk; m0 < large; m0 += blocks * kThinChunk) {
        load_thin(x, g, small, large, tall, m0);
        __syncthreads();
        four_doubles sum[kTiles] = {};
#pragma unroll
        for (int n = 0; n < kRows / 4; ++n) {
            const double b = static_cast<double>(x[n * 4 + q4][m]);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) sum[t] = __builtin_amdgcn_mfma_f64_16x16x4f64(q[t][n], b, sum[t], 0, 0, 0);
        }
        // (a wave's columns are its own: it has read them; rows behind the last stay zeros)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (t * 16 + thin_row(r) < small) x[t * 16 + thin_row(r)][m] = static_cast<float>(sum[t][r]);
        __syncthreads();
        const int there = min(large - m0, kThinChunk);
        if (tall) {
            G* const to = result + static_cast<int64_t>(m0) * small;
            for (int i = static_cast<int>(threadIdx.x); i < there * small; i += kThinThreads) to[i] = static_cast<G>(x[i % small][i / small]);
        } else {
            for (int i = static_cast<int>(threadIdx.x); i < kThinChunk * small; i += kThinThreads)
                if (i % kThinChunk < there)
                    result[static_cast<int64_t>(i / kThinChunk) * large + m0 + i % kThinChunk] = static_cast<G>(x[i / kThinChunk][i % kThinChunk]);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------
// the optimiser's own part: a pass over memory before the products and one behind them

// m += (1 - momentum) (g - m), and the update g + momentum (m - g) or m itself
template <class G>
__global__ __launch_bounds__(kThreads) void momentum_kernel(int64_t n, const G* __restrict__ grad, float* __restrict__ average, float momentum, bool nesterov,
                                                            G* __restrict__ update) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const float g = static_cast<float>(grad[i]), m = average[i] + (1.0f - momentum) * (g - average[i]);
        average[i] = m;
        update[i] = static_cast<G>(nesterov ? g + momentum * (m - g) : m);
    }
}

// p = decay p - rate o
template <class G>
__global__ __launch_bounds__(kThreads) void apply_kernel(int64_t n, G* __restrict__ params, const G* __restrict__ orthogonal, float decay, float rate) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kThreads)
        params[i] = static_cast<G>(decay * static_cast<float>(params[i]) - rate * static_cast<float>(orthogonal[i]));
}

unsigned grid_of(int64_t n) { return static_cast<unsigned>(std::min<int64_t>((n + kThreads - 1) / kThreads, 8192)); }

// ------------------------------------------------------------------------------------------
// which kernels

// How many times 16 columns of X a wave may have, for 16 kTiles rows: what fits the LDS.
template <int kTiles>
constexpr int kMostBlocks = ((kMostResident / (16 * kTiles) - 16 * kTiles * 4) / 256 * 4 + kResidentWaves - 1) / kResidentWaves;

bool is_resident(int64_t rows, int64_t columns) {
    const int64_t small = std::min(rows, columns), large = std::max(rows, columns);
    if (small > kMostSmall || large > 1 << 12) return false;
    const int s = round_to_32(static_cast<int>(small)), l = (static_cast<int>(large) + 63) / 64 * 64;
    return static_cast<int64_t>(s) * (resident_pitch(l) + resident_pitch(s)) + (s <= 32 ? kSliceBytes : 0) <= kMostResident;
}

template <class G>
int resident(int64_t matrices, int64_t rows, int64_t columns, int steps, Coefficients k, const G* g, G* result, hipStream_t stream) {
    const auto launch = [&](auto tiles) -> int {
        constexpr int kTiles = decltype(tiles)::value;
        resident_kernel<G, kTiles, kMostBlocks<kTiles>><<<static_cast<unsigned>(matrices), kResidentThreads, 0, stream>>>(
            static_cast<int>(rows), static_cast<int>(columns), steps,
                                                                                                                          k, g, result);
        return launched();
    };
    const int64_t small = std::min(rows, columns);
    if (small <= 32) return launch(std::integral_constant<int, 2>{});
    if (small <= 64) return launch(std::integral_constant<int, 4>{});
    if (small <= 96) return launch(std::integral_constant<int, 6>{});
    return launch(std::integral_constant<int, 8>{});
}

// Three launches against a chain of them, or against one workgroup that has a matrix to itself (us, fp32, so and otherwise): 14 x 2048 x 6 15 and 121, 1 x 32
// x 4096 25 and 120, 8 x 64 x 4096 81 and 125; 1 x 18 x 1104 23 and 50, 1 x 16 x 128 12 and 16, 1 x 18 x 300 21 and 22, 1 x 48 x 400 45 and 50, 1 x 64 x 400
// 67 and 53; 64 x 32 x 1100 44 and 53, 256 of them 83 and 56.
bool is_thin(int64_t matrices, int64_t rows, int64_t columns) {
    const int64_t small = std::min(rows, columns);
    return small <= kThin && (!is_resident(rows, columns) || (matrices <= 64 && small <= 48 && std::max(rows, columns) >= (small <= 16 ? 128 : small <= 32 ? 300 : 350)));
}
int thin_pieces(int64_t matrices, int64_t large) {
    return static_cast<int>(std::max<int64_t>(1, std::min({(large + 4 * kThinChunk - 1) / (4 * kThinChunk), int64_t{kMostThinPieces}, (int64_t{1} << 22) / matrices})));
}
int thin_tiles(int64_t rows, int64_t columns) { return static_cast<int>((std::min(rows, columns) + 15) / 16); }
size_t thin_workspace(int64_t matrices, int64_t rows, int64_t columns) {
    const int tiles = thin_tiles(rows, columns);
    const size_t of_piece = static_cast<size_t>((tiles * (tiles + 1) / 2 + 3) / 4) * (kThinThreads * sizeof(four_doubles));
    return static_cast<size_t>(matrices) * (thin_pieces(matrices, std::max(rows, columns)) * of_piece +
                                            256 * tiles * tiles * sizeof(double));
}
template <class G>
int thin(int64_t matrices, int64_t rows, int64_t columns, int steps, Coefficients k, const G* g, G* result, char* workspace, hipStream_t stream) {
    const bool tall = rows > columns;
    const int small = static_cast<int>(std::min(rows, columns)), large = static_cast<int>(std::max(rows, columns)),
        pieces = thin_pieces(matrices, large), tiles = thin_tiles(rows, columns);
    double* const factors = reinterpret_cast<double*>(workspace);
    four_doubles* const sums = reinterpret_cast<four_doubles*>(factors + matrices * 256 * tiles * tiles);
    const int blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((large + kThinChunk - 1) / kThinChunk, (int64_t{1} << 22) / matrices)));
    const auto launch = [&](auto tiles) -> int {
        constexpr int kTiles = decltype(tiles)::value;
        thin_gram_kernel<G, kTiles><<<static_cast<unsigned>(matrices * pieces), kThinThreads, 0, stream>>>(small, large, tall, pieces, g, sums);
        if (const int rc = launched()) return rc;
        thin_steps_kernel<kTiles><<<static_cast<unsigned>(matrices), kThinThreads, 0, stream>>>(small, pieces, steps, k, sums, factors);
        if (const int rc = launched()) return rc;
        thin_apply_kernel<G, kTiles><<<static_cast<unsigned>(matrices * blocks), kThinThreads, 0, stream>>>(small, large, tall, blocks, factors, g, result);
        return launched();
    };
    if (tiles == 1) return launch(std::integral_constant<int, 1>{});
    if (tiles == 2) return launch(std::integral_constant<int, 2>{});
    if (tiles == 3) return launch(std::integral_constant<int, 3>{});
    return launch(std::integral_constant<int, 4>{});
}

// Whether a launch takes tiles of 64 x 64: where there would not be a workgroup of 128 x 128 for each compute unit.
bool small_tiles(int64_t matrices, int64_t side_m, int64_t side_n, bool half) {
    return matrices * ((side_m + 127) / 128) * ((side_n + 127) / 128) / (half ? 2 : 1) < 256;
}
int64_t pairs_of(int64_t small, int side) {
    const int64_t tiles = (small + side - 1) / side;
    return tiles * (tiles + 1) / 2;
}
// How many workgroups share the k of a tile of S: up to one for each compute unit, each with two steps at least (1000 x 203 fp16: 14 us without, 4 and 3 for
// the sums).
int gram_splits(int64_t matrices, int64_t small, int64_t depth, int step) {
    const int64_t items = matrices * pairs_of(small, kSumSide);
    if (!small_tiles(matrices, small, small, true) || items > 64) return 1;
    return static_cast<int>(std::max<int64_t>(1, std::min({256 / items, depth / (2 * step), int64_t{16}})));
}

// The workspace of matrices that do not stay in the LDS.
struct Layout {
    int64_t padded, small, small_padded, x, s;  // x, s: bytes of all matrices'
    int pieces, splits;
    int64_t partial;  // bytes of the sums of workgroups that share tiles
    int64_t sums;     // of the squares'
    size_t total;
};
template <class E>
Layout layout_of(int64_t matrices, int64_t rows, int64_t columns) {
    constexpr int kBytes = ProductType<E>::kBytes, kDepth = ProductType<E>::kDepth;
    Layout l;
    l.padded = (columns + 31) / 32 * 32;
    l.small = std::min(rows, columns);
    l.small_padded = (l.small + 31) / 32 * 32;
    l.x = matrices * rows * l.padded * kBytes;
    l.s = matrices * l.small * l.small_padded * kBytes;
    l.pieces = static_cast<int>(std::min<int64_t>(kMostPieces, (rows * columns + 16383) / 16384));
    l.splits = gram_splits(matrices, l.small, std::max(rows, columns), kDepth);
    const auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    l.x = up(l.x), l.s = up(l.s);
    l.partial = l.splits > 1 ? matrices * pairs_of(l.small, kSumSide) * l.splits * (4 * kSumSide * kSumSide) : 0;
    l.sums = up(8 * matrices * l.pieces);
    l.total = static_cast<size_t>(2 * l.x + 2 * l.s + l.partial + l.sums + up(4 * matrices) + up(4 * matrices * l.small_padded));
    return l;
}

template <Stage kStage, bool kTall, class E, class Result>
int launch_step(StepArgs a, int64_t matrices, hipStream_t stream) {
    constexpr bool kAlongM = (kStage == kGram && kTall) || (kStage == kUpdate && !kTall), kAlongN = kStage == kGram && kTall;
    const auto launch = [&](auto product) -> int {
        using P = typename decltype(product)::type;
        int64_t each;
        if (kStage != kUpdate) {
            each = pairs_of(a.small, P::kM);
            a.tiles_m = 1;
        } else {
            a.tiles_m = static_cast<uint32_t>((a.columns + P::kM - 1) / P::kM);
            each = static_cast<int64_t>(a.tiles_m) * ((a.rows + P::kN - 1) / P::kN);
        }
        const int64_t items = each * matrices * (kStage == kGram ? a.splits : 1);
        if (items * P::kThreads >= (int64_t{1} << 32) - (1 << 18)) return PENC_ERR_BAD_LAYER_SIZE;
        a.each = static_cast<uint32_t>(each), a.spread = Spread(items, 32);
        step_kernel<kStage, kTall, E, Result, P><<<a.spread.grid(), P::kThreads, 0, stream>>>(a);
        return launched();
    };
    const int64_t side_m = kStage == kUpdate ? a.columns : a.small, side_n = kStage == kUpdate ? a.rows : a.small;
    const int64_t huge = matrices * ((side_m + 255) / 256) * ((side_n + 255) / 256) / (kStage == kUpdate ? 1 : 2);
    if constexpr (std::is_same_v<E, half_t>) {
        if (huge >= 128) return launch(std::common_type<Product<E, kAlongM, kAlongN, 256, 256, 4, 2, Chunks::kDirect>>{});
    }
    if (small_tiles(matrices, side_m, side_n, kStage != kUpdate)) {
        // (of a few workgroups each has a compute unit's LDS to itself, for loads ahead; of many, two share it)
        const int64_t items = matrices * (kStage == kUpdate ? ((side_m + 63) / 64) * ((side_n + 63) / 64) : pairs_of(a.small, 64)) * (kStage == kGram ? a.splits : 1);
        if (items > 256) return launch(std::common_type<Product<E, kAlongM, kAlongN, 64, 64, 2, 2, Chunks::kDirect, 2>>{});
        return launch(std::common_type<Product<E, kAlongM, kAlongN, 64, 64, 2, 2, Chunks::kDirect, 4>>{});
    }
    return launch(std::common_type<Product<E, kAlongM, kAlongN, 128, 128, 2, 2, Chunks::kDirect>>{});
}

// Matrices of any size.
template <class E, class G>
int large(int64_t matrices, int64_t rows, int64_t columns, int steps, Coefficients k, const G* g, G* result, char* workspace, hipStream_t stream) {
    const Layout l = layout_of<E>(matrices, rows, columns);
    char *x = workspace, *next = x + l.x, *const s = next + l.x, *const f = s + l.s;
    float* const partial = reinterpret_cast<float*>(f + l.s);
    double* const sums = reinterpret_cast<double*>(f + l.s + l.partial);
    float* const rest = reinterpret_cast<float*>(f + l.s + l.partial + l.sums);
    float* const diagonal = rest + (matrices + 63) / 64 * 64;
    squares_kernel<G><<<static_cast<unsigned>(matrices * l.pieces), kThreads, 0, stream>>>(rows * columns, l.pieces, g, sums);
    if (const int rc = launched()) return rc;
    const int64_t eights = rows * (l.padded / 8);
    const uint32_t blocks = static_cast<uint32_t>(std::min<int64_t>((eights + kThreads - 1) / kThreads, std::max<int64_t>(1, 4096 / matrices)));
    stage_kernel<E, G><<<static_cast<unsigned>(matrices * blocks), kThreads, 0, stream>>>(static_cast<int>(rows), static_cast<int>(columns), static_cast<int>(l.padded),
                                                                                         l.pieces, g, sums, k.eps, x, rest, blocks);
    if (const int rc = launched()) return rc;
    for (int step = 0; step < steps; ++step) {
        StepArgs a{x, s, f, s, nullptr, static_cast<int>(rows), static_cast<int>(columns), static_cast<int>(l.padded), static_cast<int>(l.small),
                   static_cast<int>(l.small_padded), {}, 0, 0, l.splits, l.splits > 1 ? partial : nullptr, diagonal,
                   step == 0 && std::is_same_v<E, half_t> ? rest : nullptr, k.a, k.b, k.c};
        const auto all = [&](auto tall) -> int {
            constexpr bool kTall = decltype(tall)::value;
            if (const int rc = launch_step<kGram, kTall, E, G>(a, matrices, stream)) return rc;
            if (l.splits > 1) {
                a.each = static_cast<uint32_t>(pairs_of(l.small, kSumSide));
                gram_sum_kernel<E><<<static_cast<unsigned>(matrices * a.each), kSumThreads, 0, stream>>>(a);
                if (const int rc = launched()) return rc;
            }
            a.out = f;
            if (const int rc = launch_step<kSquare, false, E, G>(a, matrices, stream)) return rc;
            a.out = next;
            if (step + 1 == steps) a.result = result;
            return launch_step<kUpdate, kTall, E, G>(a, matrices, stream);
        };
        if (const int rc = rows > columns ? all(std::true_type{}) : all(std::false_type{})) return rc;
        std::swap(x, next);
    }
    return PENC_OK;
}

// What the steps make of 0 .. 1 has to stay where float16 times 2^12 has room: |X| <= 3, and F <= 15.  `growth`: the most that they make of a rounding of S.
bool bounded(double a, double b, double c, int steps, double& growth) {
    double most = 1.0;
    growth = 1.0;
    for (int step = 0; step < steps; ++step) {
        const double t = most * most;
        double p = std::max(std::abs(a), std::abs(a + b * t + c * t * t));
        double f = std::max(0.0, std::abs(b * t + c * t * t)), x = std::abs((a + b * t + c * t * t) * most);
        if (c != 0.0) {
            const double at = -b / (2.0 * c);  // of b t + c t^2
            if (at > 0.0 && at < t) f = std::max(f, std::abs(b * at + c * at * at)), p = std::max(p, std::abs(a + b * at + c * at * at));
            const double d = 9.0 * b * b - 20.0 * a * c;  // of a s + b s^3 + c s^5, whose slope is a + 3 b t + 5 c t^2
            if (d >= 0.0)
                for (const double sign : {-1.0, 1.0}) {
                    const double u = (-3.0 * b + sign * std::sqrt(d)) / (10.0 * c);
                    if (u > 0.0 && u < t) x = std::max(x, std::abs((a + b * u + c * u * u) * std::sqrt(u)));
                }
        } else if (b != 0.0) {
            const double u = -a / (3.0 * b);
            if (u > 0.0 && u < t) x = std::max(x, std::abs((a + b * u) * std::sqrt(u)));
        }
        if (!(f <= 15.0) || !(x <= 3.0)) return false;
        growth *= p * p;
        most = std::max(x, 1e-30);
    }
    return true;
}

bool bad_matrices(int64_t matrices, int64_t rows, int64_t columns) {
    return matrices < 0 || matrices > PENC_MAX_MATRICES || rows < 1 || rows > PENC_MAX_MATRIX_SIDE || columns < 1 || columns > PENC_MAX_MATRIX_SIDE;
}

// Whether the products are of float16 once.
bool in_halves(const penc_orthogonal& o) { return o.type == PENC_BF16 && o.halves != 0; }

bool bad_type(int type) { return type != PENC_FP32 && type != PENC_FP16 && type != PENC_BF16; }
bool bad_options(const penc_orthogonal& o) { return o.steps < 1 || o.steps > PENC_MAX_ORTHOGONAL_STEPS || !(o.eps >= 1e-30f) || std::isinf(o.eps); }

// Which way matrices go.
enum Way { kThinWay, kResidentWay, kLargeWay };
Way way_of(const penc_orthogonal& o, double growth) {
    if (growth <= kMostThinGrowth && is_thin(o.matrices, o.rows, o.columns)) return kThinWay;
    return is_resident(o.rows, o.columns) ? kResidentWay : kLargeWay;
}

// What it takes.  (Thin matrices that are not to go their own way take far more than they have: columns are padded to 32.)
size_t workspace_bytes(const penc_orthogonal& o, Way way) {
    if (way == kThinWay) return thin_workspace(o.matrices, o.rows, o.columns);
    if (way == kResidentWay) return 0;
    return in_halves(o) ? layout_of<half_t>(o.matrices, o.rows, o.columns).total : layout_of<split_t>(o.matrices, o.rows, o.columns).total;
}
size_t workspace_bytes(const penc_orthogonal& o) {
    double growth;
    if (bad_type(o.type) || bad_matrices(o.matrices, o.rows, o.columns) || o.matrices == 0 || bad_options(o) || !bounded(o.a, o.b, o.c, o.steps, growth)) return 0;
    return workspace_bytes(o, way_of(o, growth));
}
// What matrices take with any steps and coefficients.
size_t most_workspace_bytes(const penc_orthogonal& o) {
    if (bad_type(o.type) || bad_matrices(o.matrices, o.rows, o.columns) || o.matrices == 0) return 0;
    return std::max(workspace_bytes(o, way_of(o, 1.0)), workspace_bytes(o, way_of(o, INFINITY)));
}

int run(const penc_orthogonal& o, const void* update, void* result, void* workspace, size_t bytes, void* stream) {
    return with_type(o.type, [&](auto e) -> int {
        using G = decltype(e);
        if (bad_matrices(o.matrices, o.rows, o.columns) || o.steps < 1 || o.steps > PENC_MAX_ORTHOGONAL_STEPS) return PENC_ERR_BAD_LAYER_SIZE;
        double growth;
        if (bad_options(o) || !bounded(o.a, o.b, o.c, o.steps, growth)) return PENC_ERR_UNSUPPORTED_KIND;
        if (o.matrices == 0) return PENC_OK;
        if (!update || !result) return PENC_ERR_NULL_POINTER;
        if (!aligned_to(update, sizeof(G)) || !aligned_to(result, 4 * sizeof(G)) || !aligned_to(workspace, 256)) return PENC_ERR_MISALIGNED;
        const Way way = way_of(o, growth);
        const size_t need = workspace_bytes(o, way);
        if (bytes < need) return PENC_ERR_WORKSPACE_TOO_SMALL;
        if (need > 0 && !workspace) return PENC_ERR_NULL_POINTER;
        const Coefficients k{o.a, o.b, o.c, o.eps};
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const G* const from = static_cast<const G*>(update);
        G* const to = static_cast<G*>(result);
        char* const room = static_cast<char*>(workspace);
        if (way == kThinWay) return thin<G>(o.matrices, o.rows, o.columns, o.steps, k, from, to, room, s);
        if (way == kResidentWay) return resident<G>(o.matrices, o.rows, o.columns, o.steps, k, from, to, s);
        if constexpr (std::is_same_v<G, bf16_t>) {
            if (in_halves(o)) return large<half_t, G>(o.matrices, o.rows, o.columns, o.steps, k, from, to, room, s);
        }
        return large<split_t, G>(o.matrices, o.rows, o.columns, o.steps, k, from, to, room, s);
    });
}

}  // namespace
}  // namespace penc

using namespace penc;

extern "C" {

size_t penc_orthogonal_workspace_bytes(const penc_orthogonal* orthogonal) { return orthogonal ? workspace_bytes(*orthogonal) : 0; }

int penc_orthogonal_matrices(const penc_orthogonal* orthogonal, const void* update, void* result, void* workspace, size_t workspace_bytes, void* stream) {
    if (!orthogonal) return PENC_ERR_NULL_POINTER;
    return run(*orthogonal, update, result, workspace, workspace_bytes, stream);
}

size_t penc_orthogonalise_workspace_bytes(int type, int64_t matrices, int64_t rows, int64_t columns) {
    return most_workspace_bytes({type, 1, matrices, rows, columns, 0, 0.0f, 0.0f, 0.0f, 0.0f});
}

int penc_orthogonalise(int type, int64_t matrices, int64_t rows, int64_t columns, int steps, float a, float b, float c, float eps, const void* update, void* result,
                       void* workspace, size_t workspace_bytes, void* stream) {
    return run({type, 1, matrices, rows, columns, steps, a, b, c, eps}, update, result, workspace, workspace_bytes, stream);
}

int penc_muon_momentum(int type, int64_t n, const void* grad, float* average, float momentum, int nesterov, void* update, void* stream) {
    return with_type(type, [&](auto e) -> int {
        using G = decltype(e);
        if (n < 0) return PENC_ERR_BAD_LAYER_SIZE;
        if (n == 0) return PENC_OK;
        if (!grad || !average || !update) return PENC_ERR_NULL_POINTER;
        if (!aligned_to(grad, sizeof(G)) || !aligned_to(update, sizeof(G)) || !aligned_to(average, 4)) return PENC_ERR_MISALIGNED;
        momentum_kernel<G><<<grid_of(n), kThreads, 0, static_cast<hipStream_t>(stream)>>>(n, static_cast<const G*>(grad), average, momentum, nesterov != 0,
                                                                                         static_cast<G*>(update));
        return launched();
    });
}

int penc_muon_apply(int type, int64_t n, void* params, const void* orthogonal, float decay, float rate, void* stream) {
    return with_type(type, [&](auto e) -> int {
        using G = decltype(e);
        if (n < 0) return PENC_ERR_BAD_LAYER_SIZE;
        if (n == 0) return PENC_OK;
        if (!params || !orthogonal) return PENC_ERR_NULL_POINTER;
        if (!aligned_to(params, sizeof(G)) || !aligned_to(orthogonal, sizeof(G))) return PENC_ERR_MISALIGNED;
        apply_kernel<G><<<grid_of(n), kThreads, 0, static_cast<hipStream_t>(stream)>>>(n, static_cast<G*>(params), static_cast<const G*>(orthogonal), decay, rate);
        return launched();
    });
}

}  // extern "C"
