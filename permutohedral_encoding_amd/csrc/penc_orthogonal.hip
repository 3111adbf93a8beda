// Nearly orthogonal matrices from updates, by Newton-Schulz products (K. Jordan et al., "Muon: an optimizer for hidden layers in neural networks", 2024):
//
//     X = G / (|G|_F + eps);    `steps` times:  S = X X^T (of a tall X: X^T X),  F = b S + c S S,  X = a X + F X (X F)
//
// takes every singular value s in 0 .. 1 through as many times a s + b s^3 + c s^5.  What is small in X is taken up by a factor a in each step, and so is what a rounding has
// added to it.  In 16 bits with 8 of them behind the point (bfloat16) the result is off by 1e-2 of it, in float16 by 1.4e-3, in float16 twice (22 bits) by 2.7e-7, of
// which float32 itself has 1.8e-7 (random matrices of 32 to 1024 rows, 5 steps).  So X, S and F are kept
//
//     for bfloat16 results     as float16, one product for each: with the result's own rounding (1.66e-3) 2.1e-3
//     for float16 and float32  as two float16 values, hi + lo, three products for each
//
// times 2^12: with |X| <= 1.2, S <= 1.5 and F <= 3 they stay under 2^14 (a bound on the coefficients sees to that), and what matters of lo is no subnormal number.
// The matrix cores run float16 8 times as fast as float32, so that three products take 3/8 of the time.
//
// S and S S are symmetric: tiles on one side of the diagonal are computed and stored twice.  Matrices of up to 128 rows (or columns) that fit the LDS go through all of their
// steps there, one to a workgroup.
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

// Four numbers at `column` of a stored row.
template <class E>
__device__ __forceinline__ int column_at(int column) {
    if constexpr (std::is_same_v<E, split_t>) return column / 32 * 128 + column % 32 * 2;
    else return column * 2;
}
using half_four = half_t __attribute__((ext_vector_type(4)));
template <class E>
__device__ __forceinline__ tile_acc load_stored(const char* row, int column) {
    const char* const p = row + column_at<E>(column);
    tile_acc v = __builtin_convertvector(*reinterpret_cast<const half_four*>(p), tile_acc);
    if constexpr (std::is_same_v<E, split_t>) v += __builtin_convertvector(*reinterpret_cast<const half_four*>(p + 64), tile_acc);
    return v;
}
template <class E>
__device__ __forceinline__ void store_stored(char* row, int column, tile_acc v) {
    char* const p = row + column_at<E>(column);
    const half_four hi = __builtin_convertvector(v, half_four);
    *reinterpret_cast<half_four*>(p) = hi;
    if constexpr (std::is_same_v<E, split_t>) *reinterpret_cast<half_four*>(p + 64) = __builtin_convertvector(v - __builtin_convertvector(hi, tile_acc), half_four);
}
template <class E>
__device__ __forceinline__ void store_stored(char* row, int column, float v) {
    char* const p = row + column_at<E>(column);
    const half_t hi = static_cast<half_t>(v);
    *reinterpret_cast<half_t*>(p) = hi;
    if constexpr (std::is_same_v<E, split_t>) *reinterpret_cast<half_t*>(p + 64) = static_cast<half_t>(v - static_cast<float>(hi));
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

template <class G>
__global__ __launch_bounds__(kThreads) void squares_kernel(int64_t values, int pieces, const G* __restrict__ g, double* __restrict__ sums) {
    const int64_t each = (values + pieces - 1) / pieces, piece = blockIdx.x % pieces;
    const int64_t first = piece * each, last = min(first + each, values);
    const G* const from = g + blockIdx.x / pieces * values;
    double sum = 0.0;
    for (int64_t i = first + threadIdx.x; i < last; i += kThreads) {
        const double v = static_cast<double>(static_cast<float>(from[i]));
        sum += v * v;
    }
    sum = workgroup_sum<kThreads>(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// X 2^12 as it is stored, zeros behind each row's end.
template <class E, class G>
__global__ __launch_bounds__(kThreads) void stage_kernel(int rows, int columns, int padded, int pieces, const G* __restrict__ g, const double* __restrict__ sums,
                                                         float eps, char* __restrict__ x, uint32_t blocks) {
    const int64_t matrix = blockIdx.x / blocks;
    const double* const mine = sums + matrix * pieces;
    double squares = 0.0;
    for (int i = static_cast<int>(threadIdx.x); i < pieces; i += kThreads) squares += mine[i];
    const double factor = per_norm(workgroup_sum<kThreads>(squares), eps);
    const G* const from = g + matrix * rows * columns;
    const int64_t stride = static_cast<int64_t>(padded) * ProductType<E>::kBytes;
    char* const to = x + matrix * rows * stride;
    const int64_t fours = static_cast<int64_t>(rows) * (padded / 4);
    for (int64_t i = static_cast<int64_t>(blockIdx.x % blocks) * kThreads + threadIdx.x; i < fours; i += static_cast<int64_t>(blocks) * kThreads) {
        const int64_t row = i / (padded / 4);
        const int column = static_cast<int>(i % (padded / 4)) * 4;
        tile_acc v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = column + k < columns ? scaled(from[row * columns + column + k], factor) : 0.0f;
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
    float a, b, c;
};

// Pair `t` of tiles on and behind the diagonal: i <= j.
__device__ __forceinline__ void pair_of(uint32_t t, uint32_t& i, uint32_t& j) {
    j = static_cast<uint32_t>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
    while (j * (j + 1) / 2 > t) --j;
    while ((j + 1) * (j + 2) / 2 <= t) ++j;
    i = t - j * (j + 1) / 2;
}

template <Stage kStage, bool kTall, class E, class Result, class P>
__global__ __launch_bounds__(P::kThreads) void step_kernel(StepArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    constexpr int kBytes = ProductType<E>::kBytes;
    const uint32_t item = a.spread.item(), t = item % a.each;
    if (item >= a.spread.items) return;
    const int64_t matrix = item / a.each;
    const int64_t stride = static_cast<int64_t>(a.padded) * kBytes, small_stride = static_cast<int64_t>(a.small_padded) * kBytes;
    const char *const x = a.x + matrix * a.rows * stride, *const s = a.s + matrix * a.small * small_stride, *const f = a.f + matrix * a.small * small_stride;
    uint32_t i = t % a.tiles_m, j = t / a.tiles_m;
    if constexpr (kStage != kUpdate) pair_of(t, i, j);
    const int m0 = uniform(static_cast<int>(i)) * P::kM, n0 = uniform(static_cast<int>(j)) * P::kN;
    const auto rows_from = [&](const char* p, int64_t row_bytes, int rows, int first, int most) { return Operand{p + first * row_bytes, row_bytes, min(rows - first, most), static_cast<int>(row_bytes)}; };
    const auto columns_from = [&](int first, int most) { return Operand{x + first * kBytes, stride, a.rows, min(a.padded - first, most) * kBytes}; };
    P p;
    if constexpr (kStage == kGram && !kTall) p.run(lds, rows_from(x, stride, a.rows, m0, P::kM), rows_from(x, stride, a.rows, n0, P::kN), a.padded, P::kZero, P::kNothing);
    else if constexpr (kStage == kGram) p.run(lds, columns_from(m0, P::kM), columns_from(n0, P::kN), a.rows, P::kZero, P::kNothing);
    else if constexpr (kStage == kSquare) p.run(lds, rows_from(s, small_stride, a.small, m0, P::kM), rows_from(s, small_stride, a.small, n0, P::kN), a.small_padded, P::kZero, P::kNothing);
    else if constexpr (!kTall) p.run(lds, columns_from(m0, P::kM), rows_from(f, small_stride, a.small, n0, P::kN), a.small, P::kZero, P::kNothing);
    else p.run(lds, rows_from(f, small_stride, a.small, m0, P::kM), rows_from(x, stride, a.rows, n0, P::kN), a.padded, P::kZero, P::kNothing);
    if constexpr (kStage != kUpdate) {
        char* const out = a.out + matrix * a.small * small_stride;
        p.each([&](int m, int n, tile_acc v) {
            m += m0, n += n0;
            if (n >= a.small || m >= a.small_padded) return;
            v *= kPerScale;
            if constexpr (kStage == kSquare) v = a.b * load_stored<E>(s + n * small_stride, m) + a.c * v;
            store_stored<E>(out + n * small_stride, m, v);
            if (i == j) return;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (m + k < a.small) store_stored<E>(out + (m + k) * small_stride, n, v[k]);
        });
        // (columns behind the last one, of rows that only the other side of the diagonal has)
        if (i != j && n0 + P::kN >= a.small) {
            const int behind = a.small_padded - a.small;
            for (int k = static_cast<int>(threadIdx.x); k < behind * P::kM; k += P::kThreads) {
                const int row = m0 + k / behind;
                if (row < a.small) store_stored<E>(out + row * small_stride, a.small + k % behind, 0.0f);
            }
        }
    } else {
        char* const out = a.out + matrix * a.rows * stride;
        using result_four = Result __attribute__((ext_vector_type(4)));
        Result* const result = static_cast<Result*>(a.result) + matrix * a.rows * a.columns;
        p.each([&](int m, int n, tile_acc v) {
            m += m0, n += n0;
            if (n >= a.rows || m >= a.padded) return;
            v = a.a * load_stored<E>(x + n * stride, m) + v * kPerScale;
            if (a.result == nullptr) store_stored<E>(out + n * stride, m, v);
            else if (m < a.columns) store_values<Result, 4>(result + static_cast<int64_t>(n) * a.columns + m, __builtin_convertvector(v * kPerScale, result_four), a.columns - m);
        });
    }
}

// ------------------------------------------------------------------------------------------
// matrices that stay in the LDS

constexpr int kResidentThreads = 512, kResidentWaves = kResidentThreads / 64;
constexpr int kMostSmall = 128;

// A matrix of Split numbers in the LDS.  Chunks of a row's 128 bytes are permuted by the row, so that neither 8 rows of one chunk nor 4 rows of two chunks meet in a bank.
struct Resident {
    char* first;
    int pitch;

    __device__ __forceinline__ char* chunk(int row, int byte) const { return first + row * pitch + (byte & ~127) + ((byte >> 4 & 7) ^ ((row & 3) << 1 | (row >> 2 & 1))) * 16 + (byte & 15); }
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
    __device__ __forceinline__ tile_acc load(int row, int column) const {
        const int byte = column_at<split_t>(column);
        return __builtin_convertvector(*reinterpret_cast<const half_four*>(chunk(row, byte)), tile_acc) +
               __builtin_convertvector(*reinterpret_cast<const half_four*>(chunk(row, byte + 64)), tile_acc);
    }
    __device__ __forceinline__ void store(int row, int column, tile_acc v) const {
        const int byte = column_at<split_t>(column);
        const half_four hi = __builtin_convertvector(v, half_four);
        *reinterpret_cast<half_four*>(chunk(row, byte)) = hi;
        *reinterpret_cast<half_four*>(chunk(row, byte + 64)) = __builtin_convertvector(v - __builtin_convertvector(hi, tile_acc), half_four);
    }
    __device__ __forceinline__ void store(int row, int column, float v) const {
        const int byte = column_at<split_t>(column);
        const half_t hi = static_cast<half_t>(v);
        *reinterpret_cast<half_t*>(chunk(row, byte)) = hi;
        *reinterpret_cast<half_t*>(chunk(row, byte + 64)) = static_cast<half_t>(v - static_cast<float>(hi));
    }
};

__device__ __forceinline__ tile_acc multiply_split(chunk16 a, chunk16 a_low, chunk16 b, chunk16 b_low, tile_acc c) {
    c = multiply<half_t>(a, b_low, c);
    c = multiply<half_t>(a_low, b, c);
    return multiply<half_t>(a, b, c);
}

__host__ __device__ constexpr int resident_pitch(int padded) { return padded * 4; }
__host__ __device__ constexpr int round_to_32(int n) { return (n + 31) / 32 * 32; }

// One matrix to a workgroup, X as `small` rows of `large` numbers whichever way it lies in memory.  A wave has 16 x 32 results of S and of F, and 16 columns of X, which it
// overwrites when it has them all.
template <class G, int kLds>
__global__ __launch_bounds__(kResidentThreads) void resident_kernel(int rows, int columns, int steps, Coefficients k, const G* __restrict__ g, G* __restrict__ result) {
    __shared__ __attribute__((aligned(1024))) char lds[kLds];
    const bool tall = rows > columns;
    const int small = min(rows, columns), large = max(rows, columns), small_padded = round_to_32(small), large_padded = round_to_32(large);
    const Resident x{lds, resident_pitch(large_padded)}, s{lds + small_padded * x.pitch, resident_pitch(small_padded)};
    const int64_t values = static_cast<int64_t>(rows) * columns;
    const G* const from = g + blockIdx.x * values;
    double squares = 0.0;
    for (int i = static_cast<int>(threadIdx.x); i < values; i += kResidentThreads) {
        const double v = static_cast<double>(static_cast<float>(from[i]));
        squares += v * v;
    }
    const double factor = per_norm(workgroup_sum<kResidentThreads>(squares), k.eps);
    for (int i = static_cast<int>(threadIdx.x); i < small_padded * large_padded; i += kResidentThreads) {
        // (neighbouring lanes read neighbours in memory)
        const int row = tall ? i % small_padded : i / large_padded, column = tall ? i / small_padded : i % large_padded;
        const bool there = row < small && column < large;
        x.store(row, column, there ? scaled(from[tall ? column * columns + row : row * columns + column], factor) : 0.0f);
    }
    __syncthreads();
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), q4 = lane / 16 * 4, l16 = lane % 16;
    const int units_m = small_padded / 16, units = units_m * (small_padded / 32);
    constexpr int kMostUnits = kMostSmall / 16 * (kMostSmall / 32) / kResidentWaves;
    for (int step = 0; step < steps; ++step) {
        tile_acc of_s[kMostUnits][2];
#pragma unroll
        for (int u = 0; u < kMostUnits; ++u) {
            const int unit = u * kResidentWaves + wave, m = unit % units_m * 16, n = unit / units_m * 32;
            if (unit >= units) continue;
            of_s[u][0] = of_s[u][1] = tile_acc{};
            for (int line = 0; line < large_padded / 32; ++line) {
                const chunk16 a = x.across(m, line, 0), a_low = x.across(m, line, 1);
#pragma unroll
                for (int h = 0; h < 2; ++h) of_s[u][h] = multiply_split(a, a_low, x.across(n + 16 * h, line, 0), x.across(n + 16 * h, line, 1), of_s[u][h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                of_s[u][h] *= kPerScale;
                s.store(n + 16 * h + l16, m + q4, of_s[u][h]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMostUnits; ++u) {
            const int unit = u * kResidentWaves + wave, m = unit % units_m * 16, n = unit / units_m * 32;
            if (unit >= units) continue;
            tile_acc square[2] = {};
            for (int line = 0; line < small_padded / 32; ++line) {
                const chunk16 a = s.across(m, line, 0), a_low = s.across(m, line, 1);
#pragma unroll
                for (int h = 0; h < 2; ++h) square[h] = multiply_split(a, a_low, s.across(n + 16 * h, line, 0), s.across(n + 16 * h, line, 1), square[h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) of_s[u][h] = k.b * of_s[u][h] + (k.c * kPerScale) * square[h];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMostUnits; ++u) {
            const int unit = u * kResidentWaves + wave, m = unit % units_m * 16, n = unit / units_m * 32;
            if (unit >= units) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) s.store(n + 16 * h + l16, m + q4, of_s[u][h]);
        }
        __syncthreads();
        const bool last = step + 1 == steps;
        for (int m = wave * 16; m < large_padded; m += kResidentWaves * 16) {
            constexpr int kMostTiles = kMostSmall / 16;
            tile_acc acc[kMostTiles];
#pragma unroll
            for (int n = 0; n < kMostTiles; ++n) acc[n] = tile_acc{};
            for (int line = 0; line < small_padded / 32; ++line) {
                const chunk16 a = x.along(line * 32, m, 0), a_low = x.along(line * 32, m, 1);
#pragma unroll
                for (int n = 0; n < kMostTiles; ++n)
                    if (n * 16 < small_padded) acc[n] = multiply_split(a, a_low, s.across(n * 16, line, 0), s.across(n * 16, line, 1), acc[n]);
            }
#pragma unroll
            for (int n = 0; n < kMostTiles; ++n) {
                if (n * 16 >= small_padded) continue;
                const int row = n * 16 + l16, column = m + q4;
                const tile_acc v = k.a * x.load(row, column) + acc[n] * kPerScale;
                if (!last) {
                    x.store(row, column, v);
                } else if (row < small) {
                    G* const to = result + blockIdx.x * values;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (column + i < large) to[tall ? (column + i) * columns + row : row * columns + column + i] = static_cast<G>(v[i] * kPerScale);
                }
            }
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

int64_t resident_bytes(int64_t small, int64_t large) {
    if (small > kMostSmall || large > 1 << 12) return int64_t{1} << 40;
    const int s = round_to_32(static_cast<int>(small)), l = round_to_32(static_cast<int>(large));
    return static_cast<int64_t>(s) * (resident_pitch(l) + resident_pitch(s));
}
constexpr int kMostResident = 160 * 1024 - 256;

// The workspace of matrices that do not stay in the LDS.
struct Layout {
    int64_t padded, small, small_padded, x, s;  // x, s: bytes of all matrices'
    int pieces;
    size_t total;
};
template <class E>
Layout layout_of(int64_t matrices, int64_t rows, int64_t columns) {
    constexpr int kBytes = ProductType<E>::kBytes, kDepth = ProductType<E>::kDepth;
    Layout l;
    l.padded = (columns + kDepth - 1) / kDepth * kDepth;
    l.small = std::min(rows, columns);
    l.small_padded = (l.small + kDepth - 1) / kDepth * kDepth;
    l.x = matrices * rows * l.padded * kBytes;
    l.s = matrices * l.small * l.small_padded * kBytes;
    l.pieces = static_cast<int>(std::min<int64_t>(kMostPieces, (rows * columns + 16383) / 16384));
    const auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    l.x = up(l.x), l.s = up(l.s);
    l.total = static_cast<size_t>(2 * l.x + 2 * l.s + up(8 * matrices * l.pieces));
    return l;
}

template <Stage kStage, bool kTall, class E, class Result>
int launch_step(StepArgs a, int64_t matrices, hipStream_t stream) {
    constexpr bool kAlongM = (kStage == kGram && kTall) || (kStage == kUpdate && !kTall), kAlongN = kStage == kGram && kTall;
    const auto launch = [&](auto product) -> int {
        using P = typename decltype(product)::type;
        int64_t each;
        if (kStage != kUpdate) {
            const int64_t tiles = (a.small + P::kM - 1) / P::kM;
            each = tiles * (tiles + 1) / 2;
            a.tiles_m = 1;
        } else {
            a.tiles_m = static_cast<uint32_t>((a.columns + P::kM - 1) / P::kM);
            each = static_cast<int64_t>(a.tiles_m) * ((a.rows + P::kN - 1) / P::kN);
        }
        const int64_t items = each * matrices;
        if (items * P::kThreads >= (int64_t{1} << 32) - (1 << 18)) return PENC_ERR_BAD_LAYER_SIZE;
        a.each = static_cast<uint32_t>(each), a.spread = Spread(items, 32);
        step_kernel<kStage, kTall, E, Result, P><<<a.spread.grid(), P::kThreads, 0, stream>>>(a);
        return launched();
    };
    // tiles of 64 x 64 where there would not be a workgroup of 128 x 128 for each compute unit
    const int64_t side_m = kStage == kUpdate ? a.columns : a.small, side_n = kStage == kUpdate ? a.rows : a.small;
    const int64_t large = matrices * ((side_m + 127) / 128) * ((side_n + 127) / 128) / (kStage == kUpdate ? 1 : 2);
    const int64_t huge = matrices * ((side_m + 255) / 256) * ((side_n + 255) / 256) / (kStage == kUpdate ? 1 : 2);
    if constexpr (std::is_same_v<E, half_t>) {
        if (huge >= 128) return launch(std::common_type<Product<E, kAlongM, kAlongN, 256, 256, 4, 2, Chunks::kDirect>>{});
    }
    if (large < 256) return launch(std::common_type<Product<E, kAlongM, kAlongN, 64, 64, 2, 2, Chunks::kDirect>>{});
    return launch(std::common_type<Product<E, kAlongM, kAlongN, 128, 128, 2, 2, Chunks::kDirect>>{});
}

template <class E, class G>
int orthogonalise(int64_t matrices, int64_t rows, int64_t columns, int steps, Coefficients k, const G* g, G* result, char* workspace, hipStream_t stream) {
    const Layout l = layout_of<E>(matrices, rows, columns);
    char *x = workspace, *next = x + l.x, *const s = next + l.x, *const f = s + l.s;
    double* const sums = reinterpret_cast<double*>(f + l.s);
    squares_kernel<G><<<static_cast<unsigned>(matrices * l.pieces), kThreads, 0, stream>>>(rows * columns, l.pieces, g, sums);
    if (const int rc = launched()) return rc;
    const int64_t fours = rows * (l.padded / 4);
    const uint32_t blocks = static_cast<uint32_t>(std::min<int64_t>((fours + kThreads - 1) / kThreads, std::max<int64_t>(1, 4096 / matrices)));
    stage_kernel<E, G><<<static_cast<unsigned>(matrices * blocks), kThreads, 0, stream>>>(static_cast<int>(rows), static_cast<int>(columns), static_cast<int>(l.padded),
                                                                                         l.pieces, g, sums, k.eps, x, blocks);
    if (const int rc = launched()) return rc;
    for (int step = 0; step < steps; ++step) {
        StepArgs a{x, s, f, s, nullptr, static_cast<int>(rows), static_cast<int>(columns), static_cast<int>(l.padded), static_cast<int>(l.small),
                   static_cast<int>(l.small_padded), {}, 0, 0, k.a, k.b, k.c};
        const auto all = [&](auto tall) -> int {
            constexpr bool kTall = decltype(tall)::value;
            if (const int rc = launch_step<kGram, kTall, E, G>(a, matrices, stream)) return rc;
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

// What the steps make of 0 .. 1 has to stay where float16 times 2^12 has room: |X| <= 3, and F <= 15.
bool bounded(double a, double b, double c, int steps) {
    double most = 1.0;
    for (int step = 0; step < steps; ++step) {
        const double t = most * most;
        double f = std::max(0.0, std::abs(b * t + c * t * t)), x = std::abs((a + b * t + c * t * t) * most);
        if (c != 0.0) {
            const double at = -b / (2.0 * c);  // of b t + c t^2
            if (at > 0.0 && at < t) f = std::max(f, std::abs(b * at + c * at * at));
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
        most = std::max(x, 1e-30);
    }
    return true;
}

bool bad_matrices(int64_t matrices, int64_t rows, int64_t columns) {
    return matrices < 0 || matrices > PENC_MAX_MATRICES || rows < 1 || rows > PENC_MAX_MATRIX_SIDE || columns < 1 || columns > PENC_MAX_MATRIX_SIDE;
}

}  // namespace
}  // namespace penc

using namespace penc;

extern "C" {

size_t penc_orthogonalise_workspace_bytes(int type, int64_t matrices, int64_t rows, int64_t columns) {
    if (bad_matrices(matrices, rows, columns) || resident_bytes(std::min(rows, columns), std::max(rows, columns)) <= kMostResident) return 0;
    return type == PENC_BF16 ? layout_of<half_t>(matrices, rows, columns).total : layout_of<split_t>(matrices, rows, columns).total;
}

int penc_orthogonalise(int type, int64_t matrices, int64_t rows, int64_t columns, int steps, float a, float b, float c, float eps, const void* update, void* result,
                       void* workspace, size_t workspace_bytes, void* stream) {
    return with_type(type, [&](auto e) -> int {
        using G = decltype(e);
        if (bad_matrices(matrices, rows, columns) || steps < 1 || steps > PENC_MAX_ORTHOGONAL_STEPS) return PENC_ERR_BAD_LAYER_SIZE;
        if (!(eps >= 1e-30f) || std::isinf(eps) || !bounded(a, b, c, steps)) return PENC_ERR_UNSUPPORTED_KIND;
        if (matrices == 0) return PENC_OK;
        if (!update || !result) return PENC_ERR_NULL_POINTER;
        if (!aligned_to(update, sizeof(G)) || !aligned_to(result, 4 * sizeof(G)) || !aligned_to(workspace, 256)) return PENC_ERR_MISALIGNED;
        const size_t need = penc_orthogonalise_workspace_bytes(type, matrices, rows, columns);
        if (workspace_bytes < need) return PENC_ERR_WORKSPACE_TOO_SMALL;
        if (need > 0 && !workspace) return PENC_ERR_NULL_POINTER;
        const Coefficients k{a, b, c, eps};
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const G* const from = static_cast<const G*>(update);
        G* const to = static_cast<G*>(result);
        if (need == 0) {
            const int64_t bytes = resident_bytes(std::min(rows, columns), std::max(rows, columns));
            const auto launch = [&](auto size) -> int {
                resident_kernel<G, decltype(size)::value><<<static_cast<unsigned>(matrices), kResidentThreads, 0, s>>>(static_cast<int>(rows), static_cast<int>(columns),
                                                                                                                    steps, k, from, to);
                return launched();
            };
            // (two workgroups to a compute unit, where they fit)
            if (bytes <= kMostResident / 2) return launch(std::integral_constant<int, kMostResident / 2>{});
            return launch(std::integral_constant<int, kMostResident>{});
        }
        using E = std::conditional_t<std::is_same_v<G, bf16_t>, half_t, split_t>;
        return orthogonalise<E, G>(matrices, rows, columns, steps, k, from, to, static_cast<char*>(workspace), s);
    });
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
