// Matrix products of a workgroup: D[m][n] = sum over k of A[m][k] B[n][k], for a tile of kM x kN results that stay in the registers of its waves.
//
// Operands come in steps of k through the LDS, one step on its way while the one before is multiplied.  An operand is
//
//     Across   rows of adjacent k: 128 bytes of each row in a step, 64 k of a 16-bit type and 32 of fp32
//     Along    rows of one k, adjacent in m (or n): as many k in a step, transposed on the way from the LDS into registers
//
// 16-bit types are multiplied by v_mfma_f32_16x16x32, fp32 by v_mfma_f32_16x16x4_f32.  A Split number is two halves, hi = the nearest to x and lo = the nearest to x - hi
// (22 bits of x together, where x - hi is no less than 2^-14): of every 32 numbers the hi and behind them the lo, so that a row has 4 bytes for each; a product is
// hi hi + hi lo + lo hi, and what is left out is 2^-22 of it.
//
// Chunks of 16 bytes go from memory into the LDS directly, where rows and their ends are on 16 bytes, each lane its own: where a chunk stands in the LDS is fixed by the lane that brings it, so
// a lane brings the chunk that belongs there.  Addresses behind an operand's end (rows, k, or columns) read zeros, which the buffer's bounds see to.  Of operands that
// begin anywhere, lanes load what is there into registers and write it into the LDS.
//
// Where a chunk stands: fragments are read by 16 lanes at a time, which should meet 64 banks of 4 bytes each once.  Across: lanes read one chunk c of 16 rows of 128 bytes; c
// stands at c ^ (row / 2 mod 8).  Along: 16 lanes read 32 bytes (fp32: 64) of 4 neighbouring k, and 16 more those of the k 8 (fp32: 4) behind; pieces of 32 (64)
// bytes are permuted by these bits of k.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "penc_kept.hpp"

namespace penc {

struct split_t {
    half_t part;  // (rows are counted in 4 bytes a number; this is what they are made of)
};

template <class E>
struct ProductType {
    static constexpr int kBytes = 2;  // of a number
    static constexpr int kDepth = 64; // k of a step
};
template <>
struct ProductType<float> {
    static constexpr int kBytes = 4;
    static constexpr int kDepth = 32;
};
template <>
struct ProductType<split_t> {
    static constexpr int kBytes = 4;
    static constexpr int kDepth = 32;
};

using tile_acc = float __attribute__((ext_vector_type(4)));
using chunk16 = uint32_t __attribute__((ext_vector_type(4)));

template <class E>
__device__ __forceinline__ tile_acc multiply(chunk16 a, chunk16 b, tile_acc c) {
    if constexpr (std::is_same_v<E, bf16_t>) {
        using V = bf16_t __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    } else if constexpr (std::is_same_v<E, float>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    } else {
        using V = half_t __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
}

// One operand of a workgroup's tile, from its first row (Across: of the tile, Along: of k).
struct Operand {
    const char* first;
    int64_t stride;  // bytes between rows
    int rows;        // Across: that are there from the first on; Along: k
    int bytes;       // of a row from `first` on: Across: of k; Along: of columns
};

constexpr int kMostOperandStride = 1 << 24;  // bytes: 256 rows are within a buffer's 2^32

// kAlong; kWide: rows (Across) or columns (Along) of the tile.
template <class E, bool kAlong, int kWide>
struct OperandTile {
    using T = ProductType<E>;
    static constexpr int kRowBytes = kAlong ? kWide * T::kBytes : 128;
    static constexpr int kRows = kAlong ? T::kDepth : kWide;
    static constexpr int kSize = kRows * kRowBytes;
    static constexpr int kChunks = kSize / 16, kRowChunks = kRowBytes / 16;

    // where chunk c of a row stands in it
    __device__ __forceinline__ static int place(int row, int c) {
        if constexpr (!kAlong) return c ^ (row >> 1 & 7);
        else if constexpr (std::is_same_v<E, float>) return c ^ (row >> 2 & 3) << 2;
        else if constexpr (kRowBytes >= 256) return c ^ ((row & 3) | (row >> 3 & 1) << 2) << 1;
        else return c ^ ((row >> 1 & 1) | (row >> 3 & 1) << 1) << 1;
    }

    // 16 rows (columns) from `at` on, as the matrix instruction takes them: lane 16 g + i has row i; half q of a step (Split: hi or lo).
    __device__ __forceinline__ static chunk16 fragment(const char* lds, int at, int q) {
        const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
        if constexpr (!kAlong) {
            const int row = at + i;
            return *reinterpret_cast<const chunk16*>(lds + row * 128 + place(row, q * 4 + g) * 16);
        } else if constexpr (std::is_same_v<E, float>) {
            chunk16 f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = q * 16 + g * 4 + j, column = at + i;
                f[j] = *reinterpret_cast<const uint32_t*>(lds + row * kRowBytes + place(row, column / 4) * 16 + column % 4 * 4);
            }
            return f;
        } else {
            constexpr bool kSplit = std::is_same_v<E, split_t>;
            const int byte = (kSplit ? at / 32 * 128 + at % 32 * 2 + q * 64 : at * 2) + i % 4 * 8;
            using V = short __attribute__((ext_vector_type(4)));
            using Lds = __attribute__((address_space(3))) V;
            chunk16 f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = (kSplit ? 0 : q * 32) + g * 8 + h * 4 + i / 4;
                const char* const p = lds + row * kRowBytes + place(row, byte / 16) * 16 + byte % 16;
                const V v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p));
                const uint2 w = __builtin_bit_cast(uint2, v);
                f[2 * h] = w.x, f[2 * h + 1] = w.y;
            }
            return f;
        }
    }
};

// Brings an operand's steps into the LDS.
template <class E, bool kAlong, int kWide, int kThreads, bool kDirect>
struct Loader {
    using Tile = OperandTile<E, kAlong, kWide>;
    using T = ProductType<E>;
    static constexpr int kEach = Tile::kChunks / kThreads;
    static_assert(Tile::kChunks % kThreads == 0);

    Operand o;
    int row[kEach], byte[kEach];  // of the chunks that this lane brings
    chunk16 held[kDirect ? 1 : kEach];

    __device__ __forceinline__ explicit Loader(const Operand& operand) : o(operand) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int slot = j * kThreads + static_cast<int>(threadIdx.x);
            row[j] = slot / Tile::kRowChunks;
            byte[j] = Tile::place(row[j], slot % Tile::kRowChunks) * 16;
        }
    }

    // The chunks of a step are on their way, into the LDS or into registers.
    __device__ __forceinline__ void begin(char* lds, int step) {
        // (rows, bytes of a row, and the first of them that this step has)
        const int64_t past = kAlong ? static_cast<int64_t>(step) * T::kDepth * o.stride : static_cast<int64_t>(step) * 128;
        const char* const first = o.first + past;
        const int rows = kAlong ? o.rows - step * T::kDepth : o.rows, bytes = kAlong ? o.bytes : o.bytes - step * 128;
        if constexpr (kDirect) {
            const int64_t there = rows > 0 && bytes > 0 ? (rows - 1) * o.stride + bytes : 0;
            const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(first), 0, static_cast<int>(there < 0x7FFFFFFF ? there : 0x7FFFFFFF), 0x00020000);
            const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int at = byte[j] < bytes ? row[j] * static_cast<int>(o.stride) + byte[j] : -1;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (__attribute__((address_space(3))) void*)(lds + (j * kThreads + wave * 64) * 16), 16, at, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const char* const p = first + row[j] * o.stride + byte[j];
                const int left = row[j] < rows ? bytes - byte[j] : 0;
                chunk16 v{};
                if (left >= 16) {
                    using Unaligned = uint32_t __attribute__((ext_vector_type(4), aligned(T::kBytes == 2 ? 2 : 4)));
                    v = *reinterpret_cast<const Unaligned*>(p);
                } else if (left > 0) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if constexpr (T::kBytes == 4) {
                            if (4 * w < left) v[w] = *reinterpret_cast<const uint32_t*>(p + 4 * w);
                        } else {
                            if (4 * w < left) v[w] = *reinterpret_cast<const uint16_t*>(p + 4 * w);
                            if (4 * w + 2 < left) v[w] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 4 * w + 2)) << 16;
                        }
                    }
                }
                held[j] = v;
            }
        }
    }
    // What was on its way is in the LDS (of this wave; a barrier makes it so for the others).
    __device__ __forceinline__ void end(char* lds) {
        if constexpr (!kDirect) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) *reinterpret_cast<chunk16*>(lds + (j * kThreads + static_cast<int>(threadIdx.x)) * 16) = held[j];
        }
    }
};

// A workgroup of kWavesM x kWavesN waves, each with kM / kWavesM x kN / kWavesN results.
template <class E, bool kAlongM, bool kAlongN, int kM_, int kN_, int kWavesM, int kWavesN, bool kDirect>
struct Product {
    static constexpr int kM = kM_, kN = kN_, kThreads = 64 * kWavesM * kWavesN;
    static constexpr int kTilesM = kM / kWavesM / 16, kTilesN = kN / kWavesN / 16;
    using TileM = OperandTile<E, kAlongM, kM>;
    using TileN = OperandTile<E, kAlongN, kN>;
    static constexpr int kStage = TileM::kSize + TileN::kSize;
    static constexpr int kLds = 2 * kStage;
    static constexpr int kDepth = ProductType<E>::kDepth;

    tile_acc acc[kTilesM][kTilesN];

    __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x / 64); }
    __device__ __forceinline__ static int wave_m() { return wave() / kWavesN * (kM / kWavesM); }
    __device__ __forceinline__ static int wave_n() { return wave() % kWavesN * (kN / kWavesN); }

    __device__ __forceinline__ void multiply_step(const char* lds) {
        const char *const m = lds, *const n = lds + TileM::kSize;
        if constexpr (std::is_same_v<E, split_t>) {
            chunk16 a[kTilesM], b[kTilesN], low[kTilesN];
#pragma unroll
            for (int i = 0; i < kTilesM; ++i) a[i] = TileM::fragment(m, wave_m() + 16 * i, 0);
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) b[j] = TileN::fragment(n, wave_n() + 16 * j, 0);
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) low[j] = TileN::fragment(n, wave_n() + 16 * j, 1);
#pragma unroll
            for (int i = 0; i < kTilesM; ++i)
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) acc[i][j] = multiply<half_t>(a[i], low[j], acc[i][j]);
#pragma unroll
            for (int i = 0; i < kTilesM; ++i) {
                const chunk16 a_low = TileM::fragment(m, wave_m() + 16 * i, 1);
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) acc[i][j] = multiply<half_t>(a_low, b[j], acc[i][j]);
            }
#pragma unroll
            for (int i = 0; i < kTilesM; ++i)
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) acc[i][j] = multiply<half_t>(a[i], b[j], acc[i][j]);
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                chunk16 a[kTilesM], b[kTilesN];
#pragma unroll
                for (int i = 0; i < kTilesM; ++i) a[i] = TileM::fragment(m, wave_m() + 16 * i, q);
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) b[j] = TileN::fragment(n, wave_n() + 16 * j, q);
#pragma unroll
                for (int i = 0; i < kTilesM; ++i)
#pragma unroll
                    for (int j = 0; j < kTilesN; ++j) acc[i][j] = multiply<E>(a[i], b[j], acc[i][j]);
            }
        }
    }

    // `also(lds, step)` may look at each step while it is there.
    template <class F>
    __device__ __forceinline__ void run(char* lds, const Operand& m, const Operand& n, int depth, F&& also) {
#pragma unroll
        for (int i = 0; i < kTilesM; ++i)
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) acc[i][j] = tile_acc{};
        const int steps = (depth + kDepth - 1) / kDepth;
        if (steps == 0) return;
        Loader<E, kAlongM, kM, kThreads, kDirect> load_m(m);
        Loader<E, kAlongN, kN, kThreads, kDirect> load_n(n);
        load_m.begin(lds, 0);
        load_n.begin(lds + TileM::kSize, 0);
        for (int step = 0; step < steps; ++step) {
            char* const here = lds + (step & 1) * kStage;
            char* const next = lds + ((step & 1) ^ 1) * kStage;
            load_m.end(here);
            load_n.end(here + TileM::kSize);
            if constexpr (kDirect) __builtin_amdgcn_s_waitcnt(0x0F70);  // (what this wave's loads bring is there)
            __syncthreads();  // so it is for all of them, and none still reads the other half
            if (step + 1 < steps) {
                load_m.begin(next, step + 1);
                load_n.begin(next + TileM::kSize, step + 1);
            }
            multiply_step(here);
            also(here, step);
        }
    }

    // Calls f(m, n, v) for the results of this lane: v of m .. m + 3 and n, within the tile.
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        const int lane = threadIdx.x % 64;
#pragma unroll
        for (int j = 0; j < kTilesN; ++j)
#pragma unroll
            for (int i = 0; i < kTilesM; ++i) f(wave_m() + 16 * i + lane / 16 * 4, wave_n() + 16 * j + lane % 16, acc[i][j]);
    }
};

// Stores v, of m .. m + 3 of `valid`, rounded once.
template <class E>
__device__ __forceinline__ void store_four(E* p, tile_acc v, int valid, bool aligned) {
    using Four = E __attribute__((ext_vector_type(4)));
    const Four y = __builtin_convertvector(v, Four);
    if (valid >= 4 && aligned) {
        *reinterpret_cast<Four*>(p) = y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = y[i];
    }
}

// The work of a workgroup of `items`.  Consecutive workgroups go to the 8 dies in turn: each die gets neighbouring items, whose operands its cache then holds.
__device__ __forceinline__ uint32_t item_of(uint32_t items) {
    constexpr uint32_t kDies = 8;
    const uint32_t die = blockIdx.x % kDies, each = items / kDies, rest = items % kDies;
    return die * each + min(die, rest) + blockIdx.x / kDies;
}

}  // namespace penc
