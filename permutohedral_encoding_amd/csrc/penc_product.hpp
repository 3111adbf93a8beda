// Matrix products of a workgroup: D[m][n] = sum over k of A[m][k] B[n][k], for a tile of kM x kN results that stay in the registers of its waves.
//
// Operands come in steps of k through the LDS; one or more steps are on their way while one is multiplied, and the fragments of each half of a step are read
// from the LDS while the half before is.  An operand is
//
//     Across   rows of adjacent k: 128 bytes of each row in a step, 64 k of a 16-bit type and 32 of fp32
//     Along    rows of one k, adjacent in m (or n): as many k in a step, transposed on the way from the LDS into registers
//
// 16-bit types are multiplied by v_mfma_f32_16x16x32, fp32 by v_mfma_f32_16x16x4_f32.  A Split number is two halves, hi = the nearest to x and lo = the
// nearest to x - hi (22 bits of x together, where x - hi is no less than 2^-14): of every 32 numbers the hi and behind them the lo, twice 128 bytes in a
// step; a product is hi hi + hi lo + lo hi, and what is left out is 2^-22 of it.
//
// Chunks of 16 bytes go from memory into the LDS directly, where rows and their ends are on 16 bytes.  Where a chunk stands in the LDS is fixed by the lane
// that brings it, so a lane brings the chunk that belongs there.  Addresses behind an operand's end (rows, k, or columns) read zeros, which the buffer's
// bounds see to.  Of rows that begin anywhere, lanes load chunks into registers and write them into the LDS a step later; where a row ends, its last 16
// bytes, of which what the chunk does not have is moved out then.
//
// Where a chunk stands: a read of 16 bytes takes 8 lanes at a time, one of 8 bytes 16 and one of 4 bytes 32, which should meet the 32 banks of 4 bytes once.
// Across: lanes read one chunk c of 8 rows; c stands at c ^ (row mod 8).  Along: 16 lanes read 32 bytes (fp32: 64) of each of 4 neighbouring k (fp32: 32
// lanes of two k, 4 apart); pieces of 32 (64) bytes are permuted by these bits of k.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "penc_kept.hpp"

namespace penc {

struct split_t {
    half_t part;  // (rows are counted in 4 bytes a number; this is what they are made of)
};

template <class E>
struct ProductType {
    static constexpr int kBytes = 2;   // of a number
    static constexpr int kDepth = 64;  // k of a step
    static constexpr int kParts = 1;   // fragments of 16 rows and half a step
};
template <>
struct ProductType<float> {
    static constexpr int kBytes = 4;
    static constexpr int kDepth = 32;
    static constexpr int kParts = 1;
};
template <>
struct ProductType<split_t> {
    static constexpr int kBytes = 4;
    static constexpr int kDepth = 64;
    static constexpr int kParts = 2;
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

constexpr int kMostOperandStride = 1 << 22;  // bytes: 256 rows end before kNowhere
constexpr int kNowhere = 1 << 30;            // behind every buffer's end

// kAlong; kWide: rows (Across) or columns (Along) of the tile.
template <class E, bool kAlong, int kWide>
struct OperandTile {
    using T = ProductType<E>;
    static constexpr int kLine = T::kDepth * T::kBytes;
    static constexpr int kRowBytes = kAlong ? kWide * T::kBytes : kLine;
    static constexpr int kRows = kAlong ? T::kDepth : kWide;
    static constexpr int kSize = kRows * kRowBytes;
    static constexpr int kChunks = kSize / 16, kRowChunks = kRowBytes / 16;

    // where chunk c of a row stands in it
    __device__ __forceinline__ static int place(int row, int c) {
        if constexpr (!kAlong) return c ^ (row & 7);
        else if constexpr (std::is_same_v<E, float>) return c ^ (row >> 2 & 3) << 2;
        else if constexpr (kRowBytes >= 256) return c ^ ((row & 3) | (row >> 3 & 1) << 2) << 1;
        else return c ^ ((row >> 1 & 1) | (row >> 3 & 1) << 1) << 1;
    }

    // 16 rows (columns) from `at` on, of half a step, as the matrix instruction takes them: lane 16 g + i has row i.  Split: hi (part 0) or lo.
    __device__ __forceinline__ static chunk16 fragment(const char* lds, int at, int half, int part) {
        const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
        if constexpr (!kAlong) {
            const int row = at + i;
            return *reinterpret_cast<const chunk16*>(lds + row * kLine + place(row, half * (4 * T::kParts) + part * 4 + g) * 16);
        } else if constexpr (std::is_same_v<E, float>) {
            chunk16 f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = half * 16 + g * 4 + j, column = at + i;
                f[j] = *reinterpret_cast<const uint32_t*>(lds + row * kRowBytes + place(row, column / 4) * 16 + column % 4 * 4);
            }
            return f;
        } else {
            const int byte = (std::is_same_v<E, split_t> ? at / 32 * 128 + at % 32 * 2 + part * 64 : at * 2) + i % 4 * 8;
            using V = short __attribute__((ext_vector_type(4)));
            using Lds = __attribute__((address_space(3))) V;
            chunk16 f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = half * 32 + g * 8 + h * 4 + i / 4;
                const V v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(lds + row * kRowBytes + place(row, byte / 16) * 16 + byte % 16));
                const uint2 w = __builtin_bit_cast(uint2, v);
                f[2 * h] = w.x, f[2 * h + 1] = w.y;
            }
            return f;
        }
    }
};

// 16 bytes to each lane from buffer + at + more, to the LDS from `to` on, lane after lane.  (Not the builtin: of that the compiler knows that it writes to
// the LDS, but not where, and has every read of the LDS wait for it.  It has no result: what it brings is waited for by wait_for_loads.  The wait states are
// those that a scalar register written by a vector instruction needs before it is an address, and M0 before it is used.)
__device__ __forceinline__ void load_to_lds(__attribute__((ext_vector_type(4))) uint32_t buffer, int at, int more, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(to), "v"(at), "s"(buffer), "s"(more) : "memory");
}

// What is the same in all lanes, in a scalar register (the compiler does not see it of all that is computed from a division).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint32_t low = static_cast<uint32_t>(uniform(static_cast<int>(x)));
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(x >> 32)))) << 32 | low);
}

// How chunks come: directly, through registers, or (rows of less than 16 bytes) value by value.
enum class Chunks { kDirect, kHeld, kSingle };

// The last 16 - by of 16 bytes, and zeros behind them (by: a multiple of two).
__device__ __forceinline__ chunk16 to_front(chunk16 m, int by) {
    const bool eight = by & 8, four = by & 4, two = by & 2;
    m = {eight ? m[2] : m[0], eight ? m[3] : m[1], eight ? 0u : m[2], eight ? 0u : m[3]};
    m = {four ? m[1] : m[0], four ? m[2] : m[1], four ? m[3] : m[2], four ? 0u : m[3]};
    if (two) m = {m[0] >> 16 | m[1] << 16, m[1] >> 16 | m[2] << 16, m[2] >> 16 | m[3] << 16, m[3] >> 16};
    return by >= 16 ? chunk16{} : m;
}

// Brings an operand's steps into the LDS, one after the other.
template <class E, bool kAlong, int kWide, int kThreads, Chunks kChunksCome>
struct Loader {
    static constexpr bool kDirect = kChunksCome == Chunks::kDirect;
    using Tile = OperandTile<E, kAlong, kWide>;
    using T = ProductType<E>;
    static constexpr int kEach = Tile::kChunks / kThreads;
    static_assert(Tile::kChunks % kThreads == 0 && kThreads % 128 == 0);

    const char* first;  // of the next step
    int64_t step_bytes;
    int left;           // Across: bytes of a row, Along: rows
    int stride, rest;   // rest: what the buffer has beside: Across: the rows before the last, Along: how much longer a row is than they are apart
    int rows, wide;     // of the operand; bytes of a row (Along)
    // this lane's chunks from `first` on: rows kSameRows apart, where a chunk stands alike in those (else each has its own)
    static constexpr int kSameRows = kThreads / Tile::kRowChunks;
    static constexpr bool kSame = kSameRows % 16 == 0;
    int at[kDirect && !kSame ? kEach : 1];
    int byte;  // Across: in a row
    chunk16 held[kDirect ? 1 : kEach];

    __device__ __forceinline__ static int slot_of(int j) { return j * kThreads + static_cast<int>(threadIdx.x); }
    __device__ __forceinline__ static int row_of(int j) { return slot_of(j) / Tile::kRowChunks; }
    __device__ __forceinline__ static int byte_of(int j) { return Tile::place(row_of(j), slot_of(j) % Tile::kRowChunks) * 16; }

    __device__ __forceinline__ explicit Loader(const Operand& o)
        : first(reinterpret_cast<const char*>(uniform(reinterpret_cast<int64_t>(o.first)))), step_bytes(kAlong ? T::kDepth * uniform(o.stride) : Tile::kLine),
          left(uniform(kAlong ? o.rows : o.bytes)), stride(uniform(static_cast<int>(o.stride))), rest(kAlong ? uniform(o.bytes) - stride : uniform(o.rows - 1) * stride),
          rows(uniform(o.rows)), wide(uniform(o.bytes)), byte(byte_of(0)) {
        static_assert(kAlong || kSameRows % 8 == 0);
        if constexpr (kDirect) {
#pragma unroll
            for (int j = 0; j < (kSame ? 1 : kEach); ++j) at[j] = kAlong && byte_of(j) >= wide ? kNowhere : row_of(j) * stride + byte_of(j);
        }
    }

    // The chunks of the next step are on their way, into the LDS or into registers.
    __device__ __forceinline__ void begin(uint32_t lds) {
        if constexpr (kDirect) {
            const int there = left <= 0 ? 0 : kAlong ? min(left, T::kDepth) * stride + rest : rest + left;
            const uint64_t p = reinterpret_cast<uint64_t>(first);
            const __attribute__((ext_vector_type(4))) uint32_t buffer = {static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32) & 0xFFFFu,
                static_cast<uint32_t>(there), 0x00020000u};
            const uint32_t to = lds + static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / 64)) * 1024;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int from = at[kSame ? 0 : j];
                load_to_lds(buffer, kAlong || byte < left ? from : kNowhere, kSame ? j * kSameRows * stride : 0, to + j * kThreads * 16);
            }
        } else if constexpr (kChunksCome == Chunks::kHeld) {
            // (loads have no conditions: where there is nothing, the operand's last row or a row's last 16 bytes are read)
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                using Unaligned = uint32_t __attribute__((ext_vector_type(4), aligned(T::kBytes == 2 ? 2 : 4)));
                const int row = min(row_of(j), (kAlong ? left : rows) - 1), in_row = min(byte_of(j), (kAlong ? wide : left) - 16);
                held[j] = *reinterpret_cast<const Unaligned*>(first + (static_cast<int64_t>(row) * stride + in_row));
            }
        } else {
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int row = row_of(j), n = (row < (kAlong ? left : rows) ? (kAlong ? wide : left) : 0) - byte_of(j);
                const char* const p = first + static_cast<int64_t>(row) * stride + byte_of(j);
                chunk16 v{};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    if constexpr (T::kBytes == 4) {
                        if (4 * w < n) v[w] = *reinterpret_cast<const uint32_t*>(p + 4 * w);
                    } else {
                        if (4 * w < n) v[w] = *reinterpret_cast<const uint16_t*>(p + 4 * w);
                        if (4 * w + 2 < n) v[w] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 4 * w + 2)) << 16;
                    }
                }
                held[j] = v;
            }
        }
        first += step_bytes;
        left -= kAlong ? T::kDepth : Tile::kLine;
    }
    // What is held goes into the LDS (a barrier makes it so for the other waves).
    __device__ __forceinline__ void end(char* lds) {
        if constexpr (!kDirect) {
            if constexpr (kChunksCome == Chunks::kHeld) {
                const int there = left + (kAlong ? T::kDepth : Tile::kLine);  // as it was
                if (kAlong ? there < T::kDepth || wide < Tile::kRowBytes : there < Tile::kLine) {
#pragma unroll
                    for (int j = 0; j < kEach; ++j) {
                        const int in_row = (kAlong ? wide : there) - byte_of(j);
                        held[j] = to_front(held[j], kAlong && row_of(j) >= there ? 16 : min(max(16 - in_row, 0), 16));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kEach; ++j) *reinterpret_cast<chunk16*>(lds + slot_of(j) * 16) = held[j];
        }
    }
};

// Until all but kLoads of this wave's loads have come (they come in order), and it has read what it asked the LDS for.
template <int kLoads>
__device__ __forceinline__ void wait_for_loads() {
    static_assert(kLoads < 64);
    __builtin_amdgcn_s_waitcnt((kLoads & 15) | 7 << 4 | (kLoads >> 4) << 14);
}

// A workgroup of kWavesM x kWavesN waves, each with kM / kWavesM x kN / kWavesN results; kRing steps have room in the LDS.
template <class E, bool kAlongM, bool kAlongN, int kM_, int kN_, int kWavesM_, int kWavesN_, Chunks kChunksM, int kRing = 2, Chunks kChunksN = kChunksM>
struct Product {
    static constexpr int kWavesM = kWavesM_, kWavesN = kWavesN_;
    static constexpr int kM = kM_, kN = kN_, kThreads = 64 * kWavesM * kWavesN;
    static constexpr int kTilesM = kM / kWavesM / 16, kTilesN = kN / kWavesN / 16;
    using TileM = OperandTile<E, kAlongM, kM>;
    using TileN = OperandTile<E, kAlongN, kN>;
    static constexpr bool kDirect = kChunksM == Chunks::kDirect;
    static_assert(kDirect == (kChunksN == Chunks::kDirect));
    using LoadM = Loader<E, kAlongM, kM, kThreads, kChunksM>;
    using LoadN = Loader<E, kAlongN, kN, kThreads, kChunksN>;
    static constexpr int kStage = TileM::kSize + TileN::kSize;
    static constexpr int kLds = kRing * kStage;
    static constexpr int kDepth = ProductType<E>::kDepth, kParts = ProductType<E>::kParts;
    static constexpr int kLoads = LoadM::kEach + LoadN::kEach;  // of a lane, for a step

    // What a wave multiplies in half a step.
    struct Fragments {
        chunk16 m[kParts][kTilesM], n[kParts][kTilesN];

        __device__ __forceinline__ void read(const char* lds, int half) {
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) n[p][j] = TileN::fragment(lds + TileM::kSize, wave_n() + 16 * j, half, p);
#pragma unroll
                for (int i = 0; i < kTilesM; ++i) m[p][i] = TileM::fragment(lds, wave_m() + 16 * i, half, p);
            }
        }
    };

    // Reads of the LDS of half a step, and products.
    template <bool kAlong>
    static constexpr int kReadsOf = !kAlong ? 1 : std::is_same_v<E, float> ? 4 : 2;
    static constexpr int kReads = kParts * (kTilesM * kReadsOf<kAlongM> + kTilesN * kReadsOf<kAlongN>);
    static constexpr int kProducts = kTilesM * kTilesN * (kParts == 2 ? 3 : std::is_same_v<E, float> ? 4 : 1);
    // A wave issues in order: reads of the LDS, which all waves begin at the same time, are spread over the products, which go on meanwhile.
    template <size_t... kRead>
    __device__ __forceinline__ static void alternate(std::index_sequence<kRead...>) {
        ((__builtin_amdgcn_sched_group_barrier(0x008, (kRead + 1) * kProducts / kReads - kRead * kProducts / kReads, 0),
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0)), ...);
    }

    tile_acc acc[kTilesM][kTilesN];

    __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x / 64); }
    __device__ __forceinline__ static int wave_m() { return wave() / kWavesN * (kM / kWavesM); }
    __device__ __forceinline__ static int wave_n() { return wave() % kWavesN * (kN / kWavesN); }

    // Sums of products with a lo, 2^-11 of the others: on their own they round as much less, and the others a third as often.
    tile_acc low[kParts == 2 ? kTilesM : 1][kParts == 2 ? kTilesN : 1];

    template <int kI, int kJ>
    __device__ __forceinline__ static void multiply_all(const chunk16 (&m)[kTilesM], const chunk16 (&n)[kTilesN], tile_acc (&to)[kI][kJ]) {
        using Part = std::conditional_t<std::is_same_v<E, split_t>, half_t, E>;
#pragma unroll
        for (int i = 0; i < kTilesM; ++i)
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) to[i][j] = multiply<Part>(m[i], n[j], to[i][j]);
    }
    __device__ __forceinline__ void multiply_half(const Fragments& f) {
        if constexpr (kParts == 2) {
            multiply_all(f.m[0], f.n[1], low);
            multiply_all(f.m[1], f.n[0], low);
        }
        multiply_all(f.m[0], f.n[0], acc);
    }
    __device__ __forceinline__ void add_low() {
        if constexpr (kParts == 2) {
#pragma unroll
            for (int i = 0; i < kTilesM; ++i)
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) acc[i][j] += low[i][j];
        }
    }

    // Where the sums begin: f(m), for the four results from m on, of every n.
    template <class F>
    __device__ __forceinline__ void start(F&& f) {
#pragma unroll
        for (int i = 0; i < kTilesM; ++i) {
            const tile_acc v = f(wave_m() + 16 * i + static_cast<int>(threadIdx.x) % 64 / 16 * 4);
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) {
                acc[i][j] = v;
                if constexpr (kParts == 2) low[i][j] = tile_acc{};
            }
        }
    }
    static constexpr auto kZero = [](int) { return tile_acc{}; };
    static constexpr auto kNothing = [](const auto&) {};

    // The sums begin at first(m).  `also(n)` may look at the fragments of N of each step.
    template <class First, class F>
    __device__ __forceinline__ void run(char* lds, const Operand& m, const Operand& n, int depth, First&& first, F&& also) {
        const int steps = (depth + kDepth - 1) / kDepth;
        if (steps == 0) return start(first);
        LoadM load_m(m);
        LoadN load_n(n);
        // Steps behind the last one are loaded too, and are zeros: each wave always has as many loads on their way.
        const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
        int room = 0, here = 0;  // where the next step goes, and the present one is
        const auto behind = [](int at) { return at + kStage == kLds ? 0 : at + kStage; };
        const auto begin = [&] {
            load_m.begin(lds_at + room);
            load_n.begin(lds_at + room + TileM::kSize);
            if constexpr (kDirect) room = behind(room);
        };
        const auto end = [&] {
            load_m.end(lds + room);
            load_n.end(lds + room + TileM::kSize);
            room = behind(room);
        };
        const auto meet = [&] {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        };
        if constexpr (kDirect) {
#pragma unroll
            for (int k = 0; k < kRing; ++k) begin();
            start(first);
            wait_for_loads<kLoads * (kRing - 1)>();
        } else {
            static_assert(kRing == 2);
            begin();
            start(first);
            end();
            begin();
        }
        meet();
        Fragments even, odd;
        even.read(lds, 0);
        const auto turn = [&](const Fragments& now, Fragments& next, const char* from, int half) {
            __builtin_amdgcn_sched_barrier(0);
            next.read(from, half);
            multiply_half(now);
            also(now.n[0]);
            alternate(std::make_index_sequence<kReads>{});
            __builtin_amdgcn_sched_barrier(0);
        };
        for (int step = 1; step < steps; ++step) {
            turn(even, odd, lds + here, 1);
            // What is brought for the next step is there for all waves, and all have read the second half of this one, whose room the step kRing behind it
            // takes.
            if constexpr (kDirect) wait_for_loads<kLoads * (kRing - 2)>();
            else end();
            meet();
            begin();
            here = behind(here);
            turn(odd, even, lds + here, 0);
        }
        turn(even, odd, lds + here, 1);
        multiply_half(odd);
        also(odd.n[0]);
        add_low();
        if constexpr (kDirect) wait_for_loads<0>();  // (nothing is on its way into the LDS when the workgroup ends)
    }

    // Calls f(m, n, v) for eight results m .. m + 7 of n at a time: lanes 16 apart have four neighbouring m each, and exchange those of two tiles.
    template <class F>
    __device__ __forceinline__ void each_eight(F&& f) const {
        static_assert(kTilesM % 2 == 0);
        using Eight = float __attribute__((ext_vector_type(8)));
        const int lane = threadIdx.x % 64, g = lane / 16;
#pragma unroll
        for (int j = 0; j < kTilesN; ++j)
#pragma unroll
            for (int i = 0; i < kTilesM; i += 2) {
                Eight v;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][r]), __float_as_uint(acc[i + 1][j][r]), false, false);
                    v[r] = __uint_as_float(x[0]), v[4 + r] = __uint_as_float(x[1]);
                }
                f(wave_m() + 16 * (i + g % 2) + g / 2 * 8, wave_n() + 16 * j + lane % 16, v);
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

// Stores the first `valid` of kWide values, wherever they are.
template <class E, int kWide>
__device__ __forceinline__ void store_values(E* p, E __attribute__((ext_vector_type(kWide))) v, int valid) {
    using Unaligned = E __attribute__((ext_vector_type(kWide), aligned(sizeof(E))));
    if (valid >= kWide) {
        *reinterpret_cast<Unaligned*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < kWide; ++i)
            if (i < valid) p[i] = v[i];
    }
}

// Stores a workgroup's results as rows of n, `stride` values apart: `rows` of them and `columns` of m, rounded once.
// 16-bit results: lanes 16 apart have four neighbouring m each, of one n; they exchange those of two tiles, and each stores eight of one of them.
template <class E, class P>
__device__ __forceinline__ void store_rows(const P& p, E* out, int64_t stride, int rows, int columns) {
    using Four = E __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(E) == 2 && P::kTilesM % 2 == 0) {
        using Eight = E __attribute__((ext_vector_type(8)));
        const int lane = threadIdx.x % 64, g = lane / 16;
#pragma unroll
        for (int j = 0; j < P::kTilesN; ++j) {
            const int n = P::wave_n() + 16 * j + lane % 16;
#pragma unroll
            for (int i = 0; i < P::kTilesM; i += 2) {
                const uint2 a = __builtin_bit_cast(uint2, __builtin_convertvector(p.acc[i][j], Four)),
                    b = __builtin_bit_cast(uint2, __builtin_convertvector(p.acc[i + 1][j], Four));
                const auto x = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false), y = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
                const int m = P::wave_m() + 16 * (i + g % 2) + g / 2 * 8;
                if (n < rows && m < columns) store_values<E, 8>(out + n * stride + m, __builtin_bit_cast(Eight, make_uint4(x[0], y[0], x[1], y[1])), columns - m);
            }
        }
    } else {
        p.each([&](int m, int n, tile_acc v) {
            if (n < rows && m < columns) store_values<E, 4>(out + n * stride + m, __builtin_convertvector(v, Four), columns - m);
        });
    }
}

// How items are spread over a launch.  Consecutive workgroups go to the 8 dies in turn; each die gets `run` neighbouring items at a time, whose operands its
// cache then holds, and all of them go through the items alike: items take different times, and of some there is nothing to do.
struct Spread {
    uint32_t items, run;
    static constexpr uint32_t kDies = 8;

    Spread() = default;
    Spread(int64_t n, int64_t most) : items(static_cast<uint32_t>(n)), run(static_cast<uint32_t>(std::max<int64_t>(1, std::min((n + kDies - 1) / kDies, most)))) {}
    uint32_t grid() const { return (items + kDies * run - 1) / (kDies * run) * (kDies * run); }
    __device__ __forceinline__ uint32_t item() const {
        const uint32_t at = blockIdx.x / kDies;
        return (at / run * kDies + blockIdx.x % kDies) * run + at % run;
    }
};

}  // namespace penc
