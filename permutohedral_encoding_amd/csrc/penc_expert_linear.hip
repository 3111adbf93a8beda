// A linear layer of each expert on its own rows, of rows sorted by expert: for offsets[e] <= r < offsets[e + 1]
//
//     y[r][o] = sum over c of W[e][o][c] x[r][c] + b[e][o],      dx[r][c] = sum over o of W[e][o][c] dy[r][o],
//     dW[e][o][c] = sum over these r of dy[r][o] x[r][c],        db[e][o] = sum of dy[r][o].
//
// Which rows a workgroup has it finds from the offsets, which are on the device: tiles of rows do not cross from one expert to the next, and the grid has
// room for one tile of each expert that is not full.  Rows behind the last expert's are zero in y and dx and not read otherwise.
//
// The type of values (PENC_TYPE: those of penc.h) is one compilation each.
#include <algorithm>
#include <cmath>

#include "penc_expert_linear.hpp"
#include "penc_product.hpp"

#ifndef PENC_TYPE
#error "PENC_TYPE: PENC_FP32, PENC_FP16 or PENC_BF16"
#endif

namespace penc {
namespace {

using Value = std::conditional_t<PENC_TYPE == PENC_FP32, float, std::conditional_t<PENC_TYPE == PENC_FP16, half_t, bf16_t>>;
constexpr int kSize = sizeof(Value);
static_assert(PENC_MAX_EXPERT_STRIDE * kSize <= kMostOperandStride && PENC_MAX_EXPERT_CHANNELS * kSize <= kMostOperandStride);

// The sum of a wave's values up to each lane.
__device__ __forceinline__ uint32_t sum_to_lane(uint32_t v) {
    const auto moved = [](uint32_t x, auto control, auto rows) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(control)::value, decltype(rows)::value, 0xF, false));
    };
    constexpr std::integral_constant<int, 0xF> all{};
    v += moved(v, std::integral_constant<int, 0x111>{}, all);  // from 1, 2, 4 and 8 lanes before, of 16
    v += moved(v, std::integral_constant<int, 0x112>{}, all);
    v += moved(v, std::integral_constant<int, 0x114>{}, all);
    v += moved(v, std::integral_constant<int, 0x118>{}, all);
    v += moved(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // the last of 16 lanes to the next 16
    v += moved(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // the last of 32 to the others
    return v;
}

// Tile `t` of rows: those of an expert (`experts`: the rows behind the last one's), cut every `most` rows.
struct RowTile {
    int expert, first, rows, tiles;  // tiles: the expert's; expert < 0: there is no such tile
    int64_t slot;                    // pieces: which it is of those of experts with several, whose sums go through memory
};

// All lanes of a wave call it.  kWhole: tiles of the rows behind the last expert's too; else each expert has a tile at least, be it one of no rows.
template <bool kWhole>
__device__ __forceinline__ RowTile row_tile(const int32_t* __restrict__ offsets, int experts, int rows, uint32_t t, int most) {
    const int lane = threadIdx.x % 64;
    uint32_t before = 0, cut_before = 0;
    for (int base = 0; base < experts + (kWhole ? 1 : 0); base += 64) {
        const int e = base + lane;
        int from = 0, to = 0;
        if (e <= experts) from = min(max(offsets[e], 0), rows);
        if (e < experts) to = min(max(offsets[e + 1], 0), rows);
        else if (kWhole && e == experts) to = rows;
        const int n = max(to - from, 0);
        uint32_t tiles = (static_cast<uint32_t>(n) + most - 1) / most;
        if (!kWhole && e < experts) tiles = max(tiles, 1u);
        if (e > experts || (!kWhole && e == experts)) tiles = 0;
        const uint32_t cut = !kWhole && tiles > 1 ? tiles : 0u;
        const uint32_t sum = sum_to_lane(tiles), sum_of_cut = kWhole ? 0u : sum_to_lane(cut);
        const uint64_t behind = __ballot(t < before + sum);
        if (behind != 0) {
            const int found = __builtin_ctzll(behind);
            const auto its_own = [&](int v) { return __builtin_amdgcn_readlane(v, found); };
            const int first = its_own(from), count = its_own(n);
            const uint32_t its = its_own(tiles), at = t - before - (its_own(sum) - its);
            // (tiles of rows are full but for the last one; pieces for the weights' gradient are alike)
            const int each = kWhole ? most : (count / static_cast<int>(its) / 64 + 1) * 64, skip = min(static_cast<int>(at) * each, count);
            return {base + found, first + skip, min(count - skip, each), static_cast<int>(its),
                    int64_t{cut_before} + static_cast<uint32_t>(its_own(sum_of_cut)) - static_cast<uint32_t>(its_own(cut)) + at};
        }
        before += __builtin_amdgcn_readlane(sum, 63), cut_before += __builtin_amdgcn_readlane(sum_of_cut, 63);
    }
    return {-1, 0, 0, 0, 0};
}

// Piece `t` of all experts' (row_tile<false>), the largest pieces first, in classes of an eighth of `most`: workgroups that begin last are short then.
// (dW in the experts' order and so, experts in uneven demand: 32768 x 1024 by 4096 bf16 of 16 experts 363 and 306 us, 65536 x 512 by 2048 bf16 of 32 198 and
// 175, 32768 x 1024 by 1024 fp32 of 16 723 and 570; 131072 x 1024 by 1024 bf16 of 8, which are cut for whole rounds, 347 and 340, 50000 x 512 by 512 fp32 of
// 20 247 and 242.)  For the experts of a wave's lanes; more of them have more pieces than matter.
__device__ __forceinline__ RowTile row_tile_by_size(const int32_t* __restrict__ offsets, int experts, int rows, uint32_t t, int most) {
    if (experts > 64) return row_tile<false>(offsets, experts, rows, t, most);
    const int lane = threadIdx.x % 64, from = lane < experts ? min(max(offsets[lane], 0), rows) : 0, to = lane < experts ? min(max(offsets[lane + 1], 0), rows) : 0;
    const int n = max(to - from, 0);
    const uint32_t tiles = lane < experts ? max((static_cast<uint32_t>(n) + most - 1) / most, 1u) : 0u, cut = tiles > 1 ? tiles : 0u, cut_before = sum_to_lane(cut) - cut;
    const int each = tiles > 0 ? (n / static_cast<int>(tiles) / 64 + 1) * 64 : 0, size = static_cast<int>(static_cast<int64_t>(each) * 8 / most);  // 0 to 9
    uint32_t done = 0;
    for (int s = 9; s >= 0; --s) {
        const uint32_t mine = size == s ? tiles : 0u, sum = sum_to_lane(mine);
        const uint64_t here = __ballot(t >= done && t < done + sum);
        if (here != 0) {
            const int found = __builtin_ctzll(here);
            const auto its_own = [&](uint32_t v) { return static_cast<int>(__builtin_amdgcn_readlane(static_cast<int>(v), found)); };
            const int its = its_own(tiles), at = static_cast<int>(t - done) - (its_own(sum) - its), rows_each = its_own(each), count = its_own(n),
                skip = min(at * rows_each, count);
            return {found, its_own(from) + skip, min(count - skip, rows_each), its, int64_t{static_cast<uint32_t>(its_own(cut_before))} + at};
        }
        done += __builtin_amdgcn_readlane(static_cast<int>(sum), 63);
    }
    return {-1, 0, 0, 0, 0};
}

// How many tiles row_tile<true> has.
__device__ __forceinline__ uint32_t row_tiles(const int32_t* __restrict__ offsets, int experts, int rows, int most) {
    const int lane = threadIdx.x % 64;
    uint32_t tiles = 0;
    for (int e = lane; e <= experts; e += 64) {
        const int from = min(max(offsets[e], 0), rows), to = e < experts ? min(max(offsets[e + 1], 0), rows) : rows;
        tiles += (static_cast<uint32_t>(max(to - from, 0)) + most - 1) / most;
    }
    return __builtin_amdgcn_readlane(sum_to_lane(tiles), 63);
}

constexpr uint32_t kUnits = 256;  // compute units

struct RowsArgs {
    const void *rows_in, *weight, *bias;
    void* rows_out;
    int64_t stride;                // of rows_in, in values
    const int32_t* offsets;
    int experts, rows, wide, deep; // wide: values of a row of the result; deep: of the operand
    Spread spread;
    uint32_t tiles;                // of a row of the result
};

constexpr uint32_t kGroup = 8;

// A tile of results: those of P::kN rows from `skip` rows into t on, and P::kM columns from m0 on.
template <bool kBack, class P>
__device__ __forceinline__ void rows_tile(const RowsArgs& a, char* lds, const RowTile& t, int skip, int m0) {
    P p;
    const int columns = a.wide - m0, first_row = t.first + skip, rows = t.rows - skip;
    if (t.expert == a.experts) {
        p.start(P::kZero);
    } else {
        const Value* const bias = !kBack && a.bias != nullptr ? static_cast<const Value*>(a.bias) + static_cast<int64_t>(t.expert) * a.wide + m0 : nullptr;
        const char* const weight = static_cast<const char*>(a.weight) + static_cast<int64_t>(t.expert) * a.wide * a.deep * kSize;
        const int m_rows = min(columns, P::kM);
        const Operand m = kBack ? Operand{weight + static_cast<int64_t>(m0) * kSize, static_cast<int64_t>(a.wide) * kSize, a.deep, m_rows * kSize}
                                : Operand{weight + static_cast<int64_t>(m0) * a.deep * kSize, static_cast<int64_t>(a.deep) * kSize, m_rows, a.deep * kSize};
        const Operand n{static_cast<const char*>(a.rows_in) + static_cast<int64_t>(first_row) * a.stride * kSize, a.stride * kSize, min(rows, P::kN), a.deep * kSize};
        const auto first = [&](int m) {
            tile_acc v{};
            if (bias != nullptr) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = m + k < columns ? static_cast<float>(bias[m + k]) : 0.0f;
            }
            return v;
        };
        p.run(lds, m, n, a.deep, first, P::kNothing);
    }
    store_rows(p, static_cast<Value*>(a.rows_out) + static_cast<int64_t>(first_row) * a.wide + m0, a.wide, rows, columns);
}

// kSplit: with as many tiles as compute units, or twice or three times as many, and a few more, those few take as long as all before them; where the last
// round has at most half of the compute units, its tiles go in quarters, which then are one round or two of a third of the time (32768 x 4096 by 1024 bf16,
// 544 tiles: 310 -> 250 us).
template <bool kBack, class P, class Quarter>
__global__ __launch_bounds__(P::kThreads) void expert_rows_kernel(RowsArgs a) {
    constexpr bool kSplit = !std::is_same_v<P, Quarter>;
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    const uint32_t item = a.spread.item();
    if (item >= a.spread.items) return;
    uint32_t tile = item, quarter = 0, tiles = a.spread.items;
    bool whole = true;
    if constexpr (kSplit) {
        static_assert(Quarter::kM * 2 == P::kM && Quarter::kN * 2 == P::kN && Quarter::kThreads == P::kThreads && Quarter::kLds <= P::kLds);
        tiles = row_tiles(a.offsets, a.experts, a.rows, P::kN) * a.tiles;
        const uint32_t last = tiles % kUnits;
        if (last <= kUnits / 2 && item >= tiles - last) {
            whole = false;
            tile = tiles - last + (item - (tiles - last)) / 4, quarter = (item - (tiles - last)) % 4;
        }
        if (tile >= tiles) return;
    }
    // eight tiles of rows to each tile of weights, one after the other: what a die works on at a time fits its cache
    const uint32_t of_group = kGroup * a.tiles, group = tile / of_group, in_group = tile % of_group, grouped = min(kGroup, tiles / a.tiles - group * kGroup);
    const RowTile t = row_tile<true>(a.offsets, a.experts, a.rows, group * kGroup + in_group % grouped, P::kN);
    if (t.expert < 0) return;
    const int m0 = static_cast<int>(in_group / grouped) * P::kM;
    if (whole) {
        rows_tile<kBack, P>(a, lds, t, 0, m0);
    } else {
        const int skip = static_cast<int>(quarter / 2) * Quarter::kN, m1 = m0 + static_cast<int>(quarter % 2) * Quarter::kM;
        if (skip < t.rows && m1 < a.wide) rows_tile<kBack, Quarter>(a, lds, t, skip, m1);
    }
}

// ------------------------------------------------------------------------------------------
// narrow layers, and few rows

// 16 bytes of a buffer, zeros behind its end.
__device__ __forceinline__ chunk16 load_chunk16(__amdgpu_buffer_rsrc_t buffer, int at) {
    return __builtin_bit_cast(chunk16, __builtin_amdgcn_raw_buffer_load_b128(buffer, at, 0, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const char* first, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(first), 0, static_cast<int>(min(max(bytes, int64_t{0}), int64_t{0x7FFFFFFF})), 0x00020000);
}

// Stores what a wave has of 16 rows (v[t]: four of 16 results to a lane), `columns` of each.
template <class E, int kTiles>
__device__ __forceinline__ void store_sixteen_rows(const tile_acc (&v)[kTiles], E* out, int64_t stride, int rows, int columns) {
    using Four = E __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x % 64, n = lane % 16, g = lane / 16;
    if constexpr (sizeof(E) == 2 && kTiles % 2 == 0) {
        using Eight = E __attribute__((ext_vector_type(8)));
#pragma unroll
        for (int t = 0; t < kTiles; t += 2) {
            const uint2 a = __builtin_bit_cast(uint2, __builtin_convertvector(v[t], Four)), b = __builtin_bit_cast(uint2, __builtin_convertvector(v[t + 1], Four));
            const auto x = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false), y = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
            const int m = 16 * (t + g % 2) + g / 2 * 8;
            if (n < rows && m < columns) store_values<E, 8>(out + n * stride + m, __builtin_bit_cast(Eight, make_uint4(x[0], y[0], x[1], y[1])), columns - m);
        }
    } else {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int m = 16 * t + g * 4;
            if (n < rows && m < columns) store_values<E, 4>(out + n * stride + m, __builtin_convertvector(v[t], Four), columns - m);
        }
    }
}

constexpr int kNarrowThreads = 256, kNarrowLines = 4, kNarrowTiles = 4;  // 64 results of 256 bytes
constexpr int kNarrowGroups = kSize == 2 ? 2 : 1;                       // of 16 rows that a wave has at a time

// Layers whose weights fit a wave's registers: at most 64 results of rows of at most 256 bytes.  The weights come through the LDS once; then waves walk over
// rows, 16 (or twice 16) at a time, straight from memory into the fragments' registers, the next ones on their way.
template <bool kBack, int kLines, int kTiles>
__global__ __launch_bounds__(kNarrowThreads) void expert_narrow_kernel(RowsArgs a, int most) {
    using Load = Loader<Value, kBack, 64, kNarrowThreads, Chunks::kDirect>;
    using Tile = typename Load::Tile;
    static_assert(kLines % 2 == 0);
    __shared__ __attribute__((aligned(1024))) char lds[kLines / 2 * Tile::kSize];
    const uint32_t item = a.spread.item();
    if (item >= a.spread.items) return;
    const RowTile t = row_tile<true>(a.offsets, a.experts, a.rows, item, most);
    if (t.expert < 0) return;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    Value* const out = static_cast<Value*>(a.rows_out) + static_cast<int64_t>(t.first) * a.wide;
    constexpr int kStep = 16 * kNarrowGroups * kNarrowThreads / 64;
    if (t.expert == a.experts) {
        const tile_acc zero[kTiles] = {};
        for (int row = wave * 16; row < t.rows; row += 16 * kNarrowThreads / 64)
            store_sixteen_rows(zero, out + static_cast<int64_t>(row) * a.wide, a.wide, t.rows - row, a.wide);
        return;
    }
    const char* const weight = static_cast<const char*>(a.weight) + static_cast<int64_t>(t.expert) * a.wide * a.deep * kSize;
    Load load(kBack ? Operand{weight, static_cast<int64_t>(a.wide) * kSize, a.deep, a.wide * kSize}
                    : Operand{weight, static_cast<int64_t>(a.deep) * kSize, a.wide, a.deep * kSize});
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
#pragma unroll
    for (int l = 0; l < kLines / 2; ++l) load.begin(lds_at + l * Tile::kSize);

    // this lane's chunks of a row, and of the rows of a group
    const int deep_bytes = a.deep * kSize, stride = static_cast<int>(a.stride) * kSize;
    int at[kLines];
#pragma unroll
    for (int l = 0; l < kLines; ++l) {
        const int byte = l * 64 + lane / 16 * 16;
        at[l] = byte < deep_bytes ? lane % 16 * stride + byte : kNowhere;
    }
    const char* const in = static_cast<const char*>(a.rows_in) + static_cast<int64_t>(t.first) * a.stride * kSize;
    chunk16 rows[kNarrowGroups][kLines], next[kNarrowGroups][kLines];
    const auto begin = [&](chunk16 (&r)[kNarrowGroups][kLines], int row) {
#pragma unroll
        for (int k = 0; k < kNarrowGroups; ++k) {
            const int first = row + 16 * k, left = t.rows - first;
            const auto buffer = buffer_of(in + static_cast<int64_t>(first) * stride, left <= 0 ? 0 : (min(left, 16) - 1) * stride + deep_bytes);
#pragma unroll
            for (int l = 0; l < kLines; ++l) r[k][l] = load_chunk16(buffer, at[l]);
        }
    };
    int row = wave * 16 * kNarrowGroups;
    begin(next, row);
    tile_acc bias[kTiles] = {};
    if (!kBack && a.bias != nullptr) {
        const Value* const from = static_cast<const Value*>(a.bias) + static_cast<int64_t>(t.expert) * a.wide;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int m = 16 * i + lane / 16 * 4 + k;
                bias[i][k] = m < a.wide ? static_cast<float>(from[m]) : 0.0f;
            }
    }
    wait_for_loads<0>();
    __syncthreads();
    chunk16 w[kTiles][kLines];
#pragma unroll
    for (int l = 0; l < kLines; ++l)
#pragma unroll
        for (int i = 0; i < kTiles; ++i) w[i][l] = Tile::fragment(lds + l / 2 * Tile::kSize, 16 * i, l % 2, 0);
    for (; row < t.rows; row += kStep) {
#pragma unroll
        for (int k = 0; k < kNarrowGroups; ++k)
#pragma unroll
            for (int l = 0; l < kLines; ++l) rows[k][l] = next[k][l];
        begin(next, row + kStep);
#pragma unroll
        for (int k = 0; k < kNarrowGroups; ++k) {
            tile_acc acc[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) acc[i] = bias[i];
#pragma unroll
            for (int l = 0; l < kLines; ++l)
#pragma unroll
                for (int i = 0; i < kTiles; ++i) acc[i] = multiply<Value>(w[i][l], rows[k][l], acc[i]);
            const int first = row + 16 * k;
            store_sixteen_rows(acc, out + static_cast<int64_t>(first) * a.wide, a.wide, t.rows - first, a.wide);
        }
    }
}

constexpr int kFewRows = 16, kFewOutputs = 64, kFewThreads = 256, kFewWaves = kFewThreads / 64;

// A few rows of an expert, whose weights are what there is to read: 64 outputs of 16 rows to a workgroup, whose waves take each fourth line of 64 bytes of
// all of them straight into the fragments' registers, four lines on their way, and add their sums in order.
__global__ __launch_bounds__(kFewThreads) void expert_few_kernel(RowsArgs a) {
    constexpr int kTiles = kFewOutputs / 16, kAhead = 4;
    __shared__ tile_acc lds[kFewWaves - 1][kTiles][64];
    const uint32_t item = a.spread.item();
    if (item >= a.spread.items) return;
    const RowTile t = row_tile<true>(a.offsets, a.experts, a.rows, item / a.tiles, kFewRows);
    if (t.expert < 0) return;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), m0 = static_cast<int>(item % a.tiles) * kFewOutputs,
        columns = a.wide - m0;
    tile_acc acc[kTiles] = {};
    if (t.expert < a.experts) {
        const int deep_bytes = a.deep * kSize, stride = static_cast<int>(a.stride) * kSize;
        const auto weights = buffer_of(static_cast<const char*>(a.weight) + (static_cast<int64_t>(t.expert) * a.wide + m0) * deep_bytes,
            static_cast<int64_t>(min(columns, kFewOutputs)) * deep_bytes);
        const auto rows = buffer_of(static_cast<const char*>(a.rows_in) + static_cast<int64_t>(t.first) * stride, static_cast<int64_t>(t.rows - 1) * stride + deep_bytes);
        const int w_at = lane % 16 * deep_bytes + lane / 16 * 16, x_at = lane % 16 * stride + lane / 16 * 16;
        for (int first = wave * 64; first < deep_bytes; first += kAhead * kFewWaves * 64) {
            chunk16 w[kAhead][kTiles], x[kAhead];
#pragma unroll
            for (int l = 0; l < kAhead; ++l) {
                const int byte = first + l * kFewWaves * 64;
                const bool there = byte + lane / 16 * 16 < deep_bytes;
                x[l] = load_chunk16(rows, there ? x_at + byte : kNowhere);
#pragma unroll
                for (int i = 0; i < kTiles; ++i) w[l][i] = load_chunk16(weights, there ? w_at + 16 * i * deep_bytes + byte : kNowhere);
            }
#pragma unroll
            for (int l = 0; l < kAhead; ++l)
#pragma unroll
                for (int i = 0; i < kTiles; ++i) acc[i] = multiply<Value>(w[l][i], x[l], acc[i]);
        }
    }
    if (wave > 0) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) lds[wave - 1][i][lane] = acc[i];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
        for (int k = 0; k < kFewWaves - 1; ++k) acc[i] += lds[k][i][lane];
        if (a.bias != nullptr && t.expert < a.experts) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int m = m0 + 16 * i + lane / 16 * 4 + k;
                if (m < a.wide) acc[i][k] += static_cast<float>(static_cast<const Value*>(a.bias)[static_cast<int64_t>(t.expert) * a.wide + m]);
            }
        }
    }
    store_sixteen_rows(acc, static_cast<Value*>(a.rows_out) + static_cast<int64_t>(t.first) * a.wide + m0, a.wide, t.rows, columns);
}

struct WeightArgs {
    const void *x, *grad;
    int64_t x_stride, grad_stride;
    const int32_t* offsets;
    int experts, rows, channels, outputs, most;  // most: rows of a piece
    Spread spread;
    uint32_t channel_tiles, tiles;
    void *weight, *bias;  // results, written where an expert's rows are one piece
    float* sums;          // [slots][outputs][channels], and behind them [slots][outputs]: of pieces of experts with several
    int64_t slots;
};

// A wave's sums of dy itself: of 16-bit types its products with ones, of fp32, whose products take eight times as long, each lane's own k, in 64 bits.
template <int kTilesN>
struct BiasGrads {
    static constexpr bool kWide = PENC_TYPE == PENC_FP32;
    tile_acc acc[kWide ? 1 : kTilesN] = {};
    double wide[kWide ? kTilesN : 1] = {};

    __device__ __forceinline__ void add(const chunk16 (&grad)[kTilesN]) {
        const uint32_t one = PENC_TYPE == PENC_FP16 ? 0x3C003C00u : 0x3F803F80u;
        const chunk16 ones = {one, one, one, one};
#pragma unroll
        for (int j = 0; j < kTilesN; ++j) {
            const auto value = [&](int k) { return __uint_as_float(grad[j][k]); };
            if constexpr (kWide) wide[j] += static_cast<double>((value(0) + value(1)) + (value(2) + value(3)));
            else acc[j] = multiply<Value>(ones, grad[j], acc[j]);
        }
    }
    // The sum of tile j, where lanes 16 apart have a part each (fp32; of 16-bit types all have all).
    __device__ __forceinline__ float sum(int j) const {
        if constexpr (kWide) {
            double v = wide[j];
            v += __shfl_xor(v, 16);
            v += __shfl_xor(v, 32);
            return static_cast<float>(v);
        } else {
            return acc[j][0];
        }
    }
};

// Stores what a workgroup has of dW, and the waves with `bias` of db: the results where the expert's rows are one piece, else the piece's sums.
template <class P>
__device__ __forceinline__ void store_weight_grads(const WeightArgs& a, const RowTile& t, int c0, int o0, const P& p, bool bias, const BiasGrads<P::kTilesN>& of_bias) {
    const int64_t n_weights = static_cast<int64_t>(a.outputs) * a.channels;
    const bool whole = t.tiles == 1;
    const int64_t at = static_cast<int64_t>(o0) * a.channels + c0;
    if (whole) store_rows(p, static_cast<Value*>(a.weight) + t.expert * n_weights + at, a.channels, a.outputs - o0, a.channels - c0);
    else store_rows(p, a.sums + t.slot * n_weights + at, a.channels, a.outputs - o0, a.channels - c0);
    if (!bias) return;
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int j = 0; j < P::kTilesN; ++j) {
        const float sum = of_bias.sum(j);
        const int o = o0 + P::wave_n() + 16 * j + lane;
        if (lane >= 16 || o >= a.outputs) continue;
        if (whole) static_cast<Value*>(a.bias)[static_cast<int64_t>(t.expert) * a.outputs + o] = static_cast<Value>(sum);
        else a.sums[a.slots * n_weights + t.slot * a.outputs + o] = sum;
    }
}

// dW and db of a piece of an expert's rows.
template <class P>
__global__ __launch_bounds__(P::kThreads) void expert_weights_kernel(WeightArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    const uint32_t item = a.spread.item(), tile = item % a.tiles;
    if (item >= a.spread.items) return;
    const RowTile t = row_tile_by_size(a.offsets, a.experts, a.rows, item / a.tiles, a.most);
    if (t.expert < 0 || (t.tiles > 1 && t.slot >= a.slots)) return;  // (the second: offsets that no plan has)
    const int c0 = static_cast<int>(tile % a.channel_tiles) * P::kM, o0 = static_cast<int>(tile / a.channel_tiles) * P::kN;
    const bool bias = a.bias != nullptr && c0 == 0 && P::wave_m() == 0;
    const Operand m{static_cast<const char*>(a.x) + (static_cast<int64_t>(t.first) * a.x_stride + c0) * kSize, a.x_stride * kSize, t.rows,
        min(a.channels - c0, P::kM) * kSize};
    const Operand n{static_cast<const char*>(a.grad) + (static_cast<int64_t>(t.first) * a.grad_stride + o0) * kSize, a.grad_stride * kSize, t.rows,
                    min(a.outputs - o0, P::kN) * kSize};
    P p;
    BiasGrads<P::kTilesN> of_bias;
    p.run(lds, m, n, t.rows, P::kZero, [&](const chunk16 (&grad)[P::kTilesN]) {
        if (bias) of_bias.add(grad);
    });
    store_weight_grads(a, t, c0, o0, p, bias, of_bias);
}

constexpr int kNarrowRing = 3, kTailBlocks = 256;

// All gradients of a narrow layer, of at most 64 channels and outputs: x and dy are read once, where dx and dW on their own read dy twice.  A wave has the
// weights for some of dx's columns in registers and reads, of each step that the workgroup brings into the LDS, the fragments for both products.  Workgroups
// behind those of the pieces clear dx behind the last expert's rows.  2^20 x 64 by 64 fp32 (8 experts): 175 us, 4.7 TB/s, and 8 for the sums; dx and dW on
// their own 119 and 136, and 13.
__global__ __launch_bounds__(kNarrowThreads) void expert_narrow_grads_kernel(WeightArgs a, const void* weight, void* dx) {
    using P = Product<Value, true, true, 64, 64, 2, 2, Chunks::kDirect, kNarrowRing>;
    using Load = Loader<Value, true, 64, kNarrowThreads, Chunks::kDirect>;
    using Tile = typename Load::Tile;
    constexpr int kDepth = P::kDepth, kWeightSteps = 64 / kDepth;
    constexpr int kRowTiles = kDepth / 16, kShare = 4 / kRowTiles, kTiles = 4 / kShare;  // of a step; waves to each; tiles of 16 columns that a wave has
    constexpr int kLines = 64 * kSize / 64;                                             // 64 bytes of a row of dy
    // the weights, until all waves have read them, have the room of the step that is loaded first in the loop
    constexpr int kWeightsAt = (kNarrowRing - 1) * P::kStage;
    static_assert(P::kThreads == kNarrowThreads && kWeightSteps * Tile::kSize <= P::kStage);
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    if (blockIdx.x >= gridDim.x - kTailBlocks) {
        const int routed = min(max(a.offsets[a.experts], 0), a.rows);
        const int64_t chunks = static_cast<int64_t>(a.rows - routed) * a.channels * kSize / 16;
        chunk16* const to = reinterpret_cast<chunk16*>(static_cast<Value*>(dx) + static_cast<int64_t>(routed) * a.channels);
        const uint32_t block = blockIdx.x - (gridDim.x - kTailBlocks);
        for (int64_t i = static_cast<int64_t>(block) * kNarrowThreads + threadIdx.x; i < chunks; i += kTailBlocks * kNarrowThreads) to[i] = chunk16{};
        return;
    }
    const uint32_t piece = a.spread.item();
    if (piece >= a.spread.items) return;
    const RowTile t = row_tile<false>(a.offsets, a.experts, a.rows, piece, a.most);
    if (t.expert < 0 || (t.tiles > 1 && t.slot >= a.slots)) return;  // (the second: offsets that no plan has)
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    const int64_t row_bytes = static_cast<int64_t>(a.channels) * kSize;
    Load load_w(Operand{static_cast<const char*>(weight) + t.expert * a.outputs * row_bytes, row_bytes, a.outputs, static_cast<int>(row_bytes)});
    Load load_m(Operand{static_cast<const char*>(a.x) + t.first * a.x_stride * kSize, a.x_stride * kSize, t.rows, static_cast<int>(row_bytes)});
    Load load_n(Operand{static_cast<const char*>(a.grad) + t.first * a.grad_stride * kSize, a.grad_stride * kSize, t.rows, a.outputs * kSize});
#pragma unroll
    for (int k = 0; k < kWeightSteps; ++k) load_w.begin(lds_at + kWeightsAt + k * Tile::kSize);
    int room = 0, here = 0;
    const auto behind = [](int at) { return at + P::kStage == P::kLds ? 0 : at + P::kStage; };
    const auto begin = [&] {
        load_m.begin(lds_at + room);
        load_n.begin(lds_at + room + Tile::kSize);
        room = behind(room);
    };
    const auto meet = [&] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
#pragma unroll
    for (int k = 0; k < kNarrowRing - 1; ++k) begin();
    const int lane = threadIdx.x % 64, wave = P::wave(), row16 = wave / kShare * 16, m0 = wave % kShare * (16 * kTiles);
    P p;
    p.start(P::kZero);
    const bool bias = a.bias != nullptr && P::wave_m() == 0;
    BiasGrads<P::kTilesN> of_bias;
    wait_for_loads<P::kLoads * (kNarrowRing - 1)>();
    meet();
    chunk16 w[kTiles][kLines];
#pragma unroll
    for (int l = 0; l < kLines; ++l)
#pragma unroll
        for (int i = 0; i < kTiles; ++i) w[i][l] = Tile::fragment(lds + kWeightsAt + l / 2 * Tile::kSize, m0 + 16 * i, l % 2, 0);
    Value* const out = static_cast<Value*>(dx) + static_cast<int64_t>(t.first) * a.channels;
    for (int first = 0; first < t.rows; first += kDepth) {
        // This step is there for all waves, and all have read the one before, whose room the step kNarrowRing - 1 behind this one takes.
        wait_for_loads<P::kLoads * (kNarrowRing - 2)>();
        meet();
        begin();
        typename P::Fragments f[2];
        f[0].read(lds + here, 0);
        f[1].read(lds + here, 1);
        chunk16 rows[kLines];
        const int mine = row16 + lane % 16;
        const char* const its = lds + here + Tile::kSize + mine * Tile::kRowBytes;
#pragma unroll
        for (int l = 0; l < kLines; ++l) rows[l] = *reinterpret_cast<const chunk16*>(its + Tile::place(mine, l * 4 + lane / 16) * 16);
        here = behind(here);
        tile_acc acc[kTiles] = {};
#pragma unroll
        for (int l = 0; l < kLines; ++l)
#pragma unroll
            for (int i = 0; i < kTiles; ++i) acc[i] = multiply<Value>(w[i][l], rows[l], acc[i]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            p.multiply_half(f[h]);
            if (bias) of_bias.add(f[h].n[0]);
        }
        const int row = first + row16;
        store_sixteen_rows(acc, out + static_cast<int64_t>(row) * a.channels + m0, a.channels, t.rows - row, a.channels - m0);
    }
    wait_for_loads<0>();  // (nothing is on its way into the LDS when the workgroup ends)
    store_weight_grads(a, t, 0, 0, p, bias, of_bias);
}

constexpr int kBiasThreads = 256;

// db alone, of pieces of experts' rows: kLanes neighbouring outputs to as many lanes, whose others take the next rows; sums in 64 bits.  Memory bounds it:
// 32768 x 4096 bf16 of 16 experts 50 us with the sums, 5.4 TB/s (dW with it, and thrown away, 290), 2^20 x 64 fp32 47.
template <int kLanes>
__global__ __launch_bounds__(kBiasThreads) void expert_bias_kernel(WeightArgs a) {
    constexpr int kRows = kBiasThreads / kLanes;
    __shared__ double lds[kRows][kLanes];
    const uint32_t item = a.spread.item();
    if (item >= a.spread.items) return;
    const RowTile t = row_tile<false>(a.offsets, a.experts, a.rows, item / a.tiles, a.most);
    if (t.expert < 0 || (t.tiles > 1 && t.slot >= a.slots)) return;  // (the second: offsets that no plan has)
    const int row = static_cast<int>(threadIdx.x) / kLanes, lane = static_cast<int>(threadIdx.x) % kLanes, o = static_cast<int>(item % a.tiles) * kLanes + lane;
    // (lanes behind the last output read it too)
    const Value* const from = static_cast<const Value*>(a.grad) + static_cast<int64_t>(t.first) * a.grad_stride + min(o, a.outputs - 1);
    double sum = 0.0;
#pragma unroll 8
    for (int r = row; r < t.rows; r += kRows) sum += static_cast<double>(static_cast<float>(from[r * a.grad_stride]));
    lds[row][lane] = sum;
    __syncthreads();
    if (row > 0 || o >= a.outputs) return;
    for (int k = 1; k < kRows; ++k) sum += lds[k][lane];
    if (t.tiles == 1) static_cast<Value*>(a.bias)[static_cast<int64_t>(t.expert) * a.outputs + o] = static_cast<Value>(static_cast<float>(sum));
    else a.sums[t.slot * a.outputs + o] = static_cast<float>(sum);
}

constexpr int kSumThreads = 256;

// The sums of experts whose rows are several pieces (of db alone: with no channels), in 64 bits: kSlices lanes share a result's pieces, each taking every
// kSlices-th in order, and their sums are added in order.
template <int kSlices>
__global__ __launch_bounds__(kSumThreads) void expert_sums_kernel(WeightArgs a, uint32_t blocks) {
    constexpr int kResults = kSumThreads / kSlices;
    __shared__ double lds[kSlices][kResults];
    const int e = static_cast<int>(blockIdx.x / blocks);
    // the slot of the expert's first piece, and how many pieces there are
    uint32_t first = 0, mine = 0;
    for (int i = static_cast<int>(threadIdx.x) % 64; i <= e; i += 64) {
        const int from = min(max(a.offsets[i], 0), a.rows), to = min(max(a.offsets[i + 1], 0), a.rows);
        const uint32_t n = max((static_cast<uint32_t>(max(to - from, 0)) + a.most - 1) / a.most, 1u);
        if (i < e) first += n > 1 ? n : 0u;
        else mine = n;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) first += __shfl_xor(first, d), mine = max(mine, static_cast<uint32_t>(__shfl_xor(mine, d)));
    if (mine <= 1 || int64_t{first} + mine > a.slots) return;  // (the second: offsets that no plan has)
    const int64_t weights = static_cast<int64_t>(a.outputs) * a.channels, n = weights + (a.bias != nullptr ? a.outputs : 0);
    const int slice = static_cast<int>(threadIdx.x) / kResults, result = static_cast<int>(threadIdx.x) % kResults;
    // (a lane has kWide results: with one slice four, where those of every piece and expert begin on four)
    constexpr int kWide = kSlices == 1 ? 4 : 1;
    const bool fours = kWide == 4 && weights % 4 == 0;
    if (fours) {
        using Four = float __attribute__((ext_vector_type(4)));
        using Doubles = double __attribute__((ext_vector_type(4)));
        for (int64_t i = (static_cast<int64_t>(blockIdx.x % blocks) * kResults + result) * 4; i < weights; i += static_cast<int64_t>(blocks) * kResults * 4) {
            const float* const from = a.sums + first * weights + i;
            Doubles sum{};
#pragma unroll 4
            for (uint32_t k = 0; k < mine; ++k) sum += __builtin_convertvector(*reinterpret_cast<const Four*>(from + k * weights), Doubles);
            store_values<Value, 4>(static_cast<Value*>(a.weight) + e * weights + i,
                                   __builtin_convertvector(__builtin_convertvector(sum, Four), Value __attribute__((ext_vector_type(4)))), 4);
        }
    }
    for (int64_t begin = static_cast<int64_t>(blockIdx.x % blocks) * kResults + (fours ? weights : 0); begin < n; begin += static_cast<int64_t>(blocks) * kResults) {
        const int64_t i = begin + result;
        const bool there = i < n, weight = i < weights;
        const int64_t each = weight ? weights : a.outputs, at = weight ? i : i - weights;
        double sum = 0.0;
        if (there) {
            const float* const from = a.sums + (weight ? 0 : a.slots * weights) + first * each + at;
#pragma unroll 4
            for (uint32_t k = slice; k < mine; k += kSlices) sum += static_cast<double>(from[k * each]);
        }
        if constexpr (kSlices > 1) {
            lds[slice][result] = sum;
            __syncthreads();
            sum = lds[0][result];
#pragma unroll
            for (int k = 1; k < kSlices; ++k) sum += lds[k][result];
            __syncthreads();
        }
        if (there && slice == 0) static_cast<Value*>(weight ? a.weight : a.bias)[e * each + at] = static_cast<Value>(static_cast<float>(sum));
    }
}

// ------------------------------------------------------------------------------------------
// which kernel

// How chunks of rows of `values` values, `stride` apart, come.
Chunks chunks_of(const void* p, int64_t stride, int64_t values) {
    if (aligned_to(p, 16) && stride * kSize % 16 == 0 && values * kSize % 16 == 0) return Chunks::kDirect;
    return values * kSize >= 16 ? Chunks::kHeld : Chunks::kSingle;
}

// (a launch has less than 2^32 threads, and a spread rounds up)
constexpr int64_t kMostThreads = (int64_t{1} << 32) - (1 << 18);

// The most tiles of `most` rows that there are.
int64_t row_tiles(const RowsArgs& a, int most) { return a.rows / most + std::min(a.experts, a.rows) + 1; }

template <bool kBack, class P, class Quarter = P>
int launch_rows(RowsArgs a, hipStream_t stream) {
    a.tiles = static_cast<uint32_t>((a.wide + P::kM - 1) / P::kM);
    const int64_t items = row_tiles(a, P::kN) * a.tiles + (std::is_same_v<P, Quarter> ? 0 : 3 * kUnits / 2);
    if (items * P::kThreads >= kMostThreads) return PENC_ERR_BAD_LAYER_SIZE;
    a.spread = Spread(items, 32);
    expert_rows_kernel<kBack, P, Quarter><<<a.spread.grid(), P::kThreads, 0, stream>>>(a);
    return launched();
}

template <bool kBack>
int launch_narrow(RowsArgs a, hipStream_t stream) {
    // (1024 workgroups, as many as the card holds, have some that begin late: 2^20 x 64 by 64 fp32 140 us, 4096 of them 125)
    const int most = static_cast<int>(std::min<int64_t>(std::max<int64_t>((a.rows / 4096 + 63) / 64 * 64, 256), 1 << 16));
    a.spread = Spread(row_tiles(a, most), 1);
    const auto launch = [&](auto lines, auto tiles) -> int {
        expert_narrow_kernel<kBack, decltype(lines)::value, decltype(tiles)::value><<<a.spread.grid(), kNarrowThreads, 0, stream>>>(a, most);
        return launched();
    };
    const auto with_tiles = [&](auto lines) -> int {
        if (a.wide <= 16) return launch(lines, std::integral_constant<int, 1>{});
        if (a.wide <= 32) return launch(lines, std::integral_constant<int, 2>{});
        return launch(lines, std::integral_constant<int, 4>{});
    };
    return a.deep * kSize <= 128 ? with_tiles(std::integral_constant<int, 2>{}) : with_tiles(std::integral_constant<int, 4>{});
}

int launch_few(RowsArgs a, hipStream_t stream) {
    a.tiles = static_cast<uint32_t>((a.wide + kFewOutputs - 1) / kFewOutputs);
    const int64_t items = row_tiles(a, kFewRows) * a.tiles;
    if (items * kFewThreads >= kMostThreads) return PENC_ERR_BAD_LAYER_SIZE;
    a.spread = Spread(items, 32);
    expert_few_kernel<<<a.spread.grid(), kFewThreads, 0, stream>>>(a);
    return launched();
}

// kChunks: of the weights' rows; kChunksN: of the others.
template <bool kBack, Chunks kChunks, Chunks kChunksN = kChunks>
int rows_of_experts(const RowsArgs& a, hipStream_t stream) {
    if constexpr (kChunks == Chunks::kDirect) {
        if (a.wide <= 16 * kNarrowTiles && a.deep * kSize <= 64 * kNarrowLines && a.stride * kSize * 64 < 1 << 30) return launch_narrow<kBack>(a, stream);
        // A few rows: 64 experts of 1024 by 4096 bf16, 4 rows to an expert, 99 us, and 122 without; 16 to an expert 140 and 108.  More of them where the
        // workgroups would be few otherwise, each with all of a long row: 1257 rows of 82 experts, 2048 by 24 fp32, 23 us and 135.
        if (!kBack && (a.rows <= kFewRows / 2 * static_cast<int64_t>(a.experts) ||
                       (a.rows <= 2 * kFewRows * static_cast<int64_t>(a.experts) && row_tiles(a, 256) * ((a.wide + 63) / 64) < kUnits)))
            return launch_few(a, stream);
    }
    // Where tiles of 128 x 128 would leave half of the compute units without one, tiles of 64 x 64, loaded three steps ahead where they come directly: 500
    // rows of 4096 by 64 bf16 39 us -> 21, of fp32 264 -> 84, 1000 rows of 512 by 512 fp32 with 3 experts, y and dx, 76 -> 29; with 180 such tiles (5000
    // rows, 4 experts, bf16) 20 -> 23.
    if constexpr (kChunks != Chunks::kSingle && kChunksN != Chunks::kSingle) {
        if (row_tiles(a, 128) * ((a.wide + 127) / 128) < static_cast<int64_t>(kUnits / 2))
            return launch_rows<kBack, Product<Value, kBack, false, 64, 64, 2, 2, kChunks, kChunks == Chunks::kDirect ? 4 : 2>>(a, stream);
    }
    // (129 to 192 results of rows that begin anywhere: three tiles of 64, where they are two rounds of compute units at least, 33.6 us of 70001 x 203 by 130
    // fp16, two of 128 35.7; 34.6 and 37.7 of 203 by 190; of 200000 x 513 by 132 bf16 113 and 120; but of 30000 x 1001 by 160 fp16, which has 366 such tiles,
    // 37.0 and 31.8.  Of rows on 16 bytes, 208 by 136, 22.3 and 21.0.)
    const bool threes = kChunks == Chunks::kHeld && a.wide > 128 && a.wide <= 192 && 3 * row_tiles(a, 256) >= 2 * kUnits;
    if (a.wide <= 64 || threes || kChunks == Chunks::kSingle) return launch_rows<kBack, Product<Value, kBack, false, 64, 256, 1, 4, kChunks, 2, kChunksN>>(a, stream);
    if constexpr (kChunks != Chunks::kSingle) {
        if constexpr (kChunks == Chunks::kDirect && kSize == 2) {
            // (1024 by 4096 bf16, 16 experts, of 2048 rows each: 302 us and 347 without; of 512 89 and 86, of 256 58 and 50: tiles of 256 rows that are not
            // full. 2^18 rows of 1024, 4 experts, y and dx: of 72 results 144 and 152 us, without 129 and 130; of 128 152 and 153, 139 and 140; of 264 232
            // and 239, 232 and 248; 2^17 of 640 189 and 192, 211 and 216)
            if (a.wide > 128 && a.rows >= 1024 * static_cast<int64_t>(a.experts) && static_cast<int64_t>(a.rows / 256) * ((a.wide + 255) / 256) >= 512)
                return launch_rows<kBack, Product<Value, kBack, false, 256, 256, 4, 2, kChunks>, Product<Value, kBack, false, 128, 128, 4, 2, kChunks>>(a, stream);
        }
        return launch_rows<kBack, Product<Value, kBack, false, 128, 128, 2, 2, kChunks, 2, kChunksN>>(a, stream);
    }
}

// Both operands come directly, or both through registers; value by value only the one whose rows are that short (363113 x 1032 by 4 bf16, with gradients: 915
// us, both so 1430).
template <bool kBack>
int rows_of_experts(const RowsArgs& a, Chunks weight, Chunks rows, hipStream_t stream) {
    constexpr Chunks kHeld = Chunks::kHeld, kSingle = Chunks::kSingle;
    if (weight == Chunks::kDirect && rows == Chunks::kDirect) return rows_of_experts<kBack, Chunks::kDirect>(a, stream);
    if (weight != kSingle && rows != kSingle) return rows_of_experts<kBack, kHeld>(a, stream);
    if constexpr (kBack) {
        if (weight != kSingle) return rows_of_experts<kBack, kHeld, kSingle>(a, stream);
        if (rows != kSingle) return rows_of_experts<kBack, kSingle, kHeld>(a, stream);
    }
    return rows_of_experts<kBack, kSingle>(a, stream);
}

// How rows are cut for db alone: for four workgroups to a compute unit, where one has all outputs.
struct BiasPlan {
    int64_t most, pieces, slots;
};
BiasPlan bias_plan(int64_t rows, int64_t experts) {
    BiasPlan p;
    p.most = std::max<int64_t>((rows / (4 * kUnits) + 63) / 64 * 64, 512);
    p.pieces = rows / p.most + experts;
    p.slots = rows / p.most + std::min(experts, rows / (p.most + 1));
    return p;
}

// How the rows of the weights' gradient are cut, and the tiles.  A time is in rows that a workgroup multiplies.
struct WeightPlan {
    int side;      // of a tile
    int64_t tiles; // of an expert
    int64_t most;  // rows of a piece
    int64_t pieces;
    int64_t slots; // the most pieces of experts of more than `most` rows
    double time;
};
// Workgroups go in rounds of as many as have room at a time.  Beside its rows a workgroup takes as long as for two steps, and where its sums go through
// memory, as long again as kCut rows.  Either an expert's rows are one piece (up to twice as many as experts have on average, or 3/4 of all that a workgroup
// has if that is more: dW of 32768 x 1024 by 4096 bf16, 16 experts in uneven demand, 324 us and then 304, of 16384 x 2048 by 2048 bf16, 16 experts, 205 and
// 185, of 16384 x 1024 by 2048 fp32 568 and 556; and a quarter of the time for experts that are not alike), or they are cut for whole rounds, as few as there
// can be or up to three more.  (Four workgroups to a compute unit whatever their tiles: 70001 x 203 by 130 fp16, where 600 of them are two rounds, 38 us and
// 6 for the sums, now 28 and 5; 2^20 x 64 by 64 fp32, all of the layer, with 2, 4, 6 and 8 to a compute unit 347, 325, 305 and 316 us, with 3 299.  16384 x
// 1024 by 2048 bf16, 4 experts, y and dW: cut for three rounds 216 us, in one piece 165.) No piece is longer than kLongest.  A chain of n additions of one
// sign is off by n / 2 times 2^-24 of it at the most: fp32, whose products are added one by one, by 2^-12 (in one chain of 98304 rows 1.2e-3 was seen),
// 16-bit types, which add 32 products at a time, by 2^-14.  Pieces are added in 64 bits.  (2^20 x 256 by 256 fp32, 4 experts: 3400 us in two rounds of
// shorter pieces, 3350 without a limit, 3860 with the limit alone.)
constexpr int64_t kLongest = kSize == 2 ? 1 << 16 : 1 << 13;
WeightPlan weight_plan_of(int side, int64_t rows, int64_t experts, int64_t channels, int64_t outputs) {
    constexpr double kBeside = 128.0, kCut = kSize == 2 ? 512.0 : 128.0;
    WeightPlan p;
    p.side = side;
    p.tiles = ((channels + side - 1) / side) * ((outputs + side - 1) / side);
    const int64_t room = (side == 256 ? 1 : side == 128 ? 2 : 3) * kUnits, own = (rows + experts - 1) / experts;
    p.most = std::max(2 * own, rows / 4 * 3 * p.tiles / room);
    p.time = static_cast<double>((experts * p.tiles + room - 1) / room) * 1.25 * (static_cast<double>(own) + kBeside);
    if (own > kLongest) p.time = INFINITY;
    const int64_t least = (((rows + kLongest - 1) / kLongest + experts) * p.tiles + room - 1) / room;  // with pieces of kLongest rows
    for (int64_t rounds = std::max<int64_t>(least, 1); rounds < std::max<int64_t>(least, 1) + 4; ++rounds) {
        const int64_t pieces = rounds * room / p.tiles - experts;
        if (pieces <= 0) continue;
        const int64_t each = std::max<int64_t>((rows + pieces - 1) / pieces, 512);
        const double time = static_cast<double>(rounds) * (static_cast<double>(each) + kBeside + kCut);
        if (time < p.time) p.time = time, p.most = each;
    }
    p.most = std::min<int64_t>(std::max<int64_t>((p.most + 63) / 64 * 64, 512), kLongest);
    p.pieces = rows / p.most + experts;
    p.slots = rows / p.most + std::min(experts, rows / (p.most + 1));
    return p;
}
WeightPlan weight_plan(int64_t rows, int64_t experts, int64_t channels, int64_t outputs) {
    if (channels <= 64 || outputs <= 64) return weight_plan_of(64, rows, experts, channels, outputs);
    const WeightPlan p = weight_plan_of(128, rows, experts, channels, outputs);
    // (half of the compute units without a workgroup: 1000 x 512 by 512 fp32, 3 experts, y and dW, 47 us, 30 so; 4000 x 512 by 512 bf16, 4 experts, 28 and 26)
    if (std::max(experts, rows / p.most) * p.tiles < static_cast<int64_t>(kUnits / 2)) return weight_plan_of(64, rows, experts, channels, outputs);
    if (kSize != 2 || channels % 8 != 0 || outputs % 8 != 0 || channels < 256 || outputs < 256) return p;
    // Two tiles of 128 have half of the work of one of 256 a row, which they do in 0.6 of its time (32768 x 1024 by 4096 bf16, 16 experts, all of the layer:
    // 256 897 us, 128 940).
    const WeightPlan large = weight_plan_of(256, rows, experts, channels, outputs);
    return large.time < 0.6 * p.time ? large : p;
}

template <class P>
int launch_weights(WeightArgs a, const WeightPlan& plan, hipStream_t stream) {
    a.channel_tiles = static_cast<uint32_t>((a.channels + P::kM - 1) / P::kM);
    a.tiles = a.channel_tiles * static_cast<uint32_t>((a.outputs + P::kN - 1) / P::kN);
    const int64_t items = plan.pieces * a.tiles;
    if (items * P::kThreads >= kMostThreads) return PENC_ERR_BAD_LAYER_SIZE;
    // (pieces take different times: all dies work on the same ones)
    a.spread = Spread(items, a.tiles / 8);
    expert_weights_kernel<P><<<a.spread.grid(), P::kThreads, 0, stream>>>(a);
    return launched();
}

int launch_narrow_grads(WeightArgs a, const WeightPlan& plan, const void* weight, void* dx, hipStream_t stream) {
    a.spread = Spread(plan.pieces, 1);
    expert_narrow_grads_kernel<<<a.spread.grid() + kTailBlocks, kNarrowThreads, 0, stream>>>(a, weight, dx);
    return launched();
}

int launch_sums(const WeightArgs& a, int64_t pieces, hipStream_t stream) {
    const int64_t results = int64_t{a.outputs} * (a.channels + 1);
    // (many pieces: a few results, and lanes that share them)
    const auto sum = [&](auto slices) -> int {
        constexpr int kSlices = decltype(slices)::value, kResults = kSumThreads / kSlices;
        const uint32_t blocks = static_cast<uint32_t>(std::min<int64_t>((results + kResults - 1) / kResults, std::max<int64_t>(16, 8192 / a.experts)));
        expert_sums_kernel<kSlices><<<static_cast<uint32_t>(a.experts) * blocks, kSumThreads, 0, stream>>>(a, blocks);
        return launched();
    };
    return pieces >= 32 * int64_t{a.experts} ? sum(std::integral_constant<int, 16>{}) : sum(std::integral_constant<int, 1>{});
}

template <Chunks kChunks, Chunks kChunksN = kChunks>
int weights_of_experts(const WeightArgs& a, const WeightPlan& plan, hipStream_t stream) {
    if (plan.side == 64) return launch_weights<Product<Value, true, true, 64, 64, 2, 2, kChunks, 2, kChunksN>>(a, plan, stream);
    if constexpr (kChunks != Chunks::kSingle && kChunksN != Chunks::kSingle) {
        if constexpr (kChunks == Chunks::kDirect && kSize == 2) {
            if (plan.side == 256) return launch_weights<Product<Value, true, true, 256, 256, 2, 4, kChunks>>(a, plan, stream);
        }
        return launch_weights<Product<Value, true, true, 128, 128, 2, 2, kChunks>>(a, plan, stream);
    }
    return PENC_ERR_BAD_LAYER_SIZE;  // (not reached: rows of less than 16 bytes have less than 64 values)
}
int weights_of_experts(const WeightArgs& a, const WeightPlan& plan, Chunks x, Chunks grad, hipStream_t stream) {
    constexpr Chunks kHeld = Chunks::kHeld, kSingle = Chunks::kSingle;
    if (x == Chunks::kDirect && grad == Chunks::kDirect) return weights_of_experts<Chunks::kDirect>(a, plan, stream);
    if (x != kSingle && grad != kSingle) return weights_of_experts<kHeld>(a, plan, stream);
    if (x != kSingle) return weights_of_experts<kHeld, kSingle>(a, plan, stream);
    if (grad != kSingle) return weights_of_experts<kSingle, kHeld>(a, plan, stream);
    return weights_of_experts<kSingle>(a, plan, stream);
}

}  // namespace

template <>
int expert_rows<PENC_TYPE>(bool back, int64_t rows, int experts, int64_t wide, int64_t deep, const void* in, int64_t stride, const void* weight, const void* bias,
                           const int32_t* offsets, void* out, hipStream_t stream) {
    if (rows == 0) return PENC_OK;
    RowsArgs a{in, weight, bias, out, stride, offsets, experts, static_cast<int>(rows), static_cast<int>(wide), static_cast<int>(deep), {}, 0};
    const Chunks of_weight = chunks_of(weight, back ? wide : deep, back ? wide : deep), of_rows = chunks_of(in, stride, deep);
    return back ? rows_of_experts<true>(a, of_weight, of_rows, stream) : rows_of_experts<false>(a, of_weight, of_rows, stream);
}

template <>
size_t expert_weights_workspace<PENC_TYPE>(int64_t rows, int64_t experts, int64_t channels, int64_t outputs) {
    const WeightPlan p = weight_plan(rows, experts, channels, outputs);
    if (rows <= p.most) return 0;  // no expert's rows are cut
    return 4 * static_cast<size_t>(p.slots) * static_cast<size_t>(outputs) * (static_cast<size_t>(channels) + 1);
}

template <>
int expert_grads<PENC_TYPE>(int64_t rows, int experts, int64_t channels, int64_t outputs, const void* x, int64_t x_stride, const void* grad, int64_t grad_stride,
                            const void* weight, const int32_t* offsets, void* dx, void* dweight, void* dbias, void* workspace, hipStream_t stream) {
    const WeightPlan plan = weight_plan(rows, experts, channels, outputs);
    WeightArgs a{x, grad, x_stride, grad_stride, offsets, experts, static_cast<int>(rows), static_cast<int>(channels), static_cast<int>(outputs),
                 static_cast<int>(plan.most), {}, 0, 0, dweight, dbias, static_cast<float*>(workspace), plan.slots};
    const Chunks of_x = chunks_of(x, x_stride, channels), of_grad = chunks_of(grad, grad_stride, outputs);
    const bool together = dx != nullptr && channels <= 64 && outputs <= 64 && of_x == Chunks::kDirect && of_grad == Chunks::kDirect &&
        aligned_to(weight, 16) && aligned_to(dx, 16);
    if (dx != nullptr && !together) {
        if (const int rc = expert_rows<PENC_TYPE>(true, rows, experts, channels, outputs, grad, grad_stride, weight, nullptr, offsets, dx, stream)) return rc;
    }
    if (const int rc = together ? launch_narrow_grads(a, plan, weight, dx, stream) : weights_of_experts(a, plan, of_x, of_grad, stream))
        return rc;
    return rows <= plan.most ? PENC_OK : launch_sums(a, plan.pieces, stream);
}

template <>
size_t expert_bias_workspace<PENC_TYPE>(int64_t rows, int64_t experts, int64_t outputs) {
    const BiasPlan p = bias_plan(rows, experts);
    return rows <= p.most ? 0 : 4 * static_cast<size_t>(p.slots) * static_cast<size_t>(outputs);
}

template <>
int expert_bias<PENC_TYPE>(int64_t rows, int experts, int64_t outputs, const void* grad, int64_t grad_stride, const int32_t* offsets, void* dbias, void* workspace,
                           hipStream_t stream) {
    const BiasPlan plan = bias_plan(rows, experts);
    WeightArgs a{nullptr, grad, 0, grad_stride, offsets, experts, static_cast<int>(rows), 0, static_cast<int>(outputs), static_cast<int>(plan.most), {}, 0, 0,
                 nullptr, dbias, static_cast<float*>(workspace), plan.slots};
    const auto launch = [&](auto lanes) -> int {
        constexpr int kLanes = decltype(lanes)::value;
        a.tiles = static_cast<uint32_t>((outputs + kLanes - 1) / kLanes);
        const int64_t items = plan.pieces * a.tiles;
        if (items * kBiasThreads >= kMostThreads) return PENC_ERR_BAD_LAYER_SIZE;
        a.spread = Spread(items, 1);
        expert_bias_kernel<kLanes><<<a.spread.grid(), kBiasThreads, 0, stream>>>(a);
        return launched();
    };
    if (const int rc = outputs <= 16 ? launch(std::integral_constant<int, 16>{}) : launch(std::integral_constant<int, 64>{})) return rc;
    return rows <= plan.most ? PENC_OK : launch_sums(a, plan.pieces, stream);
}

}  // namespace penc
