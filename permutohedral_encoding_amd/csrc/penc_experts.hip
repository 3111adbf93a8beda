// Rows that go to experts and come back: which experts a row takes, where its choices stand when they are sorted by expert, and the rows themselves,
// there and back.
//
//     route      the k largest of a row's logits l, the lowest index first among equal ones, and w_j = exp(l_j - top) / sum of exp(l_i - top) over the chosen
//                (or over all experts).  dl_j = w_j (g_j - sum_i w_i g_i) at the chosen (over all: less p_i sum_j w_j g_j everywhere, p_i every expert's share)
//     plan       choice i of N k (row i / k) stands at position p(i): those of one expert in their order, expert by expert, those of none last
//     dispatch   s[p(i)] = x[i / k], zeros for a choice without an expert;    dx[t] = sum of ds[p] over t's choices
//     combine    o[t] = sum of w y[p] over t's choices;                      dy[p] = w do[t],  dw = <do[t], y[p]>
//
// All but some of route is bound by memory.  Results, and the logits, go past the caches (nontemporal), but for short rows that go to places of their own
// (with_past): a pass over rows of 256 MiB that leaves what it wrote in them has the next pass wait until that is in memory.  Route and its gradient of 2^20
// x 64 fp32: 160 us without, 115 so; rows of 2^20 x 64 fp32 there and back, two choices, with gradients 729 and 698, of 16381 x 2048 bf16 195 and 181.  With
// rows that the caches hold (a decoder of 2^11 to 2^17 points, its passes one after the other) the two are within 1%.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "penc_expert_linear.hpp"
#include "penc_kept.hpp"

namespace penc {
namespace {

constexpr int kThreads = 256, kLog2Threads = 8;
constexpr int kWave = 64;

// ------------------------------------------------------------------------------------------
// route

// The lanes of a row's group bring it to all of them: kLanes is a power of two.
template <int kLanes, class T, class F>
__device__ __forceinline__ T over_lanes(T v, F&& f) {
    const auto moved = [](T x, auto control) {
        return __builtin_bit_cast(T, dpp<decltype(control)::value>(__builtin_bit_cast(uint32_t, x)));
    };
    if constexpr (kLanes > 1) v = f(v, moved(v, std::integral_constant<int, kSwapPairs>{}));
    if constexpr (kLanes > 2) v = f(v, moved(v, std::integral_constant<int, kSwapTwos>{}));
    if constexpr (kLanes > 4) v = f(v, moved(v, std::integral_constant<int, kMirrorHalfRow>{}));
    if constexpr (kLanes > 8) v = f(v, moved(v, std::integral_constant<int, kMirrorRow>{}));
    if constexpr (kLanes > 16) v = f(v, __shfl_xor(v, 16));
    if constexpr (kLanes > 32) v = f(v, __shfl_xor(v, 32));
    return v;
}

// A logit as an integer that is larger where the logit is: a NaN is the largest, -0 is 0.  Up to kNone nothing is chosen: -inf, and 0 for what has been
// chosen before.
constexpr uint32_t kNone = 0x007FFFFFu;
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f), key = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return v != v ? 0xFFFFFFFFu : key;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return key == 0xFFFFFFFFu ? __builtin_nanf("") : __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}

// A lane of kLanes has 8 kChunks logits of a row, in pieces of 16 bytes: neighbouring lanes have neighbouring pieces.
template <class E, int kLanes, int kChunks>
struct LogitRow {
    static constexpr int kWide = 16 / sizeof(E), kPieces = kChunk * kChunks / kWide, kValues = kWide * kPieces;
    using Unaligned = E __attribute__((ext_vector_type(kWide), aligned(sizeof(E))));
    float v[kValues];

    // where value i is in the row
    __device__ __forceinline__ static int index_of(int i) { return (i / kWide * kLanes + static_cast<int>(threadIdx.x) % kLanes) * kWide + i % kWide; }

    __device__ __forceinline__ LogitRow(const E* __restrict__ row, int experts) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int at = index_of(p * kWide);
            if (at + kWide <= experts) {
                const Unaligned piece = __builtin_nontemporal_load(reinterpret_cast<const Unaligned*>(row + at));
#pragma unroll
                for (int i = 0; i < kWide; ++i) v[p * kWide + i] = static_cast<float>(piece[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kWide; ++i) v[p * kWide + i] = at + i < experts ? static_cast<float>(row[at + i]) : -__builtin_inff();
            }
        }
    }
    // Stores results as the logits lie.
    __device__ __forceinline__ static void store(E* __restrict__ row, int experts, const float (&out)[kValues]) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int at = index_of(p * kWide);
            using Floats = float __attribute__((ext_vector_type(kWide)));
            Floats f;
#pragma unroll
            for (int i = 0; i < kWide; ++i) f[i] = out[p * kWide + i];
            const auto y = __builtin_convertvector(f, E __attribute__((ext_vector_type(kWide))));
            if (at + kWide <= experts) {
                __builtin_nontemporal_store(y, reinterpret_cast<Unaligned*>(row + at));
            } else {
#pragma unroll
                for (int i = 0; i < kWide; ++i)
                    if (at + i < experts) row[at + i] = y[i];
            }
        }
    }
    // exp(l - top) of all of them (top: the largest, and not -inf)
    __device__ __forceinline__ float total(float top) const {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kValues; ++i) sum += expf(v[i] - top);
        return over_lanes<kLanes>(sum, [](float a, float b) { return a + b; });
    }
};

// A logit of 16 bits, which has the last 13 bits of a float free, and its expert in one integer: the largest of them is the largest logit's, and of equal
// ones the lowest expert's.
constexpr uint32_t kPackedIndex = 0x1FFFu;
static_assert(PENC_MAX_EXPERTS <= kPackedIndex);
__device__ __forceinline__ uint32_t packed_key(float v, int index) { return (key_of(v) & ~kPackedIndex) | (kPackedIndex - static_cast<uint32_t>(index)); }
__device__ __forceinline__ float packed_logit(uint32_t key) {
    const uint32_t k = key & ~kPackedIndex;
    return k == ~kPackedIndex ? __builtin_nanf("") : logit_of(k >> 31 ? k : k | kPackedIndex);
}

// A row to kLanes lanes, which have it in registers: k times the largest key, and the lowest index that has it.  Of 16 bits both are one integer.
// Instructions bound it but for a few choices of a few experts: 435701 x 144 bf16, four choices, 65 us (with both apart, 32 lanes and 64 logits more than
// there are 120), 2^20 x 64 fp32, two choices, 52 (5.5 TB/s).
template <class E, int kLanes, int kChunks, int kMost>
__global__ __launch_bounds__(kThreads) void route_kernel(row_t rows, int experts, int choices, bool normalise, const E* __restrict__ logits, uint32_t stride,
                                                         float* __restrict__ weights, int32_t* __restrict__ chosen) {
    for (row_t row = blockIdx.x * static_cast<row_t>(kThreads / kLanes) + threadIdx.x / kLanes; row < rows; row += gridDim.x * static_cast<row_t>(kThreads / kLanes)) {
        using Row = LogitRow<E, kLanes, kChunks>;
        const Row r(logits + offset_of(row, stride), experts);
        constexpr bool kPacked = sizeof(E) == 2;
        uint32_t keys[Row::kValues];
#pragma unroll
        for (int i = 0; i < Row::kValues; ++i) {
            if constexpr (kPacked) keys[i] = packed_key(r.v[i], Row::index_of(i));
            else keys[i] = key_of(r.v[i]);
        }
        const auto largest = [](uint32_t a, uint32_t b) { return max(a, b); };
        const auto logit = [](uint32_t key) {
            if constexpr (kPacked) return packed_logit(key);
            else return logit_of(key);
        };
        uint32_t best[kMost];
        int at[kMost];
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
            best[j] = 0, at[j] = -1;
            if (j >= choices) continue;
            uint32_t key = keys[0];
            if constexpr (kPacked) {
#pragma unroll
                for (int i = 1; i < Row::kValues; ++i) key = max(key, keys[i]);
                best[j] = over_lanes<kLanes>(key, largest);
                at[j] = static_cast<int>(kPackedIndex - (best[j] & kPackedIndex));
                if (j + 1 == kMost) continue;
#pragma unroll
                for (int i = 0; i < Row::kValues; ++i) keys[i] = keys[i] == best[j] ? 0u : keys[i];
            } else {
                int index = Row::index_of(0);
#pragma unroll
                for (int i = 1; i < Row::kValues; ++i)
                    if (keys[i] > key) key = keys[i], index = Row::index_of(i);
                best[j] = over_lanes<kLanes>(key, largest);
                const uint32_t mine = key == best[j] ? static_cast<uint32_t>(index) : 0x7FFFFFFFu;
                at[j] = static_cast<int>(over_lanes<kLanes>(mine, [](uint32_t a, uint32_t b) { return min(a, b); }));
                if (j + 1 == kMost) continue;
#pragma unroll
                for (int i = 0; i < Row::kValues; ++i) keys[i] = at[j] == Row::index_of(i) ? 0u : keys[i];
            }
        }
        const float top = logit(best[0]);
        float w[kMost], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
            w[j] = best[j] > kNone ? expf(logit(best[j]) - top) : 0.0f;
            sum += w[j];
        }
        if (!normalise) sum = best[0] > kNone ? r.total(top) : 1.0f;
        if (best[0] <= kNone) sum = 1.0f;
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
            if (j >= choices || static_cast<int>(threadIdx.x) % kLanes != j % kLanes) continue;
            const uint64_t to = offset_of(row, static_cast<uint32_t>(choices)) + j;
            weights[to] = w[j] / sum;
            chosen[to] = best[j] > kNone ? at[j] : -1;
        }
    }
}

// From the weights and their gradients those of all logits.
template <class E, int kLanes, int kChunks, int kMost>
__global__ __launch_bounds__(kThreads) void route_backward_kernel(row_t rows, int experts, int choices, bool normalise, const E* __restrict__ logits,
                                                                  uint32_t stride, const float* __restrict__ weights, const int32_t* __restrict__ chosen,
                                                                  const float* __restrict__ grad, E* __restrict__ dlogits) {
    for (row_t row = blockIdx.x * static_cast<row_t>(kThreads / kLanes) + threadIdx.x / kLanes; row < rows; row += gridDim.x * static_cast<row_t>(kThreads / kLanes)) {
        using Row = LogitRow<E, kLanes, kChunks>;
        constexpr int kValues = Row::kValues;
        float d[kMost], w[kMost], mean = 0.0f;
        int at[kMost];
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
            const uint64_t from = offset_of(row, static_cast<uint32_t>(choices)) + j;
            const bool there = j < choices;
            at[j] = there ? chosen[from] : -1;
            w[j] = there ? weights[from] : 0.0f;
            d[j] = at[j] >= 0 ? w[j] * grad[from] : 0.0f;
            mean += d[j];
        }
        float out[kValues];
        if (normalise || at[0] < 0) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) out[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < kMost; ++j) d[j] -= w[j] * mean;
        } else {
            const Row r(logits + offset_of(row, stride), experts);
            uint32_t key = 0;
#pragma unroll
            for (int i = 0; i < kValues; ++i) key = max(key, key_of(r.v[i]));
            const float top = logit_of(over_lanes<kLanes>(key, [](uint32_t a, uint32_t b) { return max(a, b); })), total = r.total(top);
#pragma unroll
            for (int i = 0; i < kValues; ++i) out[i] = -(expf(r.v[i] - top) / total) * mean;
        }
#pragma unroll
        for (int j = 0; j < kMost; ++j)
#pragma unroll
            for (int i = 0; i < kValues; ++i) out[i] += at[j] == Row::index_of(i) ? d[j] : 0.0f;
        Row::store(dlogits + offset_of(row, static_cast<uint32_t>(experts)), experts, out);
    }
}

// Runs f with how a row of `experts` logits is laid out over lanes, and the most choices that the kernel holds.
template <class F>
int with_row_layout(int experts, int choices, F&& f) {
    const auto with_most = [&](auto lanes, auto chunks) {
        if (choices <= 1) return f(lanes, chunks, std::integral_constant<int, 1>{});
        if (choices <= 2) return f(lanes, chunks, std::integral_constant<int, 2>{});
        if (choices <= 4) return f(lanes, chunks, std::integral_constant<int, 4>{});
        return f(lanes, chunks, std::integral_constant<int, 8>{});
    };
    const int chunks = (experts + kChunk - 1) / kChunk;
    constexpr std::integral_constant<int, 1> one{};
    if (chunks <= 1) return with_most(std::integral_constant<int, 1>{}, one);
    if (chunks <= 2) return with_most(std::integral_constant<int, 2>{}, one);
    if (chunks <= 4) return with_most(std::integral_constant<int, 4>{}, one);
    if (chunks <= 8) return with_most(std::integral_constant<int, 8>{}, one);
    if (chunks <= 16) return with_most(std::integral_constant<int, 16>{}, one);
    if (chunks <= 24) return with_most(std::integral_constant<int, 8>{}, std::integral_constant<int, 3>{});
    // (more lanes exchange what they have through the LDS: 200000 x 512 bf16, 8 choices, 187 us, with 64 of them 287; of 50000 x 1000, which would not fit
    // the registers, 113 and 187)
    constexpr std::integral_constant<int, 16> sixteen{};
    if (chunks <= 32) return with_most(sixteen, std::integral_constant<int, 2>{});
    if (chunks <= 48) return with_most(sixteen, std::integral_constant<int, 3>{});
    if (chunks <= 64) return with_most(sixteen, std::integral_constant<int, 4>{});
    return with_most(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
}

// (a launch has less than 2^32 threads: workgroups go on from there)
unsigned grid_of(int64_t rows, int per_workgroup) { return static_cast<unsigned>(std::min<int64_t>((rows + per_workgroup - 1) / per_workgroup, 1 << 23)); }

// ------------------------------------------------------------------------------------------
// plan

constexpr int kPlanItems = 4;                           // of a lane
constexpr int kPlanChunk = kThreads * kPlanItems;       // of a workgroup
constexpr int kPlanAlone = 1024, kPlanMost = 16;        // one workgroup alone: its lanes, and the most items of a lane
constexpr int kClasses = PENC_MAX_EXPERTS + 1;          // the experts, and none

template <class I>
__device__ __forceinline__ int class_of(const I* __restrict__ chosen, int64_t item, int experts) {
    const int64_t e = chosen[item];
    return e >= 0 && e < experts ? static_cast<int>(e) : experts;
}

// How many of a chunk's choices go to each expert: counts[expert][chunk].
template <class I>
__global__ __launch_bounds__(kThreads) void plan_count_kernel(int64_t items, int experts, const I* __restrict__ chosen, uint32_t* __restrict__ counts) {
    __shared__ uint32_t lds[kClasses];
    for (int e = threadIdx.x; e <= experts; e += kThreads) lds[e] = 0;
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlanChunk;
    int expert[kPlanItems];
    bool there[kPlanItems];
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
        const int64_t item = first + i * kThreads + threadIdx.x;
        expert[i] = class_of(chosen, min(item, items - 1), experts);
        there[i] = item < items;
    }
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i)
        if (there[i]) atomicAdd(&lds[expert[i]], 1u);
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += kThreads) counts[static_cast<int64_t>(e) * gridDim.x + blockIdx.x] = lds[e];
}

// The exclusive sums of kWaves waves' lanes' values, and their total.
template <int kWaves>
__device__ __forceinline__ uint32_t sums_before(uint32_t v, uint32_t (&of_waves)[kWaves], uint32_t& total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t sum = v;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const uint32_t other = __shfl_up(sum, d);
        sum += lane >= d ? other : 0u;
    }
    __syncthreads();
    if (lane == kWave - 1) of_waves[wave] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? of_waves[w] : 0u;
        total += of_waves[w];
    }
    return before + sum - v;
}

// A workgroup to an expert: each chunk's count becomes the sum of those before it; totals[expert].
__global__ __launch_bounds__(kThreads) void plan_scan_kernel(int64_t chunks, uint32_t* __restrict__ counts, uint32_t* __restrict__ totals) {
    __shared__ uint32_t of_waves[kThreads / kWave];
    uint32_t* const mine = counts + blockIdx.x * chunks;
    uint32_t before = 0;
    for (int64_t first = 0; first < chunks; first += kThreads) {
        const int64_t i = first + threadIdx.x;
        const uint32_t v = i < chunks ? mine[i] : 0u;
        uint32_t total;
        const uint32_t sum = sums_before(v, of_waves, total);
        if (i < chunks) mine[i] = before + sum;
        before += total;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// Where each choice of a chunk stands.  A wave takes 64 consecutive choices after the other; lanes of one expert find each other by a ballot for each bit of
// its number, and each stands behind those of the wave's choices before.  Without `counts` there is one chunk, which counts for itself.
template <class I, int kLanes, int kItems>
__global__ __launch_bounds__(kLanes) void plan_place_kernel(int64_t items, int experts, int bits, const I* __restrict__ chosen,
                                                              const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                                                              int32_t* __restrict__ positions, int32_t* __restrict__ offsets) {
    constexpr int kWaves = kLanes / kWave;
    __shared__ uint32_t lds[kWaves][kClasses];
    __shared__ uint32_t of_waves[kWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    for (int e = threadIdx.x; e <= experts; e += kLanes)
#pragma unroll
        for (int w = 0; w < kWaves; ++w) lds[w][e] = 0;
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kLanes * kItems) + wave * (kWave * kItems) + lane;
    int expert[kItems];
    uint32_t rank[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        // (read without a condition: a branch for each would have them come one after the other)
        const int64_t item = first + i * kWave;
        const int e = items > 0 ? class_of(chosen, min(item, items - 1), experts) : 0;
        expert[i] = item < items ? e : -1;
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        uint64_t same = __ballot(expert[i] >= 0);
        if (same == 0) break;  // (nothing behind it either)
        for (int b = 0; b < bits; ++b) {
            const bool set = expert[i] >> b & 1;
            const uint64_t those = __ballot(set);
            same &= set ? those : ~those;
        }
        const uint32_t before = __popcll(same & ((1ull << lane) - 1));
        const uint32_t counted = expert[i] >= 0 ? lds[wave][expert[i]] : 0u;
        rank[i] = counted + before;
        // (a wave's LDS operations keep their order: all lanes have read before the first of each expert writes)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        if (expert[i] >= 0 && before == 0) lds[wave][expert[i]] = counted + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    __syncthreads();
    // what stands before each wave's choices of an expert: the experts before, the chunks before, the waves before
    uint32_t of_experts = 0;
    for (int begin = 0; begin <= experts; begin += kLanes) {
        const int e = begin + static_cast<int>(threadIdx.x);
        uint32_t mine = 0;
        if (e <= experts) {
            if (counts != nullptr) {
                mine = totals[e];
            } else {
#pragma unroll
                for (int w = 0; w < kWaves; ++w) mine += lds[w][e];
            }
        }
        uint32_t total;
        uint32_t at = of_experts + sums_before(mine, of_waves, total);
        of_experts += total;
        if (e <= experts) {
            if (blockIdx.x == 0) offsets[e] = static_cast<int32_t>(at);
            if (counts != nullptr) at += counts[static_cast<int64_t>(e) * gridDim.x + blockIdx.x];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const uint32_t n = lds[w][e];
                lds[w][e] = at;
                at += n;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int64_t item = first + i * kWave;
        if (item < items) positions[item] = static_cast<int32_t>(lds[wave][expert[i]] + rank[i]);
    }
}

// ------------------------------------------------------------------------------------------
// dispatch and combine

struct RowPlan {
    row_t rows, items;
    int choices, channels;
    const int32_t* positions;
    const int32_t* routed;  // how many choices have an expert

    __device__ __forceinline__ uint32_t position(row_t row, int j) const { return static_cast<uint32_t>(positions[offset_of(row, static_cast<uint32_t>(choices)) + j]); }
    __device__ __forceinline__ uint32_t most() const { return min(static_cast<uint32_t>(max(*routed, 0)), items); }
};

// A lane's kWide channels of a row, 16 bytes or what a shorter row has of 8 and 4, wherever they are.  The last lane of a row that has no whole number of
// those takes some that its neighbour has too.  (2^20 x 7 bf16 there and back with gradients, two choices: 136 us channel by channel, 67 so.)
template <class E, int kWide_ = 16 / sizeof(E)>
struct Piece {
    static constexpr int kWide = kWide_;
    using Vector = E __attribute__((ext_vector_type(kWide)));
    using Unaligned = E __attribute__((ext_vector_type(kWide), aligned(sizeof(E))));
    using Floats = float __attribute__((ext_vector_type(kWide)));

    __device__ __forceinline__ static Vector load(const E* p) { return *reinterpret_cast<const Unaligned*>(p); }
    // (the two in one function, chosen by a flag, would become one store)
    template <bool kPast>
    __device__ __forceinline__ static void store(E* p, Vector v) {
        if constexpr (kPast) __builtin_nontemporal_store(v, reinterpret_cast<Unaligned*>(p));
        else *reinterpret_cast<Unaligned*>(p) = v;
    }
    __device__ __forceinline__ static Floats floats(Vector v) { return __builtin_convertvector(v, Floats); }
    __device__ __forceinline__ static Vector rounded(Floats v) { return __builtin_convertvector(v, Vector); }
};
// The same of a single channel.
template <class E>
struct Single {
    static constexpr int kWide = 1;
    using Vector = E __attribute__((ext_vector_type(1)));
    using Floats = float __attribute__((ext_vector_type(1)));

    __device__ __forceinline__ static Vector load(const E* p) { return Vector{*p}; }
    template <bool kPast>
    __device__ __forceinline__ static void store(E* p, Vector v) { *p = v[0]; }
    __device__ __forceinline__ static Floats floats(Vector v) { return Floats{static_cast<float>(v[0])}; }
    __device__ __forceinline__ static Vector rounded(Floats v) { return Vector{static_cast<E>(v[0])}; }
};

// A row to neighbouring lanes, a power of two of them, and from there on every `step`-th.
struct Group {
    row_t first, step;
    int lane;
    __device__ __forceinline__ Group(int log2_lanes)
        : first(blockIdx.x * static_cast<row_t>(kThreads >> log2_lanes) + (threadIdx.x >> log2_lanes)),
          step(gridDim.x * static_cast<row_t>(kThreads >> log2_lanes)),
          lane(threadIdx.x & ((1 << log2_lanes) - 1)) {}
};

// Each row is read once and written to the places of its choices.
template <class P, class E, bool kPast>
__global__ __launch_bounds__(kThreads) void dispatch_kernel(RowPlan plan, int log2_lanes, const E* __restrict__ x, uint32_t stride, E* __restrict__ sorted) {
    const Group g(log2_lanes);
    const uint32_t most = plan.most();
    for (row_t row = g.first; row < plan.rows; row += g.step) {
        const E* const from = x + offset_of(row, stride);
        for (int c = g.lane * P::kWide; c < plan.channels; c += P::kWide << log2_lanes) {
            const int at = min(c, plan.channels - P::kWide);
            const typename P::Vector v = P::load(from + at);
            for (int j = 0; j < plan.choices; ++j) {
                const uint32_t to = plan.position(row, j);
                if (to < plan.items) P::template store<kPast>(sorted + offset_of(to, plan.channels) + at, to < most ? v : typename P::Vector{});
            }
        }
    }
}

// out[t] = the sum, with weights or without, of the rows at t's choices; kMost at a time are on their way.
template <class P, class E, class W, int kMost>
__global__ __launch_bounds__(kThreads) void gather_kernel(RowPlan plan, int log2_lanes, const E* __restrict__ y, uint32_t stride, const W* __restrict__ weights,
                                                          E* __restrict__ out) {
    const Group g(log2_lanes);
    const uint32_t most = plan.most();
    const int step = P::kWide << log2_lanes;
    for (row_t row = g.first; row < plan.rows; row += g.step) {
        const E* from[kMost];
        float w[kMost];
        const auto choose = [&](int first) {
#pragma unroll
            for (int j = 0; j < kMost; ++j) {
                const bool there = first + j < plan.choices;
                const uint32_t at = there ? plan.position(row, first + j) : most;
                from[j] = at < most ? y + offset_of(at, stride) : nullptr;
                w[j] = from[j] != nullptr && weights != nullptr ? static_cast<float>(weights[offset_of(row, static_cast<uint32_t>(plan.choices)) + first + j]) : 1.0f;
            }
        };
        choose(0);
        for (int c = g.lane * P::kWide; c < plan.channels; c += step) {
            const int at = min(c, plan.channels - P::kWide);
            typename P::Floats sum{};
            for (int first = 0; first < plan.choices; first += kMost) {
                if (plan.choices > kMost) choose(first);
                typename P::Vector v[kMost];
#pragma unroll
                for (int j = 0; j < kMost; ++j)
                    if (from[j] != nullptr) v[j] = P::load(from[j] + at);
#pragma unroll
                for (int j = 0; j < kMost; ++j)
                    if (from[j] != nullptr) sum += P::floats(v[j]) * w[j];
            }
            P::template store<true>(out + offset_of(row, plan.channels) + at, P::rounded(sum));
        }
    }
}

// dy[p] = w do[t] (zeros behind the last choice that has an expert), dw = <do[t], y[p]>: each row of do is read once for kMost choices.
template <class P, class E, class W, int kMost, bool kPast>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(RowPlan plan, int log2_lanes, const E* __restrict__ grad, uint32_t grad_stride,
                                                                    const E* __restrict__ y, uint32_t stride, const W* __restrict__ weights,
                                                                    E* __restrict__ dy, W* __restrict__ dweights) {
    const Group g(log2_lanes);
    const uint32_t most = plan.most();
    for (row_t row = g.first; row < plan.rows; row += g.step) {
        for (int first = 0; first < plan.choices; first += kMost) {
            uint32_t position[kMost];
            float w[kMost], dot[kMost];
    #pragma unroll
            for (int j = 0; j < kMost; ++j) {
                const bool there = first + j < plan.choices;
                position[j] = there ? plan.position(row, first + j) : plan.items;
                w[j] = there && position[j] < most ? static_cast<float>(weights[offset_of(row, static_cast<uint32_t>(plan.choices)) + first + j]) : 0.0f;
                dot[j] = 0.0f;
            }
            for (int c = g.lane * P::kWide; c < plan.channels; c += P::kWide << log2_lanes) {
                const int at = min(c, plan.channels - P::kWide);
                const typename P::Floats d = P::floats(P::load(grad + offset_of(row, grad_stride) + at));
                typename P::Vector v[kMost];
                if (dweights != nullptr) {
    #pragma unroll
                    for (int j = 0; j < kMost; ++j)
                        if (position[j] < most) v[j] = P::load(y + offset_of(position[j], stride) + at);
                }
    #pragma unroll
                for (int j = 0; j < kMost; ++j) {
                    if (dy != nullptr && position[j] < plan.items)
                        P::template store<kPast>(dy + offset_of(position[j], plan.channels) + at, position[j] < most ? P::rounded(d * w[j]) : typename P::Vector{});
                    if (dweights != nullptr && position[j] < most) {
                        const typename P::Floats f = P::floats(v[j]);
    #pragma unroll
                        for (int i = 0; i < P::kWide; ++i) dot[j] += at + i >= c ? d[i] * f[i] : 0.0f;  // (each channel in one lane)
                    }
                }
            }
            if (dweights == nullptr) continue;
    #pragma unroll
            for (int j = 0; j < kMost; ++j) {
                for (int d = 1; d < 1 << log2_lanes; d *= 2) dot[j] += __shfl_xor(dot[j], d);
                if (g.lane == 0 && first + j < plan.choices) dweights[offset_of(row, static_cast<uint32_t>(plan.choices)) + first + j] = static_cast<W>(dot[j]);
            }
        }
    }
}

bool bad_plan(int64_t rows, int choices, int64_t channels) {
    return bad_rows(rows) || choices < 1 || choices > PENC_MAX_CHOICES || bad_rows(rows * choices) || channels < 1 || channels > PENC_MAX_CHANNELS;
}

// Runs f with the kind of piece that a row takes, and the lanes of a row, at most 2^most.
template <class E, class F>
int with_pieces(int64_t channels, int most, F&& f) {
    constexpr int kWide = Piece<E>::kWide;
    const auto log2_lanes = [most](int64_t pieces) {
        int n = 0;
        while (n < most && (1 << n) < pieces) ++n;
        return n;
    };
    if (channels >= kWide) return f(Piece<E>{}, log2_lanes((channels + kWide - 1) / kWide));
    if constexpr (kWide == 8) {
        if (channels >= 4) return f(Piece<E, 4>{}, log2_lanes((channels + 3) / 4));
    }
    if (channels >= 2) return f(Piece<E, 2>{}, log2_lanes((channels + 1) / 2));
    return f(Single<E>{}, 0);
}

// Rows that go to places of their own go past the caches where they are whole lines, or long; the ends of short ones would be read back from memory (2^20 x
// 48 bf16 to two places each: 61 us, past them 102; 64 channels 77 and 62; 50000 x 1000 fp16 53 and 50).
template <class F>
int with_past(const void* to, size_t row_bytes, F&& f) {
    if (aligned_to(to, 64) && (row_bytes % 64 == 0 || row_bytes >= 1024)) return f(std::true_type{});
    return f(std::false_type{});
}

template <class F>
int with_most(int choices, F&& f) {
    if (choices <= 1) return f(std::integral_constant<int, 1>{});
    if (choices <= 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 4>{});
}

RowPlan row_plan(int64_t rows, int choices, int64_t channels, const int32_t* positions, const int32_t* routed) {
    return {static_cast<row_t>(rows), static_cast<row_t>(rows * choices), choices, static_cast<int>(channels), positions, routed};
}

}  // namespace
}  // namespace penc

using namespace penc;

extern "C" {

int penc_route(int type, int64_t rows, int experts, int choices, int normalise, const void* logits, int64_t row_stride, float* weights, int32_t* chosen,
               void* stream) {
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        if (bad_rows(rows) || bad_stride(row_stride) || experts < 1 || experts > PENC_MAX_EXPERTS || choices < 1 || choices > experts ||
            choices > PENC_MAX_ROUTED || bad_rows(rows * choices))
            return PENC_ERR_BAD_LAYER_SIZE;
        if (rows == 0) return PENC_OK;
        if (!logits || !weights || !chosen) return PENC_ERR_NULL_POINTER;
        if (!aligned_to(logits, sizeof(E)) || !aligned_to(weights, 4) || !aligned_to(chosen, 4)) return PENC_ERR_MISALIGNED;
        return with_row_layout(experts, choices, [&](auto lanes, auto chunks, auto most) -> int {
            constexpr int kLanes = decltype(lanes)::value;
            route_kernel<E, kLanes, decltype(chunks)::value, decltype(most)::value>
                <<<grid_of(rows, kThreads / kLanes), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                    static_cast<row_t>(rows), experts, choices, normalise != 0, static_cast<const E*>(logits), static_cast<uint32_t>(row_stride), weights, chosen);
            return launched();
        });
    });
}

int penc_route_backward(int type, int64_t rows, int experts, int choices, int normalise, const void* logits, int64_t row_stride, const float* weights,
                        const int32_t* chosen, const float* grad, void* dlogits, void* stream) {
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        if (bad_rows(rows) || bad_stride(row_stride) || experts < 1 || experts > PENC_MAX_EXPERTS || choices < 1 || choices > experts ||
            choices > PENC_MAX_ROUTED || bad_rows(rows * choices))
            return PENC_ERR_BAD_LAYER_SIZE;
        if (rows == 0) return PENC_OK;
        if ((!normalise && !logits) || !weights || !chosen || !grad || !dlogits) return PENC_ERR_NULL_POINTER;
        if (!aligned_to(logits, sizeof(E)) || !aligned_to(dlogits, sizeof(E)) || !aligned_to(weights, 4) || !aligned_to(chosen, 4) || !aligned_to(grad, 4))
            return PENC_ERR_MISALIGNED;
        return with_row_layout(experts, choices, [&](auto lanes, auto chunks, auto most) -> int {
            constexpr int kLanes = decltype(lanes)::value;
            route_backward_kernel<E, kLanes, decltype(chunks)::value, decltype(most)::value>
                <<<grid_of(rows, kThreads / kLanes), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                    static_cast<row_t>(rows), experts, choices, normalise != 0, static_cast<const E*>(logits), static_cast<uint32_t>(row_stride), weights, chosen,
                    grad, static_cast<E*>(dlogits));
            return launched();
        });
    });
}

size_t penc_plan_workspace_bytes(int64_t items, int experts) {
    if (bad_rows(items) || experts < 1 || experts > PENC_MAX_EXPERTS || items <= kPlanAlone * kPlanMost) return 0;
    return 4 * (static_cast<size_t>(experts) + 1) * (static_cast<size_t>((items + kPlanChunk - 1) / kPlanChunk) + 1);
}

int penc_plan(int index_bytes, int64_t items, int experts, const void* chosen, int32_t* positions, int32_t* offsets, void* workspace, size_t workspace_bytes,
              void* stream) {
    if (index_bytes != 4 && index_bytes != 8) return PENC_ERR_UNSUPPORTED_TYPE;
    if (bad_rows(items) || experts < 1 || experts > PENC_MAX_EXPERTS) return PENC_ERR_BAD_LAYER_SIZE;
    if (!offsets || (items > 0 && (!chosen || !positions))) return PENC_ERR_NULL_POINTER;
    if (!aligned_to(chosen, index_bytes) || !aligned_to(positions, 4) || !aligned_to(offsets, 4) || !aligned_to(workspace, 4)) return PENC_ERR_MISALIGNED;
    const size_t need = penc_plan_workspace_bytes(items, experts);
    if (workspace_bytes < need) return PENC_ERR_WORKSPACE_TOO_SMALL;
    if (need > 0 && !workspace) return PENC_ERR_NULL_POINTER;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int bits = 1;
    while ((1 << bits) <= experts) ++bits;
    const auto plan = [&](auto index) -> int {
        using I = decltype(index);
        const I* const from = static_cast<const I*>(chosen);
        // up to 16384 choices: one workgroup, one launch
        const auto alone = [&](auto n) -> int {
            plan_place_kernel<I, kPlanAlone, decltype(n)::value><<<1, kPlanAlone, 0, s>>>(items, experts, bits, from, nullptr, nullptr, positions, offsets);
            return launched();
        };
        if (items <= kPlanAlone) return alone(std::integral_constant<int, 1>{});
        if (items <= kPlanAlone * 4) return alone(std::integral_constant<int, 4>{});
        if (items <= kPlanAlone * kPlanMost) return alone(std::integral_constant<int, kPlanMost>{});
        const int64_t chunks = (items + kPlanChunk - 1) / kPlanChunk;
        uint32_t* const totals = static_cast<uint32_t*>(workspace);
        uint32_t* const counts = totals + experts + 1;
        plan_count_kernel<I><<<static_cast<unsigned>(chunks), kThreads, 0, s>>>(items, experts, from, counts);
        if (const int rc = launched()) return rc;
        plan_scan_kernel<<<static_cast<unsigned>(experts + 1), kThreads, 0, s>>>(chunks, counts, totals);
        if (const int rc = launched()) return rc;
        plan_place_kernel<I, kThreads, kPlanItems><<<static_cast<unsigned>(chunks), kThreads, 0, s>>>(items, experts, bits, from, counts, totals, positions, offsets);
        return launched();
    };
    return index_bytes == 4 ? plan(int32_t{}) : plan(int64_t{});
}

int penc_dispatch(int type, int64_t rows, int choices, int64_t channels, const void* x, int64_t row_stride, const int32_t* positions, const int32_t* routed,
                  void* sorted, void* stream) {
    if (type != PENC_FP32 && type != PENC_FP16 && type != PENC_BF16) return PENC_ERR_UNSUPPORTED_TYPE;
    if (bad_plan(rows, choices, channels) || bad_stride(row_stride)) return PENC_ERR_BAD_LAYER_SIZE;
    if (rows == 0) return PENC_OK;
    if (!x || !positions || !routed || !sorted) return PENC_ERR_NULL_POINTER;
    const auto copy = [&](auto e) -> int {
        using E = decltype(e);
        if (!aligned_to(x, sizeof(E)) || !aligned_to(sorted, sizeof(E)) || !aligned_to(positions, 4) || !aligned_to(routed, 4)) return PENC_ERR_MISALIGNED;
        return with_pieces<E>(channels, kLog2Threads, [&](auto piece, int log2_lanes) -> int {
            return with_past(sorted, channels * sizeof(E), [&](auto past) -> int {
                dispatch_kernel<decltype(piece), E, decltype(past)::value><<<grid_of(rows, kThreads >> log2_lanes), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                    row_plan(rows, choices, channels, positions, routed), log2_lanes, static_cast<const E*>(x), static_cast<uint32_t>(row_stride),
                        static_cast<E*>(sorted));
                return launched();
            });
        });
    };
    return type == PENC_FP32 ? copy(uint32_t{}) : copy(uint16_t{});
}

int penc_combine(int type, int weight_type, int64_t rows, int choices, int64_t channels, const void* y, int64_t row_stride, const void* weights,
                 const int32_t* positions, const int32_t* routed, void* out, void* stream) {
    if (weight_type != type && weight_type != PENC_FP32) return PENC_ERR_UNSUPPORTED_TYPE;
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        if (bad_plan(rows, choices, channels) || bad_stride(row_stride)) return PENC_ERR_BAD_LAYER_SIZE;
        if (rows == 0) return PENC_OK;
        if (!y || !positions || !routed || !out) return PENC_ERR_NULL_POINTER;
        if (!aligned_to(y, sizeof(E)) || !aligned_to(out, sizeof(E)) || !aligned_to(weights, weight_type == PENC_FP32 ? 4 : 2) || !aligned_to(positions, 4) ||
            !aligned_to(routed, 4))
            return PENC_ERR_MISALIGNED;
        return with_pieces<E>(channels, kLog2Threads, [&](auto piece, int log2_lanes) -> int {
            return with_most(choices, [&](auto most) -> int {
                const auto launch = [&](auto w) -> int {
                    using W = decltype(w);
                    gather_kernel<decltype(piece), E, W, decltype(most)::value><<<grid_of(rows, kThreads >> log2_lanes), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                        row_plan(rows, choices, channels, positions, routed), log2_lanes, static_cast<const E*>(y), static_cast<uint32_t>(row_stride),
                        static_cast<const W*>(weights), static_cast<E*>(out));
                    return launched();
                };
                return weight_type == PENC_FP32 ? launch(float{}) : launch(e);
            });
        });
    });
}

int penc_combine_backward(int type, int weight_type, int64_t rows, int choices, int64_t channels, const void* grad, int64_t grad_row_stride, const void* y,
                          int64_t row_stride, const void* weights, const int32_t* positions, const int32_t* routed, void* dy, void* dweights, void* stream) {
    if (weight_type != type && weight_type != PENC_FP32) return PENC_ERR_UNSUPPORTED_TYPE;
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        if (bad_plan(rows, choices, channels) || bad_stride(row_stride) || bad_stride(grad_row_stride)) return PENC_ERR_BAD_LAYER_SIZE;
        if (rows == 0 || (!dy && !dweights)) return PENC_OK;
        if (!grad || !weights || !positions || !routed || (dweights && !y)) return PENC_ERR_NULL_POINTER;
        const size_t weight = weight_type == PENC_FP32 ? 4 : 2;
        if (!aligned_to(y, sizeof(E)) || !aligned_to(grad, sizeof(E)) || !aligned_to(dy, sizeof(E)) || !aligned_to(weights, weight) ||
            !aligned_to(dweights, weight) || !aligned_to(positions, 4) || !aligned_to(routed, 4))
            return PENC_ERR_MISALIGNED;
        return with_pieces<E>(channels, 6, [&](auto piece, int log2_lanes) -> int {
            return with_most(choices, [&](auto most) -> int {
                const auto launch = [&](auto w) -> int {
                    using W = decltype(w);
                    return with_past(dy, channels * sizeof(E), [&](auto past) -> int {
                        combine_backward_kernel<decltype(piece), E, W, decltype(most)::value, decltype(past)::value>
                            <<<grid_of(rows, kThreads >> log2_lanes), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                                row_plan(rows, choices, channels, positions, routed), log2_lanes, static_cast<const E*>(grad), static_cast<uint32_t>(grad_row_stride),
                                static_cast<const E*>(y), static_cast<uint32_t>(row_stride), static_cast<const W*>(weights), static_cast<E*>(dy),
                                    static_cast<W*>(dweights));
                        return launched();
                    });
                };
                return weight_type == PENC_FP32 ? launch(float{}) : launch(e);
            });
        });
    });
}

}  // extern "C"

// ------------------------------------------------------------------------------------------
// the experts' products (penc_expert_linear.hip)

namespace {

// Runs f with the type as a constant.
template <class F>
int with_constant_type(int type, F&& f) {
    switch (type) {
        case PENC_FP32: return f(std::integral_constant<int, PENC_FP32>{});
        case PENC_FP16: return f(std::integral_constant<int, PENC_FP16>{});
        case PENC_BF16: return f(std::integral_constant<int, PENC_BF16>{});
        default: return PENC_ERR_UNSUPPORTED_TYPE;
    }
}

bool bad_layer(int64_t rows, int experts, int64_t channels, int64_t outputs) {
    return bad_rows(rows) || experts < 1 || experts > PENC_MAX_EXPERTS || channels < 1 || channels > PENC_MAX_EXPERT_CHANNELS || outputs < 1 ||
           outputs > PENC_MAX_EXPERT_CHANNELS;
}
// (rows that overlap would not end where one is told that they do)
bool bad_row_stride(int64_t rows, int64_t stride, int64_t values) { return rows > 1 && (stride < values || stride > PENC_MAX_EXPERT_STRIDE); }

}  // namespace

extern "C" {

int penc_expert_linear(int type, int64_t rows, int experts, int64_t channels, int64_t outputs, const void* x, int64_t row_stride, const void* weight,
                       const void* bias, const int32_t* offsets, void* y, void* stream) {
    return with_constant_type(type, [&](auto constant) -> int {
        constexpr int kType = decltype(constant)::value;
        if (bad_layer(rows, experts, channels, outputs) || bad_row_stride(rows, row_stride, channels)) return PENC_ERR_BAD_LAYER_SIZE;
        if (rows == 0) return PENC_OK;
        if (!x || !weight || !offsets || !y) return PENC_ERR_NULL_POINTER;
        const size_t size = kType == PENC_FP32 ? 4 : 2;
        if (!aligned_to(x, size) || !aligned_to(weight, size) || !aligned_to(bias, size) || !aligned_to(y, size) || !aligned_to(offsets, 4))
            return PENC_ERR_MISALIGNED;
        return expert_rows<kType>(false, rows, experts, outputs, channels, x, rows > 1 ? row_stride : channels, weight, bias, offsets, y,
                                  static_cast<hipStream_t>(stream));
    });
}

int penc_expert_linear_input_grad(int type, int64_t rows, int experts, int64_t channels, int64_t outputs, const void* grad, int64_t grad_row_stride,
                                  const void* weight, const int32_t* offsets, void* dx, void* stream) {
    return with_constant_type(type, [&](auto constant) -> int {
        constexpr int kType = decltype(constant)::value;
        if (bad_layer(rows, experts, channels, outputs) || bad_row_stride(rows, grad_row_stride, outputs)) return PENC_ERR_BAD_LAYER_SIZE;
        if (rows == 0) return PENC_OK;
        if (!grad || !weight || !offsets || !dx) return PENC_ERR_NULL_POINTER;
        const size_t size = kType == PENC_FP32 ? 4 : 2;
        if (!aligned_to(grad, size) || !aligned_to(weight, size) || !aligned_to(dx, size) || !aligned_to(offsets, 4)) return PENC_ERR_MISALIGNED;
        return expert_rows<kType>(true, rows, experts, channels, outputs, grad, rows > 1 ? grad_row_stride : outputs, weight, nullptr, offsets, dx,
                                  static_cast<hipStream_t>(stream));
    });
}

size_t penc_expert_weight_grad_workspace_bytes(int type, int64_t rows, int experts, int64_t channels, int64_t outputs) {
    if (bad_layer(rows, experts, channels, outputs)) return 0;
    switch (type) {
        case PENC_FP32: return expert_weights_workspace<PENC_FP32>(rows, experts, channels, outputs);
        case PENC_FP16: return expert_weights_workspace<PENC_FP16>(rows, experts, channels, outputs);
        case PENC_BF16: return expert_weights_workspace<PENC_BF16>(rows, experts, channels, outputs);
        default: return 0;
    }
}

int penc_expert_linear_grads(int type, int64_t rows, int experts, int64_t channels, int64_t outputs, const void* x, int64_t row_stride, const void* grad,
                             int64_t grad_row_stride, const void* weight, const int32_t* offsets, void* dx, void* weight_grad, void* bias_grad, void* workspace,
                             size_t workspace_bytes, void* stream) {
    return with_constant_type(type, [&](auto constant) -> int {
        constexpr int kType = decltype(constant)::value;
        if (bad_layer(rows, experts, channels, outputs) || bad_row_stride(rows, row_stride, channels) || bad_row_stride(rows, grad_row_stride, outputs))
            return PENC_ERR_BAD_LAYER_SIZE;
        if ((rows > 0 && (!x || !grad || (dx && !weight))) || !offsets || !weight_grad) return PENC_ERR_NULL_POINTER;
        const size_t size = kType == PENC_FP32 ? 4 : 2, need = penc_expert_weight_grad_workspace_bytes(type, rows, experts, channels, outputs);
        if (!aligned_to(x, size) || !aligned_to(grad, size) || !aligned_to(weight, size) || !aligned_to(dx, size) || !aligned_to(weight_grad, size) ||
            !aligned_to(bias_grad, size) || !aligned_to(offsets, 4) || !aligned_to(workspace, 16))
            return PENC_ERR_MISALIGNED;
        if (workspace_bytes < need) return PENC_ERR_WORKSPACE_TOO_SMALL;
        if (need > 0 && !workspace) return PENC_ERR_NULL_POINTER;
        return expert_grads<kType>(rows, experts, channels, outputs, x, rows > 1 ? row_stride : channels, grad, rows > 1 ? grad_row_stride : outputs, weight, offsets,
                                   rows > 0 ? dx : nullptr, weight_grad, bias_grad, workspace, static_cast<hipStream_t>(stream));
    });
}

int penc_expert_weight_grad(int type, int64_t rows, int experts, int64_t channels, int64_t outputs, const void* x, int64_t row_stride, const void* grad,
                            int64_t grad_row_stride, const int32_t* offsets, void* weight_grad, void* bias_grad, void* workspace, size_t workspace_bytes,
                            void* stream) {
    return penc_expert_linear_grads(type, rows, experts, channels, outputs, x, row_stride, grad, grad_row_stride, nullptr, offsets, nullptr, weight_grad, bias_grad,
                                    workspace, workspace_bytes, stream);
}

size_t penc_expert_bias_grad_workspace_bytes(int type, int64_t rows, int experts, int64_t outputs) {
    if (bad_layer(rows, experts, 1, outputs)) return 0;
    switch (type) {
        case PENC_FP32: return expert_bias_workspace<PENC_FP32>(rows, experts, outputs);
        case PENC_FP16: return expert_bias_workspace<PENC_FP16>(rows, experts, outputs);
        case PENC_BF16: return expert_bias_workspace<PENC_BF16>(rows, experts, outputs);
        default: return 0;
    }
}

int penc_expert_bias_grad(int type, int64_t rows, int experts, int64_t outputs, const void* grad, int64_t grad_row_stride, const int32_t* offsets, void* bias_grad,
                          void* workspace, size_t workspace_bytes, void* stream) {
    return with_constant_type(type, [&](auto constant) -> int {
        constexpr int kType = decltype(constant)::value;
        if (bad_layer(rows, experts, 1, outputs) || bad_row_stride(rows, grad_row_stride, outputs)) return PENC_ERR_BAD_LAYER_SIZE;
        if ((rows > 0 && !grad) || !offsets || !bias_grad) return PENC_ERR_NULL_POINTER;
        const size_t size = kType == PENC_FP32 ? 4 : 2, need = penc_expert_bias_grad_workspace_bytes(type, rows, experts, outputs);
        if (!aligned_to(grad, size) || !aligned_to(bias_grad, size) || !aligned_to(offsets, 4) || !aligned_to(workspace, 16)) return PENC_ERR_MISALIGNED;
        if (workspace_bytes < need) return PENC_ERR_WORKSPACE_TOO_SMALL;
        if (need > 0 && !workspace) return PENC_ERR_NULL_POINTER;
        return expert_bias<kType>(rows, experts, outputs, grad, rows > 1 ? grad_row_stride : outputs, offsets, bias_grad, workspace, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
