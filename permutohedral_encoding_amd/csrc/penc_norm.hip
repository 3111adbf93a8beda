// What stands between a block and the next one, for rows of one type (PENC_TYPE: PENC_FP32, PENC_FP16 or PENC_BF16).
//
//     p = post norm(f),  y = s x + gate p,  n = pre norm(y);     norm(v) = v~ w + b,  v~ = (v - mean) r,  r = 1 / sqrt(mean (v - mean)^2 + eps)
//
// ("rms": without the mean).  Backward, at the checkpoints x^ and f^, statistics recomputed from them:
//
//     d = dn w_pre,  dY = dy + r_y (d - mean d - y~ mean(d y~)),  dx = s dY,  dp = dY gate
//     d = dp w_post, df = r_f (d - mean d - f~ mean(d f~))                                     (the "mean d" for "layer" alone)
//     sums over rows: dgate = dY p, dw_post = dp f~, db_post = dp, dw_pre = dn y~, db_pre = dn
//
// One pass over the rows in either direction, bound by memory: a row stays in the registers of its lanes, 8 channels each, from its first load to its
// last store.  The means go through the lanes (and, from 513 channels on, through the LDS), each wait for them serving all sums that are known by
// then: two on the way there, three back (rms; a mean has one more, before the squares around it).  The next row is loaded while a row is worked on.
//
// The sums over rows stay in registers while a workgroup walks over its rows; each workgroup leaves one row of partial sums, added up in a
// fixed order by sum_partials_kernel.  No atomics: results are the same in every run.
//
// Measured, with the checkpoints of x and f written and read (us, and the rate of the bytes that this takes; a copy on this card reaches 5.5 TB/s):
//
//     1048576 x 64 fp32 "rms"                              forward 234, 5.2 TB/s      backward 252, 4.8 TB/s
//     16384 x 4096 bf16 "rms"                                      121, 5.5                    156, 4.3
//     130944 x 203 fp16 "layer", a gate per 128 rows                66, 4.0                    102, 2.6
//
// The last is bound by instructions: 570 of the vector units for 8 channels of the backward, 60% of its time, in the three waves a SIMD has
// registers for.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "penc_kept.hpp"
#include "penc_norm.hpp"

namespace penc {
namespace {

__device__ __forceinline__ float across_rows(float v) {  // of 16 lanes: one from each such row of a wave
    // (v_permlane16_swap and v_permlane32_swap exchange rows between two registers: with one value in both, their sum is a row's and its partner's)
    const uint32_t u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float across_halves(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// The lanes of a workgroup, and sums over those of a row, the same in each of them.
template <int kLanes>
struct Row {
    static constexpr int kThreads = row_threads(kLanes);
    static constexpr int kRows = kThreads / kLanes;               // at a time
    static constexpr int kWaves = kLanes > 64 ? kLanes / 64 : 1;  // of one row

    float2* exchange;  // [2][kWaves]: a sum may begin while slow waves still read the one before it
    int turn = 0;

    template <int kOver>
    __device__ __forceinline__ static float in_wave(float v) {
        if constexpr (kOver >= 2) v += __uint_as_float(dpp<kSwapPairs>(__float_as_uint(v)));
        if constexpr (kOver >= 4) v += __uint_as_float(dpp<kSwapTwos>(__float_as_uint(v)));
        if constexpr (kOver >= 8) v += __uint_as_float(dpp<kMirrorHalfRow>(__float_as_uint(v)));
        if constexpr (kOver >= 16) v += __uint_as_float(dpp<kMirrorRow>(__float_as_uint(v)));
        if constexpr (kOver >= 32) v = across_rows(v);
        if constexpr (kOver >= 64) v = across_halves(v);
        return v;
    }
    __device__ __forceinline__ float2 sums(float a, float b) {
        float2 v = make_float2(in_wave<kLanes>(a), in_wave<kLanes>(b));
        if constexpr (kWaves > 1) {
            float2* const e = exchange + turn * kWaves;
            turn ^= 1;
            if (threadIdx.x % 64 == 0) e[threadIdx.x / 64] = v;
            __syncthreads();
            v = e[threadIdx.x % kWaves];
            v.x = in_wave<kWaves>(v.x), v.y = in_wave<kWaves>(v.y);
        }
        return v;
    }
    __device__ __forceinline__ float sum(float a) {
        if constexpr (kWaves == 1) return in_wave<kLanes>(a);
        else return sums(a, 0.0f).x;
    }
};

using Values = float[kChunk];

#define PENC_EACH _Pragma("unroll") for (int i = 0; i < kChunk; ++i)

// The eight channels that a lane has of a row.  Loads have no conditions, so that they can be under way while something else is done: a lane
// that would read behind the row reads its last eight channels, and `bring` moves those it has to the front.
template <class E, int kEnd>
struct Place {
    static constexpr bool kNarrow = kEnd == kNarrowRow, kWhole = kEnd == kWholeChunks;
    int channels, first, valid;
    float per_channel;

    template <class T>
    struct Fetched {
        uint32_t __attribute__((ext_vector_type(kChunk * sizeof(T) / 4))) w;
    };
    struct FetchedKept {
        uint2 q;
        uint32_t exponent;
    };

    __device__ __forceinline__ Place(int channels_, int lane)
        : channels(channels_), first(lane * kChunk), valid(max(0, min(channels_ - lane * kChunk, kChunk))), per_channel(1.0f / channels_) {}

    template <class T>
    __device__ __forceinline__ Fetched<T> fetch(const T* __restrict__ row) const {
        using Words = decltype(Fetched<T>::w);
        if constexpr (kNarrow) {
            T __attribute__((ext_vector_type(kChunk))) v;
            PENC_EACH v[i] = i < valid ? row[i] : static_cast<T>(0.0f);
            return {__builtin_bit_cast(Words, v)};
        } else {
            using Unaligned = uint32_t __attribute__((ext_vector_type(kChunk * sizeof(T) / 4), aligned(sizeof(T))));
            return {*reinterpret_cast<const Unaligned*>(row + min(first, channels - kChunk))};
        }
    }
    __device__ __forceinline__ FetchedKept fetch(const KeptArray& kept, row_t row) const {
        const int c = min(first, static_cast<int>(kept.pitch) - kChunk);
        return {*reinterpret_cast<const uint2*>(kept.values + offset_of(row, kept.pitch) + c), kept.exponents[offset_of(row, kept.blocks) + c / kKeptBlock]};
    }
    template <class T>
    __device__ __forceinline__ void bring(const Fetched<T>& f, Values& x) const {
        auto w = f.w;
        if constexpr (!kNarrow) {
            const uint32_t whole = valid == kChunk ? ~0u : 0u;
            if constexpr (kWhole) {  // (word by word: of the vectors' own operators the backward spills 38 registers and not 4, 16384 x 4096 bf16 156 -> 165 us)
#pragma unroll
                for (int i = 0; i < static_cast<int>(kChunk * sizeof(T) / 4); ++i) w[i] &= whole;
            } else {  // the row's last lane
                const auto m = to_front<T>(w, kChunk - (channels & 7));
                const uint32_t part = ~whole & (valid > 0 ? ~0u : 0u);
#pragma unroll
                for (int i = 0; i < static_cast<int>(kChunk * sizeof(T) / 4); ++i) w[i] = (w[i] & whole) | (m[i] & part);
            }
        }
        const float8 v = __builtin_convertvector(__builtin_bit_cast(T __attribute__((ext_vector_type(kChunk))), w), float8);
        PENC_EACH x[i] = v[i];
    }
    __device__ __forceinline__ void bring(const FetchedKept& f, Values& x, float scale = 1.0f) const {
        const uint32_t here = valid > 0 ? ~0u : 0u;
        restore(make_uint2(f.q.x & here, f.q.y & here), f.exponent & here, x, scale);
    }
    template <class T>
    __device__ __forceinline__ void store(T* __restrict__ row, const Values& x) const {
        if (valid <= 0) return;
        const auto y = rounded<T>(x);
        if (kWhole || valid == kChunk) store_whole(row + first, y);
        else store_part(row + first, channels & 7, y);
    }
    // a parameter, 0 behind the row's end
    __device__ __forceinline__ void given(const void* p, bool fp32, Values& x, uint64_t at = 0) const {
        if (fp32) bring(fetch(static_cast<const float*>(p) + at), x);
        else bring(fetch(static_cast<const E*>(p) + at), x);
    }
    // the same, or `none` for each channel; 0 behind the row's end takes away what the mean of a "layer" leaves there of a gradient
    __device__ __forceinline__ void param(const void* p, bool fp32, float none, Values& x) const {
        if (p != nullptr) given(p, fp32, x);
        else PENC_EACH x[i] = i < valid ? none : 0.0f;
    }
    // (a difference to the mean is zero behind the row's end)
    __device__ __forceinline__ void centre(Values& x, float mean) const {
        PENC_EACH x[i] = __uint_as_float(__float_as_uint(x[i] - mean) & static_cast<uint32_t>((kWhole ? -valid : i - valid) >> 31));
    }
};

__device__ __forceinline__ float total(const Values& x) {
    float s = 0.0f;
    PENC_EACH s += x[i];
    return s;
}
__device__ __forceinline__ float dot(const Values& x, const Values& y) {
    float s = 0.0f;
    PENC_EACH s = __builtin_fmaf(x[i], y[i], s);
    return s;
}

// Parameters of all rows, in the LDS: read again for every row, where registers for them would cost waves.
template <int kLanes, int kParams>
struct Shared {
    float4 v[kParams][2][kLanes];

    // (by the lanes of the workgroup's first row; a barrier follows)
    template <class P>
    __device__ __forceinline__ void load(int k, const P& at, const void* param, bool fp32, float none) {
        if (threadIdx.x >= kLanes) return;
        Values x;
        at.param(param, fp32, none, x);
        v[k][0][threadIdx.x] = make_float4(x[0], x[1], x[2], x[3]);
        v[k][1][threadIdx.x] = make_float4(x[4], x[5], x[6], x[7]);
    }
    __device__ __forceinline__ void get(int k, Values& x) const {
        const int lane = threadIdx.x % kLanes;
        const float4 a = v[k][0][lane], b = v[k][1][lane];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
};

// v becomes v~; returns r.
template <bool kFull, class P, class R>
__device__ __forceinline__ float normalise(Values& x, const NormArgs& a, const P& at, R& row) {
    if (kFull && a.layer) at.centre(x, row.sum(total(x)) * at.per_channel);
    const float r = rsqrtf(row.sum(dot(x, x)) * at.per_channel + a.eps);
    PENC_EACH x[i] *= r;
    return r;
}

// The rows that the lanes of a row go through: `run` consecutive ones, then the next run `stride` runs on, up to `end`; body(row, the first of
// its run, the last of its run, fetched).  `fetch` is called for a row while the one before it is worked on.
template <int kLanes, class Fetch, class Body>
__device__ __forceinline__ void walk(row_t row, row_t end, row_t run, row_t stride, Fetch&& fetch, Body&& body) {
    // (from a wave on, a row's number is that of all lanes: its addresses are computed once)
    const auto same = [](row_t v) { return kLanes < 64 ? v : static_cast<row_t>(__builtin_amdgcn_readfirstlane(v)); };
    row = same(row);
    if (row >= end) return;
    auto now = fetch(row);
    for (row_t k = 0; row < end;) {
        const bool ends = k + 1 == run;
        const row_t next = same(ends ? row + 1 + (stride - 1) * run : row + 1);
        auto ahead = fetch(min(next, end - 1));
        body(row, k == 0, ends, now);
        now = ahead;
        row = next;
        k = ends ? 0 : k + 1;
    }
}

// kFull: any kind of norm; else "rms" without biases, whose sums and parameters need 32 registers less (backward of 16384 x 4096 bf16 as "layer": 232 us
// instead of 156).
template <class E, int kLanes, int kEnd, bool kFull>
__global__ __launch_bounds__(Row<kLanes>::kThreads) void norm_kernel(NormArgs a, E* __restrict__ y_out, E* __restrict__ n_out) {
    using R = Row<kLanes>;
    using P = Place<E, kEnd>;
    __shared__ float2 exchange[2 * R::kWaves];
    R across{exchange};
    const P at(a.channels, threadIdx.x % kLanes);
    Values gate, post_weight, post_bias, pre_weight, pre_bias;
    at.param(a.post_weight, a.param_fp32, 1.0f, post_weight);
    at.param(a.pre_weight, a.param_fp32, 1.0f, pre_weight);
    if constexpr (kFull) {
        at.param(a.post_bias, a.param_fp32, 0.0f, post_bias);
        at.param(a.pre_bias, a.param_fp32, 0.0f, pre_bias);
    }
    at.param(a.gate, a.gate_fp32, 1.0f, gate);
    struct Fetched {
        typename P::template Fetched<E> x, f;
    };
    const auto fetch = [&](row_t row) {
        Fetched r;
        r.x = at.fetch(static_cast<const E*>(a.x) + offset_of(row, a.x_stride));
        if (a.has_branch) r.f = at.fetch(static_cast<const E*>(a.branch) + offset_of(row, a.branch_stride));
        return r;
    };
    // One gate: workgroups take rows in turn.  Else each takes rows that follow each other, and the gate changes seldom.
    row_t first = blockIdx.x * R::kRows + threadIdx.x / kLanes, end = a.rows, stride = gridDim.x * R::kRows, gate_until = 0;
    if (a.rows_per_gate != 0) {
        const row_t each = ((a.rows - 1) / stride + 1) * R::kRows, begin = min(blockIdx.x * each, a.rows);
        first = begin + threadIdx.x / kLanes, end = min(begin + each, a.rows), stride = R::kRows;
    }
    walk<kLanes>(first, end, 1, stride, fetch, [&](row_t row, bool, bool, const Fetched& fetched) {
        Values x, f;
        if (a.rows_per_gate != 0 && row >= gate_until) {
            const row_t group = row / a.rows_per_gate;
            gate_until = (group + 1) * a.rows_per_gate;
            if (a.gate != nullptr) at.given(a.gate, a.gate_fp32, gate, offset_of(group, a.channels));
        }
        at.bring(fetched.x, x);
        if (a.kept_x.values != nullptr) a.kept_x.store(row, at.first, x);
        PENC_EACH x[i] *= a.scale;
        if (a.has_branch) {
            at.bring(fetched.f, f);
            if (a.kept_branch.values != nullptr) a.kept_branch.store(row, at.first, f);
            if (a.post_norm) {
                normalise<kFull>(f, a, at, across);
                PENC_EACH f[i] = kFull ? __builtin_fmaf(f[i], post_weight[i], post_bias[i]) : f[i] * post_weight[i];
            }
            PENC_EACH x[i] = __builtin_fmaf(gate[i], f[i], x[i]);
        }
        if (y_out != nullptr) at.store(y_out + offset_of(row, a.channels), x);
        if (a.pre_norm) {
            // (of y before it is rounded)
            normalise<kFull>(x, a, at, across);
            PENC_EACH x[i] = kFull ? __builtin_fmaf(x[i], pre_weight[i], pre_bias[i]) : x[i] * pre_weight[i];
            at.store(n_out + offset_of(row, a.channels), x);
        }
    });
}

// The sums of one of a lane's accumulators over the rows that a workgroup has at a time: `store` gets them in the lanes of the first.
template <int kLanes, class F>
__device__ __forceinline__ void write_sum(const Values& sum, float (*__restrict__ lds)[kChunk], F&& store) {
    constexpr int kRows = Row<kLanes>::kRows;
    Values all;
    PENC_EACH all[i] = sum[i];
    if constexpr (kRows > 1) {
        PENC_EACH lds[threadIdx.x][i] = all[i];
        __syncthreads();
        if (threadIdx.x < kLanes) {
#pragma unroll 1
            for (int r = 1; r < kRows; ++r) PENC_EACH all[i] += lds[r * kLanes + threadIdx.x][i];
        }
        __syncthreads();
    }
    if (threadIdx.x < kLanes) store(all);
}

// kKept: x and the branch are read from their checkpoints.
//
// Waves to a SIMD, by what the kernel needs in registers: four, of 128, for "rms" without biases, which 16-bit rows of up to 512 channels fit, wider ones but for 2 to
// 4 registers that are spilled, fp32 but for up to 14; three, of 168, for the others, which spill none; and two where a workgroup is eight waves, of which a
// compute unit holds one or two and not one and a half.  Rows of more than 4096 channels are workgroups of 16 waves, which have 128 registers and no choice:
// "layer" spills 18 to 64 there.  (Four waves of "layer" with 4096 channels spill: 331 us instead of 232.)
//
// Gates of groups of rows: with few rows in a group (a.gate_by_lanes) the lanes of a row take whole groups and write their sums themselves; else a
// workgroup takes a piece of a group, `pieces` of them to a group, and leaves a row of partial sums.  One gate for all rows is one more sum over rows.
template <class E, int kLanes, int kEnd, bool kFull, bool kKept>
__global__ __launch_bounds__(Row<kLanes>::kThreads, !kFull ? 4 : kLanes == 512 ? 2 : 3) void norm_backward_kernel(NormArgs a, NormGrads g) {
    using R = Row<kLanes>;
    using P = Place<E, kEnd>;
    __shared__ float2 exchange[2 * R::kWaves];
    __shared__ float lds[R::kRows > 1 ? R::kThreads : 1][kChunk];
    __shared__ Shared<kLanes, kFull ? 4 : 2> params;
    constexpr int kPostWeight = 0, kPreWeight = 1, kPostBias = 2, kPreBias = 3;
    R across{exchange};
    const P at(a.channels, threadIdx.x % kLanes);
    params.load(kPostWeight, at, a.post_weight, a.param_fp32, 1.0f);
    params.load(kPreWeight, at, a.pre_weight, a.param_fp32, 1.0f);
    if constexpr (kFull) {
        params.load(kPostBias, at, a.post_bias, a.param_fp32, 0.0f);
        params.load(kPreBias, at, a.pre_bias, a.param_fp32, 0.0f);
    }
    Values gate;
    at.param(a.gate, a.gate_fp32, 1.0f, gate);
    __syncthreads();
    Values d_gate{}, d_post_weight{}, d_post_bias{}, d_pre_weight{}, d_pre_bias{};

    using Input = std::conditional_t<kKept, typename P::FetchedKept, typename P::template Fetched<E>>;
    struct Fetched {
        Input x, f;
        typename P::template Fetched<E> dy, dn;
    };
    const auto fetch = [&](row_t row) {
        Fetched r;
        if constexpr (kKept) {
            r.x = at.fetch(a.kept_x, row);
            if (a.has_branch) r.f = at.fetch(a.kept_branch, row);
        } else {
            r.x = at.fetch(static_cast<const E*>(a.x) + offset_of(row, a.x_stride));
            if (a.has_branch) r.f = at.fetch(static_cast<const E*>(a.branch) + offset_of(row, a.branch_stride));
        }
        if (g.y != nullptr) r.dy = at.fetch(static_cast<const E*>(g.y) + offset_of(row, g.y_stride));
        if (g.n != nullptr) r.dn = at.fetch(static_cast<const E*>(g.n) + offset_of(row, g.n_stride));
        return r;
    };
    const auto one_row = [&](row_t row, const Fetched& fetched) {
        Values y, f, dy;
        float r_f = 1.0f;
        // p, computed twice: its registers would be held all the way
        const auto inner = [&](Values& p) {
            PENC_EACH p[i] = f[i];
            if (!a.post_norm) return;
            Values w;
            params.get(kPostWeight, w);
            PENC_EACH p[i] *= w[i];
            if constexpr (kFull) {
                params.get(kPostBias, w);
                PENC_EACH p[i] += w[i];
            }
        };
        if constexpr (kKept) {
            at.bring(fetched.x, y, a.scale);
        } else {
            at.bring(fetched.x, y);
            PENC_EACH y[i] *= a.scale;
        }
        if (a.has_branch) {
            at.bring(fetched.f, f);
            if (a.post_norm) {
                r_f = normalise<kFull>(f, a, at, across);
            }
            Values p;
            inner(p);
            PENC_EACH y[i] = __builtin_fmaf(gate[i], p[i], y[i]);
        }
        if (g.y != nullptr) at.bring(fetched.dy, dy);
        else PENC_EACH dy[i] = 0.0f;
        if (g.n != nullptr) {
            Values dn, d;
            at.bring(fetched.dn, dn);
            params.get(kPreWeight, d);
            PENC_EACH d[i] *= dn[i];
            float mean = 0.0f;
            if (kFull && a.layer) {
                const float2 s = across.sums(total(y), total(d));
                at.centre(y, s.x * at.per_channel);
                mean = s.y * at.per_channel;
            }
            const float2 s = across.sums(dot(y, y), dot(d, y));
            const float r_y = rsqrtf(s.x * at.per_channel + a.eps), along = s.y * at.per_channel * r_y;
            PENC_EACH {
                y[i] *= r_y;
                d_pre_weight[i] = __builtin_fmaf(dn[i], y[i], d_pre_weight[i]);
                if (kFull) d_pre_bias[i] += dn[i];
                dy[i] = __builtin_fmaf(r_y, d[i] - mean - y[i] * along, dy[i]);
            }
        }
        if (g.x != nullptr) {
            Values dx;
            PENC_EACH dx[i] = a.scale * dy[i];
            at.store(static_cast<E*>(g.x) + offset_of(row, a.channels), dx);
        }
        if (!a.has_branch) return;
        Values p;
        inner(p);
        PENC_EACH {
            d_gate[i] = __builtin_fmaf(dy[i], p[i], d_gate[i]);
            dy[i] *= gate[i];
        }
        if (a.post_norm) {
            params.get(kPostWeight, p);
            PENC_EACH {
                d_post_weight[i] = __builtin_fmaf(dy[i], f[i], d_post_weight[i]);
                if (kFull) d_post_bias[i] += dy[i];
                dy[i] *= p[i];
            }
            if (g.branch != nullptr) {
                const float2 s = across.sums(dot(dy, f), kFull ? total(dy) : 0.0f);
                const float along = s.x * at.per_channel, mean = kFull && a.layer ? s.y * at.per_channel : 0.0f;
                PENC_EACH dy[i] = r_f * (dy[i] - mean - f[i] * along);
            }
        }
        if (g.branch != nullptr) at.store(static_cast<E*>(g.branch) + offset_of(row, a.channels), dy);
    };

    const auto store_gate = [&](row_t group, const Values& v) {
        if (a.gate_fp32) at.store(static_cast<float*>(g.gate) + offset_of(group, a.channels), v);
        else at.store(static_cast<E*>(g.gate) + offset_of(group, a.channels), v);
    };
    const auto leave = [&](float* sums, row_t at_row, const Values& v) {
        if (sums != nullptr) write_sum<kLanes>(v, lds, [&](const Values& t) { at.store(sums + offset_of(at_row, a.channels), t); });
    };
    // one gate, or gates by lanes: a workgroup has one unit of rows; else it has pieces of groups, one after the other
    const bool pieces = a.rows_per_gate != 0 && !a.gate_by_lanes;
    const row_t units = pieces ? a.rows / a.rows_per_gate * g.pieces : gridDim.x;
    const row_t run = a.gate_by_lanes ? a.rows_per_gate : 1;
    for (row_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        row_t group = unit * R::kRows + threadIdx.x / kLanes, first = group * run, end = a.rows, stride = gridDim.x * R::kRows;
        if (pieces) {
            group = unit / g.pieces;
            first = group * a.rows_per_gate + unit % g.pieces * g.piece_rows;
            end = min(first + g.piece_rows, (group + 1) * a.rows_per_gate);
            first += threadIdx.x / kLanes;
            stride = R::kRows;
            if (a.gate != nullptr) at.given(a.gate, a.gate_fp32, gate, offset_of(group, a.channels));
        }
        walk<kLanes>(first, end, run, stride, fetch, [&](row_t row, bool begins, bool ends, const Fetched& fetched) {
            if (a.gate_by_lanes && begins && a.gate != nullptr) at.given(a.gate, a.gate_fp32, gate, offset_of(group, a.channels));
            one_row(row, fetched);
            if (!a.gate_by_lanes || !ends) return;
            if (g.gate != nullptr) store_gate(group, d_gate);
            PENC_EACH d_gate[i] = 0.0f;
            group += stride;
        });
        if (a.gate_by_lanes) break;
        if (pieces && g.pieces == 1 && g.gate != nullptr) write_sum<kLanes>(d_gate, lds, [&](const Values& v) { store_gate(group, v); });
        else leave(g.gate_sums, unit, d_gate);
        PENC_EACH d_gate[i] = 0.0f;
    }
    leave(g.sums[0], blockIdx.x, d_post_weight);
    leave(g.sums[2], blockIdx.x, d_pre_weight);
    if constexpr (kFull) {
        leave(g.sums[1], blockIdx.x, d_post_bias);
        leave(g.sums[3], blockIdx.x, d_pre_bias);
    }
}

#undef PENC_EACH

// to[group][c] = the sum over `rows` rows of partial sums of a group, in a fixed order; 32 channels and 32 strands of rows to a workgroup, which waits
// for memory and not for its bytes: 5 us behind the backward of 1048576 x 64.
template <class E>
__global__ __launch_bounds__(1024) void sum_partials_kernel(SumPartials s) {
    __shared__ float lds[32][33];
    const Sum sum = s.sums[blockIdx.y];
    const int64_t tiles = (s.channels + 31) / 32;
    const int64_t group = blockIdx.x / tiles;
    const int c = static_cast<int>(blockIdx.x % tiles) * 32 + threadIdx.x % 32, strand = threadIdx.x / 32;
    if (group >= sum.groups) return;
    float total = 0.0f;
    if (c < s.channels) {
        const float* const from = sum.from + group * sum.rows * s.channels + c;
#pragma unroll 8
        for (int64_t r = strand; r < sum.rows; r += 32) total += from[r * s.channels];
    }
    lds[strand][threadIdx.x % 32] = total;
    __syncthreads();
    if (strand != 0 || c >= s.channels) return;
    for (int i = 1; i < 32; ++i) total += lds[i][threadIdx.x];
    if (sum.fp32) static_cast<float*>(sum.to)[group * s.channels + c] = total;
    else static_cast<E*>(sum.to)[group * s.channels + c] = static_cast<E>(total);
}

template <class E>
int launch_norm(const NormArgs& a, void* y, void* n, hipStream_t stream) {
    return with_row_shape(a.channels, [&](auto lanes, auto end) {
        constexpr int kLanes = decltype(lanes)::value, kEnd = decltype(end)::value;
        const dim3 grid(static_cast<unsigned>(std::min<int64_t>((a.rows + Row<kLanes>::kRows - 1) / Row<kLanes>::kRows, most_groups(kLanes, false)))), threads(Row<kLanes>::kThreads);
        if (is_full(a)) hipLaunchKernelGGL((norm_kernel<E, kLanes, kEnd, true>), grid, threads, 0, stream, a, static_cast<E*>(y), static_cast<E*>(n));
        else hipLaunchKernelGGL((norm_kernel<E, kLanes, kEnd, false>), grid, threads, 0, stream, a, static_cast<E*>(y), static_cast<E*>(n));
        return launched();
    });
}

template <class E>
int launch_norm_backward(const NormArgs& a, const NormGrads& g, unsigned grid, hipStream_t stream) {
    return with_row_shape(a.channels, [&](auto lanes, auto end) {
        constexpr int kLanes = decltype(lanes)::value, kEnd = decltype(end)::value;
        const auto launch = [&](auto full, auto kept) {
            hipLaunchKernelGGL((norm_backward_kernel<E, kLanes, kEnd, decltype(full)::value, decltype(kept)::value>), dim3(grid), dim3(Row<kLanes>::kThreads), 0,
                               stream, a, g);
            return launched();
        };
        const auto with_kept = [&](auto full) { return a.kept_x.values != nullptr ? launch(full, std::true_type{}) : launch(full, std::false_type{}); };
        return is_full(a) || g.sums[1] != nullptr || g.sums[3] != nullptr ? with_kept(std::true_type{}) : with_kept(std::false_type{});
    });
}

template <class E>
int launch_sum_partials(const SumPartials& s, unsigned grid, int n, hipStream_t stream) {
    hipLaunchKernelGGL(sum_partials_kernel<E>, dim3(grid, n), dim3(1024), 0, stream, s);
    return launched();
}

}  // namespace

#if PENC_TYPE == PENC_FP32
using Element = float;
#elif PENC_TYPE == PENC_FP16
using Element = half_t;
#else
using Element = bf16_t;
#endif

template <>
NormLaunches norm_launches<PENC_TYPE>() {
    return {launch_norm<Element>, launch_norm_backward<Element>, launch_sum_partials<Element>};
}

}  // namespace penc
