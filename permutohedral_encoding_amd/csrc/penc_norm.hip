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
// One pass over the rows in either direction: a row stays in the registers of its lanes, 8 or 16 channels each, from its first load to its last
// store, and the means go through the lanes (and, from 1025 channels on, through the LDS).  Bound by memory.
//
// The sums over rows stay in registers while a workgroup walks over its rows; each workgroup leaves one row of partial sums, added up in a
// fixed order by sum_partials_kernel.  No atomics: results are the same in every run.
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


// The lanes of a workgroup, and the sum over those of a row.
template <int kLanes>
struct Row {
    static constexpr int kThreads = kLanes > 256 ? kLanes : 256;
    static constexpr int kRows = kThreads / kLanes;           // at a time
    static constexpr int kWaves = kLanes > 64 ? kLanes / 64 : 1;  // of one row

    float2* exchange;  // [2][kWaves]: a reduction may begin while slow waves still read the one before it
    int turn = 0;

    __device__ __forceinline__ static float in_wave(float v) {
        v += __uint_as_float(dpp<kSwapPairs>(__float_as_uint(v)));
        v += __uint_as_float(dpp<kSwapTwos>(__float_as_uint(v)));
        if constexpr (kLanes >= 8) v += __uint_as_float(dpp<kMirrorHalfRow>(__float_as_uint(v)));
        if constexpr (kLanes >= 16) v += __uint_as_float(dpp<kMirrorRow>(__float_as_uint(v)));
        if constexpr (kLanes >= 32) v = across_rows(v);
        if constexpr (kLanes >= 64) v = across_halves(v);
        return v;
    }
    __device__ __forceinline__ float2 sums(float a, float b) {
        float2 v = make_float2(in_wave(a), in_wave(b));
        if constexpr (kWaves > 1) {
            float2* const e = exchange + turn * kWaves;
            turn ^= 1;
            if (threadIdx.x % 64 == 0) e[threadIdx.x / 64] = v;
            __syncthreads();
            v = e[0];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) v.x += e[i].x, v.y += e[i].y;
        }
        return v;
    }
    __device__ __forceinline__ float sum(float a) {
        if constexpr (kWaves == 1) return in_wave(a);
        else return sums(a, 0.0f).x;
    }
};

template <int kVectors>
struct Values {
    float v[kVectors][kChunk];
};

// What a lane has of a row: kVectors times 8 channels, kLanes chunks apart.
template <class E, int kLanes, int kVectors>
struct Place {
    int channels, first;
    float per_channel;
    __device__ __forceinline__ Place(int channels_, int lane) : channels(channels_), first(lane * kChunk), per_channel(1.0f / channels_) {}
    __device__ __forceinline__ int channel(int j) const { return first + j * kLanes * kChunk; }
    __device__ __forceinline__ int valid(int j) const { return min(channels - channel(j), kChunk); }

    __device__ __forceinline__ void load(const E* row, Values<kVectors>& x) const {
#pragma unroll
        for (int j = 0; j < kVectors; ++j) load_chunk(row + channel(j), valid(j), x.v[j]);
    }
    __device__ __forceinline__ void load(const KeptArray& kept, int64_t row, Values<kVectors>& x) const {
#pragma unroll
        for (int j = 0; j < kVectors; ++j) kept.load(row, channel(j), valid(j), x.v[j]);
    }
    __device__ __forceinline__ void keep(const KeptArray& kept, int64_t row, const Values<kVectors>& x) const {
#pragma unroll
        for (int j = 0; j < kVectors; ++j) kept.store(row, channel(j), x.v[j]);
    }
    __device__ __forceinline__ void store(E* row, const Values<kVectors>& x) const {
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
            if (valid(j) > 0) store_chunk(row + channel(j), valid(j), x.v[j]);
    }
    __device__ __forceinline__ void load(const void* param, bool fp32, float none, Values<kVectors>& x, int64_t at = 0) const {
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
            if (param != nullptr) {
                load_param<E>(param, fp32, at + channel(j), valid(j), x.v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < kChunk; ++i) x.v[j][i] = none;
            }
        }
    }
    // v becomes v~; returns r.  Channels behind the row's end stay zero.
    __device__ __forceinline__ float normalise(Values<kVectors>& x, bool layer, float eps, Row<kLanes>& row) const {
        if (layer) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) s += x.v[j][i];
            const float mean = row.sum(s) * per_channel;
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) x.v[j][i] = i < valid(j) ? x.v[j][i] - mean : 0.0f;
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) s = __builtin_fmaf(x.v[j][i], x.v[j][i], s);
        const float r = rsqrtf(row.sum(s) * per_channel + eps);
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) x.v[j][i] *= r;
        return r;
    }
    // d becomes r (d - mean d - v~ mean(d v~))
    __device__ __forceinline__ void through_norm(Values<kVectors>& d, const Values<kVectors>& normed, float r, bool layer, Row<kLanes>& row) const {
        float s = 0.0f, t = 0.0f;
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
                s += d.v[j][i];
                t = __builtin_fmaf(d.v[j][i], normed.v[j][i], t);
            }
        const float2 sums = row.sums(s, t);
        const float mean = layer ? sums.x * per_channel : 0.0f, along = sums.y * per_channel;
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) d.v[j][i] = r * (d.v[j][i] - mean - normed.v[j][i] * along);
    }
};

// The parameters of a lane's channels, loaded again for every row where a lane has more than 8 of them: they come from the caches, and
// their registers would cost waves.
template <class E, int kLanes, int kVectors>
struct Params {
    Values<kVectors> gate, post_weight, post_bias, pre_weight, pre_bias;

    __device__ __forceinline__ void load_shared(const NormArgs& a, const Place<E, kLanes, kVectors>& at) {
        at.load(a.post_weight, a.param_fp32, 1.0f, post_weight);
        at.load(a.post_bias, a.param_fp32, 0.0f, post_bias);
        at.load(a.pre_weight, a.param_fp32, 1.0f, pre_weight);
        at.load(a.pre_bias, a.param_fp32, 0.0f, pre_bias);
    }
    __device__ __forceinline__ void load_gate(const NormArgs& a, const Place<E, kLanes, kVectors>& at, int64_t group) {
        at.load(a.gate, a.gate_fp32, 1.0f, gate, group * a.channels);
    }
};

template <class E, int kLanes, int kVectors>
__global__ __launch_bounds__(Row<kLanes>::kThreads) void norm_kernel(NormArgs a, E* __restrict__ y_out, E* __restrict__ n_out) {
    using R = Row<kLanes>;
    __shared__ float2 exchange[2 * R::kWaves];
    R across{exchange};
    const Place<E, kLanes, kVectors> at(a.channels, threadIdx.x % kLanes);
    Params<E, kLanes, kVectors> p;
    if constexpr (kVectors == 1) {
        p.load_shared(a, at);
        if (a.rows_per_gate == 0) p.load_gate(a, at, 0);
    }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * R::kRows + threadIdx.x / kLanes; row < a.rows;
         row += static_cast<int64_t>(gridDim.x) * R::kRows) {
        Values<kVectors> x, f;
        at.load(static_cast<const E*>(a.x) + row * a.x_stride, x);
        if (a.has_branch) at.load(static_cast<const E*>(a.branch) + row * a.branch_stride, f);
        if constexpr (kVectors > 1) p.load_shared(a, at);
        if (a.rows_per_gate != 0) p.load_gate(a, at, group_of(row, a.rows_per_gate));
        else if constexpr (kVectors > 1) p.load_gate(a, at, 0);
        if (a.kept_x.values != nullptr) at.keep(a.kept_x, row, x);
        if (a.kept_branch.values != nullptr) at.keep(a.kept_branch, row, f);
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) x.v[j][i] *= a.scale;
        if (a.has_branch) {
            if (a.post_norm) {
                at.normalise(f, a.layer, a.eps, across);
#pragma unroll
                for (int j = 0; j < kVectors; ++j)
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) f.v[j][i] = __builtin_fmaf(f.v[j][i], p.post_weight.v[j][i], p.post_bias.v[j][i]);
            }
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) x.v[j][i] = __builtin_fmaf(p.gate.v[j][i], f.v[j][i], x.v[j][i]);
        }
        if (y_out != nullptr) at.store(y_out + row * a.channels, x);
        if (a.pre_norm) {
            // (of y before it is rounded)
            at.normalise(x, a.layer, a.eps, across);
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) x.v[j][i] = __builtin_fmaf(x.v[j][i], p.pre_weight.v[j][i], p.pre_bias.v[j][i]);
            at.store(n_out + row * a.channels, x);
        }
    }
}

// The sums of one of a lane's accumulators over the rows that a workgroup has at a time: `store` gets them from the lanes of the first.
template <int kLanes, int kVectors, class F>
__device__ __forceinline__ void write_sum(const Values<kVectors>& sum, float (*__restrict__ lds)[kChunk], int channels, F&& store) {
    constexpr int kRows = Row<kLanes>::kRows;
    const int lane = threadIdx.x % kLanes;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
        float total[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) total[i] = sum.v[j][i];
        if constexpr (kRows > 1) {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) lds[threadIdx.x][i] = total[i];
            __syncthreads();
            if (threadIdx.x < kLanes) {
#pragma unroll 1
                for (int r = 1; r < kRows; ++r)
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) total[i] += lds[r * kLanes + lane][i];
            }
            __syncthreads();
        }
        const int c = (lane + j * kLanes) * kChunk;
        if (threadIdx.x < kLanes && c < channels) store(c, min(channels - c, kChunk), total);
    }
}

// kKept: x and the branch are read from their checkpoints.
//
// Gates of groups of rows: with few rows in a group (a.gate_by_lanes) the lanes of a row take whole groups and write their sums themselves; else a
// workgroup takes a piece of a group, `pieces` of them to a group, and leaves a row of partial sums.  One gate for all rows is one more sum over rows.
template <class E, int kLanes, int kVectors, bool kKept>
__global__ __launch_bounds__(Row<kLanes>::kThreads) void norm_backward_kernel(NormArgs a, NormGrads g) {
    using R = Row<kLanes>;
    __shared__ float2 exchange[2 * R::kWaves];
    __shared__ float lds[R::kRows > 1 ? R::kThreads : 1][kChunk];
    R across{exchange};
    const Place<E, kLanes, kVectors> at(a.channels, threadIdx.x % kLanes);
    Params<E, kLanes, kVectors> p;
    if constexpr (kVectors == 1) {
        p.load_shared(a, at);
        p.load_gate(a, at, 0);
    }
    Values<kVectors> d_gate{}, d_post_weight{}, d_post_bias{}, d_pre_weight{}, d_pre_bias{};

    const auto one_row = [&](int64_t row, int64_t group, bool new_gate) {
        Values<kVectors> x, f, dn, dy;
        if constexpr (kKept) {
            at.load(a.kept_x, row, x);
            if (a.has_branch) at.load(a.kept_branch, row, f);
        } else {
            at.load(static_cast<const E*>(a.x) + row * a.x_stride, x);
            if (a.has_branch) at.load(static_cast<const E*>(a.branch) + row * a.branch_stride, f);
        }
        if (g.y != nullptr) at.load(static_cast<const E*>(g.y) + row * g.y_stride, dy);
        else at.load(nullptr, false, 0.0f, dy);
        if (g.n != nullptr) at.load(static_cast<const E*>(g.n) + row * g.n_stride, dn);
        if constexpr (kVectors > 1) p.load_shared(a, at);
        if (kVectors > 1 || new_gate) p.load_gate(a, at, group);
        float r_f = 1.0f;
        Values<kVectors> inner;
        if (a.has_branch) {
            if (a.post_norm) r_f = at.normalise(f, a.layer, a.eps, across);
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    inner.v[j][i] = a.post_norm ? __builtin_fmaf(f.v[j][i], p.post_weight.v[j][i], p.post_bias.v[j][i]) : f.v[j][i];
                    x.v[j][i] = __builtin_fmaf(p.gate.v[j][i], inner.v[j][i], a.scale * x.v[j][i]);
                }
        } else {
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) x.v[j][i] *= a.scale;
        }
        if (g.n != nullptr) {
            const float r_y = at.normalise(x, a.layer, a.eps, across);
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    d_pre_weight.v[j][i] = __builtin_fmaf(dn.v[j][i], x.v[j][i], d_pre_weight.v[j][i]);
                    d_pre_bias.v[j][i] += dn.v[j][i];
                    dn.v[j][i] *= p.pre_weight.v[j][i];
                }
            at.through_norm(dn, x, r_y, a.layer, across);
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) dy.v[j][i] += dn.v[j][i];
        }
        if (g.x != nullptr) {
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) x.v[j][i] = a.scale * dy.v[j][i];
            at.store(static_cast<E*>(g.x) + row * a.channels, x);
        }
        if (!a.has_branch) return;
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
                d_gate.v[j][i] = __builtin_fmaf(dy.v[j][i], inner.v[j][i], d_gate.v[j][i]);
                dy.v[j][i] *= p.gate.v[j][i];
            }
        if (a.post_norm) {
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    d_post_weight.v[j][i] = __builtin_fmaf(dy.v[j][i], f.v[j][i], d_post_weight.v[j][i]);
                    d_post_bias.v[j][i] += dy.v[j][i];
                    dy.v[j][i] *= p.post_weight.v[j][i];
                }
            if (g.branch != nullptr) at.through_norm(dy, f, r_f, a.layer, across);
        }
        if (g.branch != nullptr) at.store(static_cast<E*>(g.branch) + row * a.channels, dy);
    };

    const auto store_gate = [&](int64_t group, int c, int valid, const float(&v)[kChunk]) {
        if (a.gate_fp32) store_chunk(static_cast<float*>(g.gate) + group * a.channels + c, valid, v);
        else store_chunk(static_cast<E*>(g.gate) + group * a.channels + c, valid, v);
    };
    const auto leave = [&](float* sums, int64_t at_row, const Values<kVectors>& v) {
        if (sums != nullptr)
            write_sum<kLanes, kVectors>(v, lds, a.channels,
                                        [&](int c, int valid, const float(&t)[kChunk]) { store_chunk(sums + at_row * a.channels + c, valid, t); });
    };
    const int sub = threadIdx.x / kLanes;
    if (a.rows_per_gate == 0) {
        for (int64_t row = static_cast<int64_t>(blockIdx.x) * R::kRows + sub; row < a.rows; row += static_cast<int64_t>(gridDim.x) * R::kRows)
            one_row(row, 0, false);
    } else if (a.gate_by_lanes) {
        const int64_t groups = a.rows / a.rows_per_gate;
        for (int64_t group = static_cast<int64_t>(blockIdx.x) * R::kRows + sub; group < groups; group += static_cast<int64_t>(gridDim.x) * R::kRows) {
            for (int64_t k = 0; k < a.rows_per_gate; ++k) one_row(group * a.rows_per_gate + k, group, k == 0);
            if (g.gate != nullptr) {
#pragma unroll
                for (int j = 0; j < kVectors; ++j)
                    if (at.valid(j) > 0) store_gate(group, at.channel(j), at.valid(j), d_gate.v[j]);
            }
            d_gate = Values<kVectors>{};
        }
    } else {
        const int64_t units = a.rows / a.rows_per_gate * g.pieces;
        for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
            const int64_t group = unit / g.pieces, piece = unit % g.pieces;
            const int64_t first = group * a.rows_per_gate + piece * g.piece_rows;
            const int64_t last = min(first + g.piece_rows, (group + 1) * a.rows_per_gate);
            p.load_gate(a, at, group);
            for (int64_t row = first + sub; row < last; row += R::kRows) one_row(row, group, false);
            if (g.gate != nullptr) {
                if (g.pieces == 1)
                    write_sum<kLanes, kVectors>(d_gate, lds, a.channels, [&](int c, int valid, const float(&v)[kChunk]) { store_gate(group, c, valid, v); });
                else
                    leave(g.gate_sums, unit, d_gate);
            }
            d_gate = Values<kVectors>{};
        }
    }
    if (a.rows_per_gate == 0) leave(g.gate_sums, blockIdx.x, d_gate);
    leave(g.sums[0], blockIdx.x, d_post_weight);
    leave(g.sums[1], blockIdx.x, d_post_bias);
    leave(g.sums[2], blockIdx.x, d_pre_weight);
    leave(g.sums[3], blockIdx.x, d_pre_bias);
}

// to[group][c] = the sum over `rows` rows of partial sums of a group, in a fixed order; 32 channels and 32 strands of rows to a workgroup.
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
    return with_row_shape(a.channels, [&](auto lanes, auto vectors) {
        constexpr int kLanes = decltype(lanes)::value, kVectors = decltype(vectors)::value;
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>((a.rows + Row<kLanes>::kRows - 1) / Row<kLanes>::kRows, 8192));
        hipLaunchKernelGGL((norm_kernel<E, kLanes, kVectors>), dim3(grid), dim3(Row<kLanes>::kThreads), 0, stream, a, static_cast<E*>(y),
                           static_cast<E*>(n));
        return launched();
    });
}

template <class E>
int launch_norm_backward(const NormArgs& a, const NormGrads& g, unsigned grid, hipStream_t stream) {
    return with_row_shape(a.channels, [&](auto lanes, auto vectors) {
        constexpr int kLanes = decltype(lanes)::value, kVectors = decltype(vectors)::value;
        const dim3 threads(Row<kLanes>::kThreads);
        if (a.kept_x.values != nullptr)
            hipLaunchKernelGGL((norm_backward_kernel<E, kLanes, kVectors, true>), dim3(grid), threads, 0, stream, a, g);
        else
            hipLaunchKernelGGL((norm_backward_kernel<E, kLanes, kVectors, false>), dim3(grid), threads, 0, stream, a, g);
        return launched();
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
