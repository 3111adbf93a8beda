// What the kernels of penc_norm.hip take, and how lanes are laid over a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "penc_kept.hpp"

namespace penc {

struct NormArgs {
    row_t rows, rows_per_gate;
    uint32_t x_stride, branch_stride;
    int channels;
    float scale, eps;
    bool layer, post_norm, pre_norm, has_branch, param_fp32, gate_fp32, gate_by_lanes;
    const void *x, *branch, *gate, *post_weight, *post_bias, *pre_weight, *pre_bias;
    KeptArray kept_x, kept_branch;
};

// Whether a norm is more than "rms" without biases.
inline bool is_full(const NormArgs& a) { return a.layer || a.post_bias != nullptr || a.pre_bias != nullptr; }

struct NormGrads {
    const void *y, *n;
    uint32_t y_stride, n_stride;
    void *x, *branch, *gate;
    float* gate_sums;              // a row for each workgroup (one gate) or piece of a group
    float* sums[4];                // a row for each workgroup: post weight, post bias, pre weight, pre bias; null where not wanted
    uint32_t pieces;               // of a group of rows that share a gate
    row_t piece_rows;
};

struct Sum {
    const float* from;  // [groups][rows][channels]
    void* to;           // [groups][channels]
    int64_t groups, rows;
    bool fp32;
};
struct SumPartials {
    Sum sums[5];
    int channels;
};

// How a row ends: in a whole chunk of 8 channels, in a part of one, or before the first is whole.
enum RowEnd { kWholeChunks, kPartOfChunk, kNarrowRow };

// Lanes to a row, 8 channels each, and how it ends.  A wave or less up to 512 channels: nothing goes through the LDS; from there on
// a workgroup.
template <class F>
int with_row_shape(int channels, F&& f) {
    if (channels < kChunk) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, kNarrowRow>{});
#define PENC_SHAPE(lanes)                                                                                                                     \
    if (channels <= lanes * kChunk)                                                                                                           \
        return channels % kChunk == 0 ? f(std::integral_constant<int, lanes>{}, std::integral_constant<int, kWholeChunks>{})                  \
                                      : f(std::integral_constant<int, lanes>{}, std::integral_constant<int, kPartOfChunk>{})
    PENC_SHAPE(4);
    PENC_SHAPE(8);
    PENC_SHAPE(16);
    PENC_SHAPE(32);
    PENC_SHAPE(64);
    PENC_SHAPE(128);
    PENC_SHAPE(256);
    PENC_SHAPE(512);
    PENC_SHAPE(1024);
#undef PENC_SHAPE
    return PENC_ERR_BAD_LAYER_SIZE;
}
static_assert(PENC_MAX_NORM_CHANNELS == 1024 * kChunk, "the widest row");

__host__ __device__ constexpr int row_threads(int lanes) { return lanes > 64 ? lanes : 256; }
// Workgroups that the card's 256 compute units hold at a time: 16 waves each, of the backward of any kind of norm 12, or 8 where a workgroup has as many.
inline int64_t most_groups(int lanes, bool full_backward) {
    return 256 * ((full_backward && lanes < 1024 ? lanes == 512 ? 8 : 12 : 16) * 64 / row_threads(lanes));
}

inline int lanes_of_row(int channels) {
    int n = 0;
    with_row_shape(channels, [&](auto lanes, auto) { return n = decltype(lanes)::value; });
    return n;
}

struct NormLaunches {
    int (*forward)(const NormArgs&, void* y, void* n, hipStream_t);
    int (*backward)(const NormArgs&, const NormGrads&, unsigned grid, hipStream_t);
    int (*sum_partials)(const SumPartials&, unsigned grid, int n, hipStream_t);
};

template <int kType>
NormLaunches norm_launches();

}  // namespace penc
