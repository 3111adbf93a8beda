// What the kernels of penc_norm.hip take, and how lanes are laid over a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "penc_kept.hpp"

namespace penc {

struct NormArgs {
    int64_t rows, rows_per_gate, x_stride, branch_stride;
    int channels;
    float scale, eps;
    bool layer, post_norm, pre_norm, has_branch, param_fp32, gate_fp32, gate_by_lanes;
    const void *x, *branch, *gate, *post_weight, *post_bias, *pre_weight, *pre_bias;
    KeptArray kept_x, kept_branch;
};

struct NormGrads {
    const void *y, *n;
    int64_t y_stride, n_stride;
    void *x, *branch, *gate;
    float* gate_sums;              // a row for each workgroup (one gate) or piece of a group
    float* sums[4];                // a row for each workgroup: post weight, post bias, pre weight, pre bias; null where not wanted
    int64_t pieces, piece_rows;    // of a group of rows that share a gate
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

__device__ __forceinline__ int64_t group_of(int64_t row, int64_t rows_per_gate) {
    if (((row | rows_per_gate) >> 32) == 0) return static_cast<uint32_t>(row) / static_cast<uint32_t>(rows_per_gate);
    return row / rows_per_gate;
}

// Lanes to a row and vectors of 8 channels to a lane.  A wave or less per row up to 1024 channels: nothing goes through the LDS.  From there on a
// workgroup per row, wide before deep, so that a lane's sums over the rows (5 x 8 registers a vector) leave room for waves.
template <class F>
int with_row_shape(int channels, F&& f) {
    const auto shape = [&](auto lanes, auto vectors) { return f(lanes, vectors); };
#define PENC_SHAPE(most, lanes, vectors) \
    if (channels <= most) return shape(std::integral_constant<int, lanes>{}, std::integral_constant<int, vectors>{})
    PENC_SHAPE(32, 4, 1);
    PENC_SHAPE(64, 8, 1);
    PENC_SHAPE(128, 16, 1);
    PENC_SHAPE(256, 32, 1);
    PENC_SHAPE(512, 64, 1);
    PENC_SHAPE(1024, 64, 2);
    PENC_SHAPE(2048, 256, 1);
    PENC_SHAPE(4096, 512, 1);
    PENC_SHAPE(PENC_MAX_NORM_CHANNELS, 512, 2);
#undef PENC_SHAPE
    return PENC_ERR_BAD_LAYER_SIZE;
}

inline int rows_at_a_time(int channels) {
    int rows = 1;
    with_row_shape(channels, [&](auto lanes, auto) { return rows = decltype(lanes)::value < 256 ? 256 / decltype(lanes)::value : 1; });
    return rows;
}

struct NormLaunches {
    int (*forward)(const NormArgs&, void* y, void* n, hipStream_t);
    int (*backward)(const NormArgs&, const NormGrads&, unsigned grid, hipStream_t);
    int (*sum_partials)(const SumPartials&, unsigned grid, int n, hipStream_t);
};

template <int kType>
NormLaunches norm_launches();

}  // namespace penc
