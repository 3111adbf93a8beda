// The products of penc_expert_linear.hip, one compilation for each type of include/penc.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace penc {

// y of `deep` channels and `wide` outputs, or (back) dx of `deep` outputs and `wide` channels; weight [experts][outputs][channels].
template <int kType>
int expert_rows(bool back, int64_t rows, int experts, int64_t wide, int64_t deep, const void* in, int64_t stride, const void* weight, const void* bias,
                const int32_t* offsets, void* out, hipStream_t stream);
template <int kType>
size_t expert_weights_workspace(int64_t rows, int64_t experts, int64_t channels, int64_t outputs);
// dW, db (may be null) and, where it is not null, dx.
template <int kType>
int expert_grads(int64_t rows, int experts, int64_t channels, int64_t outputs, const void* x, int64_t x_stride, const void* grad, int64_t grad_stride, const void* weight,
                 const int32_t* offsets, void* dx, void* dweight, void* dbias, void* workspace, hipStream_t stream);
// db alone.
template <int kType>
size_t expert_bias_workspace(int64_t rows, int64_t experts, int64_t outputs);
template <int kType>
int expert_bias(int64_t rows, int experts, int64_t outputs, const void* grad, int64_t grad_stride, const int32_t* offsets, void* dbias, void* workspace, hipStream_t stream);

}  // namespace penc
