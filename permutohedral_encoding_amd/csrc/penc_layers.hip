// Checkpoints in 8 bits, and activations whose backward reads them.
//
//     y = act(x), or act(a) b of rows [a | b];     dx = g act'(x^), da = g b^ act'(a^), db = g act(a^)
//     gelu  x Phi(x)                act' = Phi(x) + x phi(x)
//     silu  x s, s = 1/(1+exp(-x))  act' = s (1 + x (1 - s))
//     softplus  log(1 + exp(x))     act' = s
//
// All of them are one pass over their rows: bound by memory.  A lane has 8 channels, the lanes of a row are a multiple of four up to 256, so that
// a block of a checkpoint is always four neighbours of one wave, and a workgroup has as many rows as it has lanes for.  Measured, us and bytes read and
// written (a copy on this card reaches 5.5 TB/s; what fits the 256 MB cache in front of the memory, more):
//
//     pack, channels adjacent     65536 x 1024 bf16  38, 5.3 TB/s      1048576 x 48 fp32  44, 5.8 TB/s
//     pack, rows adjacent                                              1048576 x 48 fp32  60, 4.2 TB/s
//     unpack                      65536 x 1024 bf16  31, 6.6 TB/s      1048576 x 48 fp32  38, 6.7 TB/s
//     gated silu                  32765 x 2 2048 bf16: forward with its checkpoints 93, 5.8 TB/s; backward from them 93, 5.8 TB/s
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "penc_kept.hpp"
#include "penc_norm.hpp"

namespace penc {
namespace {

constexpr int kThreads = 256;

// How lanes are laid over rows: `lanes` on a row, a multiple of four, which take its `chunks` of eight channels (another) in as many turns as there must be.
// (With powers of two, silu of 1048576 x 70 bf16 and back with its checkpoint 211 us instead of 180.)
struct Lanes {
    row_t rows;
    int channels, last_channels, chunks;  // last_channels: of the last row
    int lanes, per_group, per_lane;       // per_group: rows at a time; per_lane: 2^16 / lanes, rounded up
    unsigned grid;
};

Lanes lanes_for(int64_t rows, int64_t channels) {
    Lanes l{static_cast<row_t>(rows), static_cast<int>(channels), static_cast<int>(channels), static_cast<int>(4 * kept_blocks(channels)), 0, 0, 0, 0};
    const int turns = (l.chunks + kThreads - 1) / kThreads;
    l.lanes = ((l.chunks + turns - 1) / turns + 3) / 4 * 4;
    l.per_group = kThreads / l.lanes;
    l.per_lane = ((1 << 16) + l.lanes - 1) / l.lanes;
    // (a workgroup for every row or group of rows, up to the threads that a launch may have; each walking over its share of the rows, 8192 of them: gated silu
    // of 32765 x 2 2048 bf16 and back 200 us instead of 192, unpack of 1048576 x 64 fp32 91 instead of 71)
    l.grid = static_cast<unsigned>(std::min<int64_t>((rows + l.per_group - 1) / l.per_group, 1 << 22));
    return l;
}

// Values one behind the other, where no block matters: rows of 2048, the last one shorter.  (Silu of 1048576 x 3 fp32 20 us row by row and 6 like this, of
// x 70 118 and 103, bf16 77 and 50.)
constexpr int64_t kFlatRow = 2048;
bool lies_flat(int64_t rows, int64_t channels, int64_t stride) { return stride == channels && rows * channels <= kFlatRow * kMostRows; }
Lanes flat_lanes(int64_t values) {
    Lanes l = lanes_for((values + kFlatRow - 1) / kFlatRow, kFlatRow);
    l.last_channels = static_cast<int>(values - (static_cast<int64_t>(l.rows) - 1) * kFlatRow);
    return l;
}

// f(row, first channel, channels of the row), four lanes of a block together, and behind the row's end too
template <class F>
__device__ __forceinline__ void over_chunks(const Lanes& l, F&& f) {
    // (exact: both are at most 256)
    const int among = static_cast<int>(threadIdx.x * l.per_lane >> 16), lane = threadIdx.x - among * l.lanes;
    if (among >= l.per_group) return;
    for (row_t row = blockIdx.x * l.per_group + among; row < l.rows; row += gridDim.x * l.per_group)
        for (int chunk = lane; chunk < l.chunks; chunk += l.lanes) f(row, chunk * kChunk, row + 1 == l.rows ? l.last_channels : l.channels);
}

template <class E>
__global__ __launch_bounds__(kThreads) void pack_kernel(Lanes l, const E* __restrict__ x, uint32_t stride, KeptArray kept) {
    over_chunks(l, [&](row_t row, int c, int channels) {
        float v[kChunk];
        load_chunk(x + offset_of(row, stride), c, channels, v);
        kept.store(row, c, v);
    });
}

// The encoding's own result: channels of consecutive rows next to each other.  A workgroup has kThreads rows and up to 128 of their channels: a lane has a
// row and walks over its blocks, reading 32 channels, each with the 63 lanes beside it, and what it makes of them waits in the LDS until all rows' can be
// written one after the other.  (Written by the lanes themselves, 16 bytes a row: 1000003 x 48 fp32 48.7 us instead of 38.6; 2^20 x 48 54 instead of 50, where
// channels 4 MiB apart meet in the same memory channels.  All 8192 channels of 10 rows by one workgroup: 515 us instead of 7.)
constexpr int kPiece = 128;
template <class E>
__global__ __launch_bounds__(kThreads) void pack_channels_kernel(row_t rows, int channels, const E* __restrict__ x, int64_t stride, KeptArray kept) {
    extern __shared__ uint4 staged[];  // the rows, and behind them their exponents
    const int begin = blockIdx.y * kPiece;
    const uint32_t pitch = min(static_cast<uint32_t>(kPiece), kept.pitch - begin), blocks = min(static_cast<uint32_t>(kPiece / kKeptBlock), kept.blocks - begin / kKeptBlock);
    uint8_t* const exponents = reinterpret_cast<uint8_t*>(staged) + kThreads * pitch;
    const row_t row0 = blockIdx.x * kThreads, row = row0 + threadIdx.x;
    if (row < rows) {
        for (uint32_t block = 0; block < blocks; ++block) {
            const int first = begin + block * kKeptBlock;
            float v[kKeptBlock];
#pragma unroll
            for (int i = 0; i < kKeptBlock; ++i) v[i] = first + i < channels ? static_cast<float>(x[(first + i) * stride + row]) : 0.0f;
            uint32_t a = 0;
#pragma unroll
            for (int i = 0; i < kKeptBlock; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
            const BlockStep s(a);
            s.saturate(v);
#pragma unroll
            for (int i = 0; i < kKeptBlock; i += 16) {
                if (block * kKeptBlock + i >= pitch) break;
                uint4 q;
                q.x = s.quantised(v + i), q.y = s.quantised(v + i + 4), q.z = s.quantised(v + i + 8), q.w = s.quantised(v + i + 12);
                staged[(threadIdx.x * pitch + block * kKeptBlock + i) / 16] = q;
            }
            exponents[threadIdx.x * blocks + block] = static_cast<uint8_t>(s.exponent);
        }
    }
    __syncthreads();
    const uint32_t n = min(static_cast<uint32_t>(kThreads), rows - row0), vectors = pitch / 16;
    for (uint32_t i = threadIdx.x; i < n * vectors; i += kThreads)
        *reinterpret_cast<uint4*>(kept.values + offset_of(row0 + i / vectors, kept.pitch) + begin + i % vectors * 16) = staged[i];
    for (uint32_t i = threadIdx.x; i < n * blocks; i += kThreads)
        kept.exponents[offset_of(row0 + i / blocks, kept.blocks) + begin / kKeptBlock + i % blocks] = exponents[i];
}

template <class E>
__global__ __launch_bounds__(kThreads) void unpack_kernel(Lanes l, KeptArray kept, E* __restrict__ x) {
    over_chunks(l, [&](row_t row, int c, int channels) {
        if (c >= channels) return;
        float v[kChunk];
        kept.load(row, c, v);
        if constexpr (sizeof(E) == 2 && !std::is_same_v<E, bf16_t>) {
            // (65520 and more round to 64 * 2^10 = 65536 in a block, which fp16 does not have)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[i] = v[i] > 65504.0f ? 65504.0f : v[i] < -65504.0f ? -65504.0f : v[i];
        }
        store_chunk(x + offset_of(row, l.channels) + c, channels - c, v);
    });
}

// act(x) and act'(x)
template <int kKind>
__device__ __forceinline__ void activate(float x, float& value, float& slope) {
    if constexpr (kKind == PENC_GELU) {
        const float below = 0.5f * (1.0f + erff(x * 0.70710678f));
        value = x * below;
        slope = below + x * (0.39894228f * expf(-0.5f * x * x));
    } else if constexpr (kKind == PENC_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + expf(-x));
        value = x * s;
        slope = s * (1.0f + x * (1.0f - s));
    } else {
        // log(1 + e) with e in 0..1: u = 1 + e leaves c = e - (u - 1) of e behind, both differences exact, and log(u + c) = log(u) + c / u up to c^2.
        // (69757 x 2 161 fp16 gated, forward and back: log1pf 54 and 61 us, this 23 and 24)
        const float e = expf(-fabsf(x)), u = 1.0f + e, c = e - (u - 1.0f), r = __builtin_amdgcn_rcpf(u);
        value = fmaxf(x, 0.0f) + __builtin_fmaf(c, r, 0.69314718f * __builtin_amdgcn_logf(u));
        slope = x < 0.0f ? e * r : r;
        if (x != x) value = slope = x;
    }
}

template <class E, int kKind, bool kGated>
__global__ __launch_bounds__(kThreads) void activation_kernel(Lanes l, const E* __restrict__ x, uint32_t stride, E* __restrict__ y, KeptArray kept,
                                                              KeptArray kept_gate) {
    over_chunks(l, [&](row_t row, int c, int channels) {
        float a[kChunk], b[kChunk], unused;
        load_chunk(x + offset_of(row, stride), c, channels, a);
        if constexpr (kGated) load_chunk(x + offset_of(row, stride) + l.channels, c, channels, b);
        if (kept.values != nullptr) {
            kept.store(row, c, a);
            if constexpr (kGated) kept_gate.store(row, c, b);
        }
        if (c >= channels) return;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            activate<kKind>(a[i], a[i], unused);
            if constexpr (kGated) a[i] *= b[i];
        }
        store_chunk(y + offset_of(row, l.channels) + c, channels - c, a);
    });
}

// x: the input itself, or null where it is kept in 8 bits
template <class E, int kKind, bool kGated>
__global__ __launch_bounds__(kThreads) void activation_backward_kernel(Lanes l, const E* __restrict__ x, uint32_t stride, KeptArray kept,
                                                                       KeptArray kept_gate, const E* __restrict__ grad, uint32_t grad_stride,
                                                                       E* __restrict__ dx) {
    over_chunks(l, [&](row_t row, int c, int channels) {
        if (c >= channels) return;
        float a[kChunk], b[kChunk], g[kChunk], value, slope;
        load_chunk(grad + offset_of(row, grad_stride), c, channels, g);
        if (x != nullptr) {
            load_chunk(x + offset_of(row, stride), c, channels, a);
            if constexpr (kGated) load_chunk(x + offset_of(row, stride) + l.channels, c, channels, b);
        } else {
            kept.load(row, c, a);
            if constexpr (kGated) kept_gate.load(row, c, b);
        }
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            activate<kKind>(a[i], value, slope);
            if constexpr (kGated) {
                a[i] = g[i] * b[i] * slope;
                b[i] = g[i] * value;
            } else {
                a[i] = g[i] * slope;
            }
        }
        E* const to = dx + offset_of(row, l.channels * (kGated ? 2 : 1)) + c;
        store_chunk(to, channels - c, a);
        if constexpr (kGated) store_chunk(to + l.channels, channels - c, b);
    });
}

template <class F>
int with_kind(int kind, int gated, F&& f) {
    const auto with_gate = [&](auto k) { return gated ? f(k, std::true_type{}) : f(k, std::false_type{}); };
    switch (kind) {
        case PENC_GELU: return with_gate(std::integral_constant<int, PENC_GELU>{});
        case PENC_SILU: return with_gate(std::integral_constant<int, PENC_SILU>{});
        case PENC_SOFTPLUS: return with_gate(std::integral_constant<int, PENC_SOFTPLUS>{});
        default: return PENC_ERR_UNSUPPORTED_KIND;
    }
}

bool bad_size(int64_t rows, int64_t channels) { return bad_rows(rows) || channels <= 0 || channels > PENC_MAX_CHANNELS; }
bool misplaced(const int8_t* values) { return !aligned_to(values, kKeptPitch); }

// How the backward of a norm is cut up: workgroups, pieces of a group of rows that share a gate, and the rows of partial sums they leave.
struct NormPlan {
    unsigned grid;
    int64_t pieces, piece_rows, gate_rows;
    bool gate_by_lanes;
};
NormPlan norm_plan(int64_t rows, int64_t channels, int64_t rows_per_gate, bool full) {
    const int lanes = lanes_of_row(static_cast<int>(channels));
    const int64_t at_a_time = row_threads(lanes) / lanes, most = most_groups(lanes, full);
    const auto groups_of = [&](int64_t n) { return std::max<int64_t>(1, (n + at_a_time - 1) / at_a_time); };
    NormPlan p{0, 1, rows_per_gate, 0, false};
    if (rows_per_gate == 0) {
        p.grid = static_cast<unsigned>(std::min(most, groups_of(rows)));
        p.gate_rows = p.grid;
    } else if (rows_per_gate < 2 * at_a_time) {
        p.gate_by_lanes = true;
        p.grid = static_cast<unsigned>(std::min(most, groups_of(rows / rows_per_gate)));
    } else {
        const int64_t groups = std::max<int64_t>(1, rows / rows_per_gate);
        const int64_t wanted = groups >= most / 2 ? 1 : std::min((most + groups - 1) / groups, groups_of(rows_per_gate));
        p.piece_rows = groups_of((rows_per_gate + wanted - 1) / wanted) * at_a_time;
        p.pieces = (rows_per_gate + p.piece_rows - 1) / p.piece_rows;
        p.grid = static_cast<unsigned>(std::min(most, groups * p.pieces));
        p.gate_rows = p.pieces > 1 ? groups * p.pieces : 0;
    }
    return p;
}

// The checks and the kernels' arguments that the two directions share; false with `status` where there is nothing to launch.
bool norm_args(const penc_norm* n, NormArgs& a, int& status) {
    status = PENC_ERR_NULL_POINTER;
    if (!n) return false;
    status = PENC_ERR_UNSUPPORTED_KIND;
    if (n->kind != PENC_RMS && n->kind != PENC_LAYER) return false;
    status = PENC_ERR_UNSUPPORTED_TYPE;
    if ((n->type != PENC_FP32 && n->type != PENC_FP16 && n->type != PENC_BF16) || (n->param_type != n->type && n->param_type != PENC_FP32) ||
        (n->gate_type != n->type && n->gate_type != PENC_FP32))
        return false;
    status = PENC_ERR_BAD_LAYER_SIZE;
    if (bad_rows(n->rows) || bad_stride(n->x_stride) || bad_stride(n->branch_stride) || n->channels <= 0 || n->channels > PENC_MAX_NORM_CHANNELS || n->rows_per_gate < 0 ||
        (n->rows_per_gate > 0 && n->rows % n->rows_per_gate != 0))
        return false;
    status = PENC_ERR_NULL_POINTER;
    if ((n->x_values == nullptr) != (n->x_exponents == nullptr) || (n->branch_values == nullptr) != (n->branch_exponents == nullptr)) return false;
    status = PENC_ERR_MISALIGNED;
    const size_t size = n->type == PENC_FP32 ? 4 : 2, param = n->param_type == PENC_FP32 ? 4 : 2, gate = n->gate_type == PENC_FP32 ? 4 : 2;
    if (misplaced(n->x_values) || misplaced(n->branch_values) || !aligned_to(n->x, size) || !aligned_to(n->branch, size) || !aligned_to(n->gate, gate) ||
        !aligned_to(n->post_weight, param) || !aligned_to(n->post_bias, param) || !aligned_to(n->pre_weight, param) || !aligned_to(n->pre_bias, param))
        return false;
    a = {static_cast<row_t>(n->rows), static_cast<row_t>(n->rows_per_gate), static_cast<uint32_t>(n->x_stride), static_cast<uint32_t>(n->branch_stride),
         static_cast<int>(n->channels), n->residual_scale, n->eps, n->kind == PENC_LAYER,
         n->post_norm != 0, n->pre_norm != 0, n->has_branch != 0, n->param_type == PENC_FP32, n->gate_type == PENC_FP32, false, n->x, n->branch, n->gate,
         n->post_weight, n->post_bias, n->pre_weight, n->pre_bias, kept_array(n->x_values, n->x_exponents, n->channels),
         kept_array(n->branch_values, n->branch_exponents, n->channels)};
    status = PENC_OK;
    return true;
}

NormLaunches norm_launches_of(int type) {
    return type == PENC_FP32 ? norm_launches<PENC_FP32>() : type == PENC_FP16 ? norm_launches<PENC_FP16>() : norm_launches<PENC_BF16>();
}

}  // namespace
}  // namespace penc

using namespace penc;

extern "C" {

int64_t penc_kept_pitch(int64_t channels) { return kept_pitch(channels); }
int64_t penc_kept_blocks(int64_t channels) { return kept_blocks(channels); }

int penc_keep(int type, int64_t rows, int64_t channels, const void* x, int64_t row_stride, int64_t channel_stride, int8_t* values,
              uint8_t* exponents, void* stream) {
    if (bad_size(rows, channels) || (channel_stride != 1 && row_stride != 1) || (channel_stride == 1 && bad_stride(row_stride)) || channel_stride < 0)
        return PENC_ERR_BAD_LAYER_SIZE;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        if (rows == 0) return PENC_OK;
        if (!x || !values || !exponents) return PENC_ERR_NULL_POINTER;
        if (misplaced(values) || !aligned_to(x, sizeof(E))) return PENC_ERR_MISALIGNED;
        const KeptArray kept = kept_array(values, exponents, channels);
        if (channel_stride == 1) {
            const Lanes l = lanes_for(rows, channels);
            hipLaunchKernelGGL(pack_kernel<E>, dim3(l.grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream), l, static_cast<const E*>(x),
                               static_cast<uint32_t>(row_stride), kept);
        } else {
            const int64_t groups = (rows + kThreads - 1) / kThreads, pieces = (channels + kPiece - 1) / kPiece;
            if (pieces > 0xFFFF) return PENC_ERR_BAD_LAYER_SIZE;
            const uint32_t lds = kThreads * (std::min<uint32_t>(kPiece, kept.pitch) + std::min<uint32_t>(kPiece / kKeptBlock, kept.blocks));
            hipLaunchKernelGGL(pack_channels_kernel<E>, dim3(static_cast<unsigned>(groups), static_cast<unsigned>(pieces)), dim3(kThreads), lds,
                               static_cast<hipStream_t>(stream), static_cast<row_t>(rows), static_cast<int>(channels), static_cast<const E*>(x), channel_stride,
                               kept);
        }
        return launched();
    });
}

int penc_restore(int type, int64_t rows, int64_t channels, const int8_t* values, const uint8_t* exponents, void* x, void* stream) {
    if (bad_size(rows, channels)) return PENC_ERR_BAD_LAYER_SIZE;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        if (rows == 0) return PENC_OK;
        if (!x || !values || !exponents) return PENC_ERR_NULL_POINTER;
        if (misplaced(values) || !aligned_to(x, sizeof(E))) return PENC_ERR_MISALIGNED;
        const Lanes l = lanes_for(rows, channels);
        hipLaunchKernelGGL(unpack_kernel<E>, dim3(l.grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream), l, kept_array(values, exponents, channels),
                           static_cast<E*>(x));
        return launched();
    });
}

int penc_activation(int type, int kind, int gated, int64_t rows, int64_t channels, const void* x, int64_t row_stride, void* y, int8_t* values,
                    uint8_t* exponents, void* stream) {
    if (bad_size(rows, channels) || bad_stride(row_stride)) return PENC_ERR_BAD_LAYER_SIZE;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        return with_kind(kind, gated, [&](auto k, auto g) {
            if (rows == 0) return PENC_OK;
            if (!x || !y || (values == nullptr) != (exponents == nullptr)) return PENC_ERR_NULL_POINTER;
            if (misplaced(values) || !aligned_to(x, sizeof(E)) || !aligned_to(y, sizeof(E))) return PENC_ERR_MISALIGNED;
            const bool flat = !gated && values == nullptr && lies_flat(rows, channels, row_stride);
            const Lanes l = flat ? flat_lanes(rows * channels) : lanes_for(rows, channels);
            const KeptArray kept = kept_array(values, exponents, channels);
            KeptArray kept_gate = kept;
            if (values != nullptr) kept_gate.values += rows * kept.pitch, kept_gate.exponents += rows * kept.blocks;
            hipLaunchKernelGGL((activation_kernel<E, decltype(k)::value, decltype(g)::value>), dim3(l.grid), dim3(kThreads), 0,
                               static_cast<hipStream_t>(stream), l, static_cast<const E*>(x), static_cast<uint32_t>(flat ? kFlatRow : row_stride), static_cast<E*>(y), kept,
                               kept_gate);
            return launched();
        });
    });
}

int penc_activation_backward(int type, int kind, int gated, int64_t rows, int64_t channels, const void* x, int64_t row_stride, const int8_t* values,
                             const uint8_t* exponents, const void* grad, int64_t grad_row_stride, void* dx, void* stream) {
    if (bad_size(rows, channels) || bad_stride(row_stride) || bad_stride(grad_row_stride)) return PENC_ERR_BAD_LAYER_SIZE;
    return with_type(type, [&](auto e) {
        using E = decltype(e);
        return with_kind(kind, gated, [&](auto k, auto g) {
            if (rows == 0) return PENC_OK;
            if (!grad || !dx || (!x && (!values || !exponents))) return PENC_ERR_NULL_POINTER;
            if (misplaced(values) || !aligned_to(x, sizeof(E)) || !aligned_to(grad, sizeof(E)) || !aligned_to(dx, sizeof(E))) return PENC_ERR_MISALIGNED;
            const bool flat = !gated && x != nullptr && lies_flat(rows, channels, row_stride) && grad_row_stride == channels;
            const Lanes l = flat ? flat_lanes(rows * channels) : lanes_for(rows, channels);
            if (flat) row_stride = grad_row_stride = kFlatRow;
            const KeptArray kept = kept_array(values, exponents, channels);
            KeptArray kept_gate = kept;
            if (values != nullptr) kept_gate.values += rows * kept.pitch, kept_gate.exponents += rows * kept.blocks;
            hipLaunchKernelGGL((activation_backward_kernel<E, decltype(k)::value, decltype(g)::value>), dim3(l.grid), dim3(kThreads), 0,
                               static_cast<hipStream_t>(stream), l, static_cast<const E*>(x), static_cast<uint32_t>(row_stride), kept, kept_gate, static_cast<const E*>(grad),
                               static_cast<uint32_t>(grad_row_stride), static_cast<E*>(dx));
            return launched();
        });
    });
}

int penc_residual_norm(const penc_norm* norm, void* y, void* n, void* stream) {
    NormArgs a;
    int status;
    if (!norm_args(norm, a, status)) return status;
    if (a.rows == 0) return PENC_OK;
    if (!a.x || (a.pre_norm && !n) || (!a.pre_norm && !y) || (a.has_branch && !a.branch)) return PENC_ERR_NULL_POINTER;
    if (!a.has_branch) a.kept_branch.values = nullptr;
    const size_t size = norm->type == PENC_FP32 ? 4 : 2;
    if (!aligned_to(y, size) || !aligned_to(n, size)) return PENC_ERR_MISALIGNED;
    return norm_launches_of(norm->type).forward(a, y, n, static_cast<hipStream_t>(stream));
}

size_t penc_residual_norm_workspace_bytes(int64_t rows, int64_t channels, int64_t rows_per_gate) {
    if (bad_rows(rows) || channels <= 0 || channels > PENC_MAX_NORM_CHANNELS || rows_per_gate < 0) return 0;
    size_t most = 0;
    for (const bool full : {false, true}) {
        const NormPlan p = norm_plan(rows, channels, rows_per_gate, full);
        most = std::max(most, 4 * static_cast<size_t>(p.grid) + static_cast<size_t>(p.gate_rows));
    }
    return 4 * static_cast<size_t>(channels) * most;
}

int penc_residual_norm_backward(const penc_norm* norm, const penc_norm_grads* grads, void* workspace, size_t workspace_bytes, void* stream) {
    NormArgs a;
    int status;
    if (!norm_args(norm, a, status)) return status;
    if (!grads || (grads->gate && !norm->has_branch)) return PENC_ERR_NULL_POINTER;
    const bool kept = a.kept_x.values != nullptr;
    if (a.rows > 0 && !kept && (!a.x || (a.has_branch && !a.branch))) return PENC_ERR_NULL_POINTER;
    if (a.rows > 0 && kept && a.has_branch && !a.kept_branch.values) return PENC_ERR_NULL_POINTER;
    const size_t size = norm->type == PENC_FP32 ? 4 : 2, param = norm->param_type == PENC_FP32 ? 4 : 2, gate = norm->gate_type == PENC_FP32 ? 4 : 2;
    for (const void* p : {grads->y, grads->n, static_cast<const void*>(grads->x), static_cast<const void*>(grads->branch)})
        if (!aligned_to(p, size)) return PENC_ERR_MISALIGNED;
    for (const void* p : {grads->post_weight, grads->post_bias, grads->pre_weight, grads->pre_bias})
        if (!aligned_to(p, param)) return PENC_ERR_MISALIGNED;
    if (!aligned_to(grads->gate, gate) || !aligned_to(workspace, 16)) return PENC_ERR_MISALIGNED;
    if (bad_stride(grads->y_stride) || bad_stride(grads->n_stride)) return PENC_ERR_BAD_LAYER_SIZE;
    const NormPlan plan = norm_plan(a.rows, a.channels, a.rows_per_gate, is_full(a) || grads->post_bias || grads->pre_bias);
    if (workspace_bytes < penc_residual_norm_workspace_bytes(a.rows, a.channels, a.rows_per_gate)) return PENC_ERR_WORKSPACE_TOO_SMALL;
    if (!workspace) return PENC_ERR_NULL_POINTER;
    a.gate_by_lanes = plan.gate_by_lanes;
    if (a.rows == 0) a.gate = nullptr;  // (there may be no group's gate either)
    NormGrads g{grads->y, a.pre_norm ? grads->n : nullptr, static_cast<uint32_t>(grads->y_stride), static_cast<uint32_t>(grads->n_stride), grads->x, a.has_branch ? grads->branch : nullptr, grads->gate,
                nullptr, {}, static_cast<uint32_t>(plan.pieces), static_cast<row_t>(plan.piece_rows)};
    // partial sums of what is wanted, one array after the other
    float* next = static_cast<float*>(workspace);
    SumPartials sums{};
    sums.channels = a.channels;
    int n = 0;
    const auto wanted = [&](void* to, int64_t groups, int64_t rows, bool fp32) {
        if (!to || groups == 0) return static_cast<float*>(nullptr);
        float* const from = next;
        next += groups * rows * a.channels;
        sums.sums[n++] = {from, to, groups, rows, fp32};
        return from;
    };
    void* const to[4] = {grads->post_weight, grads->post_bias, grads->pre_weight, grads->pre_bias};
    for (int i = 0; i < 4; ++i) g.sums[i] = wanted(to[i], 1, plan.grid, a.param_fp32);
    if (a.rows_per_gate == 0) g.gate_sums = wanted(g.gate, 1, plan.grid, a.gate_fp32);
    else if (plan.gate_rows > 0 && a.rows > 0) g.gate_sums = wanted(g.gate, a.rows / a.rows_per_gate, plan.pieces, a.gate_fp32);
    const NormLaunches launches = norm_launches_of(norm->type);
    // (without rows the workgroups leave sums of nothing)
    if (a.rows > 0 || n > 0)
        if (const int rc = launches.backward(a, g, plan.grid, static_cast<hipStream_t>(stream))) return rc;
    if (n == 0) return PENC_OK;
    int64_t groups = 1;
    for (int i = 0; i < n; ++i) groups = std::max(groups, sums.sums[i].groups);
    const int64_t grid = groups * ((a.channels + 31) / 32);
    if (grid > 0x7FFFFFFF) return PENC_ERR_BAD_LAYER_SIZE;
    return launches.sum_partials(sums, static_cast<unsigned>(grid), n, static_cast<hipStream_t>(stream));
}

}  // extern "C"
