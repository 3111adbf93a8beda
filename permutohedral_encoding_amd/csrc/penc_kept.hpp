// Values in 32, 16 and 8 bits, as the kernels of the layers behind the encoding load and store them.
//
// A checkpoint keeps a row of C channels in blocks of 32 (the last one shorter).  With a the largest magnitude of a block,
//
//     e = the least integer of at least -126 with a / 2^e < 127.5,     q = round to even (x / 2^e), in -127..127,     x^ = q 2^e.
//
// (e is at most 121: from 127.5 2^121 on, the last 0.4% of what fp32 has, a value is kept as 127 2^121, where 64 2^122 would be infinite.)
// The step is a power of two, so that x / 2^e and q 2^e are exact and q does not depend on how it is computed; x^ is off by at most half a
// step, and is exact in bfloat16.  Off by, in blocks of normally distributed values (rms, in deviations): 0.0083; with a step of a / 127 0.0053, with
// values in e4m3 and a scale for every 32 of them 0.029.
// A block with an infinity or a NaN comes back as NaN.
//
//     values     int8  [rows][pitch]                     pitch: C rounded up to 16, the rest of a row zero
//     exponents  uint8 [rows][ceil(C / 32)]              e + 127, 255 for a block that is not finite
//
// A lane works on 8 consecutive channels, four lanes on a block: 16 bytes of a 16-bit type in a load, 8 of a checkpoint.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/penc.h"

namespace penc {

using half_t = _Float16;
using bf16_t = __bf16;

constexpr int kChunk = 8;   // channels of a lane
constexpr int kKeptBlock = 32;
constexpr int kKeptPitch = 16;

__host__ __device__ __forceinline__ int64_t kept_pitch(int64_t channels) { return (channels + kKeptPitch - 1) / kKeptPitch * kKeptPitch; }
__host__ __device__ __forceinline__ int64_t kept_blocks(int64_t channels) { return (channels + kKeptBlock - 1) / kKeptBlock; }

// Eight values, aligned as one is: rows of any length and stride (gfx950 takes such an address in one 16-byte access).
template <class E>
using chunk_t = E __attribute__((ext_vector_type(kChunk), aligned(sizeof(E))));
using float8 = float __attribute__((ext_vector_type(kChunk)));

template <class E>
using chunk_words = uint32_t __attribute__((ext_vector_type(kChunk * sizeof(E) / 4)));

// A chunk's values moved to its front by `by` places (1 to 7; what follows them is anything).  With masks in place of conditions: of those the
// compiler makes a branch for each value.
template <class E>
__device__ __forceinline__ chunk_words<E> to_front(chunk_words<E> m, int by) {
    constexpr int kWords = kChunk * sizeof(E) / 4;
    const uint32_t by4 = by & 4 ? ~0u : 0u, by2 = by & 2 ? ~0u : 0u, by1 = by & 1 ? ~0u : 0u;
    const auto forward = [&](int n, uint32_t mask) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) m[i] = (i + n < kWords ? m[i + n < kWords ? i + n : 0] & mask : 0u) | (m[i] & ~mask);
    };
    forward(kWords / 2, by4);
    forward(kWords / 4, by2);
    if constexpr (kWords == kChunk) {
        forward(1, by1);
    } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) m[i] = __builtin_amdgcn_alignbit(i + 1 < kWords ? m[i + 1 < kWords ? i + 1 : 0] : 0u, m[i], by1 & 16u);
    }
    return m;
}

// The chunk at channel `c` of a row of `channels`, zeros from the row's end on.  A lane that would read behind the end reads the row's last eight channels
// and moves those it has to the front (a load for each of them: silu of 1048576 x 70 fp32, forward and back with its checkpoint, 429 us instead of 287).
template <class E>
__device__ __forceinline__ void load_chunk(const E* __restrict__ row, int c, int channels, float (&v)[kChunk]) {
    if (channels >= kChunk) {
        using Unaligned = uint32_t __attribute__((ext_vector_type(kChunk * sizeof(E) / 4), aligned(sizeof(E))));
        chunk_words<E> w = *reinterpret_cast<const Unaligned*>(row + min(c, channels - kChunk));
        const uint32_t whole = c + kChunk <= channels ? ~0u : 0u;
        if (channels % kChunk == 0) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(kChunk * sizeof(E) / 4); ++i) w[i] &= whole;
        } else {
            const chunk_words<E> m = to_front<E>(w, kChunk - channels % kChunk);
            const uint32_t part = ~whole & (c < channels ? ~0u : 0u);
#pragma unroll
            for (int i = 0; i < static_cast<int>(kChunk * sizeof(E) / 4); ++i) w[i] = (w[i] & whole) | (m[i] & part);
        }
        const float8 x = __builtin_convertvector(__builtin_bit_cast(E __attribute__((ext_vector_type(kChunk))), w), float8);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) v[i] = x[i];
    } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) v[i] = c + i < channels ? static_cast<float>(row[c + i]) : 0.0f;
    }
}

template <class E>
using chunk_vector = E __attribute__((ext_vector_type(kChunk)));
// (rounded to nearest, ties to even: the only rounding to 16 bits)
template <class E>
__device__ __forceinline__ chunk_vector<E> rounded(const float (&v)[kChunk]) {
    float8 x;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) x[i] = v[i];
    return __builtin_convertvector(x, chunk_vector<E>);
}
template <class E>
__device__ __forceinline__ void store_whole(E* __restrict__ p, chunk_vector<E> y) {
    *reinterpret_cast<chunk_t<E>*>(p) = y;
}
// The first n (1 to 7) of a chunk in fours, twos and ones.
template <class E>
__device__ __forceinline__ void store_part(E* __restrict__ p, int n, chunk_vector<E> y) {
    using Four = E __attribute__((ext_vector_type(4), aligned(sizeof(E))));
    using Two = E __attribute__((ext_vector_type(2), aligned(sizeof(E))));
    if (n & 4) *reinterpret_cast<Four*>(p) = __builtin_shufflevector(y, y, 0, 1, 2, 3);
    if (n & 2) {
        if (n & 4) *reinterpret_cast<Two*>(p + 4) = __builtin_shufflevector(y, y, 4, 5);
        else *reinterpret_cast<Two*>(p) = __builtin_shufflevector(y, y, 0, 1);
    }
    if (n & 1) {
        if (n == 1) p[0] = y[0];
        else if (n == 3) p[2] = y[2];
        else if (n == 5) p[4] = y[4];
        else p[6] = y[6];
    }
}
// The first `valid` (1 or more) of a chunk.
template <class E>
__device__ __forceinline__ void store_chunk(E* __restrict__ p, int valid, const float (&v)[kChunk]) {
    const chunk_vector<E> y = rounded<E>(v);
    if (valid >= kChunk) store_whole(p, y);
    else store_part(p, valid, y);
}

template <int kControl>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kControl, 0xF, 0xF, true));
}
constexpr int kSwapPairs = 0xB1, kSwapTwos = 0x4E;  // quad_perm: lane ^ 1, lane ^ 2
constexpr int kMirrorHalfRow = 0x141, kMirrorRow = 0x140;

// What a block's largest magnitude (as an integer: an infinity or a NaN is the largest) makes of its values.
struct BlockStep {
    uint32_t exponent;
    float per_step;
    bool finite, top;

    __device__ __forceinline__ explicit BlockStep(uint32_t largest) {
        finite = largest < 0x7F800000u;
        // a = m 2^k with m in [1, 2): e = k - 6, and one more from m = 127.5 / 64 on, where the sum below carries into the exponent
        exponent = max((largest + 0x10000u) >> 23, 7u) - 6u;
        top = exponent > 248u;
        exponent = min(exponent, 248u);
        per_step = __uint_as_float((254u - exponent) << 23);
        if (!finite) exponent = 255u;
    }
    // Before the values of a block at the top of the range are quantised (all but never).
    template <int kValues>
    __device__ __forceinline__ void saturate(float (&v)[kValues]) const {
        if (!top) return;
        constexpr float kMost = 0x1.FCp+127f;  // 127 2^121
#pragma unroll
        for (int i = 0; i < kValues; ++i) v[i] = fminf(fmaxf(v[i], -kMost), kMost);
    }
    // Four of the block's values: round(x 2^-e) in the low bits of x 2^-e + 1.5 2^23, one rounding, to even.
    __device__ __forceinline__ uint32_t quantised(const float* v) const {
        uint32_t t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = __float_as_uint(__builtin_fmaf(v[i], per_step, 12582912.0f));
        const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(t[3], t[2], 0x0C0C0400u);
        return finite ? __builtin_amdgcn_perm(hi, lo, 0x05040100u) : 0u;
    }
};

struct Kept {
    uint2 q;
    uint32_t exponent;
};

// The four lanes of a block bring its 32 values, zeros behind the row's end.
__device__ __forceinline__ Kept keep(const float (&x)[kChunk]) {
    float v[kChunk];
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = x[i];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    a = max(a, dpp<kSwapPairs>(a));
    a = max(a, dpp<kSwapTwos>(a));
    const BlockStep s(a);
    s.saturate(v);
    return {make_uint2(s.quantised(v), s.quantised(v + 4)), s.exponent};
}

// (255 gives an infinite step, and 0 times that the NaN)
__device__ __forceinline__ float kept_step(uint32_t exponent) { return __uint_as_float(exponent << 23); }
__device__ __forceinline__ void restore(uint2 q, uint32_t exponent, float (&v)[kChunk], float scale = 1.0f) {
    const float step = kept_step(exponent) * scale;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? q.x : q.y) >> 8 * (i % 4))) * step;
}

// Rows are numbered in 32 bits, and so are their strides: where a row begins takes one multiplication.
using row_t = uint32_t;
constexpr int64_t kMostRows = (int64_t{1} << 31) - 1;
__device__ __forceinline__ uint64_t offset_of(row_t row, uint32_t stride) { return static_cast<uint64_t>(row) * stride; }

// Where a checkpoint is, or null.
struct KeptArray {
    int8_t* values;
    uint8_t* exponents;
    uint32_t pitch, blocks;

    // The lane of the chunk that begins at channel `c` of a row; all four lanes of a block call it.
    __device__ __forceinline__ void store(row_t row, int c, const float (&v)[kChunk]) const {
        const Kept k = keep(v);
        const uint32_t at = static_cast<uint32_t>(c);
        if (at < pitch) *reinterpret_cast<uint2*>(values + offset_of(row, pitch) + at) = k.q;
        if (at % kKeptBlock == 0 && at / kKeptBlock < blocks) exponents[offset_of(row, blocks) + at / kKeptBlock] = static_cast<uint8_t>(k.exponent);
    }
    // (of a chunk that begins before the row's end; from there on it is zeros, or NaN as the rest of its block)
    __device__ __forceinline__ void load(row_t row, int c, float (&v)[kChunk]) const {
        restore(*reinterpret_cast<const uint2*>(values + offset_of(row, pitch) + c), exponents[offset_of(row, blocks) + c / kKeptBlock], v);
    }
};

inline KeptArray kept_array(const int8_t* values, const uint8_t* exponents, int64_t channels) {
    return {const_cast<int8_t*>(values), const_cast<uint8_t*>(exponents), static_cast<uint32_t>(kept_pitch(channels)),
            static_cast<uint32_t>(kept_blocks(channels))};
}

// Runs `f` with a value of the type that an entry point's `type` names.
template <class F>
int with_type(int type, F&& f) {
    switch (type) {
        case PENC_FP32: return f(float{});
        case PENC_FP16: return f(half_t{});
        case PENC_BF16: return f(bf16_t{});
        default: return PENC_ERR_UNSUPPORTED_TYPE;
    }
}

inline bool bad_rows(int64_t rows) { return rows < 0 || rows > kMostRows; }
inline bool bad_stride(int64_t stride) { return stride < 0 || stride > kMostRows; }
inline int launched() { return hipGetLastError() == hipSuccess ? PENC_OK : PENC_ERR_LAUNCH; }
inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace penc
