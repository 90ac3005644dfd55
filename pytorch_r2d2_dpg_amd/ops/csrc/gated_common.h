// Shared by the layer norm, gated recurrence and gated linear kernels.
#pragma once

#include "common.h"

#include <cstdint>
#include <type_traits>

using bf16 = __hip_bfloat16;

DEV_INLINE float to_f(float v) { return v; }
DEV_INLINE float to_f(bf16 v) { return bf2f(v); }
template <typename E> DEV_INLINE E from_f(float v);
template <> DEV_INLINE float from_f<float>(float v) { return v; }
template <> DEV_INLINE bf16 from_f<bf16>(float v) { return f2bf(v); }

// sigma(x) and sigma(-x) = 1 - sigma(x) from one exponential of -|x|: neither
// cancels where the other is near one, and a NaN is both. The exp2 and rcp
// instructions are within 1 ulp, the argument's rounding adds |x| * 2^-24.
DEV_INLINE void sigmoid_pair(float x, float& pos, float& neg) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * 1.44269504f);
    const float big = __builtin_amdgcn_rcpf(1.0f + e);
    const float small = e * big;
    pos = x >= 0.0f ? big : small;
    neg = x >= 0.0f ? small : big;
}

// silu(x) = x * sigma(x) and its derivative sigma + x sigma (1 - sigma). Where
// sigma nears one, 1 - sigma is off by a rounding of one, as is what it is added to.
DEV_INLINE void silu_grad(float x, float& val, float& grad) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
    val = x * s;
    grad = s + val * (1.0f - s);
}

// N consecutive elements in one memory instruction, whatever their alignment
// (global loads and stores need none beyond the element's on this target).
template <typename E, int N>
struct __attribute__((packed, aligned(sizeof(E)))) Run {
    E v[N];
};

// Elements p[0..N) of which the first `have` exist; the others read as 0.
template <typename E, int N>
DEV_INLINE void load_run(const E* p, int have, E (&out)[N]) {
    if (have >= N) {
        const Run<E, N> r = *reinterpret_cast<const Run<E, N>*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = r.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = i < have ? p[i] : from_f<E>(0.0f);
    }
}

template <typename E, int N>
DEV_INLINE void store_run(E* p, int have, const E (&in)[N]) {
    if (have >= N) {
        Run<E, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = in[i];
        *reinterpret_cast<Run<E, N>*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < have) p[i] = in[i];
    }
}

// Two values as they lie in memory; a register of two bf16 until they are used.
template <typename E> struct Two;
template <> struct Two<float> {
    float v[2];
    DEV_INLINE float operator[](int i) const { return v[i]; }
    static DEV_INLINE Two of(float a, float b) { return {{a, b}}; }
};
template <> struct Two<bf16> {
    unsigned v;
    DEV_INLINE float operator[](int i) const {
        return __uint_as_float(i ? v & 0xffff0000u : v << 16);
    }
    static DEV_INLINE Two of(float a, float b) {
        using f2 = __attribute__((ext_vector_type(2))) float;
        using b2 = __attribute__((ext_vector_type(2))) __bf16;
        return {__builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, b2))};
    }
};

// Sum over a row of 16 lanes, the same in each: operands of the additions are
// the other lanes' values, none goes through LDS.
DEV_INLINE float row_sum16(float v) {
#ifdef __HIP_DEVICE_COMPILE__
    const auto turned = [](float x, auto control) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x),
                                                          decltype(control)::value, 0xf, 0xf, true));
    };
    v += turned(v, std::integral_constant<int, 0xb1>());   // lane ^ 1
    v += turned(v, std::integral_constant<int, 0x4e>());   // lane ^ 2
    v += turned(v, std::integral_constant<int, 0x141>());  // half a row mirrored
    v += turned(v, std::integral_constant<int, 0x140>());  // a row mirrored
#endif
    return v;
}

// Sum over a wave, the same in each lane: across the rows by lane swaps.
DEV_INLINE float wave_sum(float v) {
    v = row_sum16(v);
#ifdef __HIP_DEVICE_COMPILE__
    const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                       false, false);
    v = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                         false, false);
    v = __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
#endif
    return v;
}

// out[c] = sum over r of part[r][c] in a fixed order: the second stage of a
// reduction over rows, in place of atomics whose order would change results.
// A block of 1024 threads has 16 columns, which 64 groups of threads walk 64 rows
// apart, eight loads at a time.
template <typename E>
DEV_INLINE void sum_columns(const float* __restrict__ part, E* __restrict__ out, int rows,
                            int cols, int block) {
    __shared__ float sums[64][17];
    const int in = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int c = block * 16 + in;
    const float* p = part + (c < cols ? c : cols - 1);
    float s = 0.0f;
    for (int r0 = group; r0 < rows; r0 += 8 * 64) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int r = r0 + 64 * k;
            v[k] = p[(int64_t)(r < rows ? r : rows - 1) * cols];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) s += r0 + 64 * k < rows ? v[k] : 0.0f;
    }
    sums[group][in] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < cols) {
        float t[4] = {};
#pragma unroll
        for (int g = 0; g < 64; ++g) t[g & 3] += sums[g][in];
        out[c] = from_f<E>((t[0] + t[1]) + (t[2] + t[3]));
    }
}
constexpr int column_blocks(int cols) { return cols / 16 + (cols % 16 != 0); }
