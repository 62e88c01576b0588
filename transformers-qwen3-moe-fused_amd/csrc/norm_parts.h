// What the norm's kernels (norm.hip) and the expert layer's first kernel (layer.hip) share: rows eight elements a lane at a time,
// the stream's rounding and the normalised value.
//
// s = x + residual rounded to the tensors' type; y = s r w with r = 1 / sqrt(sum(s^2) / H + eps), rounded to 32 bits and from
// there to the type.  The sum, r and the products are in 64 bits: the vector units take them at the rate of ordinary 32-bit
// operations, a row's time is its memory's either way, and what comes out is the definition's value up to its last rounding in
// the type, which matters where it is rounded again: the 8-bit grid, and the router's logits, where a last bit decides between two
// experts.
#pragma once
#include "common.h"

namespace mfl {

// Eight elements of a row.  WHOLE: rows are whole eights long (and stay packed in registers).  They may start anywhere: loads and
// stores are 16 bytes wide whatever the alignment.
template <typename T, bool WHOLE>
struct alignas(16) Eight {
    T v[8];
    // those from column k on; zeros behind column H
    __device__ __forceinline__ void load(const T *row, int k, int H) {
        if (WHOLE ? k < H : k + 8 <= H) {
            __builtin_memcpy(v, row + k, sizeof(v));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = !WHOLE && k + i < H ? row[k + i] : (T)0.0f;
        }
    }
    __device__ __forceinline__ void store(T *row, int k, int H) const {
        if (WHOLE ? k < H : k + 8 <= H) {
            __builtin_memcpy(row + k, v, sizeof(v));
        } else if (!WHOLE) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < H) row[k + i] = v[i];
        }
    }
};

// s of two rows' elements.  (The sum of two 16-bit values is rounded twice here, to 32 bits and to the type; the first rounding
// cannot bring it onto or across a border of the second: 24 bits are more than twice the type's and two.)
template <typename T, bool WHOLE>
__device__ __forceinline__ void add_rounded(Eight<T, WHOLE> &x, const Eight<T, WHOLE> &residual) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = from_f32<T>(to_f32(x.v[i]) + to_f32(residual.v[i]));
}

template <typename T, bool WHOLE>
__device__ __forceinline__ double sum_of_squares(const Eight<T, WHOLE> &s, double sum) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double v = (double)to_f32(s.v[i]);
        sum = __builtin_fma(v, v, sum);
    }
    return sum;
}

// 1 / sqrt(m) to the last bits of a double: the hardware's estimate and two of Newton's steps r <- r + r (1 - m r^2) / 2.
__device__ __forceinline__ double inverse_root(double m) {
    double r = __builtin_amdgcn_rsq(m);
    if (r == 0.0 || __builtin_isinf(r)) return r;  // (m infinite or zero)
#pragma unroll
    for (int i = 0; i < 2; ++i) r = __builtin_fma(0.5 * r, __builtin_fma(-m * r, r, 1.0), r);
    return r;
}

template <typename T, typename TW>
__device__ __forceinline__ T normed(T s, double r, TW w) {
    return from_f32<T>((float)((double)to_f32(s) * r * (double)to_f32(w)));
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

}  // namespace mfl
