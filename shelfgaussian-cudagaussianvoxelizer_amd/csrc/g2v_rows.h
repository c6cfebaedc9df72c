// Rows that a group of lanes reads, sums and writes (g2v_qknorm.hip, g2v_layernorm.hip): 16 bytes a lane.
#pragma once
#include "g2v_internal.h"

namespace g2v {

template <typename T>
struct RowVec;
template <>
struct RowVec<float> {
    static constexpr int n = 4;
    typedef f32x4 raw;
};
template <>
struct RowVec<__bf16> {
    static constexpr int n = 8;
    typedef bf16x8 raw;
};

// Elements [d, d + n) of a row, zero past the end.  AL: rows and D are whole 16-byte vectors; else a vector within the row
// is still one access (global memory takes any alignment), and only the row's last elements go one by one.
template <typename T, bool AL>
__device__ __forceinline__ typename RowVec<T>::raw row_load(const T* row, int d, int D) {
    typedef typename RowVec<T>::raw raw;
    typedef raw raw_any __attribute__((aligned(sizeof(T))));
    raw v;
#pragma unroll
    for (int j = 0; j < RowVec<T>::n; ++j) v[j] = (T)0.0f;
    if constexpr (AL) {
        if (d < D) v = *reinterpret_cast<const raw*>(row + d);
    } else if (d + RowVec<T>::n <= D) {
        v = *reinterpret_cast<const raw_any*>(row + d);
    } else {
#pragma unroll
        for (int j = 0; j < RowVec<T>::n; ++j)
            if (d + j < D) v[j] = row[d + j];
    }
    return v;
}
template <typename T, bool AL>
__device__ __forceinline__ void row_store(T* row, int d, int D, const float (&o)[RowVec<T>::n]) {
    constexpr int n = RowVec<T>::n;
    typedef typename RowVec<T>::raw raw;
    typedef raw raw_any __attribute__((aligned(sizeof(T))));
    raw v;
#pragma unroll
    for (int j = 0; j < n; ++j) v[j] = (T)o[j];
    if constexpr (AL) {
        if (d < D) *reinterpret_cast<raw*>(row + d) = v;
    } else if (d + n <= D) {
        *reinterpret_cast<raw_any*>(row + d) = v;
    } else {
#pragma unroll
        for (int j = 0; j < n; ++j)
            if (d + j < D) row[d + j] = v[j];
    }
}

// Sums over the 2^shift lanes of a row.  Within 16 lanes by data-parallel moves: after the steps before it every
// lane of a mirrored half holds the same sum, so a mirror serves as the exchange of the next size.
template <int kCtrl>
__device__ __forceinline__ float dpp_add(float v) {
    const int o = __builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xF, 0xF, true);
    return v + __int_as_float(o);
}
template <int M>
__device__ __forceinline__ void row_sums(float (&v)[M], int shift) {
    if (shift > 0)    // quad_perm 1 0 3 2
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = dpp_add<0xB1>(v[m]);
    if (shift > 1)    // quad_perm 2 3 0 1
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = dpp_add<0x4E>(v[m]);
    if (shift > 2)    // row_half_mirror
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = dpp_add<0x141>(v[m]);
    if (shift > 3)    // row_mirror
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = dpp_add<0x140>(v[m]);
    if (shift > 4)
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] += __shfl_xor(v[m], 16);
    if (shift > 5)
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] += __shfl_xor(v[m], 32);
}

}  // namespace g2v
