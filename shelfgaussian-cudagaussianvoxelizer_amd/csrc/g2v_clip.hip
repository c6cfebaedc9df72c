// The norm of many gradient tensors taken together, and clipping by it:
//
//   n = (sum over tensors of sum g^2)^1/2,   c = min(1, max_norm / (n + 1e-6)),   out = c g.
//
// Bound by bytes (gradients read for the norm; read again and written for the scaling) or, where tensors are small, by launches:
// the tensors' addresses go along as kernel arguments, kClipTensors a launch, so that two launches serve a small model.  Tensors
// are cut into chunks; a workgroup of the norm's kernel takes every gridDim-th of them and leaves one partial sum, and each
// workgroup of the scaling adds the partial sums by itself, in one order, instead of waiting for a launch that does.  Squares
// are summed in 64 bits: no float32 value overflows them, and a multiply-add of 64 bits an element takes less than its load.
#include <algorithm>

#include "../../include/g2v.h"
#include "g2v_internal.h"

namespace g2v {
namespace {

constexpr int kClipThreads = 256;
// Most workgroups of a launch of the norm: partial sums that every scaling workgroup adds.  12 layers of 1024 channels, 302 MB of
// bfloat16 gradients: the norm takes 112, 100, 89 and 91 us with 512, 1024, 2048 and 4096 (3.4 TB/s), writing 604 MB of float32
// 221, 198, 184 and 187 (4.9 TB/s).
constexpr int kClipParts = 2048;

// As many elements of a row of memory as 16 bytes hold.
template <typename T>
struct ClipVec {
    static constexpr int n = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(n), aligned(sizeof(T))));
};

// Tensor and first element of a chunk.
struct ClipAt {
    int k;
    int64_t first, last;
};
__device__ __forceinline__ ClipAt clip_at(const ClipArgs& a, int chunk) {
    int lo = 0, hi = a.count - 1;     // the last tensor that begins at or before the chunk (tensors without elements hold none)
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.start[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    ClipAt r;
    r.k = lo;
    r.first = (int64_t)(chunk - a.start[lo]) * a.chunk;
    r.last = min(r.first + a.chunk, a.n[lo]);
    return r;
}

__device__ __forceinline__ double wave_sum64(double v) {
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ double block_sum64(double v, double* red) {
    v = wave_sum64(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int k = 0; k < kClipThreads / 64; ++k) v += red[k];
    return v;
}

template <typename T>
__device__ __forceinline__ double clip_squares(const T* g, int64_t first, int64_t last) {
    typedef typename ClipVec<T>::vec vec;
    constexpr int N = ClipVec<T>::n, U = 4;
    double s[U] = {0.0, 0.0, 0.0, 0.0};
    int64_t i = first + (int64_t)threadIdx.x * N;
    for (; i + (U - 1) * kClipThreads * N + N <= last; i += U * kClipThreads * N) {
        vec x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const vec*>(g + i + u * kClipThreads * N);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const double v = (double)(float)x[u][j];
                s[u] = fma(v, v, s[u]);
            }
    }
    for (; i < last; i += kClipThreads * N)
        for (int j = 0; j < N; ++j)
            if (i + j < last) {
                const double v = (double)(float)g[i + j];
                s[0] = fma(v, v, s[0]);
            }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ void __launch_bounds__(kClipThreads) k_clip_norm(ClipArgs a, double* part) {
    __shared__ double red[kClipThreads / 64];
    double s = 0.0;
    for (int c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        const ClipAt at = clip_at(a, c);
        s += a.bf16[at.k] & 1 ? clip_squares(static_cast<const __bf16*>(a.g[at.k]), at.first, at.last)
                              : clip_squares(static_cast<const float*>(a.g[at.k]), at.first, at.last);
    }
    s = block_sum64(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <typename T, typename O>
__device__ __forceinline__ void clip_scale(const T* g, O* out, int64_t first, int64_t last, double c) {
    typedef typename ClipVec<T>::vec vec;
    constexpr int N = ClipVec<T>::n, U = 4;
    typedef O ovec __attribute__((ext_vector_type(N), aligned(sizeof(O))));
    int64_t i = first + (int64_t)threadIdx.x * N;
    for (; i + (U - 1) * kClipThreads * N + N <= last; i += U * kClipThreads * N) {
        vec x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const vec*>(g + i + u * kClipThreads * N);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ovec o;
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] = (O)(float)((double)(float)x[u][j] * c);
            *reinterpret_cast<ovec*>(out + i + u * kClipThreads * N) = o;
        }
    }
    for (; i < last; i += kClipThreads * N)
        for (int j = 0; j < N; ++j)
            if (i + j < last) out[i + j] = (O)(float)((double)(float)g[i + j] * c);
}

__global__ void __launch_bounds__(kClipThreads) k_clip_scale(ClipArgs a, const double* part, int parts, float max_norm, float* norm) {
    __shared__ double red[kClipThreads / 64];
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kClipThreads) s += part[i];
    const double n = sqrt(block_sum64(s, red));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double q = (double)max_norm / (n + 1e-6);
    const double c = q > 1.0 ? 1.0 : q;     // NaN stays
    for (int i = blockIdx.x; i < a.chunks; i += gridDim.x) {
        const ClipAt at = clip_at(a, a.chunks - 1 - i);    // the last ones read are the likeliest in the cache
        const void* g = a.g[at.k];
        void* out = a.out[at.k];
        if (c == 1.0 && g == out) continue;     // in place and of one type
        switch (a.bf16[at.k]) {
            case 0: clip_scale(static_cast<const float*>(g), static_cast<float*>(out), at.first, at.last, c); break;
            case 1: clip_scale(static_cast<const __bf16*>(g), static_cast<float*>(out), at.first, at.last, c); break;
            case 2: clip_scale(static_cast<const float*>(g), static_cast<__bf16*>(out), at.first, at.last, c); break;
            default: clip_scale(static_cast<const __bf16*>(g), static_cast<__bf16*>(out), at.first, at.last, c);
        }
    }
}

// Elements of a chunk: as few as give a launch's workgroups one each, in steps of a workgroup's unrolled loads, so that few
// workgroups stand idle at the end.
int64_t clip_chunk(const int64_t* numels, int64_t count) {
    int64_t all = 0;
    for (int64_t k = 0; k < count; ++k) all += numels[k];
    constexpr int64_t kStep = 4 * kClipThreads * 8;
    return std::max<int64_t>(1, ceil_div(all, kClipParts * kStep)) * kStep;
}

}  // namespace

size_t clip_workspace(int64_t count) {
    const int64_t launches = std::max<int64_t>(1, ceil_div(count, kClipTensors));
    return (size_t)launches * kClipParts * sizeof(double) + 256;
}

hipError_t launch_clip(int64_t count, const void* const* g, void* const* out, const int64_t* numels, const int* g_bf16,
                       const int* out_bf16, float max_norm, float* norm, void* ws, hipStream_t s) {
    Carver c(ws, (size_t)-1);
    const int64_t launches = std::max<int64_t>(1, ceil_div(count, kClipTensors));
    double* part = c.take<double>((size_t)launches * kClipParts);
    int parts = 0;
    ClipArgs a;
    auto fill = [&](int64_t l) {
        const int64_t first = l * kClipTensors;
        a.count = (int)std::min<int64_t>(kClipTensors, count - first);
        a.chunk = clip_chunk(numels + first, a.count);
        a.chunks = 0;
        for (int k = 0; k < a.count; ++k) {
            a.g[k] = g[first + k];
            a.out[k] = out[first + k];
            a.n[k] = numels[first + k];
            a.bf16[k] = (unsigned char)((g_bf16[first + k] ? 1 : 0) + (out_bf16[first + k] ? 2 : 0));
            a.start[k] = a.chunks;
            a.chunks += (int)ceil_div(a.n[k], a.chunk);
        }
    };
    for (int64_t l = 0; l < launches; ++l) {
        fill(l);
        const int blocks = std::min(a.chunks, kClipParts);
        if (blocks > 0) G2V_LAUNCH(k_clip_norm, dim3(blocks), dim3(kClipThreads), 0, s, a, part + parts);
        parts += blocks;
    }
    for (int64_t l = launches - 1; l >= 0; --l) {
        fill(l);
        if (l > 0 && a.chunks == 0) continue;
        G2V_LAUNCH(k_clip_scale, dim3(std::max(1, a.chunks)), dim3(kClipThreads), 0, s, a, part, parts, max_norm,
                   l == 0 ? norm : nullptr);
    }
    return hipGetLastError();
}

}  // namespace g2v
