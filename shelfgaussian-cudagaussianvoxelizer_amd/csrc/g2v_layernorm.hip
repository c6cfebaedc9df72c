// Layer norm with the residual sum before it, and its backward.  A row s has C values, weight w and bias b:
//
//   s = x + residual (rounded to the rows' type),  m = mean s,  r = (mean (s - m)^2 + eps)^-1/2,  y = (s - m) r w + b.
//
// Backward, from dy and the gradient ds that reaches s by another way, with xh = (s - m) r and g = w dy:
//   dx = ds + r (g - mean g - xh mean(g xh))   (of x and of residual),   dw = sum over rows of dy xh,   db = sum of dy.
//
// Bound by bytes: 18000 x 1024 bfloat16 with a residual takes 27 us forward and 27 + 7 backward, 5.4 TB/s, a copy's rate (and
// more than it, where inputs are still in the last cache).  A row is read once, held in registers, and the variance is taken from
// the differences to the mean (nothing cancels).  A row goes to 2^shift lanes of a wave, up to two 16-byte vectors each, or to a
// workgroup where it is longer; the next row is asked for before the present one is summed.  Weights stay in registers, as do, in
// the backward, the sums of dw and db of a workgroup's rows: their parts go to memory once a workgroup, and k_layer_norm_sums adds
// them in a fixed order.
#include <algorithm>

#include "../../include/g2v.h"
#include "g2v_internal.h"
#include "g2v_rows.h"

namespace g2v {
namespace {

constexpr int kLnThreads = 256, kLnWaves = kLnThreads / 64;

// Sums over the lanes of a row: 2^shift of a wave (WAVES 1), or all of the workgroup's.
template <int WAVES, int M>
__device__ __forceinline__ void ln_sums(float (&v)[M], int shift, float* red) {
    if constexpr (WAVES == 1) {
        row_sums(v, shift);
    } else {
        row_sums(v, 6);
        __syncthreads();    // the sums before are read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int m = 0; m < M; ++m) red[m * kLnWaves + (threadIdx.x >> 6)] = v[m];
        __syncthreads();
#pragma unroll
        for (int m = 0; m < M; ++m) {
            v[m] = 0.0f;
#pragma unroll
            for (int k = 0; k < kLnWaves; ++k) v[m] += red[m * kLnWaves + k];
        }
    }
}

// A weight's elements [d, d + N), `none` past the end or without a weight.
template <typename W, int N>
__device__ __forceinline__ void ln_weights_of(const W* w, int d, int dim, float (&o)[N]) {
    typedef W vec __attribute__((ext_vector_type(4), aligned(sizeof(W))));
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        if (d + j + 4 <= dim) {
            const vec v = *reinterpret_cast<const vec*>(w + d + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j + e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + j + e < dim) o[j + e] = (float)w[d + j + e];
        }
    }
}
template <int N>
__device__ __forceinline__ void ln_weights(const void* w, int bf16, int d, int dim, float none, float (&o)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = none;
    if (!w) return;
    if (bf16) ln_weights_of(static_cast<const __bf16*>(w), d, dim, o);
    else ln_weights_of(static_cast<const float*>(w), d, dim, o);
}

// A thread's place: lane of a row, the row's group in the workgroup, and how many groups there are.
struct LnPlace {
    int lane, lanes, group, groups;
};
template <int WAVES>
__device__ __forceinline__ LnPlace ln_place(const LayerNormArgs& a) {
    LnPlace p;
    if constexpr (WAVES == 1) {
        p.lanes = 1 << a.shift;
        p.lane = threadIdx.x & (p.lanes - 1);
        p.group = threadIdx.x >> a.shift;
        p.groups = kLnThreads >> a.shift;
    } else {
        p.lanes = kLnThreads;
        p.lane = threadIdx.x;
        p.group = 0;
        p.groups = 1;
    }
    return p;
}

template <typename T>
__device__ __forceinline__ const T* ln_row(const LayerNormArgs& a, int which, int64_t row) {
    const int64_t b = row / a.n, i = row - b * a.n;
    return static_cast<const T*>(a.in[which]) + b * a.sb[which] + i * a.sn[which];
}

template <typename T, bool AL, int V, int WAVES, bool RES>
__global__ void __launch_bounds__(kLnThreads) k_layer_norm(LayerNormArgs a) {
    constexpr int N = RowVec<T>::n;
    typedef typename RowVec<T>::raw raw;
    __shared__ float red[2 * kLnWaves];
    const LnPlace p = ln_place<WAVES>(a);
    const float inv = 1.0f / (float)a.dim;
    float w[V][N], bias[V][N];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        ln_weights(a.w, a.wbf16, (v * p.lanes + p.lane) * N, a.dim, 1.0f, w[v]);
        ln_weights(a.b, a.wbf16, (v * p.lanes + p.lane) * N, a.dim, 0.0f, bias[v]);
    }
    const int64_t step = (int64_t)gridDim.x * p.groups;
    int64_t row = (int64_t)blockIdx.x * p.groups + p.group;
    raw x[V], res[V];
    auto load = [&](int64_t at) {
        const int64_t r = at < a.rows ? at : a.rows - 1;    // groups past the end repeat the last row, unstored
        const T* xr = ln_row<T>(a, 0, r);
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = row_load<T, AL>(xr, (v * p.lanes + p.lane) * N, a.dim);
        if constexpr (RES) {
            const T* rr = ln_row<T>(a, 1, r);
#pragma unroll
            for (int v = 0; v < V; ++v) res[v] = row_load<T, AL>(rr, (v * p.lanes + p.lane) * N, a.dim);
        }
    };
    load(row);
    for (int64_t row0 = (int64_t)blockIdx.x * p.groups; row0 < a.rows; row0 += step, row += step) {
        float s[V][N], sum[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                s[v][j] = (float)x[v][j];
                if constexpr (RES) s[v][j] = (float)(T)(s[v][j] + (float)res[v][j]);
                sum[0] += s[v][j];    // zeros past the end
            }
        if (row0 + step < a.rows) load(row + step);
        ln_sums<WAVES>(sum, a.shift, red);
        const float m = sum[0] * inv;
        float sq[1] = {0.0f};
        const bool live = row < a.rows;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int d = (v * p.lanes + p.lane) * N;
            if constexpr (RES)
                if (live) row_store<T, AL>(static_cast<T*>(a.sum) + row * a.dim, d, a.dim, s[v]);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                s[v][j] -= m;
                if (d + j < a.dim) sq[0] = fmaf(s[v][j], s[v][j], sq[0]);
            }
        }
        ln_sums<WAVES>(sq, a.shift, red);
        const float r = 1.0f / sqrtf(fmaf(sq[0], inv, a.eps));
        if (live) {
            if (a.stats && p.lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(m, r);
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int j = 0; j < N; ++j) s[v][j] = fmaf(s[v][j] * r, w[v][j], bias[v][j]);
                row_store<T, AL>(static_cast<T*>(a.y) + row * a.dim, (v * p.lanes + p.lane) * N, a.dim, s[v]);
            }
        }
    }
}

// in: s, dy, ds (RES).
template <typename T, bool AL, int V, int WAVES, bool RES>
__global__ void __launch_bounds__(kLnThreads) k_layer_norm_bwd(LayerNormArgs a) {
    constexpr int N = RowVec<T>::n;
    typedef typename RowVec<T>::raw raw;
    __shared__ float red[WAVES == 1 ? kLnThreads * V * N : 2 * kLnWaves];
    const LnPlace p = ln_place<WAVES>(a);
    const float inv = 1.0f / (float)a.dim;
    float w[V][N], dw[V][N], db[V][N];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        ln_weights(a.w, a.wbf16, (v * p.lanes + p.lane) * N, a.dim, 1.0f, w[v]);
#pragma unroll
        for (int j = 0; j < N; ++j) dw[v][j] = db[v][j] = 0.0f;
    }
    const int64_t step = (int64_t)gridDim.x * p.groups;
    int64_t row = (int64_t)blockIdx.x * p.groups + p.group;
    raw x[V], g[V], e[V];
    float2 st;
    auto load = [&](int64_t at) {
        const int64_t r = at < a.rows ? at : a.rows - 1;
        const T *xr = ln_row<T>(a, 0, r), *gr = ln_row<T>(a, 1, r);
        st = *reinterpret_cast<const float2*>(a.stats + 2 * r);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = row_load<T, AL>(xr, (v * p.lanes + p.lane) * N, a.dim);
            g[v] = row_load<T, AL>(gr, (v * p.lanes + p.lane) * N, a.dim);
        }
        if constexpr (RES) {
            const T* er = ln_row<T>(a, 2, r);
#pragma unroll
            for (int v = 0; v < V; ++v) e[v] = row_load<T, AL>(er, (v * p.lanes + p.lane) * N, a.dim);
        }
    };
    load(row);
    for (int64_t row0 = (int64_t)blockIdx.x * p.groups; row0 < a.rows; row0 += step, row += step) {
        const bool live = row < a.rows;
        const float m = st.x, r = st.y;
        float xh[V][N], t[V][N], ex[V][N], s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const bool in = (v * p.lanes + p.lane) * N + j < a.dim;
                const float dy = live ? (float)g[v][j] : 0.0f;    // zero past the end
                xh[v][j] = in ? ((float)x[v][j] - m) * r : 0.0f;
                dw[v][j] = fmaf(dy, xh[v][j], dw[v][j]);
                db[v][j] += dy;
                t[v][j] = dy * w[v][j];
                s[0] += t[v][j];
                s[1] = fmaf(t[v][j], xh[v][j], s[1]);
                if constexpr (RES) ex[v][j] = (float)e[v][j];
            }
        if (row0 + step < a.rows) load(row + step);
        ln_sums<WAVES>(s, a.shift, red);
        if (live) {
            const float c0 = s[0] * inv, c1 = s[1] * inv;
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    t[v][j] = r * (t[v][j] - c0 - xh[v][j] * c1);
                    if constexpr (RES) t[v][j] += ex[v][j];
                }
                row_store<T, AL>(static_cast<T*>(a.y) + row * a.dim, (v * p.lanes + p.lane) * N, a.dim, t[v]);
            }
        }
    }
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int d = (v * p.lanes + p.lane) * N + j;
                if (d < a.dim) {
                    part[d] = dw[v][j];
                    part[a.dim + d] = db[v][j];
                }
            }
    } else {
        // lanes of the same columns: groups of a wave by exchange, the waves through LDS
        const int span = p.lanes * V * N, wave = threadIdx.x >> 6;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float(&sums)[V][N] = k ? db : dw;
            for (int o = p.lanes; o < 64; o <<= 1)
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int j = 0; j < N; ++j) sums[v][j] += __shfl_xor(sums[v][j], o);
            __syncthreads();
            if ((threadIdx.x & 63) < p.lanes)
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int j = 0; j < N; ++j) red[wave * span + (v * p.lanes + p.lane) * N + j] = sums[v][j];
            __syncthreads();
            for (int d = threadIdx.x; d < a.dim; d += kLnThreads) {
                float o = 0.0f;
#pragma unroll
                for (int i = 0; i < kLnWaves; ++i) o += red[i * span + d];
                part[k * a.dim + d] = o;
            }
        }
    }
}

// dw and db from the workgroups' parts: 16 columns a workgroup, 64 lanes a column, a fixed order.
constexpr int kLnSumThreads = 1024;
__global__ void __launch_bounds__(kLnSumThreads) k_layer_norm_sums(LayerNormArgs a, int parts) {
    __shared__ float red[kLnSumThreads];
    const int cols = 2 * a.dim, col = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
    float v = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (int r = part; r < parts; r += 64) v += a.part[(int64_t)r * cols + col];
    }
    red[threadIdx.x] = v;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (part < o) red[threadIdx.x] += red[threadIdx.x + 16 * o];
        __syncthreads();
    }
    if (part == 0 && col < cols) {
        void* dst = col < a.dim ? a.dw : a.db;
        const int d = col < a.dim ? col : col - a.dim;
        if (dst && a.wbf16) static_cast<__bf16*>(dst)[d] = (__bf16)red[threadIdx.x];
        else if (dst) static_cast<float*>(dst)[d] = red[threadIdx.x];
    }
}

template <typename T>
bool ln_aligned(const LayerNormArgs& a) {
    const int64_t n = RowVec<T>::n;
    bool ok = a.dim % n == 0;
    for (int k = 0; k < 3; ++k)
        if (a.in[k]) ok = ok && reinterpret_cast<uintptr_t>(a.in[k]) % 16 == 0 && a.sb[k] % n == 0 && a.sn[k] % n == 0;
    for (const void* p : {(const void*)a.y, (const void*)a.sum})
        if (p) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    return ok;
}

// Lanes of a row as a shift, vectors of a lane, and whether a row takes a whole workgroup.
struct LnShape {
    int shift, vectors;
    bool wide;
};
LnShape ln_shape(int dim, bool bf16) {
    LnShape g;
    const int vectors = (int)ceil_div(dim, bf16 ? 8 : 4);
    g.wide = vectors > 128;
    const int lanes = g.wide ? kLnThreads : 64;
    g.shift = 6;
    if (!g.wide)
        while (g.shift > 0 && (1 << (g.shift - 1)) >= vectors) --g.shift;
    g.vectors = 1;
    while (g.vectors * lanes < vectors) g.vectors *= 2;
    return g;
}
int ln_groups(const LnShape& g) { return g.wide ? 1 : kLnThreads >> g.shift; }

// Most workgroups: about those that fit the card, each with as many rows, so that weights are loaded and their sums left seldom and
// no workgroup has a turn more than others.  18000 x 1024 bfloat16 with a residual, forward with at most 1024, 2048, 4096 and
// 16384: 34.8, 38.0, 45.4 and 73.8 us (26.9 since weights are loaded by vectors); backward with its sums, 512, 768, 1024 and 2048:
// 34.8, 33.9, 40.8 and 41.2 us.
constexpr int kLnBlocks = 1024, kLnBwdBlocks = 768;
int ln_blocks(const LnShape& g, int64_t rows, int most) {
    const int64_t turns = ceil_div(rows, (int64_t)ln_groups(g) * most);
    return (int)ceil_div(rows, ln_groups(g) * std::max<int64_t>(turns, 1));
}

template <typename T, bool AL, int V, int WAVES>
void ln_launch(const LayerNormArgs& a, bool backward, bool res, int blocks, hipStream_t s) {
    const dim3 grid(blocks), block(kLnThreads);
    if (backward) {
        if (res) G2V_LAUNCH((k_layer_norm_bwd<T, AL, V, WAVES, true>), grid, block, 0, s, a);
        else G2V_LAUNCH((k_layer_norm_bwd<T, AL, V, WAVES, false>), grid, block, 0, s, a);
    } else {
        if (res) G2V_LAUNCH((k_layer_norm<T, AL, V, WAVES, true>), grid, block, 0, s, a);
        else G2V_LAUNCH((k_layer_norm<T, AL, V, WAVES, false>), grid, block, 0, s, a);
    }
}
template <typename T, bool AL>
void ln_vectors(const LayerNormArgs& a, const LnShape& g, bool backward, bool res, int blocks, hipStream_t s) {
    if (g.wide) {
        if (g.vectors == 1) return ln_launch<T, AL, 1, kLnWaves>(a, backward, res, blocks, s);
        if (g.vectors == 2) return ln_launch<T, AL, 2, kLnWaves>(a, backward, res, blocks, s);
        if constexpr (sizeof(T) == 4)
            if (g.vectors == 8) return ln_launch<T, AL, 8, kLnWaves>(a, backward, res, blocks, s);
        return ln_launch<T, AL, 4, kLnWaves>(a, backward, res, blocks, s);
    }
    if (g.vectors == 1) return ln_launch<T, AL, 1, 1>(a, backward, res, blocks, s);
    return ln_launch<T, AL, 2, 1>(a, backward, res, blocks, s);
}
hipError_t ln_run(LayerNormArgs& a, bool bf16, const LnShape& g, bool backward, bool res, int blocks, hipStream_t s) {
    a.shift = g.shift;
    if (bf16) {
        if (ln_aligned<__bf16>(a)) ln_vectors<__bf16, true>(a, g, backward, res, blocks, s);
        else ln_vectors<__bf16, false>(a, g, backward, res, blocks, s);
    } else {
        if (ln_aligned<float>(a)) ln_vectors<float, true>(a, g, backward, res, blocks, s);
        else ln_vectors<float, false>(a, g, backward, res, blocks, s);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_layer_norm(const LayerNormArgs& args, int dtype, hipStream_t s) {
    LayerNormArgs a = args;
    if (a.rows == 0) return hipSuccess;
    const bool bf16 = dtype == kDtBF16;
    const LnShape g = ln_shape(a.dim, bf16);
    return ln_run(a, bf16, g, false, a.in[1] != nullptr, ln_blocks(g, a.rows, kLnBlocks), s);
}

size_t layer_norm_bwd_workspace(int64_t rows, int dim, int dtype) {
    Carver c(nullptr, (size_t)-1);
    c.take<float>((size_t)ln_blocks(ln_shape(dim, dtype == kDtBF16), rows, kLnBwdBlocks) * 2 * dim);
    return c.off + 256;
}

hipError_t launch_layer_norm_bwd(const LayerNormArgs& args, int dtype, void* ws, hipStream_t s) {
    LayerNormArgs a = args;
    const bool bf16 = dtype == kDtBF16, want = a.dw || a.db;
    const LnShape g = ln_shape(a.dim, bf16);
    const int blocks = ln_blocks(g, a.rows, kLnBwdBlocks);
    Carver c(ws, (size_t)-1);
    float* part = c.take<float>((size_t)blocks * 2 * a.dim);
    a.part = want ? part : nullptr;
    if (blocks > 0) {
        const hipError_t e = ln_run(a, bf16, g, true, a.in[2] != nullptr, blocks, s);
        if (e != hipSuccess) return e;
    }
    if (want) {    // zeros without rows
        a.part = part;
        G2V_LAUNCH(k_layer_norm_sums, dim3((unsigned)ceil_div(2 * a.dim, 16)), dim3(kLnSumThreads), 0, s, a, blocks);
    }
    return hipGetLastError();
}

}  // namespace g2v
