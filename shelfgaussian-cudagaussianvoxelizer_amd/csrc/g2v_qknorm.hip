// Norms of queries and keys for each head, with the rotation by the tokens' positions in the same pass, and its
// backward.  A row is one head of one token: x (D), weight w (D, of queries or of keys), position p (axes), table
// F (axes x P), P <= D / 2:
//
//   r = (mean x^2 + eps)^-1/2,  y = w x r,  theta_i = sum_a p_a F[a][i],
//   o_2i = y_2i cos - y_2i+1 sin,  o_2i+1 = y_2i sin + y_2i+1 cos  (i < P),  o_d = y_d beyond 2P.
//
// Backward, from g = dL/do, with dy = the rotation by -theta of g:
//   dL/dw = sum over rows of dy x r,   dL/dx = r (w dy) - x r^3 / D sum(w dy x),
//   dL/dtheta_i = sum over the token's heads of dy_2i+1 y_2i - dy_2i y_2i+1  (a cross product: the same before and
//   after the rotation),   dL/dp_a = sum_i F[a][i] dL/dtheta_i.
//
// Bound by bytes: each row is read and written once (forward) or two rows read and one written (backward).  A token
// takes 2^shift neighbouring lanes of a wave, 16 bytes of its row each, and walks its heads: the sines, cosines and the
// sums over heads (dtheta, dw) stay in the lanes that need them.
#include "../../include/g2v.h"
#include "g2v_internal.h"

namespace g2v {
namespace {

constexpr int kQnThreads = 256;
constexpr int kQnUnroll = 4;       // heads whose loads are in flight together

template <typename T>
struct QnVec;
template <>
struct QnVec<float> {
    static constexpr int n = 4;
    typedef f32x4 raw;
};
template <>
struct QnVec<__bf16> {
    static constexpr int n = 8;
    typedef bf16x8 raw;
};

// Elements [d, d + n) of a row, zero past the end.
template <typename T, bool AL>
__device__ __forceinline__ typename QnVec<T>::raw qn_load(const T* row, int d, int D) {
    typename QnVec<T>::raw v;
    if constexpr (AL) {
        if (d < D) v = *reinterpret_cast<const typename QnVec<T>::raw*>(row + d);
        else
#pragma unroll
            for (int j = 0; j < QnVec<T>::n; ++j) v[j] = (T)0.0f;
    } else {
#pragma unroll
        for (int j = 0; j < QnVec<T>::n; ++j) v[j] = d + j < D ? row[d + j] : (T)0.0f;
    }
    return v;
}
// AL: the vector is stored whole (row and D are multiples of its 16 bytes).
template <typename T, bool AL>
__device__ __forceinline__ void qn_store(T* row, int d, int D, const float (&o)[QnVec<T>::n]) {
    constexpr int n = QnVec<T>::n;
    if constexpr (AL) {
        typename QnVec<T>::raw v;
#pragma unroll
        for (int j = 0; j < n; ++j) v[j] = (T)o[j];
        if (d < D) *reinterpret_cast<typename QnVec<T>::raw*>(row + d) = v;
    } else {
#pragma unroll
        for (int j = 0; j < n; ++j)
            if (d + j < D) row[d + j] = (T)o[j];
    }
}

// Sum over the 2^shift lanes of a token.
__device__ __forceinline__ float token_sum(float v, int shift) {
    for (int m = (1 << shift) >> 1; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// A workgroup's part of the problem: which tokens' side (queries, keys, or both when they share positions).
struct QnPart {
    int64_t tokens;    // B n
    int n;             // tokens of a scene
    int h0, h1;        // heads, of the heads_q query heads followed by the heads_k key heads
    const float* pos;
};

__device__ __forceinline__ QnPart qn_part(const QkNormArgs& a, int side) {
    QnPart p;
    const int all = a.heads[0] + a.heads[1];
    p.n = a.n[side];
    p.tokens = (int64_t)a.batch * p.n;
    p.h0 = side ? a.heads[0] : 0;
    p.h1 = a.shared || side ? all : a.heads[0];
    p.pos = a.pos[side];
    return p;
}

// Sines and cosines of this lane's pairs; 0 and 1 past the table.  sincosf: its reduction keeps float32
// accuracy for any angle (positions in metres reach hundreds of radians).
template <int N>
__device__ __forceinline__ void qn_angles(const QkNormArgs& a, const float* pos, int d, float (&c)[N], float (&s)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int i = d / 2 + j;
        c[j] = 1.0f;
        s[j] = 0.0f;
        if (i < a.pairs) {
            float t = 0.0f;
            for (int x = 0; x < a.axes; ++x) t = fmaf(pos[x], a.freqs[x * a.pairs + i], t);
            sincosf(t, &s[j], &c[j]);
        }
    }
}

template <typename T, bool AL>
__global__ void __launch_bounds__(kQnThreads) k_qk_norm_rotary(QkNormArgs a) {
    constexpr int N = QnVec<T>::n;
    const int side = blockIdx.x >= a.blocks0;
    const QnPart p = qn_part(a, side);
    const int lane = threadIdx.x & 63, slots = kQnThreads >> a.shift;
    const int d = (lane & ((1 << a.shift) - 1)) * N;
    const int64_t tok = (int64_t)(blockIdx.x - (side ? a.blocks0 : 0)) * slots + (threadIdx.x >> a.shift);
    const int64_t t = tok < p.tokens ? tok : p.tokens - 1;      // lanes past the end repeat the last token, unstored
    const int64_t b = t / p.n, i = t - b * p.n;
    float c[N / 2], s[N / 2];
    qn_angles(a, p.pos + t * a.axes, d, c, s);
    const int hb = p.h0 + (int)blockIdx.y * a.chunk;
    const int he = hb + a.chunk < p.h1 ? hb + a.chunk : p.h1;
    const float inv_d = 1.0f / (float)a.dim;
    for (int h0 = hb; h0 < he; h0 += kQnUnroll) {
        typename QnVec<T>::raw x[kQnUnroll];
#pragma unroll
        for (int u = 0; u < kQnUnroll; ++u) {
            const int h = h0 + u < he ? h0 + u : he - 1, k = h >= a.heads[0];
            const T* row = static_cast<const T*>(a.x[k]) + b * a.sb[k] + i * a.sn[k] +
                           (int64_t)(h - (k ? a.heads[0] : 0)) * a.sh[k];
            x[u] = qn_load<T, AL>(row, d, a.dim);
        }
#pragma unroll
        for (int u = 0; u < kQnUnroll; ++u) {
            if (h0 + u >= he) break;
            const int h = h0 + u, k = h >= a.heads[0];
            float ss = 0.0f, y[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                y[j] = (float)x[u][j];
                ss = fmaf(y[j], y[j], ss);
            }
            const float r = 1.0f / sqrtf(fmaf(token_sum(ss, a.shift), inv_d, a.eps));
            const float* w = a.w[k];
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] *= r * (w ? (d + j < a.dim ? w[d + j] : 0.0f) : 1.0f);
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const float y0 = y[2 * j], y1 = y[2 * j + 1];
                y[2 * j] = y0 * c[j] - y1 * s[j];
                y[2 * j + 1] = y0 * s[j] + y1 * c[j];
            }
            T* row = static_cast<T*>(a.out[k]) + (t * a.heads[k] + (h - (k ? a.heads[0] : 0))) * a.dim;
            if (tok < p.tokens) qn_store<T, AL>(row, d, a.dim, y);
        }
    }
}

// Workgroups stride over the tokens of their side; a workgroup's sums of dL/dw go to dw_part, a head chunk's position
// gradients to dpos_part (k_qk_norm_sums adds both in a fixed order).
template <typename T, bool AL>
__global__ void __launch_bounds__(kQnThreads) k_qk_norm_rotary_bwd(QkNormArgs a) {
    constexpr int N = QnVec<T>::n;
    __shared__ float red[kQnThreads * N];
    const int side = blockIdx.x >= a.blocks0;
    const QnPart p = qn_part(a, side);
    const int lane = threadIdx.x & 63, slots = kQnThreads >> a.shift;
    const int d = (lane & ((1 << a.shift) - 1)) * N;
    const int blk = blockIdx.x - (side ? a.blocks0 : 0), nblk = side ? gridDim.x - a.blocks0 : a.blocks0;
    const int hb = p.h0 + (int)blockIdx.y * a.chunk;
    const int he = hb + a.chunk < p.h1 ? hb + a.chunk : p.h1;
    const float inv_d = 1.0f / (float)a.dim;
    float dw[2][N];
#pragma unroll
    for (int j = 0; j < N; ++j) dw[0][j] = dw[1][j] = 0.0f;
    for (int64_t t0 = (int64_t)blk * slots; t0 < p.tokens; t0 += (int64_t)nblk * slots) {
        const int64_t tok = t0 + (threadIdx.x >> a.shift);
        const bool live = tok < p.tokens;
        const int64_t t = live ? tok : p.tokens - 1;
        const int64_t b = t / p.n, i = t - b * p.n;
        float c[N / 2], s[N / 2], dth[N / 2];
        qn_angles(a, p.pos + t * a.axes, d, c, s);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) dth[j] = 0.0f;
        for (int h = hb; h < he; ++h) {
            const int k = h >= a.heads[0], hk = h - (k ? a.heads[0] : 0);
            const T* xr = static_cast<const T*>(a.x[k]) + b * a.sb[k] + i * a.sn[k] + (int64_t)hk * a.sh[k];
            const T* gr = static_cast<const T*>(a.g[k]) + b * a.gsb[k] + i * a.gsn[k] + (int64_t)hk * a.gsh[k];
            const auto xv = qn_load<T, AL>(xr, d, a.dim);
            const auto gv = qn_load<T, AL>(gr, d, a.dim);
            const float* w = a.w[k];
            float x[N], dy[N], wv[N], ss = 0.0f, st = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[j] = (float)xv[j];
                dy[j] = live ? (float)gv[j] : 0.0f;
                wv[j] = w ? (d + j < a.dim ? w[d + j] : 0.0f) : 1.0f;
                ss = fmaf(x[j], x[j], ss);
            }
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const float g0 = dy[2 * j], g1 = dy[2 * j + 1];
                dy[2 * j] = g0 * c[j] + g1 * s[j];
                dy[2 * j + 1] = g1 * c[j] - g0 * s[j];
            }
#pragma unroll
            for (int j = 0; j < N; ++j) st = fmaf(wv[j] * dy[j], x[j], st);
            ss = token_sum(ss, a.shift);
            st = token_sum(st, a.shift);
            const float r = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
            const float q = r * r * r * inv_d * st;
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const float y0 = wv[2 * j] * x[2 * j] * r, y1 = wv[2 * j + 1] * x[2 * j + 1] * r;
                dth[j] += dy[2 * j + 1] * y0 - dy[2 * j] * y1;
            }
            float dx[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float z = dy[j] * x[j] * r;
                if (k) dw[1][j] += z;
                else dw[0][j] += z;
                dx[j] = r * wv[j] * dy[j] - x[j] * q;
            }
            T* row = static_cast<T*>(a.dx[k]) + (t * a.heads[k] + hk) * a.dim;
            if (live) qn_store<T, AL>(row, d, a.dim, dx);
        }
        if (a.dpos_part) {
            float* out = a.dpos_part + ((int64_t)blockIdx.y * a.dpos_tokens + (side ? (int64_t)a.batch * a.n[0] : 0) + t) * a.axes;
            for (int x = 0; x < a.axes; ++x) {
                float v = 0.0f;
#pragma unroll
                for (int j = 0; j < N / 2; ++j)
                    if (d / 2 + j < a.pairs) v = fmaf(a.freqs[x * a.pairs + d / 2 + j], dth[j], v);
                v = token_sum(v, a.shift);
                if (live && d == 0) out[x] = v;
            }
        }
    }
    if (!a.dw_part) return;
    // the workgroup's sums: lanes of the same elements are 2^shift apart
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) red[j * kQnThreads + threadIdx.x] = dw[k][j];
        __syncthreads();
        const int width = N << a.shift;
        for (int e = threadIdx.x; e < width; e += kQnThreads) {
            float v = 0.0f;
            for (int o = 0; o < slots; ++o) v += red[(e % N) * kQnThreads + (o << a.shift) + e / N];
            if (e < a.dim)
                a.dw_part[(((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + k) * a.dim + e] = v;
        }
    }
}

// Sums of `rows` rows of `cols` values into out (cols), each column by 16 lanes in a fixed order.
__global__ void __launch_bounds__(kQnThreads) k_qk_norm_sums(QkNormArgs a, int64_t rows, int col_blocks, int chunks) {
    if ((int)blockIdx.x < col_blocks) {   // dL/dw of queries and keys, side by side
        __shared__ float red[kQnThreads];
        const int cols = 2 * a.dim;
        const int col = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
        float v = 0.0f;
        if (col < cols)
            for (int64_t r = part; r < rows; r += 16) v += a.dw_part[r * cols + col];
        red[threadIdx.x] = v;
        __syncthreads();
        if (part == 0 && col < cols) {
            for (int o = 1; o < 16; ++o) v += red[o * 16 + (threadIdx.x & 15)];
            float* dst = a.dw[col >= a.dim];
            if (dst) dst[col >= a.dim ? col - a.dim : col] = v;
        }
        return;
    }
    const int64_t e = (int64_t)(blockIdx.x - col_blocks) * kQnThreads + threadIdx.x;
    const int64_t nq = (int64_t)a.batch * a.n[0] * a.axes, all = a.dpos_tokens * a.axes;
    if (e >= all) return;
    float v = 0.0f;
    for (int y = 0; y < chunks; ++y) v += a.dpos_part[y * all + e];
    float* dst = a.dpos[e >= nq];
    if (dst) dst[e >= nq ? e - nq : e] = v;
}

template <typename T>
bool qn_aligned(const QkNormArgs& a, bool backward) {
    const int64_t n = QnVec<T>::n;
    bool ok = a.dim % n == 0;
    auto row = [&](const void* p, const int64_t* s) {
        if (!p) return;
        ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
        if (s) ok = ok && s[0] % n == 0 && s[1] % n == 0 && s[2] % n == 0;
    };
    for (int k = 0; k < 2; ++k) {
        const int64_t sx[3] = {a.sb[k], a.sn[k], a.sh[k]}, sg[3] = {a.gsb[k], a.gsn[k], a.gsh[k]};
        row(a.x[k], sx);
        if (backward) {
            row(a.g[k], sg);
            row(a.dx[k], nullptr);
        } else {
            row(a.out[k], nullptr);
        }
    }
    return ok;
}

// Lanes of a token (as a shift), heads of a workgroup and workgroups along the tokens.  A token's lanes cover its row
// with 16 bytes each; heads are dealt to several workgroups only while the tokens alone leave most SIMDs without a wave.
struct QnGrid {
    int shift, chunk, chunks, blocks[2];
};
QnGrid qn_grid(const QkNormArgs& a, bool bf16, bool backward) {
    QnGrid g;
    const int lanes = (int)ceil_div(a.dim, bf16 ? 8 : 4);
    g.shift = 0;
    while ((1 << g.shift) < lanes) ++g.shift;
    const int slots = kQnThreads >> g.shift;
    const int most = a.shared ? a.heads[0] + a.heads[1] : (a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1]);
    const int64_t t[2] = {(int64_t)a.batch * a.n[0], a.shared ? 0 : (int64_t)a.batch * a.n[1]};
    int64_t blocks = 0;
    for (int k = 0; k < 2; ++k) {
        g.blocks[k] = (int)ceil_div(t[k], slots);
        if (backward && g.blocks[k] > kQnBwdBlocks) g.blocks[k] = kQnBwdBlocks;
        blocks += g.blocks[k];
    }
    g.chunk = most;
    while (g.chunk > kQnUnroll && blocks * ceil_div(most, g.chunk) < 1024) g.chunk = (int)ceil_div(g.chunk, 2);
    g.chunks = g.chunk > 0 ? (int)ceil_div(most, g.chunk) : 0;
    return g;
}

}  // namespace

hipError_t launch_qk_norm_rotary(const QkNormArgs& args, int dtype, hipStream_t s) {
    QkNormArgs a = args;
    const bool bf16 = dtype == kDtBF16;
    const QnGrid g = qn_grid(a, bf16, false);
    const int blocks = g.blocks[0] + g.blocks[1];
    if (blocks == 0 || g.chunks == 0) return hipSuccess;
    a.shift = g.shift;
    a.chunk = g.chunk;
    a.blocks0 = g.blocks[0];
    const dim3 grid(blocks, g.chunks), block(kQnThreads);
    if (bf16) {
        if (qn_aligned<__bf16>(a, false)) G2V_LAUNCH((k_qk_norm_rotary<__bf16, true>), grid, block, 0, s, a);
        else G2V_LAUNCH((k_qk_norm_rotary<__bf16, false>), grid, block, 0, s, a);
    } else {
        if (qn_aligned<float>(a, false)) G2V_LAUNCH((k_qk_norm_rotary<float, true>), grid, block, 0, s, a);
        else G2V_LAUNCH((k_qk_norm_rotary<float, false>), grid, block, 0, s, a);
    }
    return hipGetLastError();
}

size_t qk_norm_bwd_workspace(const QkNormArgs& a, int dtype) {
    const QnGrid g = qn_grid(a, dtype == kDtBF16, true);
    Carver c(nullptr, (size_t)-1);
    c.take<float>((size_t)(g.blocks[0] + g.blocks[1]) * g.chunks * 2 * a.dim);
    c.take<float>((size_t)g.chunks * a.batch * ((size_t)a.n[0] + (a.shared ? 0 : a.n[1])) * a.axes);
    return c.off + 256;
}

hipError_t launch_qk_norm_rotary_bwd(const QkNormArgs& args, int dtype, void* ws, hipStream_t s) {
    QkNormArgs a = args;
    const bool bf16 = dtype == kDtBF16;
    const QnGrid g = qn_grid(a, bf16, true);
    const int blocks = g.blocks[0] + g.blocks[1];
    a.shift = g.shift;
    a.chunk = g.chunk;
    a.blocks0 = g.blocks[0];
    a.dpos_tokens = (int64_t)a.batch * ((int64_t)a.n[0] + (a.shared ? 0 : a.n[1]));
    Carver c(ws, (size_t)-1);
    float* wp = c.take<float>((size_t)blocks * g.chunks * 2 * a.dim);
    float* pp = c.take<float>((size_t)g.chunks * a.dpos_tokens * a.axes);
    const bool want_w = a.dw[0] || a.dw[1], want_p = a.dpos[0] || a.dpos[1];
    a.dw_part = want_w ? wp : nullptr;
    a.dpos_part = want_p ? pp : nullptr;
    if (blocks > 0 && g.chunks > 0) {
        const dim3 grid(blocks, g.chunks), block(kQnThreads);
        if (bf16) {
            if (qn_aligned<__bf16>(a, true)) G2V_LAUNCH((k_qk_norm_rotary_bwd<__bf16, true>), grid, block, 0, s, a);
            else G2V_LAUNCH((k_qk_norm_rotary_bwd<__bf16, false>), grid, block, 0, s, a);
        } else {
            if (qn_aligned<float>(a, true)) G2V_LAUNCH((k_qk_norm_rotary_bwd<float, true>), grid, block, 0, s, a);
            else G2V_LAUNCH((k_qk_norm_rotary_bwd<float, false>), grid, block, 0, s, a);
        }
    }
    const int col_blocks = want_w ? (int)ceil_div(2 * a.dim, 16) : 0;
    const int64_t pos_blocks = want_p ? ceil_div(a.dpos_tokens * a.axes, kQnThreads) : 0;
    if (col_blocks + pos_blocks > 0)
        G2V_LAUNCH(k_qk_norm_sums, dim3((unsigned)(col_blocks + pos_blocks)), dim3(kQnThreads), 0, s, a,
                   (int64_t)blocks * g.chunks, col_blocks, g.chunks);
    return hipGetLastError();
}

}  // namespace g2v
