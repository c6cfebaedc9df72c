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
// Bound by bytes: each row is read and written once (forward), or two rows are read and one is written (backward).  A
// workgroup takes a few neighbouring tokens: their sines and cosines are computed once for all heads (a sincosf or a few a
// thread) and go through LDS.  A row is read by a group of 2^shift lanes, 16 bytes a lane; 2^heads_shift neighbouring
// groups take a token's heads in turn, so that a wave reads pieces of a few rows' length each (with all of a token's heads
// walked by one group a wave's loads fell on eight tokens' single rows and moved 2.8 TB/s instead of 4.5), and what belongs
// to the token (its angles, the sum of their gradients over its heads) stays in registers.
#include "../../include/g2v.h"
#include "g2v_internal.h"
#include "g2v_rows.h"

namespace g2v {
namespace {

constexpr int kQnThreads = 256;
constexpr int kQnUnroll = 4;       // rows whose loads a thread has in flight, forward
constexpr int kQnAhead = 1;        // the same, backward (two tensors), the next loaded while one is computed

// A workgroup's side of the problem: queries, keys, or both when they share positions.
struct QnSide {
    int64_t tokens;    // B n
    int n;             // tokens of a scene
    int h0, h1;        // heads, of the query heads followed by the key heads
    const float* pos;
};

__device__ __forceinline__ QnSide qn_side(const QkNormArgs& a, int side) {
    QnSide p;
    p.n = a.n[side];
    p.tokens = (int64_t)a.batch * p.n;
    p.h0 = side ? a.heads[0] : 0;
    p.h1 = a.shared || side ? a.heads[0] + a.heads[1] : a.heads[0];
    p.pos = a.pos[side];
    return p;
}

// Cosine and sine of this lane's pairs of its token (1 and 0 past the table), through LDS: the workgroup's tokens
// [t0, t0 + toks) have them computed once each.  sincosf: its reduction keeps float32 accuracy for any angle (positions in
// metres reach hundreds of radians).
template <int N>
__device__ __forceinline__ void qn_angles(const QkNormArgs& a, const float* positions, int64_t tokens, int64_t t0, int token, int d,
                                          float2* rot, float2 (&f)[N / 2]) {
    const int width = (N / 2) << a.shift, toks = kQnThreads >> (a.shift + a.heads_shift);
    __syncthreads();    // the last tokens' are read
    for (int e = threadIdx.x; e < toks * width; e += kQnThreads) {
        const int t = e / width, i = e - t * width;
        float c = 1.0f, s = 0.0f;
        if (i < a.pairs && t0 + t < tokens) {
            const float* pos = positions + (t0 + t) * a.axes;
            float w = 0.0f;
            for (int x = 0; x < a.axes; ++x) w = fmaf(pos[x], a.freqs[x * a.pairs + i], w);
            sincosf(w, &s, &c);
        }
        rot[e] = make_float2(c, s);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N / 2; ++j) f[j] = rot[token * width + d / 2 + j];
}

// This lane's weights of both tensors (ones without).
template <int N>
__device__ __forceinline__ void qn_weights(const QkNormArgs& a, int d, float (&w)[2][N]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) w[k][j] = a.w[k] && d + j < a.dim ? a.w[k][d + j] : 1.0f;
}

// A thread's place in its workgroup: lane of a row, token, and which of the token's groups it is in.
struct QnPlace {
    int d, token, first, step;
};
template <int N>
__device__ __forceinline__ QnPlace qn_place(const QkNormArgs& a) {
    const int group = threadIdx.x >> a.shift;
    QnPlace o;
    o.d = (threadIdx.x & ((1 << a.shift) - 1)) * N;
    o.step = 1 << a.heads_shift;
    o.token = group >> a.heads_shift;
    o.first = group & (o.step - 1);
    return o;
}

template <typename T, bool AL>
__global__ void __launch_bounds__(kQnThreads) k_qk_norm_rotary(QkNormArgs a) {
    constexpr int N = RowVec<T>::n;
    __shared__ float2 rot[kQnThreads * (N / 2)];
    const int side = blockIdx.x >= a.blocks0;
    const QnSide p = qn_side(a, side);
    const QnPlace o = qn_place<N>(a);
    const int64_t t0 = (int64_t)(blockIdx.x - (side ? a.blocks0 : 0)) * (kQnThreads >> (a.shift + a.heads_shift));
    const bool live = t0 + o.token < p.tokens;
    const int64_t t = live ? t0 + o.token : p.tokens - 1;     // groups past the end repeat the last token, unstored
    const int64_t b = t / p.n, i = t - b * p.n;
    const T* xq = static_cast<const T*>(a.x[0]) + b * a.sb[0] + i * a.sn[0];
    const T* xk = static_cast<const T*>(a.x[1]) + b * a.sb[1] + i * a.sn[1];
    float w[2][N];
    float2 f[N / 2];
    qn_weights<N>(a, o.d, w);
    qn_angles<N>(a, p.pos, p.tokens, t0, o.token, o.d, rot, f);
    const float inv_d = 1.0f / (float)a.dim;
    for (int h0 = p.h0 + o.first; h0 < p.h1; h0 += o.step * kQnUnroll) {
        typename RowVec<T>::raw x[kQnUnroll];
#pragma unroll
        for (int u = 0; u < kQnUnroll; ++u) {
            const int h = h0 + u * o.step;
            const bool k = h >= a.heads[0];
            if (h < p.h1) x[u] = row_load<T, AL>(k ? xk + (h - a.heads[0]) * a.sh[1] : xq + h * a.sh[0], o.d, a.dim);
        }
#pragma unroll
        for (int u = 0; u < kQnUnroll; ++u) {
            const int h = h0 + u * o.step;   // the same for all lanes of a group
            if (h >= p.h1) break;
            const bool k = h >= a.heads[0];
            float ss[1] = {0.0f}, y[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                y[j] = (float)x[u][j];
                ss[0] = fmaf(y[j], y[j], ss[0]);
            }
            row_sums(ss, a.shift);
            const float r = 1.0f / sqrtf(fmaf(ss[0], inv_d, a.eps));
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] *= r * (k ? w[1][j] : w[0][j]);
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const float y0 = y[2 * j], y1 = y[2 * j + 1];
                y[2 * j] = y0 * f[j].x - y1 * f[j].y;
                y[2 * j + 1] = y0 * f[j].y + y1 * f[j].x;
            }
            T* row = k ? static_cast<T*>(a.out[1]) + (t * a.heads[1] + h - a.heads[0]) * a.dim
                       : static_cast<T*>(a.out[0]) + (t * a.heads[0] + h) * a.dim;
            if (live) row_store<T, AL>(row, o.d, a.dim, y);
        }
    }
}

// Workgroups stride over the tokens of one tensor, queries or keys: a workgroup of both holds the addresses, weights and sums
// of both (139 registers instead of 112, and 70 us instead of 60 at 18000 tokens x 16 + 16 heads x 64 bfloat16, 221 MB at
// 3.8 TB/s; two rows ahead 62, five waves a SIMD with spills 74).  A workgroup's sums of dL/dw go to dw_part, and where
// the keys share the queries' positions their parts of dL/dp to a.dpos[1]; k_qk_norm_sums adds those, in a fixed order.  The
// first rows are asked for before the angles.
template <typename T, bool AL>
__global__ void __launch_bounds__(kQnThreads) k_qk_norm_rotary_bwd(QkNormArgs a) {
    constexpr int N = RowVec<T>::n;
    __shared__ float red[kQnThreads * N];
    float2* rot = reinterpret_cast<float2*>(red);
    __shared__ float dcell[kQnThreads * kQnAxes];
    const int k = blockIdx.x >= a.blocks0;
    const QnPlace o = qn_place<N>(a);
    const int toks = kQnThreads >> (a.shift + a.heads_shift), heads = a.heads[k];
    const int blk = blockIdx.x - (k ? a.blocks0 : 0), nblk = k ? gridDim.x - a.blocks0 : a.blocks0;
    const int64_t tokens = (int64_t)a.batch * a.n[k], sh = a.sh[k], gsh = a.gsh[k];
    const float* pos = a.pos[a.shared ? 0 : k];
    const float* weight = a.w[k];
    const float inv_d = 1.0f / (float)a.dim;
    float* dpos = a.dpos[k];
    float w[N], dw[N];
    float2 f[N / 2];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        w[j] = weight && o.d + j < a.dim ? weight[o.d + j] : 1.0f;
        dw[j] = 0.0f;
    }
    for (int64_t t0 = (int64_t)blk * toks; t0 < tokens; t0 += (int64_t)nblk * toks) {
        const bool live = t0 + o.token < tokens;
        const int64_t t = live ? t0 + o.token : tokens - 1;   // groups past the end repeat the last token, unstored
        const int64_t b = t / a.n[k], i = t - b * a.n[k];
        const T* x0 = static_cast<const T*>(a.x[k]) + b * a.sb[k] + i * a.sn[k];
        const T* g0 = static_cast<const T*>(a.g[k]) + b * a.gsb[k] + i * a.gsn[k];
        T* row = static_cast<T*>(a.dx[k]) + t * heads * a.dim;
        typename RowVec<T>::raw xv[kQnAhead], gv[kQnAhead];
        float dth[N / 2];
#pragma unroll
        for (int j = 0; j < N / 2; ++j) dth[j] = 0.0f;
#pragma unroll
        for (int u = 0; u < kQnAhead; ++u) {
            const int h = o.first + u * o.step;
            if (h >= heads) break;
            xv[u] = row_load<T, AL>(x0 + h * sh, o.d, a.dim);
            gv[u] = row_load<T, AL>(g0 + h * gsh, o.d, a.dim);
        }
        qn_angles<N>(a, pos, tokens, t0, o.token, o.d, rot, f);
        for (int h0 = o.first; h0 < heads; h0 += o.step * kQnAhead) {
#pragma unroll
            for (int u = 0; u < kQnAhead; ++u) {
                const int h = h0 + u * o.step;   // the same for all lanes of a group
                if (h >= heads) break;
                float x[N], dy[N], s[2] = {0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    x[j] = (float)xv[u][j];
                    dy[j] = live ? (float)gv[u][j] : 0.0f;
                    s[0] = fmaf(x[j], x[j], s[0]);
                }
                const int next = h + o.step * kQnAhead;
                if (next < heads) {
                    xv[u] = row_load<T, AL>(x0 + next * sh, o.d, a.dim);
                    gv[u] = row_load<T, AL>(g0 + next * gsh, o.d, a.dim);
                }
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    const float c = dy[2 * j], d = dy[2 * j + 1];
                    dy[2 * j] = c * f[j].x + d * f[j].y;
                    dy[2 * j + 1] = d * f[j].x - c * f[j].y;
                }
#pragma unroll
                for (int j = 0; j < N; ++j) s[1] = fmaf(w[j] * dy[j], x[j], s[1]);
                row_sums(s, a.shift);
                const float r = 1.0f / sqrtf(fmaf(s[0], inv_d, a.eps));
                const float q = r * r * inv_d * s[1];
                float dx[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float xr = x[j] * r, wdy = w[j] * dy[j];
                    dw[j] = fmaf(dy[j], xr, dw[j]);
                    dx[j] = r * wdy - xr * q;
                    x[j] = w[j] * xr;
                }
#pragma unroll
                for (int j = 0; j < N / 2; ++j) dth[j] += dy[2 * j + 1] * x[2 * j] - dy[2 * j] * x[2 * j + 1];
                if (live) row_store<T, AL>(row + (int64_t)h * a.dim, o.d, a.dim, dx);
            }
        }
        if (dpos) {   // of each of a token's groups, then of the token
            for (int e = 0; e < a.axes; ++e) {
                float v[1] = {0.0f};
#pragma unroll
                for (int j = 0; j < N / 2; ++j)
                    if (o.d / 2 + j < a.pairs) v[0] = fmaf(a.freqs[e * a.pairs + o.d / 2 + j], dth[j], v[0]);
                row_sums(v, a.shift);
                if (o.d == 0) dcell[(threadIdx.x >> a.shift) * a.axes + e] = v[0];
            }
            __syncthreads();
            for (int e = threadIdx.x; e < toks * a.axes; e += kQnThreads) {
                const int tk = e / a.axes;
                float v = 0.0f;
                for (int g = 0; g < o.step; ++g) v += dcell[(tk * o.step + g) * a.axes + e - tk * a.axes];
                if (t0 + tk < tokens) dpos[t0 * a.axes + e] = v;
            }
        }
    }
    if (!a.dw_part) return;
    // the workgroup's sums: lanes of the same elements are 2^shift apart.  Threads / width of them share an element's sum.
    // (N neighbouring lanes read one bank here, for a few reads once a workgroup.)
    const int span = N << a.shift, parts = kQnThreads > span ? kQnThreads / span : 1, slots = kQnThreads >> a.shift;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) red[j * kQnThreads + threadIdx.x] = dw[j];
    __syncthreads();
    for (int c = threadIdx.x; c < span * parts; c += kQnThreads) {
        const int e = c % span;
        float v = 0.0f;
        for (int g = c / span; g < slots; g += parts) v += red[(e % N) * kQnThreads + (g << a.shift) + e / N];
        if (parts == 1) {
            if (e < a.dim) a.dw_part[(int64_t)blockIdx.x * a.dim + e] = v;
        } else {
            dcell[c] = v;
        }
    }
    if (parts == 1) return;
    __syncthreads();
    for (int e = threadIdx.x; e < a.dim; e += kQnThreads) {
        float v = 0.0f;
        for (int g = 0; g < parts; ++g) v += dcell[g * span + e];
        a.dw_part[(int64_t)blockIdx.x * a.dim + e] = v;
    }
}

// dL/dw from the workgroups' parts (`rows` rows, the queries' before the keys'): 16 columns a workgroup, 64 lanes a column,
// a fixed order.  Workgroups from `sums` on add the keys' parts of shared positions to the queries'.
constexpr int kQnSumThreads = 1024;
__global__ void __launch_bounds__(kQnSumThreads) k_qk_norm_sums(QkNormArgs a, int rows, int sums) {
    __shared__ float red[kQnSumThreads];
    if ((int)blockIdx.x >= sums) {
        const int64_t e = (int64_t)(blockIdx.x - sums) * kQnSumThreads + threadIdx.x;
        if (e < (int64_t)a.batch * a.n[0] * a.axes) a.dpos[0][e] += a.dpos[1][e];
        return;
    }
    const int cols = 2 * a.dim;
    const int col = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
    const int k = col >= a.dim, e = k ? col - a.dim : col;
    const int last = k ? rows : a.blocks0;
    float v = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (int r = (k ? a.blocks0 : 0) + part; r < last; r += 64) v += a.dw_part[(int64_t)r * a.dim + e];
    }
    red[threadIdx.x] = v;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (part < o) red[threadIdx.x] += red[threadIdx.x + 16 * o];
        __syncthreads();
    }
    if (part == 0 && col < cols) {
        float* dst = k ? a.dw[1] : a.dw[0];
        if (dst) dst[e] = red[threadIdx.x];
    }
}

template <typename T>
bool qn_aligned(const QkNormArgs& a, bool backward) {
    const int64_t n = RowVec<T>::n;
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

constexpr int kQnWant = 2048;   // workgroups that fill the card (8 waves a SIMD)

// Lanes of a row and groups of a token (as shifts), and workgroups of each side.  A token's groups read neighbouring
// rows: as many as make 512 bytes, more where the tokens would not fill the card, never more than heads.
struct QnGrid {
    int shift, heads_shift, blocks[2];
};
QnGrid qn_grid(const QkNormArgs& a, bool bf16, bool backward) {
    QnGrid g;
    const int lanes = (int)ceil_div(a.dim, bf16 ? 8 : 4);
    g.shift = 0;
    while ((1 << g.shift) < lanes) ++g.shift;
    const bool both = a.shared && !backward;     // a workgroup's tokens have queries and keys
    const int heads = both ? a.heads[0] + a.heads[1] : std::max(a.heads[0], a.heads[1]);
    const int64_t t[2] = {a.heads[0] + (a.shared ? a.heads[1] : 0) > 0 ? (int64_t)a.batch * a.n[0] : 0,
                          both || a.heads[1] == 0 ? 0 : (int64_t)a.batch * a.n[1]};
    auto blocks = [&](int side) { return ceil_div(t[side], kQnThreads >> (g.shift + g.heads_shift)); };
    const int row = a.dim * (bf16 ? 2 : 4);
    g.heads_shift = 0;
    while (g.shift + g.heads_shift < 8 && (1 << g.heads_shift) < heads && ((row << g.heads_shift) < 512 || blocks(0) + blocks(1) < kQnWant))
        ++g.heads_shift;
    for (int k = 0; k < 2; ++k) {
        g.blocks[k] = (int)blocks(k);
        if (backward && g.blocks[k] > kQnBwdBlocks) g.blocks[k] = kQnBwdBlocks;
    }
    return g;
}

}  // namespace

hipError_t launch_qk_norm_rotary(const QkNormArgs& args, int dtype, hipStream_t s) {
    QkNormArgs a = args;
    const bool bf16 = dtype == kDtBF16;
    const QnGrid g = qn_grid(a, bf16, false);
    a.shift = g.shift;
    a.heads_shift = g.heads_shift;
    a.blocks0 = g.blocks[0];
    const dim3 grid(g.blocks[0] + g.blocks[1]), block(kQnThreads);
    if (grid.x == 0) return hipSuccess;
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
    c.take<float>((size_t)(g.blocks[0] + g.blocks[1]) * a.dim);
    if (a.shared) c.take<float>((size_t)a.batch * a.n[1] * a.axes);
    return c.off + 256;
}

hipError_t launch_qk_norm_rotary_bwd(const QkNormArgs& args, int dtype, void* ws, hipStream_t s) {
    QkNormArgs a = args;
    const bool bf16 = dtype == kDtBF16;
    const QnGrid g = qn_grid(a, bf16, true);
    a.shift = g.shift;
    a.heads_shift = g.heads_shift;
    a.blocks0 = g.blocks[0];
    const bool want_w = a.dw[0] || a.dw[1];
    const dim3 grid(g.blocks[0] + g.blocks[1]), block(kQnThreads);
    Carver c(ws, (size_t)-1);
    float* part = c.take<float>((size_t)grid.x * a.dim);
    a.dw_part = want_w ? part : nullptr;
    const bool add_pos = a.shared && a.dpos[0] && g.blocks[1] > 0;
    if (a.shared) a.dpos[1] = add_pos ? c.take<float>((size_t)a.batch * a.n[1] * a.axes) : nullptr;
    if (grid.x > 0) {
        if (bf16) {
            if (qn_aligned<__bf16>(a, true)) G2V_LAUNCH((k_qk_norm_rotary_bwd<__bf16, true>), grid, block, 0, s, a);
            else G2V_LAUNCH((k_qk_norm_rotary_bwd<__bf16, false>), grid, block, 0, s, a);
        } else {
            if (qn_aligned<float>(a, true)) G2V_LAUNCH((k_qk_norm_rotary_bwd<float, true>), grid, block, 0, s, a);
            else G2V_LAUNCH((k_qk_norm_rotary_bwd<float, false>), grid, block, 0, s, a);
        }
    }
    const int sums = want_w ? (int)ceil_div(2 * a.dim, 16) : 0;
    const int adds = add_pos ? (int)ceil_div((int64_t)a.batch * a.n[0] * a.axes, kQnSumThreads) : 0;
    if (sums + adds > 0)
        G2V_LAUNCH(k_qk_norm_sums, dim3((unsigned)(sums + adds)), dim3(kQnSumThreads), 0, s, a, (int)grid.x, sums);
    return hipGetLastError();
}

}  // namespace g2v
