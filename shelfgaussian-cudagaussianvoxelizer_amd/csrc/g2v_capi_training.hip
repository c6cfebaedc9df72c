// C ABI of what stands between a deep stack's layers and at the end of its training step (declared in include/g2v.h): argument
// checks and launches of the layer norm and of the gradients' norm and clipping.
#include <math.h>
#include <algorithm>
#include <new>
#include <vector>

#include "../../include/g2v.h"
#include "g2v_internal.h"

using namespace g2v;

namespace {

#define G2V_HIP(call)                                                                                        \
    do {                                                                                                     \
        hipError_t e_ = (call);                                                                              \
        if (e_ != hipSuccess) return api_fail(G2V_ERR_HIP, "%s: %s", #call, hipGetErrorString(e_));          \
    } while (0)

bool is_dtype(int dtype) { return dtype == G2V_DTYPE_F32 || dtype == G2V_DTYPE_BF16; }

int ln_sizes(int batch, int n, int channels, int dtype) {
    if (batch < 0 || n < 0) return api_fail(G2V_ERR_INVALID, "negative size: batch %d, n %d", batch, n);
    if (channels < 1 || channels > 8192) return api_fail(G2V_ERR_INVALID, "channels = %d (1 to 8192)", channels);
    if (!is_dtype(dtype)) return api_fail(G2V_ERR_INVALID, "dtype = %d (G2V_DTYPE_F32 or G2V_DTYPE_BF16)", dtype);
    return G2V_OK;
}

void ln_input(LayerNormArgs& a, int k, const void* p, const long long* strides) {
    a.in[k] = p;
    a.sb[k] = p ? strides[0] : 0;
    a.sn[k] = p ? strides[1] : 0;
}

// Whether an output shares memory with another output, or with a gradient other than its own at its own place and type: workgroups
// would write what others read.  The two tensors in a, b (negative: no memory to look).
bool clip_overlap(int count, const void* const* grads, const int* gd, void* const* outs, const int* od, const long long* numels,
                  int& a, int& b) {
    struct Span {
        uintptr_t at, end;
        int tensor;
    };
    auto span = [&](const void* p, int dtype, int i) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        return Span{at, at + (uintptr_t)numels[i] * (dtype == G2V_DTYPE_BF16 ? 2 : 4), i};
    };
    std::vector<Span> w;
    try {
        w.reserve(count);
        for (int i = 0; i < count; ++i)
            if (numels[i] > 0) w.push_back(span(outs[i], od[i], i));
    } catch (const std::bad_alloc&) {
        a = b = -1;
        return true;
    }
    std::sort(w.begin(), w.end(), [](const Span& x, const Span& y) { return x.at < y.at; });
    for (size_t k = 1; k < w.size(); ++k)
        if (w[k].at < w[k - 1].end) {
            a = w[k - 1].tensor;
            b = w[k].tensor;
            return true;
        }
    for (int i = 0; i < count; ++i) {
        if (numels[i] == 0) continue;
        const Span g = span(grads[i], gd[i], i);
        auto k = std::upper_bound(w.begin(), w.end(), g.at, [](uintptr_t at, const Span& x) { return at < x.end; });
        for (; k != w.end() && k->at < g.end; ++k)
            if (k->tensor != i || k->at != g.at || gd[i] != od[i]) {
                a = i;
                b = k->tensor;
                return true;
            }
    }
    return false;
}

}  // namespace

extern "C" {

int g2v_layer_norm_forward(int batch, int n, int channels, const void* x, const long long x_strides[2], const void* residual,
                           const long long residual_strides[2], int dtype, const void* weight, const void* bias,
                           int weight_dtype, float eps, void* y, void* sum, float* stats, void* stream) {
    api_begin();
    const int rc = ln_sizes(batch, n, channels, dtype);
    if (rc != G2V_OK) return rc;
    if (!is_dtype(weight_dtype)) return api_fail(G2V_ERR_INVALID, "weight_dtype = %d (G2V_DTYPE_F32 or G2V_DTYPE_BF16)", weight_dtype);
    if (!(eps >= 0.0f)) return api_fail(G2V_ERR_INVALID, "eps = %g (not negative)", (double)eps);
    LayerNormArgs a = {};
    a.rows = (int64_t)batch * n;
    if (a.rows == 0) return G2V_OK;
    if (!x || !x_strides || !y) return api_fail(G2V_ERR_INVALID, "null x, x_strides or y");
    if (residual && (!residual_strides || !sum)) return api_fail(G2V_ERR_INVALID, "residual without residual_strides or sum");
    a.n = n;
    a.dim = channels;
    ln_input(a, 0, x, x_strides);
    ln_input(a, 1, residual, residual_strides);
    a.w = weight;
    a.b = bias;
    a.wbf16 = weight_dtype == G2V_DTYPE_BF16;
    a.eps = eps;
    a.y = y;
    a.sum = residual ? sum : nullptr;
    a.stats = stats;
    G2V_HIP(launch_layer_norm(a, dtype, static_cast<hipStream_t>(stream)));
    return G2V_OK;
}

size_t g2v_layer_norm_backward_workspace(int batch, int n, int channels, int dtype) {
    if (ln_sizes(batch, n, channels, dtype) != G2V_OK) return 0;
    return layer_norm_bwd_workspace((int64_t)batch * n, channels, dtype);
}

int g2v_layer_norm_backward(int batch, int n, int channels, const void* x, const long long x_strides[2], int dtype,
                            const void* weight, int weight_dtype, const float* stats, const void* grad_y,
                            const long long grad_y_strides[2], const void* grad_sum, const long long grad_sum_strides[2],
                            void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                            void* stream) {
    api_begin();
    const int rc = ln_sizes(batch, n, channels, dtype);
    if (rc != G2V_OK) return rc;
    if (!is_dtype(weight_dtype)) return api_fail(G2V_ERR_INVALID, "weight_dtype = %d (G2V_DTYPE_F32 or G2V_DTYPE_BF16)", weight_dtype);
    LayerNormArgs a = {};
    a.rows = (int64_t)batch * n;
    if (a.rows > 0 && (!x || !x_strides || !stats || !grad_y || !grad_y_strides || !grad_x))
        return api_fail(G2V_ERR_INVALID, "null x, stats, grad_y, grad_x or strides");
    if (a.rows > 0 && grad_sum && !grad_sum_strides) return api_fail(G2V_ERR_INVALID, "grad_sum without grad_sum_strides");
    const size_t need = layer_norm_bwd_workspace(a.rows, channels, dtype);
    if (!workspace || workspace_bytes < need)
        return api_fail(G2V_ERR_INVALID, "workspace too small: %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
    a.n = n;
    a.dim = channels;
    if (a.rows > 0) {
        ln_input(a, 0, x, x_strides);
        ln_input(a, 1, grad_y, grad_y_strides);
        ln_input(a, 2, grad_sum, grad_sum_strides);
    }
    a.w = weight;
    a.wbf16 = weight_dtype == G2V_DTYPE_BF16;
    a.stats = const_cast<float*>(stats);
    a.y = grad_x;
    a.dw = grad_weight;
    a.db = grad_bias;
    G2V_HIP(launch_layer_norm_bwd(a, dtype, workspace, static_cast<hipStream_t>(stream)));
    return G2V_OK;
}

size_t g2v_clip_gradients_workspace(int count) { return count < 0 ? 0 : clip_workspace(count); }

int g2v_clip_gradients(int count, const void* const* grads, const int* grad_dtypes, void* const* outs, const int* out_dtypes,
                       const long long* numels, float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                       void* stream) {
    api_begin();
    if (count < 0) return api_fail(G2V_ERR_INVALID, "negative count %d", count);
    if (!(max_norm >= 0.0f)) return api_fail(G2V_ERR_INVALID, "max_norm = %g (not negative)", (double)max_norm);
    if (!norm) return api_fail(G2V_ERR_INVALID, "null norm");
    if (count > 0 && (!grads || !grad_dtypes || !outs || !out_dtypes || !numels)) return api_fail(G2V_ERR_INVALID, "null arrays");
    for (int i = 0; i < count; ++i) {
        if (numels[i] < 0 || numels[i] >= 1ll << 40) return api_fail(G2V_ERR_INVALID, "tensor %d has %lld elements", i, numels[i]);
        if (!is_dtype(grad_dtypes[i]) || !is_dtype(out_dtypes[i]))
            return api_fail(G2V_ERR_INVALID, "tensor %d: dtype %d / %d (G2V_DTYPE_F32 or G2V_DTYPE_BF16)", i, grad_dtypes[i],
                            out_dtypes[i]);
        if (numels[i] > 0 && (!grads[i] || !outs[i])) return api_fail(G2V_ERR_INVALID, "tensor %d: null pointer", i);
    }
    const size_t need = clip_workspace(count);
    if (!workspace || workspace_bytes < need)
        return api_fail(G2V_ERR_INVALID, "workspace too small: %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
    static_assert(sizeof(long long) == sizeof(int64_t), "64-bit sizes");
    int a, b;
    if (clip_overlap(count, grads, grad_dtypes, outs, out_dtypes, numels, a, b)) {
        if (a < 0) return api_fail(G2V_ERR_HIP, "out of host memory");
        return api_fail(G2V_ERR_INVALID, "tensors %d and %d share memory that is written", a, b);
    }
    G2V_HIP(launch_clip(count, grads, outs, reinterpret_cast<const int64_t*>(numels), grad_dtypes, out_dtypes, max_norm, norm,
                        workspace, static_cast<hipStream_t>(stream)));
    return G2V_OK;
}

}  // extern "C"
