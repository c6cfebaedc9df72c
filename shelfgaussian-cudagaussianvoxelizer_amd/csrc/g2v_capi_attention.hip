// C ABI of the operators in front of the splat (declared in include/g2v.h): argument checks, workspaces and launches of
// the query/key norms with rotary positions and of the attention.
#include <limits.h>
#include <math.h>

#include "../../include/g2v.h"
#include "g2v_internal.h"

using namespace g2v;

namespace {

#define G2V_HIP(call)                                                                                        \
    do {                                                                                                     \
        hipError_t e_ = (call);                                                                              \
        if (e_ != hipSuccess) return api_fail(G2V_ERR_HIP, "%s: %s", #call, hipGetErrorString(e_));          \
    } while (0)

int qn_sizes(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int num_axes, int num_pairs, int dtype,
             bool shared) {
    if (batch < 0 || n_q < 0 || n_k < 0 || heads_q < 0 || heads_k < 0)
        return api_fail(G2V_ERR_INVALID, "negative size: batch %d, n %d / %d, heads %d / %d", batch, n_q, n_k, heads_q, heads_k);
    if (head_dim < 1 || head_dim > 256) return api_fail(G2V_ERR_INVALID, "head_dim = %d (1 to 256)", head_dim);
    if (num_axes < 1 || num_axes > 8) return api_fail(G2V_ERR_INVALID, "num_axes = %d (1 to 8)", num_axes);
    if (num_pairs < 0 || 2 * num_pairs > head_dim)
        return api_fail(G2V_ERR_INVALID, "num_pairs = %d (0 to head_dim / 2 = %d)", num_pairs, head_dim / 2);
    if (dtype != G2V_DTYPE_F32 && dtype != G2V_DTYPE_BF16)
        return api_fail(G2V_ERR_INVALID, "dtype = %d (G2V_DTYPE_F32 or G2V_DTYPE_BF16)", dtype);
    if (shared && heads_k > 0 && n_k != n_q)
        return api_fail(G2V_ERR_INVALID, "shared positions need n_k == n_q, got %d and %d", n_k, n_q);
    // workgroups along the tokens are counted in 32 bits
    if ((double)batch * n_q > 1e9 || (double)batch * n_k > 1e9 || heads_q > 65536 || heads_k > 65536)
        return api_fail(G2V_ERR_LIMIT, "batch %d x n %d / %d tokens (limit 1e9), heads %d / %d (limit 65536)", batch, n_q, n_k,
                        heads_q, heads_k);
    return G2V_OK;
}

QkNormArgs qn_args(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int num_axes, int num_pairs,
                   bool shared) {
    QkNormArgs a = {};
    a.batch = batch;
    a.n[0] = n_q;
    a.n[1] = heads_k > 0 ? n_k : 0;
    a.heads[0] = heads_q;
    a.heads[1] = heads_k;
    a.dim = head_dim;
    a.axes = num_axes;
    a.pairs = num_pairs;
    a.shared = shared || heads_k == 0;
    if (heads_q == 0 && !a.shared) a.n[0] = 0;
    return a;
}

int qn_fill(QkNormArgs& a, const void* q, const long long* qs, const void* k, const long long* ks, const float* qw,
            const float* kw, const float* qp, const float* kp, const float* freqs, float eps) {
    const bool rows_q = (int64_t)a.batch * a.n[0] * a.heads[0] > 0, rows_k = (int64_t)a.batch * a.n[1] * a.heads[1] > 0;
    if ((rows_q && (!q || !qs || !qp)) || (rows_k && (!k || !ks || !(kp || qp))))
        return api_fail(G2V_ERR_INVALID, "null q / k, strides or positions");
    if ((rows_q || rows_k) && a.pairs > 0 && !freqs) return api_fail(G2V_ERR_INVALID, "null freqs");
    if (!(eps >= 0.0f)) return api_fail(G2V_ERR_INVALID, "eps = %g (not negative)", (double)eps);
    a.x[0] = q;
    a.x[1] = k;
    for (int i = 0; i < 2; ++i) {
        const long long* s = i ? ks : qs;
        a.sb[i] = s ? s[0] : 0;
        a.sn[i] = s ? s[1] : 0;
        a.sh[i] = s ? s[2] : 0;
    }
    a.w[0] = qw;
    a.w[1] = kw;
    a.pos[0] = qp;
    a.pos[1] = kp;
    a.freqs = freqs;
    a.eps = eps;
    return G2V_OK;
}

}  // namespace

extern "C" {

int g2v_qk_norm_rotary_forward(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int num_axes,
                               int num_pairs, const void* q, const long long q_strides[3], const void* k,
                               const long long k_strides[3], int dtype, const float* q_weight, const float* k_weight,
                               const float* q_positions, const float* k_positions, const float* freqs, float eps,
                               void* q_out, void* k_out, void* stream) {
    api_begin();
    int rc = qn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, num_axes, num_pairs, dtype, !k_positions);
    if (rc != G2V_OK) return rc;
    QkNormArgs a = qn_args(batch, n_q, n_k, heads_q, heads_k, head_dim, num_axes, num_pairs, !k_positions);
    rc = qn_fill(a, q, q_strides, k, k_strides, q_weight, k_weight, q_positions, k_positions, freqs, eps);
    if (rc != G2V_OK) return rc;
    if (((int64_t)batch * a.n[0] * heads_q > 0 && !q_out) || ((int64_t)batch * a.n[1] * heads_k > 0 && !k_out))
        return api_fail(G2V_ERR_INVALID, "null q_out / k_out");
    a.out[0] = q_out;
    a.out[1] = k_out;
    G2V_HIP(launch_qk_norm_rotary(a, dtype, static_cast<hipStream_t>(stream)));
    return G2V_OK;
}

size_t g2v_qk_norm_rotary_backward_workspace(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim,
                                             int num_axes, int dtype, int shared_positions) {
    if (qn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, num_axes, 0, dtype, shared_positions != 0) != G2V_OK) return 0;
    return qk_norm_bwd_workspace(qn_args(batch, n_q, n_k, heads_q, heads_k, head_dim, num_axes, 0, shared_positions != 0), dtype);
}

int g2v_qk_norm_rotary_backward(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int num_axes,
                                int num_pairs, const void* q, const long long q_strides[3], const void* k,
                                const long long k_strides[3], int dtype, const float* q_weight, const float* k_weight,
                                const float* q_positions, const float* k_positions, const float* freqs, float eps,
                                const void* grad_q_out, const long long grad_q_out_strides[3], const void* grad_k_out,
                                const long long grad_k_out_strides[3], void* grad_q, void* grad_k, float* grad_q_weight,
                                float* grad_k_weight, float* grad_q_positions, float* grad_k_positions, void* workspace,
                                size_t workspace_bytes, void* stream) {
    api_begin();
    int rc = qn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, num_axes, num_pairs, dtype, !k_positions);
    if (rc != G2V_OK) return rc;
    QkNormArgs a = qn_args(batch, n_q, n_k, heads_q, heads_k, head_dim, num_axes, num_pairs, !k_positions);
    rc = qn_fill(a, q, q_strides, k, k_strides, q_weight, k_weight, q_positions, k_positions, freqs, eps);
    if (rc != G2V_OK) return rc;
    if (((int64_t)batch * a.n[0] * heads_q > 0 && (!grad_q_out || !grad_q_out_strides || !grad_q)) ||
        ((int64_t)batch * a.n[1] * heads_k > 0 && (!grad_k_out || !grad_k_out_strides || !grad_k)))
        return api_fail(G2V_ERR_INVALID, "null gradient pointer or strides");
    const size_t need = qk_norm_bwd_workspace(a, dtype);
    if (!workspace || workspace_bytes < need)
        return api_fail(G2V_ERR_INVALID, "workspace too small: %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
    a.g[0] = grad_q_out;
    a.g[1] = grad_k_out;
    for (int i = 0; i < 2; ++i) {
        const long long* s = i ? grad_k_out_strides : grad_q_out_strides;
        a.gsb[i] = s ? s[0] : 0;
        a.gsn[i] = s ? s[1] : 0;
        a.gsh[i] = s ? s[2] : 0;
    }
    a.dx[0] = grad_q;
    a.dx[1] = grad_k;
    a.dw[0] = grad_q_weight;
    a.dw[1] = grad_k_weight;
    a.dpos[0] = grad_q_positions;
    a.dpos[1] = a.shared ? nullptr : grad_k_positions;
    G2V_HIP(launch_qk_norm_rotary_bwd(a, dtype, workspace, static_cast<hipStream_t>(stream)));
    return G2V_OK;
}

}  // extern "C"
