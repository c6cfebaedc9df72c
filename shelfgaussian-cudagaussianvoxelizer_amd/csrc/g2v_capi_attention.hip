// C ABI of the operators in front of the splat (declared in include/g2v.h): argument checks, workspaces and launches of
// the query/key norms with rotary positions and of the attention.
#include <limits.h>
#include <math.h>
#include <algorithm>

#include "../../include/g2v.h"
#include "g2v_attention.h"

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
    if (num_axes < 1 || num_axes > kQnAxes) return api_fail(G2V_ERR_INVALID, "num_axes = %d (1 to %d)", num_axes, kQnAxes);
    if (num_pairs < 0 || 2 * num_pairs > head_dim)
        return api_fail(G2V_ERR_INVALID, "num_pairs = %d (0 to head_dim / 2 = %d)", num_pairs, head_dim / 2);
    if (dtype != G2V_DTYPE_F32 && dtype != G2V_DTYPE_BF16)
        return api_fail(G2V_ERR_INVALID, "dtype = %d (G2V_DTYPE_F32 or G2V_DTYPE_BF16)", dtype);
    if (shared && heads_k > 0 && n_k != n_q)
        return api_fail(G2V_ERR_INVALID, "shared positions need n_k == n_q, got %d and %d", n_k, n_q);
    // workgroups and their threads are counted in 32 bits
    if ((double)batch * n_q > 8388608.0 || (double)batch * n_k > 8388608.0 || heads_q > 8192 || heads_k > 8192)
        return api_fail(G2V_ERR_LIMIT, "batch %d x n %d / %d tokens (limit 2^23), heads %d / %d (limit 8192)", batch, n_q, n_k,
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

// ---- attention --------------------------------------------------------------------------------

constexpr int kCus = 256;

// Into how many workgroups the long axis (`units` tiles) of each of `wgs` workgroups goes.  unit_us: time of a tile in a
// workgroup that shares its CU with as many others as fit (per_cu); join_us: writing and adding one split's partial
// results.  A CU's last workgroups, fewer than fit, are only a little faster, a tile's loads and barriers taking their time
// alone too: one of two is counted 0.8 of the time of two.  (3000 x 8 x 64 bfloat16 dK and dV with their join 65 us,
// dQ 60, forward 48; counted 0.6: 92, 69 and 52.)  Where a few rounds fill the card more splits only add joins.
// (18000 x 16 heads x 64 bfloat16 forward with 1 / 2 / 4 splits of every tile: 1.51 / 1.40 / 1.44 ms; 18000 x 8 x 64 dQ with
// 1 / 2 / 4: 1.59 / 1.34 / 1.26 ms; attn_run goes on from there.)
int attn_splits(int64_t wgs, int units, int per_cu, double unit_us, double join_us, double& least) {
    const int64_t most = std::min<int64_t>(units, std::min<int64_t>(128, ceil_div(4 * kCus * per_cu, std::max<int64_t>(wgs, 1))));
    int best = 1;
    least = 0.0;
    for (int s = 1; s == 1 || s <= most; ++s) {
        const int n = (int)ceil_div(wgs * s, kCus);      // workgroups of the fullest CU
        const double rounds = n / per_cu + (n % per_cu ? 0.6 + 0.4 * (n % per_cu) / per_cu : 0.0);
        double us = rounds * ((units + s - 1) / s + 2) * unit_us;
        if (s > 1) us += 5.0 + s * join_us;
        if (s == 1 || us < least) {
            best = s;
            least = us;
        }
    }
    return best;
}

struct AttnSizes {
    int batch, nq, nk, hq, hk, dim, dp, group, bhs;
    bool f32;
    int64_t rows() const { return (int64_t)group * nq; }
};

int attn_sizes(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int dtype, AttnSizes& z) {
    if (batch < 0 || n_q < 0 || n_k < 0) return api_fail(G2V_ERR_INVALID, "negative size: batch %d, n %d / %d", batch, n_q, n_k);
    if (heads_q < 1 || heads_k < 1 || heads_q % heads_k)
        return api_fail(G2V_ERR_INVALID, "heads_q = %d is not a multiple of heads_k = %d", heads_q, heads_k);
    if (head_dim < 1 || head_dim > 128) return api_fail(G2V_ERR_INVALID, "head_dim = %d (1 to 128)", head_dim);
    if (dtype != G2V_DTYPE_F32 && dtype != G2V_DTYPE_BF16)
        return api_fail(G2V_ERR_INVALID, "dtype = %d (G2V_DTYPE_F32 or G2V_DTYPE_BF16)", dtype);
    z.batch = batch;
    z.nq = n_q;
    z.nk = n_k;
    z.hq = heads_q;
    z.hk = heads_k;
    z.dim = head_dim;
    z.dp = attn_dp(head_dim);
    z.group = heads_q / heads_k;
    z.f32 = dtype == G2V_DTYPE_F32;
    // rows and workgroups are counted in 32 bits, and no launch has 2^32 threads
    const double most = 33554432.0;
    if ((double)batch * heads_q * ((double)n_q + 63.0) > most || (double)batch * heads_k * n_k > most || (double)batch * n_k > most)
        return api_fail(G2V_ERR_LIMIT, "batch %d x heads %d / %d x n %d / %d rows (limit 2^25 of queries and of keys)", batch,
                        heads_q, heads_k, n_q, n_k);
    z.bhs = batch * heads_k;
    return G2V_OK;
}

// The tiles of `mine` rows and the workgroups that share the `passing` rows (in `streams` runs that end inside a tile each);
// products: of the scores' size that the kernel takes; width: values of a row's partial result.  Where all tiles with as many
// splits would leave the card's last round half empty, the first tiles have as few splits as fill whole rounds, and the others
// as many as fill one more, short one, together; `even`: not so, as how many tiles have work is known on the GPU only (the key
// tiles of a masked call).  The space is that of either plan, so that masks only add to a workspace.  (9000 x
// 8 x 128 bfloat16 dK and dV, 568 tiles on 512 places, with their join: 851 us with 3 splits each, 714 with 512 tiles whole and 56
// in 9; its forward, 288 tiles, 400 us with 3 splits, 357 with 256 tiles in 2 and 32 in 16.)
struct AttnRun {
    attn::Parts parts;
    int64_t part_rows;
};
AttnRun attn_run(const AttnSizes& z, AttnShape g, int64_t mine, int64_t passing, int streams, int width, bool even) {
    attn::Parts r = {};
    const int own = g.waves * g.blocks * 32, slots = kCus * g.per_cu;
    r.tiles = (int)ceil_div(mine, own);
    r.head_splits = 1;
    const int units = (int)std::min<int64_t>(ceil_div(passing, g.tile) * streams, 1 << 30);
    const double flops = 2.0 * g.products * own * g.tile * z.dp;
    const double unit_us = std::max(1.0, flops * g.per_cu / ((z.f32 ? 0.15e9 : 1.0e9) / kCus));
    const double join_us = 8.0 * mine * z.bhs * width / 3e6;
    const int64_t all = (int64_t)z.bhs * r.tiles;
    double least;
    r.splits = attn_splits(all, units, g.per_cu, unit_us, join_us, least);
    const AttnRun same = {r, part_rows(r, z.bhs, mine)};
    if (least <= 1.05 * all * units * unit_us / slots) return same;
    for (int first = 1; first <= std::min(4, units); ++first) {
        const int64_t rounds = all * first / slots, head = rounds * slots / ((int64_t)z.bhs * first), tail = r.tiles - head;
        if (head == 0 || tail == 0) continue;
        double us;
        const int splits = attn_splits(z.bhs * tail, units, g.per_cu, unit_us, join_us * tail / r.tiles, us);
        if (splits == 1) continue;
        us += rounds * (ceil_div(units, first) + 2) * unit_us + (first > 1 ? first * join_us * head / r.tiles : 0.0);
        if (us < least) {
            least = us;
            r.head = (int)head;
            r.head_splits = first;
            r.splits = splits;
            r.row0 = r.head * own;
        }
    }
    return {even ? same.parts : r, std::max(same.part_rows, part_rows(r, z.bhs, mine))};
}

struct Strided {
    const void* p;
    const long long* s;
    int n, heads;
    bool keys;
};

// bfloat16 rows of whole 16-byte chunks at 16-byte boundaries are read where they are.
bool attn_in_place(const AttnSizes& z, const Strided* t, int count) {
    if (z.f32 || z.dim % 8) return false;
    for (int i = 0; i < count; ++i) {
        if (reinterpret_cast<uintptr_t>(t[i].p) % 16) return false;
        for (int k = 0; k < 3; ++k)
            if (t[i].s[k] % 8) return false;
        if (t[i].s[1] < 0 || t[i].s[1] >= (1 << 24)) return false;   // a tile's rows within 32-bit offsets
    }
    return true;
}

size_t attn_packed_bytes(const AttnSizes& z, int64_t n, int heads) {
    return (size_t)z.batch * heads * n * (z.f32 ? 3 : 1) * z.dp * 2;
}

// Keys up to which packing makes the list of valid keys by itself, every workgroup reading its scene's mask: a launch less
// (6 x 300 keys x 8 heads x 32 float32 forward: 21.6 -> 19.1 us a pass), but work that grows with the keys (4096 keys x 8
// heads x 64 float32: 20.8 us in one launch, 6.6 + 13.6 in two).
constexpr int kListInPack = 2048;

// The tensors as the kernels read them.  What cannot be read in place is packed into c's space (all of a call, or none),
// and the keys of a masked call are: the valid ones one after another.  key_list: (batch, nk) and (batch); with mask it
// is made first.
hipError_t attn_sources(const AttnSizes& z, const Strided* t, int count, bool packed, const unsigned char* mask, int* key_list,
                        Carver& c, attn::RowSrc* out, hipStream_t s) {
    AttnPack a = {};
    a.batch = z.batch;
    a.dim = z.dim;
    a.dp = z.dp;
    a.list_tensor = -1;
    if (key_list) {
        int* counts = key_list + (int64_t)z.batch * z.nk;
        if (mask && z.nk <= kListInPack) {
            a.mask = mask;
            a.list_out = key_list;
            a.count_out = counts;
        } else {
            if (mask) {
                const hipError_t e = launch_attn_list(z.batch, z.nk, mask, key_list, counts, s);
                if (e != hipSuccess) return e;
            }
            a.list = key_list;
            a.count = counts;
        }
    }
    for (int i = 0; i < count; ++i) {
        if (!packed && !(key_list && t[i].keys)) {
            out[i] = {static_cast<const char*>(t[i].p), t[i].s[0] * 2, t[i].s[1] * 2, t[i].s[2] * 2, z.dim / 8};
            continue;
        }
        const int64_t row = (int64_t)(z.f32 ? 3 : 1) * z.dp * 2;
        char* dst = c.take<char>(attn_packed_bytes(z, t[i].n, t[i].heads));
        const int k = a.tensors++;
        a.src[k] = t[i].p;
        a.sb[k] = t[i].s[0];
        a.sn[k] = t[i].s[1];
        a.sh[k] = t[i].s[2];
        a.n[k] = t[i].n;
        a.heads[k] = t[i].heads;
        a.keys[k] = t[i].keys;
        if (t[i].keys && a.list_tensor < 0) a.list_tensor = k;
        a.dst[k] = dst;
        out[i] = {dst, row * t[i].n * t[i].heads, row, row * t[i].n, z.dp / 8};
    }
    return a.tensors ? launch_attn_pack(a, z.f32, s) : hipSuccess;
}

AttnRun attn_fwd_run(const AttnSizes& z) {
    return attn_run(z, attn_fwd_shape(z.f32, z.dp, z.rows()), z.rows(), z.nk, 1, z.dp, false);
}
AttnRun attn_dq_run(const AttnSizes& z) {
    return attn_run(z, attn_dq_shape(z.f32, z.dp, z.rows()), z.rows(), z.nk, 1, z.dp, false);
}
AttnRun attn_dkv_run(const AttnSizes& z, bool masked) {
    const AttnShape g = attn_dkv_shape(z.f32, z.dp, attn_dkv_planes(z.f32, z.nk, z.rows()));
    return attn_run(z, g, z.nk, z.nq, z.group, 2 * z.dp, masked);
}

struct AttnFwdWs {
    float *part_o, *part_ml;
};
AttnFwdWs carve_attn_fwd(Carver& c, const AttnSizes& z, const AttnRun& r) {
    AttnFwdWs w = {nullptr, nullptr};
    if (const int64_t rows = r.part_rows) {
        w.part_o = c.take<float>(rows * z.dp);
        w.part_ml = c.take<float>(rows * 2);
    }
    return w;
}
// packed: all tensors; masked: k and v.
void carve_packed(Carver& c, const AttnSizes& z, bool packed, bool masked, bool backward) {
    if (packed) c.take<char>(attn_packed_bytes(z, z.nq, z.hq));
    if (packed || masked) {
        c.take<char>(attn_packed_bytes(z, z.nk, z.hk));
        c.take<char>(attn_packed_bytes(z, z.nk, z.hk));
    }
    if (packed && backward) c.take<char>(attn_packed_bytes(z, z.nq, z.hq));
}
struct AttnBwdWs {
    int nqp;
    float *lse, *delta, *part;
};
AttnBwdWs carve_attn_bwd(Carver& c, const AttnSizes& z, const AttnRun& dq, const AttnRun& dkv) {
    AttnBwdWs w;
    w.nqp = (int)((z.nq + 63) / 64 * 64);
    w.lse = c.take<float>((size_t)z.batch * z.hq * w.nqp);
    w.delta = c.take<float>((size_t)z.batch * z.hq * w.nqp);
    // one area: the two kernels run one after the other
    size_t part = (size_t)dq.part_rows * z.dp;
    part = std::max(part, (size_t)dkv.part_rows * 2 * z.dp);
    w.part = part ? c.take<float>(part) : nullptr;
    return w;
}

size_t attn_fwd_bytes(const AttnSizes& z, const AttnRun& r, bool packed, bool masked) {
    Carver c(nullptr, (size_t)-1);
    carve_attn_fwd(c, z, r);
    carve_packed(c, z, packed, masked, false);
    return c.off + 256;
}
size_t attn_bwd_bytes(const AttnSizes& z, const AttnRun& dq, const AttnRun& dkv, bool packed, bool masked) {
    Carver c(nullptr, (size_t)-1);
    carve_attn_bwd(c, z, dq, dkv);
    carve_packed(c, z, packed, masked, true);
    return c.off + 256;
}

// ---- attention within a window -----------------------------------------------------------------

// Sizes and window as the kernels take them: z.nk without the keys between the sinks and the first window, which no query sees.
struct WinSizes {
    AttnSizes z;
    AttnWindow w;
    int64_t span;    // keys of a query's window
};
int win_sizes(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int dtype, int left, int right, int sinks,
              WinSizes& x) {
    const int rc = attn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, x.z);
    if (rc != G2V_OK) return rc;
    if (left < -1 || right < -1 || sinks < 0)
        return api_fail(G2V_ERR_INVALID, "left = %d, right = %d, sinks = %d (not negative; left, right -1: no bound)", left, right, sinks);
    constexpr int kFarAway = 1 << 28;    // places are below 2^26
    x.w = {};
    x.w.left = left < 0 ? kFarAway : std::min(left, kFarAway);
    x.w.right = right < 0 ? kFarAway : std::min(right, kFarAway);
    x.w.sinks = std::min(sinks, n_k);
    x.w.shift = n_k - n_q;
    x.span = (int64_t)x.w.left + x.w.right + 1;
    x.w.gap = std::max(0, std::min(x.w.shift - x.w.left, n_k) - x.w.sinks);
    x.z.nk -= x.w.gap;
    x.w.shift -= x.w.gap;
    return G2V_OK;
}

// A workgroup's rows see a window longer by themselves, and the sinks.
int64_t win_keys(const WinSizes& x, AttnShape g) {
    return std::min<int64_t>(x.z.nk, x.span + g.waves * g.blocks * 32 / x.z.group + (x.w.sinks ? g.tile : 0));
}
// Whether the forward splits float32 rows into planes as it loads them, every workgroup that sees a row for itself, instead of
// reading planes packed before: a launch and a pass over the rows less, but each row of k and v is split again by all workgroups that see
// it.  Ten rows are split in the time that packing one takes (3.3 at 96 channels, where its registers are short), and packing takes all
// rows of q, k and v once; where a mask has tiles of planes loaded row by row, too, 32 (13).  us at 257 / 513 / 1025 / 2049 keys,
// 40,000 x 8 heads, the rule's side first: 32 channels (split) 109 for 157, 173 for 210, 295 for 320, (packed) 548 for 548; 64 (split)
// 204 for 284, 332 for 391, 593 for 617, (packed) 1033 for 1055; 96 (split) 448 for 544, 700 for 723, (packed) 1084 for 1203, 1807 for
// 2209; 72 (split) 429 for 537, 673 for 706, (packed) 1047 for 1165, 1730 for 2147; 128 (split) 532 for 750, 822 for 1011, 1408 for
// 1553, (packed) 2617 for 2592.  With a mask, at 2049 / 4097 keys: 64 channels (split) 1009 for 1077, 1902 for 1928; 96 (split) 2329
// for 2357, (packed) 4232 for 4347.  Shared heads have fewer rows of k and v to pack: 10,000 x 2 x 4 heads, 64 channels (split) 55 for
// 67, 90 for 96, (packed) 151 for 154, 251 for 275.  Few queries split each row once: one query, 4097 keys x 16 x 64 (split) 25 for 39.
// (Rows that are not whole chunks of 8 load their ends one by one: 40,000 x 8 x 75, 256 / 1024 / 2048 keys, packed 649, 1166, 1867,
// split 821, 2014, 3446.)
bool win_splits_rows(const WinSizes& x, bool masked) {
    const AttnShape g = window_fwd_shape(true, x.z.dp, x.z.rows());
    const int64_t split = ceil_div(x.z.rows(), g.waves * 32) * 2 * std::min<int64_t>(x.z.nk, x.span + x.w.sinks);
    const int64_t packed = x.z.rows() + 2 * (int64_t)x.z.nk;
    return x.z.dim % 8 == 0 && 3 * split <= (x.z.dp == 96 ? (masked ? 40 : 10) : (masked ? 96 : 30)) * packed;
}
AttnRun win_fwd_run(const WinSizes& x) {
    const AttnShape g = window_fwd_shape(x.z.f32, x.z.dp, x.z.rows());
    return attn_run(x.z, g, x.z.rows(), win_keys(x, g), 1, x.z.dp, false);
}
AttnRun win_dq_run(const WinSizes& x) {
    const AttnShape g = window_dq_shape(x.z.f32, x.z.dp, x.z.rows());
    return attn_run(x.z, g, x.z.rows(), win_keys(x, g), 1, x.z.dp, false);
}
// Planes of P and dS by the keys that a query sees (see attn_dkv_planes); two where a mask leaves fewer, how many is known on the
// GPU only.
int win_dkv_planes(const WinSizes& x, bool masked) {
    return attn_dkv_planes(x.z.f32, masked ? 1 : std::min<int64_t>(x.z.nk, x.span + x.w.sinks), x.z.rows());
}
AttnRun win_dkv_run(const WinSizes& x, int planes) {
    const AttnShape g = window_dkv_shape(x.z.f32, x.z.dp, planes, false);
    return attn_run(x.z, g, x.z.nk, std::min<int64_t>(x.z.nq, x.span + g.waves * 32), x.z.group, 2 * x.z.dp, false);
}
// The sinks' queries beyond their windows: whether there are any, and the splits of all queries for each tile of sinks.
bool win_has_far(const WinSizes& x) { return x.w.sinks > 0 && (int64_t)x.w.left - x.w.shift + 1 < x.z.nq; }
AttnRun win_sinks_run(const WinSizes& x, int planes) {
    attn::Parts r = {};
    if (!win_has_far(x)) return {r, 0};
    const AttnShape g = window_dkv_shape(x.z.f32, x.z.dp, planes, true);
    r.tiles = r.head = (int)ceil_div(x.w.sinks, 32);
    r.row0 = x.w.sinks;
    r.splits = 1;
    // as many workgroups as the card holds, of four tiles at least (200,000 queries x 8 heads x 64, 192 for 128: 116 -> 92 us)
    const int64_t units = ceil_div(x.z.nq, g.tile) * x.z.group, most = kCus * g.per_cu / std::max<int64_t>((int64_t)x.z.bhs * r.tiles, 1);
    r.head_splits = (int)std::max<int64_t>(1, std::min(units / 4, most));
    return {r, part_rows(r, x.z.bhs, x.w.sinks)};
}

struct WinBwdRuns {
    int planes;
    AttnRun dq, dkv, sinks;
};
WinBwdRuns win_bwd_runs(const WinSizes& x, bool masked) {
    WinBwdRuns r;
    r.planes = win_dkv_planes(x, masked);
    r.dq = win_dq_run(x);
    r.dkv = win_dkv_run(x, r.planes);
    r.sinks = win_sinks_run(x, r.planes);
    return r;
}
// The sinks' partial results take the area of the others' after them.
AttnBwdWs carve_win_bwd(Carver& c, const WinSizes& x, const WinBwdRuns& r) {
    AttnRun dkv = r.dkv;
    dkv.part_rows = std::max(dkv.part_rows, r.sinks.part_rows);
    return carve_attn_bwd(c, x.z, r.dq, dkv);
}
size_t win_fwd_bytes(const WinSizes& x, const AttnRun& r, bool packed) {
    Carver c(nullptr, (size_t)-1);
    carve_attn_fwd(c, x.z, r);
    carve_packed(c, x.z, packed, false, false);
    return c.off + 256;
}
size_t win_bwd_bytes(const WinSizes& x, const WinBwdRuns& r, bool packed) {
    Carver c(nullptr, (size_t)-1);
    carve_win_bwd(c, x, r);
    carve_packed(c, x.z, packed, false, true);
    return c.off + 256;
}

// The tensors as the kernels read them: all in place, or all packed without the gap and with zeros in masked keys' rows.
hipError_t win_sources(const WinSizes& x, const Strided* t, int count, bool packed, const unsigned char* mask, Carver& c,
                       attn::RowSrc* out, hipStream_t s) {
    const AttnSizes& z = x.z;
    AttnPack a = {};
    a.batch = z.batch;
    a.dim = z.dim;
    a.dp = z.dp;
    a.list_tensor = -1;
    a.sinks = x.w.sinks;
    a.gap = x.w.gap;
    a.valid = mask;
    for (int i = 0; i < count; ++i) {
        if (!packed) {
            const int size = z.f32 ? 4 : 2;
            out[i] = {static_cast<const char*>(t[i].p), t[i].s[0] * size, t[i].s[1] * size, t[i].s[2] * size, z.dim / 8};
            continue;
        }
        const int64_t row = (int64_t)(z.f32 ? 3 : 1) * z.dp * 2;
        char* dst = c.take<char>(attn_packed_bytes(z, t[i].n, t[i].heads));
        const int k = a.tensors++;
        a.src[k] = t[i].p;
        a.sb[k] = t[i].s[0];
        a.sn[k] = t[i].s[1];
        a.sh[k] = t[i].s[2];
        a.n[k] = t[i].n;
        a.heads[k] = t[i].heads;
        a.keys[k] = t[i].keys;
        a.dst[k] = dst;
        out[i] = {dst, row * t[i].n * t[i].heads, row, row * t[i].n, z.dp / 8};
    }
    return a.tensors ? launch_attn_pack(a, z.f32, s) : hipSuccess;
}

int attn_scale(float scale) {
    if (!(scale > 0.0f) || !isfinite(scale * attn::kLog2e))
        return api_fail(G2V_ERR_INVALID, "scale = %g (positive and finite)", (double)scale);
    return G2V_OK;
}

}  // namespace

extern "C" {

size_t g2v_attention_forward_workspace(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int dtype,
                                       int in_place, int masked) {
    AttnSizes z;
    if (attn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, z) != G2V_OK) return 0;
    return attn_fwd_bytes(z, attn_fwd_run(z), z.f32 || !in_place, masked != 0);
}

int g2v_attention_forward(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, const void* q,
                          const long long q_strides[3], const void* k, const long long k_strides[3], const void* v,
                          const long long v_strides[3], int dtype, const unsigned char* key_mask, float scale, void* out,
                          void* out_rest, float* lse, int* key_list, void* workspace, size_t workspace_bytes, void* stream) {
    api_begin();
    AttnSizes z;
    int rc = attn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, z);
    if (rc != G2V_OK) return rc;
    rc = attn_scale(scale);
    if (rc != G2V_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool keys = (int64_t)batch * n_k > 0;
    if (keys && key_mask && !key_list) return api_fail(G2V_ERR_INVALID, "key_mask without key_list");
    if ((int64_t)batch * n_q == 0) {
        // without queries too: the backward writes the keys' gradients by this list
        if (keys && key_mask) G2V_HIP(launch_attn_list(batch, n_k, key_mask, key_list, key_list + (int64_t)batch * n_k, s));
        return G2V_OK;
    }
    if (!out || !q || !q_strides || (keys && (!k || !v || !k_strides || !v_strides)))
        return api_fail(G2V_ERR_INVALID, "null q, k, v, strides or out");
    static const long long none[3] = {0, 0, 0};
    int* list = keys && key_mask ? key_list : nullptr;
    const Strided t[3] = {{q, q_strides, n_q, heads_q, false},
                          {k, keys ? k_strides : none, n_k, heads_k, true},
                          {v, keys ? v_strides : none, n_k, heads_k, true}};
    const bool packed = !attn_in_place(z, t, 3);
    const AttnRun r = attn_fwd_run(z);
    const size_t need = attn_fwd_bytes(z, r, packed, list != nullptr);
    if (!workspace || workspace_bytes < need)
        return api_fail(G2V_ERR_INVALID, "workspace too small: %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
    Carver c(workspace, workspace_bytes);
    const AttnFwdWs w = carve_attn_fwd(c, z, r);
    attn::RowSrc src[3];
    G2V_HIP(attn_sources(z, t, 3, packed, key_mask, list, c, src, s));
    AttnFwd a = {};
    a.q = src[0];
    a.k = src[1];
    a.v = src[2];
    if (list) a.count = list + (int64_t)batch * n_k;
    a.nq = n_q;
    a.nk = n_k;
    a.hq = heads_q;
    a.hk = heads_k;
    a.group = z.group;
    a.dim = head_dim;
    a.bhs = z.bhs;
    a.parts = r.parts;
    a.c = scale * attn::kLog2e;
    a.out = out;
    a.rest = out_rest;
    a.lse = lse;
    a.part_o = w.part_o;
    a.part_ml = w.part_ml;
    G2V_HIP(launch_attn_fwd(a, z.f32, z.dp, s));
    return G2V_OK;
}

size_t g2v_attention_backward_workspace(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int dtype,
                                        int in_place, int masked) {
    AttnSizes z;
    if (attn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, z) != G2V_OK) return 0;
    return attn_bwd_bytes(z, attn_dq_run(z), attn_dkv_run(z, masked != 0), z.f32 || !in_place, masked != 0);
}

int g2v_attention_backward(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, const void* q,
                           const long long q_strides[3], const void* k, const long long k_strides[3], const void* v,
                           const long long v_strides[3], int dtype, const int* key_list, float scale, const void* out,
                           const void* out_rest, const float* lse, const void* grad_out, const long long grad_out_strides[3], void* grad_q,
                           void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
    api_begin();
    AttnSizes z;
    int rc = attn_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, z);
    if (rc != G2V_OK) return rc;
    rc = attn_scale(scale);
    if (rc != G2V_OK) return rc;
    const bool queries = (int64_t)batch * n_q > 0, keys = (int64_t)batch * n_k > 0;
    if (!queries && !keys) return G2V_OK;
    if ((grad_k == nullptr) != (grad_v == nullptr)) return api_fail(G2V_ERR_INVALID, "grad_k and grad_v go together");
    if ((queries && (!q || !q_strides || !out || !lse || !grad_out || !grad_out_strides)) ||
        (keys && (!k || !v || !k_strides || !v_strides)))
        return api_fail(G2V_ERR_INVALID, "null q, k, v, out, lse, grad_out or strides");
    hipStream_t s = static_cast<hipStream_t>(stream);
    static const long long none[3] = {0, 0, 0};
    const long long* sq = queries ? q_strides : none;
    const long long* sg = queries ? grad_out_strides : none;
    const long long* sk = keys ? k_strides : none;
    const long long* sv = keys ? v_strides : none;
    const int* list = keys ? key_list : nullptr;
    const Strided t[4] = {{q, sq, n_q, heads_q, false}, {k, sk, n_k, heads_k, true}, {v, sv, n_k, heads_k, true},
                          {grad_out, sg, n_q, heads_q, false}};
    const bool packed = !attn_in_place(z, t, 4);
    const AttnRun rq = attn_dq_run(z), rk = attn_dkv_run(z, list != nullptr);
    const size_t need = attn_bwd_bytes(z, rq, rk, packed, list != nullptr);
    if (!workspace || workspace_bytes < need)
        return api_fail(G2V_ERR_INVALID, "workspace too small: %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
    Carver c(workspace, workspace_bytes);
    const AttnBwdWs w = carve_attn_bwd(c, z, rq, rk);
    attn::RowSrc src[4];
    G2V_HIP(attn_sources(z, t, 4, packed, nullptr, const_cast<int*>(list), c, src, s));
    G2V_HIP(launch_attn_delta(batch, n_q, w.nqp, heads_q, head_dim, out, out_rest, grad_out, sg[0], sg[1], sg[2], z.f32, lse, w.lse,
                              w.delta, s));
    AttnBwd a = {};
    a.q = src[0];
    a.k = src[1];
    a.v = src[2];
    a.g = src[3];
    if (list) a.count = list + (int64_t)batch * n_k;
    a.list = list;
    a.nq = n_q;
    a.nk = n_k;
    a.hq = heads_q;
    a.hk = heads_k;
    a.group = z.group;
    a.dim = head_dim;
    a.bhs = z.bhs;
    a.nqp = w.nqp;
    a.c = scale * attn::kLog2e;
    a.scale = scale;
    a.lse = w.lse;
    a.delta = w.delta;
    a.dq = grad_q;
    a.dk = grad_k;
    a.dv = grad_v;
    a.part = w.part;
    if (grad_k && keys) {
        a.parts = rk.parts;
        G2V_HIP(launch_attn_dkv(a, z.f32, z.dp, s));
    }
    if (grad_q && queries) {
        a.parts = rq.parts;
        G2V_HIP(launch_attn_dq(a, z.f32, z.dp, s));
    }
    return G2V_OK;
}

size_t g2v_window_attention_forward_workspace(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int dtype,
                                              int left, int right, int sinks, int in_place, int masked) {
    WinSizes x;
    if (win_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, left, right, sinks, x) != G2V_OK) return 0;
    return win_fwd_bytes(x, win_fwd_run(x), x.z.f32 ? !win_splits_rows(x, masked != 0) : !in_place);
}

int g2v_window_attention_forward(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, const void* q,
                                 const long long q_strides[3], const void* k, const long long k_strides[3], const void* v,
                                 const long long v_strides[3], int dtype, const unsigned char* key_mask, int left, int right,
                                 int sinks, float scale, void* out, void* out_rest, float* lse, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    api_begin();
    WinSizes x;
    int rc = win_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, left, right, sinks, x);
    if (rc != G2V_OK) return rc;
    rc = attn_scale(scale);
    if (rc != G2V_OK) return rc;
    if ((int64_t)batch * n_q == 0) return G2V_OK;
    const bool keys = (int64_t)batch * n_k > 0;
    if (!out || !q || !q_strides || (keys && (!k || !v || !k_strides || !v_strides)))
        return api_fail(G2V_ERR_INVALID, "null q, k, v, strides or out");
    hipStream_t s = static_cast<hipStream_t>(stream);
    static const long long none[3] = {0, 0, 0};
    const AttnSizes& z = x.z;
    const Strided t[3] = {{q, q_strides, n_q, heads_q, false},
                          {k, keys ? k_strides : none, z.nk, heads_k, true},
                          {v, keys ? v_strides : none, z.nk, heads_k, true}};
    const bool packed = z.f32 ? !win_splits_rows(x, key_mask != nullptr) : !attn_in_place(z, t, 3);
    if (!keys) key_mask = nullptr;    // (then there are no rows to pack or to split)
    const AttnRun r = win_fwd_run(x);
    const size_t need = win_fwd_bytes(x, r, packed);
    if (!workspace || workspace_bytes < need)
        return api_fail(G2V_ERR_INVALID, "workspace too small: %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
    Carver c(workspace, workspace_bytes);
    const AttnFwdWs w = carve_attn_fwd(c, z, r);
    attn::RowSrc src[3];
    G2V_HIP(win_sources(x, t, 3, packed, key_mask, c, src, s));
    WinFwd a = {};
    a.q = src[0];
    a.k = src[1];
    a.v = src[2];
    a.nq = n_q;
    a.nk = z.nk;
    a.hq = heads_q;
    a.hk = heads_k;
    a.group = z.group;
    a.dim = head_dim;
    a.bhs = z.bhs;
    a.parts = r.parts;
    a.c = scale * attn::kLog2e;
    a.out = out;
    a.rest = out_rest;
    a.lse = lse;
    a.part_o = w.part_o;
    a.part_ml = w.part_ml;
    a.win = x.w;
    a.win.mask = key_mask;
    a.win.skip = packed ? 0 : x.w.gap;
    a.floats = z.f32 && !packed;
    G2V_HIP(launch_window_fwd(a, z.f32, z.dp, s));
    return G2V_OK;
}

size_t g2v_window_attention_backward_workspace(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, int dtype,
                                               int left, int right, int sinks, int in_place, int masked) {
    WinSizes x;
    if (win_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, left, right, sinks, x) != G2V_OK) return 0;
    return win_bwd_bytes(x, win_bwd_runs(x, masked != 0), x.z.f32 || !in_place);
}

int g2v_window_attention_backward(int batch, int n_q, int n_k, int heads_q, int heads_k, int head_dim, const void* q,
                                  const long long q_strides[3], const void* k, const long long k_strides[3], const void* v,
                                  const long long v_strides[3], int dtype, const unsigned char* key_mask, int left, int right,
                                  int sinks, float scale, const void* out, const void* out_rest, const float* lse,
                                  const void* grad_out, const long long grad_out_strides[3], void* grad_q, void* grad_k,
                                  void* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
    api_begin();
    WinSizes x;
    int rc = win_sizes(batch, n_q, n_k, heads_q, heads_k, head_dim, dtype, left, right, sinks, x);
    if (rc != G2V_OK) return rc;
    rc = attn_scale(scale);
    if (rc != G2V_OK) return rc;
    const bool queries = (int64_t)batch * n_q > 0, keys = (int64_t)batch * n_k > 0;
    if (!queries && !keys) return G2V_OK;
    if ((grad_k == nullptr) != (grad_v == nullptr)) return api_fail(G2V_ERR_INVALID, "grad_k and grad_v go together");
    if ((queries && (!q || !q_strides || !out || !lse || !grad_out || !grad_out_strides)) ||
        (keys && (!k || !v || !k_strides || !v_strides)))
        return api_fail(G2V_ERR_INVALID, "null q, k, v, out, lse, grad_out or strides");
    hipStream_t s = static_cast<hipStream_t>(stream);
    static const long long none[3] = {0, 0, 0};
    const long long* sg = queries ? grad_out_strides : none;
    const Strided t[4] = {{q, queries ? q_strides : none, n_q, heads_q, false},
                          {k, keys ? k_strides : none, x.z.nk, heads_k, true},
                          {v, keys ? v_strides : none, x.z.nk, heads_k, true},
                          {grad_out, sg, n_q, heads_q, false}};
    const AttnSizes& z = x.z;
    const bool packed = !attn_in_place(z, t, 4);
    if (!keys) key_mask = nullptr;
    const WinBwdRuns r = win_bwd_runs(x, key_mask != nullptr);
    const size_t need = win_bwd_bytes(x, r, packed);
    if (!workspace || workspace_bytes < need)
        return api_fail(G2V_ERR_INVALID, "workspace too small: %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
    Carver c(workspace, workspace_bytes);
    const AttnBwdWs w = carve_win_bwd(c, x, r);
    attn::RowSrc src[4];
    G2V_HIP(win_sources(x, t, 4, packed, key_mask, c, src, s));
    WinBwd a = {};
    a.q = src[0];
    a.k = src[1];
    a.v = src[2];
    a.g = src[3];
    a.nq = n_q;
    a.nk = z.nk;
    a.gap_at = x.w.sinks;
    a.gap = x.w.gap;
    a.hq = heads_q;
    a.hk = heads_k;
    a.group = z.group;
    a.dim = head_dim;
    a.bhs = z.bhs;
    a.nqp = w.nqp;
    a.c = scale * attn::kLog2e;
    a.scale = scale;
    a.lse = w.lse;
    a.delta = w.delta;
    a.dq = grad_q;
    a.dk = grad_k;
    a.dv = grad_v;
    a.part = w.part;
    a.win = x.w;
    a.win.mask = key_mask;
    a.win.skip = packed ? 0 : x.w.gap;
    a.out = out;
    a.rest = out_rest;
    a.lse_in = lse;
    a.lse_pad = w.lse;
    a.delta_pad = w.delta;
    if (queries) {
        a.parts = r.dq.parts;
        if (!grad_q) {
            a.parts.head = 0;
            a.parts.splits = 1;
        }
        G2V_HIP(launch_window_dq(a, z.f32, z.dp, s));
    }
    if (grad_k && keys) {
        G2V_HIP(launch_window_zeros(a, batch, z.f32, s));
        WinBwd kv = a;
        if (z.nk == 1 || (x.span == 1 && x.w.sinks == 0)) kv.scale = 0.0f;    // a query's only key: its probability is 1
        kv.parts = r.dkv.parts;
        if (z.nk > 0) G2V_HIP(launch_window_dkv(kv, z.f32, z.dp, r.planes, s));    // (no queries: all keys are the gap's)
        if (queries && win_has_far(x)) {    // written anew behind them
            kv.all_queries = true;
            kv.parts = r.sinks.parts;
            G2V_HIP(launch_window_dkv(kv, z.f32, z.dp, r.planes, s));
        }
    }
    return G2V_OK;
}

}  // extern "C"

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
    hipStream_t s = static_cast<hipStream_t>(stream);
    G2V_HIP(launch_qk_norm_rotary_bwd(a, dtype, workspace, s));
    // no workgroup runs over positions that turn no head
    if (grad_q_positions && heads_q == 0 && (k_positions || heads_k == 0))
        G2V_HIP(launch_fill_i32((int64_t)batch * n_q * num_axes, 0, reinterpret_cast<int*>(grad_q_positions), s));
    if (grad_k_positions && heads_k == 0 && k_positions)
        G2V_HIP(launch_fill_i32((int64_t)batch * n_k * num_axes, 0, reinterpret_cast<int*>(grad_k_positions), s));
    return G2V_OK;
}

}  // extern "C"
