// Attention over sets of Gaussians, backward, from the inputs, the row sums of the forward (lse) and dO:
//
//   P = 2^(c S - lse),  dP = dO V^T,  dS = P (dP - delta),  delta = sum_d dO O,
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
//
// The probabilities are recomputed, twice: once by workgroups that own keys (dK, dV; the queries pass by) and once by
// workgroups that own queries (dQ; the keys pass by).  That is seven products of the scores' size instead of five, and
// nothing is added to memory that another workgroup adds to: gradients are the same on every run, and shared key heads are
// summed over their query heads in registers.  (Adding dQ up in memory, not built, would move dQ in float32 once for each
// 128 keys of a workgroup: 141 times at 18000 keys, 10 GB for 16 heads of 64, 2 ms at a copy's rate and more with atomics; the two
// products recomputed are 1.3e12 flop there, 1.2 ms.)
//
// Bound, like the forward, by matrix and vector work taking turns.  18000 x 8 heads x 64 bfloat16: dK and dV 1.27 ms (four
// products, 1050 TFLOP/s; at that launch bound 7 of its registers are spilled, 32 bytes a lane), dQ 1.17 ms (three, and the one of
// dS twice for its two planes, 1150 TFLOP/s).
#include "g2v_attention.h"

namespace g2v {
namespace {
using namespace attn;

// dQ: rows in the lanes as in the forward, S^T = K Q^T and dP^T = V dO^T, dQ^T += K^T (scale dS)^T.  (Scaled before the sum
// over the keys, which then overflows only where dQ does; the factor turns an addition into a fused one and takes no time.)
// KS: see k_attn_fwd.
template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
__global__ void __launch_bounds__(NW * 64, launch_bound(NW, dq_per_cu(NP, DP, NW))) k_attn_dq(AttnBwd a) {
    // planes of dS in its product with K: two of bfloat16 for bfloat16 inputs.  The keys that a query attends to share
    // a direction, their dS sum to zero, and what is left of dQ is small beside the terms: rounding dS to 2^-9
    // alone puts dQ 3.0e-3 off (its own rounding: 1.7e-3), a second plane leaves 2.0e-3 for a third more products here
    constexpr int NS = NP == 1 ? 2 : NP;
    constexpr int NT = NW * 64, KB = KT / 32, DB = DP / 32;
    typedef Tile<NP, DP, KT, NT> TileT;
    constexpr int kBuffers = buffers(2, TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    static_assert(dq_per_cu(NP, DP, NW) * sizeof(lds) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int rows = a.group * a.nq;
    const int r0 = (w.tile * NW + g2v::uniform(threadIdx.x >> 6)) * (NQB * 32) + (threadIdx.x & 31);
    const int n = a.count ? a.count[w.b] : a.nk;
    const char* kbase = a.k.p + w.b * a.k.sb + w.h * a.k.sh;
    const char* vbase = a.v.p + w.b * a.v.sb + w.h * a.v.sh;
    int t0, t1;
    split_range((n + KT - 1) / KT, w.split, w.splits, t0, t1);
    if (n < 2) t1 = t0;    // one key: its probability is 1 whatever q is

    bf16x8 q[NQB][KS][NP], g[NQB][KS][NP];
    float lse[NQB], delta[NQB];    // delta: negative, as it is stored, and times scale
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        const int r = r0 + 32 * b, rc = r < rows ? r : rows - 1;
        const int tok = rc / a.group, head = w.h * a.group + rc - tok * a.group;
        const char* qrow = a.q.p + w.b * a.q.sb + tok * a.q.sn + head * a.q.sh;
        const char* grow = a.g.p + w.b * a.g.sb + tok * a.g.sn + head * a.g.sh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int pl = 0; pl < NP; ++pl) {
                q[b][ks][pl] = mem_frag<DP>(qrow, r < rows, a.q.chunks, pl, ks);
                g[b][ks][pl] = mem_frag<DP>(grow, r < rows, a.g.chunks, pl, ks);
            }
        const int64_t at = ((int64_t)w.b * a.hq + head) * a.nqp + tok;
        lse[b] = a.lse[at];
        delta[b] = a.delta[at] * a.scale;
    }

    TileT tile;
    tile.init(a.k);
    Frags<DP> frags;
    frags.init(lds_off(lds));
    if (a.k.chunks < TileT::C) clear_lds<NT>(&lds[0][0][0], sizeof(lds));
    auto load = [&](int t, int buf) {
        if ((t + 1) * KT <= n) {
            tile.load(kbase, a.k.sn, (int64_t)t * KT, lds_off(lds[buf][0]));
            tile.load(vbase, a.v.sn, (int64_t)t * KT, lds_off(lds[buf][1]));
        } else {
            tile.load_tail(kbase, a.k.sn, (int64_t)t * KT, n, lds[buf][0]);
            tile.load_tail(vbase, a.v.sn, (int64_t)t * KT, n, lds[buf][1]);
        }
    };

    f32x16 dq[DB][NQB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < NQB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[d][b][i] = 0.0f;
    if (t0 < t1) load(t0, 0);
    if (kAhead > 1 && t0 + 1 < t1) load(t0 + 1, 1);
    for (int t = t0, buf = 0; t < t1; ++t, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        next_tile<kBuffers, 2 * TileT::kLoads>(t + 1 < t1 && (t + 2) * KT <= n);
        if (t + kAhead < t1) load(t + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
        const uint32_t at = buf * 2 * TileT::kBytes;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 s[NQB], dp[NQB];
#pragma unroll
            for (int b = 0; b < NQB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = dp[b][i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 fk[NP], fv[NP];
#pragma unroll
                for (int pl = 0; pl < NP; ++pl) {
                    fk[pl] = frags.rows(at, pl * KT * DP * 2, kb, ks);
                    fv[pl] = frags.rows(at, TileT::kBytes + pl * KT * DP * 2, kb, ks);
                }
#pragma unroll
                for (int b = 0; b < NQB; ++b) {
                    s[b] = mma(fk, q[b][ks], s[b]);
                    dp[b] = mma(fv, g[b][ks], dp[b]);
                }
            }
#pragma unroll
            for (int b = 0; b < NQB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[b][i] = exp2_fast(fmaf(s[b][i], a.c, -lse[b])) * fmaf(dp[b][i], a.scale, delta[b]);   // scale dS
            if ((t + 1) * KT > n) {   // the last tile's rows past the end
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (t * KT + kb * 32 + reg_row(i) >= n)
#pragma unroll
                        for (int b = 0; b < NQB; ++b) s[b][i] = 0.0f;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                bf16x8 p[NQB][NS];
#pragma unroll
                for (int b = 0; b < NQB; ++b) to_operand(s[b], st, p[b]);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    bf16x8 f[NP];
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl) f[pl] = frags.cols(at, pl * KT * DP * 2, kb, st, d);
#pragma unroll
                    for (int b = 0; b < NQB; ++b) dq[d][b] = mma(f, p[b], dq[d][b]);
                }
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        const int r = r0 + 32 * b;
        if (r >= rows) continue;
        if (w.splits > 1) {
            const PartRow pr = part_row(a.parts, a.bhs, w.bh, rows, r);
            float* out = a.part + (pr.at + w.split * pr.step) * DP;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<f32x4*>(out + 32 * d + reg_row(i)) =
                        f32x4{dq[d][b][i], dq[d][b][i + 1], dq[d][b][i + 2], dq[d][b][i + 3]};
            continue;
        }
        const int tok = r / a.group, head = w.h * a.group + r - tok * a.group;
        T* row = static_cast<T*>(a.dq) + (((int64_t)w.b * a.nq + tok) * a.hq + head) * a.dim;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                store4<T>(row, 32 * d + reg_row(i), a.dim, dq[d][b][i], dq[d][b][i + 1], dq[d][b][i + 2], dq[d][b][i + 3]);
    }
}

// Valid keys, and query rows of a key head, up to which bfloat16 P and dS go into dV and dK as two planes.  With few keys delta
// takes away most of dP, and rounding what is left to 2^-9 puts dK up to 2.7e-3 off (its own rounding: 1.7e-3; 2.4e-3 with many
// keys); with few rows it does not average out (30 rows, 3035 keys: 2.5e-3).  A half more products, of problems whose
// launches and bytes take longer: 18000 queries x 300 keys x 8 heads x 64 65 -> 74 us, 10 queries x 18000 keys 28 -> 33.
constexpr int kFewKeys = 1024, kFewRows = 64;

// dK and dV: keys in the lanes (a wave owns NKB blocks of 32), S = Q K^T and dP = dO V^T, dV^T += dO^T P,
// dK^T += Q^T dS.  The queries of each query head that shares the key head pass by, head after head.
// NS: planes of P and dS in their products.  Where the mask decides on them (a.by_count: how many keys of a scene are valid is
// known here only) both kernels are launched, and a scene's workgroups of the one that it does not belong to end at once (the
// second launch: 4 us of 9000 x 12 x 64's step of 1210; 6 scenes with 300 valid keys of 3000, 8 x 64: 228 -> 239).
template <int NP, int NS, int DP, int KS, int NKB, int NW, int QT, typename T>
__global__ void __launch_bounds__(NW * 64, dkv_per_cu(NP, NS, DP)) k_attn_dkv(AttnBwd a) {
    static_assert(NW % 2 == 0, "waves in pairs load the statistics");
    constexpr int NT = NW * 64, QB = QT / 32, DB = DP / 32;
    typedef Tile<NP, DP, QT, NT> TileT;
    constexpr int kBuffers = buffers(2, TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    __shared__ __attribute__((aligned(16))) float stat[kBuffers][2][64];   // lse and -delta of the tile's rows
    static_assert(dkv_per_cu(NP, NS, DP) * (sizeof(lds) + sizeof(stat)) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int wave = g2v::uniform(threadIdx.x >> 6);
    const int j0 = (w.tile * NW + wave) * (NKB * 32) + (threadIdx.x & 31);
    const int n = a.count ? a.count[w.b] : a.nk;
    if (NP == 1 && a.by_count && (n <= kFewKeys) != (NS > NP)) return;
    const int per = (a.nq + QT - 1) / QT;     // tiles of a query head
    int u0, u1;
    split_range(per * a.group, w.split, w.splits, u0, u1);
    if (w.tile * (NW * NKB * 32) >= n) u1 = u0;    // no valid key: nothing to add up

    bf16x8 k[NKB][KS][NP], v[NKB][KS][NP];
#pragma unroll
    for (int b = 0; b < NKB; ++b) {
        const int j = j0 + 32 * b;
        const char* krow = a.k.p + w.b * a.k.sb + w.h * a.k.sh + j * a.k.sn;
        const char* vrow = a.v.p + w.b * a.v.sb + w.h * a.v.sh + j * a.v.sn;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int pl = 0; pl < NP; ++pl) {
                k[b][ks][pl] = mem_frag<DP>(krow, j < n, a.k.chunks, pl, ks);
                v[b][ks][pl] = mem_frag<DP>(vrow, j < n, a.v.chunks, pl, ks);
            }
    }

    TileT tile;
    tile.init(a.q);
    Frags<DP> frags;
    frags.init(lds_off(lds));
    if (a.q.chunks < TileT::C) clear_lds<NT>(&lds[0][0][0], sizeof(lds));
    auto load = [&](int u, int buf) {
        const int hd = u / per, t = u - hd * per, head = w.h * a.group + hd;
        const char* qbase = a.q.p + w.b * a.q.sb + head * a.q.sh;
        const char* gbase = a.g.p + w.b * a.g.sb + head * a.g.sh;
        if ((t + 1) * QT <= a.nq) {
            tile.load(qbase, a.q.sn, (int64_t)t * QT, lds_off(lds[buf][0]));
            tile.load(gbase, a.g.sn, (int64_t)t * QT, lds_off(lds[buf][1]));
        } else {
            tile.load_tail(qbase, a.q.sn, (int64_t)t * QT, a.nq, lds[buf][0]);
            tile.load_tail(gbase, a.g.sn, (int64_t)t * QT, a.nq, lds[buf][1]);
        }
        // rows past the end are there in the padded statistics: lse +inf makes their probabilities 0
        const int64_t at = ((int64_t)w.b * a.hq + head) * a.nqp + t * QT;
        // (even waves load lse and odd ones delta, each pair the same values: every wave has as many loads)
        const uint32_t lane = threadIdx.x & 63;
        if (lane < QT) dma4(((wave & 1) ? a.delta : a.lse) + at, lane * 4, lds_off(stat[buf][wave & 1]));
    };

    f32x16 dk[DB][NKB], dv[DB][NKB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < NKB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) dk[d][b][i] = dv[d][b][i] = 0.0f;
    if (u0 < u1) load(u0, 0);
    if (kAhead > 1 && u0 + 1 < u1) load(u0 + 1, 1);
    for (int u = u0, buf = 0; u < u1; ++u, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        next_tile<kBuffers, TileT::kLoads ? 2 * TileT::kLoads + 1 : 0>(u + 1 < u1 && ((u + 1) % per + 1) * QT <= a.nq);
        if (u + kAhead < u1) load(u + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
        const uint32_t at = buf * 2 * TileT::kBytes;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const int g4 = 4 * ((threadIdx.x >> 5) & 1);
            f32x16 s[NKB], dp[NKB];    // dP begins at -delta
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 de = *reinterpret_cast<const f32x4*>(&stat[buf][1][qb * 32 + 2 * i + g4]);
#pragma unroll
                for (int b = 0; b < NKB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[b][i + j] = 0.0f;
                        dp[b][i + j] = de[j];
                    }
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 fq[NP], fg[NP];
#pragma unroll
                for (int pl = 0; pl < NP; ++pl) {
                    fq[pl] = frags.rows(at, pl * QT * DP * 2, qb, ks);
                    fg[pl] = frags.rows(at, TileT::kBytes + pl * QT * DP * 2, qb, ks);
                }
#pragma unroll
                for (int b = 0; b < NKB; ++b) {
                    s[b] = mma(fq, k[b][ks], s[b]);
                    dp[b] = mma(fg, v[b][ks], dp[b]);
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 ls = *reinterpret_cast<const f32x4*>(&stat[buf][0][qb * 32 + 2 * i + g4]);
#pragma unroll
                for (int b = 0; b < NKB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[b][i + j] = exp2_fast(fmaf(s[b][i + j], a.c, -ls[j]));
                        dp[b][i + j] *= s[b][i + j];
                    }
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                bf16x8 p[NKB][NS], ds[NKB][NS];
#pragma unroll
                for (int b = 0; b < NKB; ++b) {
                    to_operand(s[b], st, p[b]);
                    to_operand(dp[b], st, ds[b]);
                }
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    bf16x8 fg[NP], fq[NP];
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl) {
                        fg[pl] = frags.cols(at, TileT::kBytes + pl * QT * DP * 2, qb, st, d);
                        fq[pl] = frags.cols(at, pl * QT * DP * 2, qb, st, d);
                    }
#pragma unroll
                    for (int b = 0; b < NKB; ++b) {
                        dv[d][b] = mma(fg, p[b], dv[d][b]);
                        dk[d][b] = mma(fq, ds[b], dk[d][b]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NKB; ++b) {
        const int j = j0 + 32 * b;
        if (j >= a.nk) continue;
        if (w.splits > 1) {
            if (j >= n) continue;   // k_attn_dkv_join writes zeros without looking
            const PartRow pr = part_row(a.parts, a.bhs, w.bh, a.nk, j);
            float* out = a.part + (pr.at + w.split * pr.step) * (2 * DP);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    *reinterpret_cast<f32x4*>(out + 32 * d + reg_row(i)) =
                        f32x4{dk[d][b][i], dk[d][b][i + 1], dk[d][b][i + 2], dk[d][b][i + 3]};
                    *reinterpret_cast<f32x4*>(out + DP + 32 * d + reg_row(i)) =
                        f32x4{dv[d][b][i], dv[d][b][i + 1], dv[d][b][i + 2], dv[d][b][i + 3]};
                }
            continue;
        }
        const bool valid = j < n;   // a masked key's gradients are zero, whatever its row holds
        const int64_t key = a.list ? a.list[(int64_t)w.b * a.nk + j] : j;
        const int64_t at = (((int64_t)w.b * a.nk + key) * a.hk + w.h) * a.dim;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                float x[4], y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = valid && n > 1 ? dk[d][b][i + e] * a.scale : 0.0f;   // one key: its probability is 1
                    y[e] = valid ? dv[d][b][i + e] : 0.0f;
                }
                store4<T>(static_cast<T*>(a.dk) + at, 32 * d + reg_row(i), a.dim, x[0], x[1], x[2], x[3]);
                store4<T>(static_cast<T*>(a.dv) + at, 32 * d + reg_row(i), a.dim, y[0], y[1], y[2], y[3]);
            }
    }
}

// Sums of the splits: each of `parts` threads every parts-th, then in their order.
__device__ __forceinline__ f32x4 join_sum(const float* part, int64_t stride, int splits, int parts, bool live, float (*red)[256]) {
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    const int mine = threadIdx.x % parts;
    if (live) {
#pragma unroll 4
        for (int s = mine; s < splits; s += parts) o += *reinterpret_cast<const f32x4*>(part + s * stride);
    }
    if (parts > 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) red[j][threadIdx.x] = o[j];
        __syncthreads();
        if (mine == 0)
            for (int k = 1; k < parts; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] += red[j][threadIdx.x + k];
    }
    return o;
}

template <int DP, typename T>
__global__ void __launch_bounds__(256) k_attn_dq_join(AttnBwd a, int parts) {
    constexpr int kLanes = DP / 4;
    __shared__ float red[4][256];
    const int rows = a.group * a.nq, from = joined_from(a.parts, rows), own = rows - from, per = 256 / (kLanes * parts);
    const int e = threadIdx.x / parts, d = e % kLanes * 4;
    const int at = blockIdx.x * per + e / kLanes;
    const bool live = e / kLanes < per && at < a.bhs * own;
    const int bh = live ? at / own : 0, r = live ? from + at - bh * own : from;
    const PartRow pr = part_row(a.parts, a.bhs, bh, rows, r);
    const f32x4 o = join_sum(a.part + pr.at * DP + d, pr.step * DP, pr.splits, parts, live, red);
    if (!live || threadIdx.x % parts) return;
    const int b = bh / a.hk, tok = r / a.group, head = (bh % a.hk) * a.group + r % a.group;
    T* row = static_cast<T*>(a.dq) + (((int64_t)b * a.nq + tok) * a.hq + head) * a.dim;
    store4<T>(row, d, a.dim, o[0], o[1], o[2], o[3]);
}

template <int DP, typename T>
__global__ void __launch_bounds__(256) k_attn_dkv_join(AttnBwd a, int parts) {
    constexpr int kLanes = DP / 2;    // dK, then dV
    __shared__ float red[4][256];
    const int from = joined_from(a.parts, a.nk), own = a.nk - from, per = 256 / (kLanes * parts);
    const int e = threadIdx.x / parts, d = e % kLanes * 4;
    const int at = blockIdx.x * per + e / kLanes;
    const bool live = e / kLanes < per && at < a.bhs * own;
    const int bh = live ? at / own : 0, j = live ? from + at - bh * own : from, b = bh / a.hk;
    const int n = a.count ? a.count[b] : a.nk;
    const bool some = j < n && (n > 1 || d >= DP);    // one key: its probability is 1 whatever k is
    const PartRow pr = part_row(a.parts, a.bhs, bh, a.nk, j);
    const f32x4 o = join_sum(a.part + pr.at * (2 * DP) + d, pr.step * (2 * DP), pr.splits, parts, live && some, red);
    if (!live || threadIdx.x % parts) return;
    const int64_t key = a.list ? a.list[(int64_t)b * a.nk + j] : j;
    const float f = d < DP ? a.scale : 1.0f;
    T* row = static_cast<T*>(d < DP ? a.dk : a.dv) + (((int64_t)b * a.nk + key) * a.hk + bh % a.hk) * a.dim;
    store4<T>(row, d < DP ? d : d - DP, a.dim, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
}

// -delta = -sum_d dO O of a row and its lse, both padded to nqp rows of a head.  2^shift lanes a row, 16 bytes each.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_delta(int64_t rows, int nq, int nqp, int heads, int dim, int shift, const T* out,
                                                    const T* rest, const T* g, int64_t gsb, int64_t gsn, int64_t gsh,
                                                    const float* lse, float* lse_p, float* delta) {
    constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    const int64_t e = (int64_t)blockIdx.x * (256 >> shift) + (threadIdx.x >> shift);
    if (e >= rows) return;      // the same for all lanes of a row
    const int d = (threadIdx.x & ((1 << shift) - 1)) * N;
    const int64_t bh = e / nqp;
    const int i = (int)(e % nqp);
    const int64_t b = bh / heads, h = bh % heads;
    float v = 0.0f;
    if (i < nq) {
        const int64_t at = ((b * nq + i) * heads + h) * dim + d;
        const T* r = g + b * gsb + i * gsn + h * gsh + d;
        if (d + N <= dim) {
            const vec x = *reinterpret_cast<const vec*>(out + at), y = *reinterpret_cast<const vec*>(r);
            vec l;
            if (rest) l = *reinterpret_cast<const vec*>(rest + at);
#pragma unroll
            for (int j = 0; j < N; ++j) v = fmaf(rest ? (float)x[j] + (float)l[j] : (float)x[j], (float)y[j], v);
        } else {
            for (int j = 0; d + j < dim; ++j)
                v = fmaf(rest ? (float)out[at + j] + (float)rest[at + j] : (float)out[at + j], (float)r[j], v);
        }
    }
    for (int m = (1 << shift) >> 1; m > 0; m >>= 1) v += __shfl_xor(v, m);
    if (d == 0) {
        delta[e] = -v;
        lse_p[e] = i < nq ? lse[bh * nq + i] : INFINITY;
    }
}

template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
hipError_t dq_launch(const AttnBwd& a, hipStream_t s) {
    G2V_LAUNCH((k_attn_dq<NP, DP, KS, NQB, NW, KT, T>), dim3((unsigned)workgroups(a.parts, a.bhs)), dim3(NW * 64), 0, s, a);
    const int64_t rows = (int64_t)a.bhs * (a.group * a.nq - joined_from(a.parts, a.group * a.nq));
    if (rows > 0) {
        const int parts = attn_join_parts(rows, DP / 4, std::max(a.parts.head_splits, a.parts.splits));
        G2V_LAUNCH((k_attn_dq_join<DP, T>), dim3((unsigned)ceil_div(rows, 256 / (DP / 4 * parts))), dim3(256), 0, s, a, parts);
    }
    return hipGetLastError();
}
template <int NP, int NS, int DP, int NKB, int NW, int QT, typename T>
void dkv_kernel(const AttnBwd& a, hipStream_t s) {
    const dim3 grid((unsigned)workgroups(a.parts, a.bhs)), block(NW * 64);
    if (a.dim > DP - 16) G2V_LAUNCH((k_attn_dkv<NP, NS, DP, DP / 16, NKB, NW, QT, T>), grid, block, 0, s, a);
    else G2V_LAUNCH((k_attn_dkv<NP, NS, DP, DP / 16 - 1, NKB, NW, QT, T>), grid, block, 0, s, a);
}

template <int NP, int DP, int NQB, int KT, typename T>
hipError_t dq_waves(const AttnBwd& a, const AttnShape& g, hipStream_t s) {
    const bool full = a.dim > DP - 16;
    if constexpr (NP == 1)
        if (g.waves == 1)
            return full ? dq_launch<NP, DP, DP / 16, 1, 1, KT, T>(a, s) : dq_launch<NP, DP, DP / 16 - 1, 1, 1, KT, T>(a, s);
    return full ? dq_launch<NP, DP, DP / 16, NQB, 4, KT, T>(a, s) : dq_launch<NP, DP, DP / 16 - 1, NQB, 4, KT, T>(a, s);
}

template <int NP, int DP, int NKB, int NW, int QT, typename T>
hipError_t dkv_launch(AttnBwd& a, hipStream_t s) {
    const int planes = attn_dkv_planes(NP > 1, a.nk, (int64_t)a.group * a.nq);
    a.by_count = planes == 1 && a.count;
    if constexpr (NP == 1)
        if (planes == 2 || a.by_count) dkv_kernel<NP, 2, DP, NKB, NW, QT, T>(a, s);
    if (planes == NP) dkv_kernel<NP, NP, DP, NKB, NW, QT, T>(a, s);
    const int64_t rows = (int64_t)a.bhs * (a.nk - joined_from(a.parts, a.nk));
    if (rows > 0) {
        const int parts = attn_join_parts(rows, DP / 2, std::max(a.parts.head_splits, a.parts.splits));
        G2V_LAUNCH((k_attn_dkv_join<DP, T>), dim3((unsigned)ceil_div(rows, 256 / (DP / 2 * parts))), dim3(256), 0, s, a, parts);
    }
    return hipGetLastError();
}

}  // namespace

AttnShape attn_dq_shape(bool f32, int dp, int64_t rows) {
    AttnShape g;
    g.waves = !f32 && rows <= 32 ? 1 : 4;    // as in attn_fwd_shape
    g.blocks = g.waves == 4 && !f32 && dp <= 64 ? 2 : 1;
    g.tile = f32 && dp > 32 ? 32 : 64;
    g.per_cu = dq_per_cu(f32 ? 3 : 1, dp, g.waves);
    g.products = f32 ? 3 : 4;    // bfloat16: dS as two planes
    return g;
}
int attn_dkv_planes(bool f32, int64_t nk, int64_t rows) {
    return f32 ? 3 : nk <= kFewKeys || rows <= kFewRows ? 2 : 1;
}
AttnShape attn_dkv_shape(bool f32, int dp, int planes) {
    AttnShape g;
    g.waves = 4;
    g.blocks = 1;
    g.tile = (f32 && dp > 32) || dp > 96 ? 32 : 64;
    g.per_cu = dkv_per_cu(f32 ? 3 : 1, planes, dp);
    g.products = f32 ? 4 : 2 + 2 * planes;
    return g;
}

hipError_t launch_attn_dq(const AttnBwd& a, bool f32, int dp, hipStream_t s) {
    const AttnShape g = attn_dq_shape(f32, dp, (int64_t)a.group * a.nq);
    if (f32) {
        switch (dp) {
            case 32: return dq_waves<3, 32, 1, 64, float>(a, g, s);
            case 64: return dq_waves<3, 64, 1, 32, float>(a, g, s);
            case 96: return dq_waves<3, 96, 1, 32, float>(a, g, s);
            default: return dq_waves<3, 128, 1, 32, float>(a, g, s);
        }
    }
    switch (dp) {
        case 32: return dq_waves<1, 32, 2, 64, __bf16>(a, g, s);
        case 64: return dq_waves<1, 64, 2, 64, __bf16>(a, g, s);
        case 96: return dq_waves<1, 96, 1, 64, __bf16>(a, g, s);
        default: return dq_waves<1, 128, 1, 64, __bf16>(a, g, s);
    }
}

hipError_t launch_attn_dkv(const AttnBwd& args, bool f32, int dp, hipStream_t s) {
    AttnBwd a = args;
    if (f32) {
        switch (dp) {
            case 32: return dkv_launch<3, 32, 1, 4, 64, float>(a, s);
            case 64: return dkv_launch<3, 64, 1, 4, 32, float>(a, s);
            case 96: return dkv_launch<3, 96, 1, 4, 32, float>(a, s);
            default: return dkv_launch<3, 128, 1, 4, 32, float>(a, s);
        }
    }
    switch (dp) {
        case 32: return dkv_launch<1, 32, 1, 4, 64, __bf16>(a, s);
        case 64: return dkv_launch<1, 64, 1, 4, 64, __bf16>(a, s);
        case 96: return dkv_launch<1, 96, 1, 4, 64, __bf16>(a, s);
        default: return dkv_launch<1, 128, 1, 4, 32, __bf16>(a, s);
    }
}

hipError_t launch_attn_delta(int batch, int nq, int nqp, int heads, int dim, const void* out, const void* rest, const void* g,
                             int64_t gsb, int64_t gsn, int64_t gsh, bool f32, const float* lse, float* lse_p, float* delta, hipStream_t s) {
    const int64_t rows = (int64_t)batch * heads * nqp;
    if (rows == 0) return hipSuccess;
    int shift = 0;
    while ((f32 ? 4 : 8) << shift < dim) ++shift;
    const dim3 grid((unsigned)ceil_div(rows, 256 >> shift));
    if (f32)
        G2V_LAUNCH((k_attn_delta<float>), grid, dim3(256), 0, s, rows, nq, nqp, heads, dim, shift, static_cast<const float*>(out),
                   static_cast<const float*>(nullptr), static_cast<const float*>(g), gsb, gsn, gsh, lse, lse_p, delta);
    else
        G2V_LAUNCH((k_attn_delta<__bf16>), grid, dim3(256), 0, s, rows, nq, nqp, heads, dim, shift,
                   static_cast<const __bf16*>(out), static_cast<const __bf16*>(rest), static_cast<const __bf16*>(g), gsb, gsn,
                   gsh, lse, lse_p, delta);
    return hipGetLastError();
}

}  // namespace g2v
