// Attention within a window, backward (g2v_attention_window.h).
#include <algorithm>

#include "g2v_attention_window.h"

namespace g2v {
namespace {
using namespace attn;

// Workgroups that share a CU, as in g2v_attention.h, at one block of rows a wave.
constexpr int window_dq_per_cu(int np, int dp, int waves) {
    return np == 1 && waves > 1 && dp <= 64 ? (dp == 32 ? 4 : 3) : dq_per_cu(np, dp, waves);
}

// As k_attn_dq.
template <int NP, int DP, int KS, int NW, int KT, typename T>
__global__ void __launch_bounds__(NW * 64, launch_bound(NW, window_dq_per_cu(NP, DP, NW))) k_window_dq(WinBwd a) {
    constexpr int NS = NP == 1 ? 2 : NP;    // planes of dS, see k_attn_dq
    constexpr int NT = NW * 64, KB = KT / 32, DB = DP / 32;
    typedef WinTile<NP, DP, KT, NT> TileT;
    typedef TileWords<KT> Words;
    constexpr int kBuffers = buffers(window_dq_per_cu(NP, DP, NW), TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    static_assert(window_dq_per_cu(NP, DP, NW) * sizeof(lds) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int rows = a.group * a.nq, half = (threadIdx.x >> 5) & 1;
    const int first = (w.tile * NW + g2v::uniform(threadIdx.x >> 6)) * 32, r = first + (threadIdx.x & 31);
    const int g0 = w.tile * (NW * 32), g1 = min(g0 + NW * 32, rows) - 1;
    const char* kbase = a.k.p + w.b * a.k.sb + w.h * a.k.sh;
    const char* vbase = a.v.p + w.b * a.v.sb + w.h * a.v.sh;
    KeyTiles<KT> tiles;
    tiles.init(a.win, a.nk, g2v::uniform(g0 / a.group), g2v::uniform(g1 / a.group));
    int u0, u1;
    split_range(tiles.all, w.split, w.splits, u0, u1);
    if (!a.dq) u1 = u0;    // delta alone
    WaveBlocks blocks;
    blocks.init(a.win, a.nk, a.group, rows, first, tiles.sinks * KT);

    bf16x8 q[KS][NP], g[KS][NP];
    float lse, delta;    // delta = sum_d dO O, negative and times scale
    RowValues<KS, T> out, rest;
    const int rc = r < rows ? r : rows - 1;
    const int tok = rc / a.group, head = w.h * a.group + rc - tok * a.group;
    const char* qrow = a.q.p + w.b * a.q.sb + tok * a.q.sn + head * a.q.sh;
    const char* grow = a.g.p + w.b * a.g.sb + tok * a.g.sn + head * a.g.sh;
    const KeyRange see = key_range(a.win, a.nk, tok);
    load_row<DP>(qrow, a.q.chunks, q);
    load_row<DP>(grow, a.g.chunks, g);
    lse = a.lse_in[((int64_t)w.b * a.hq + head) * a.nq + tok];
    const int64_t orow = (((int64_t)w.b * a.nq + tok) * a.hq + head) * a.dim;
    out.load(static_cast<const T*>(a.out) + orow, a.dim);
    if (sizeof(T) == 2 && a.rest) rest.load(static_cast<const T*>(a.rest) + orow, a.dim);

    TileT ktile, vtile;
    ktile.init(a.k);
    vtile.init(a.v);
    Frags<DP> frags;
    frags.init(lds_off(lds));
    Words words;
    words.init(a.win, a.nk);
    const char* kfar = kbase + (int64_t)a.win.skip * a.k.sn;
    const char* vfar = vbase + (int64_t)a.win.skip * a.v.sn;
    auto load = [&](int u, int buf) __attribute__((always_inline)) {
        const int t = tiles.at(u), j0 = t * KT;
        if (words.all(t)) {
            ktile.load(a.k, kfar + (int64_t)j0 * a.k.sn, lds_off(lds[buf][0]));
            vtile.load(a.v, vfar + (int64_t)j0 * a.v.sn, lds_off(lds[buf][1]));
            return Words::kAll;
        }
        const uint64_t word = words.at(a.win, tiles, a.nk, w.b, u, u1);
        TileT::load_some(a.k, kbase, j0, word, a.win.sinks, a.win.skip, lds[buf][0]);
        TileT::load_some(a.v, vbase, j0, word, a.win.sinks, a.win.skip, lds[buf][1]);
        return word;
    };
    uint64_t word = 0, next = 0, after = 0;
    if (u0 < u1) word = load(u0, 0);
    settle_row(r < rows, a.q.chunks, q);
    settle_row(r < rows, a.g.chunks, g);
    asm volatile("" : "+v"(lse));
    float sum = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        f32x8 o = out.at(ks, a.dim);
        if (sizeof(T) == 2 && a.rest) o += rest.at(ks, a.dim);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float x = (float)g[ks][0][j];
#pragma unroll
            for (int pl = 1; pl < NP; ++pl) x += (float)g[ks][pl][j];
            sum = fmaf(o[j], x, sum);
        }
    }
    sum = half_sum(sum);
    delta = -sum * a.scale;
    if (w.split == 0 && half == 0 && r < rows) {
        const int64_t at = ((int64_t)w.b * a.hq + head) * a.nqp + tok;
        a.lse_pad[at] = lse;
        a.delta_pad[at] = -sum;
    }
    if (w.split == 0 && (w.tile + 1) * (NW * 32) >= rows) {    // the heads' padding
        const int pad = a.nqp - a.nq;
        for (int i = threadIdx.x; i < a.group * pad; i += NT) {
            const int64_t at = ((int64_t)w.b * a.hq + w.h * a.group + i / pad) * a.nqp + a.nq + i % pad;
            a.lse_pad[at] = INFINITY;
            a.delta_pad[at] = 0.0f;
        }
    }
    if (!a.dq) return;    // dK and dV alone are wanted

    f32x16 dq[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[d][i] = 0.0f;
    if (kAhead > 1 && u0 + 1 < u1) next = load(u0 + 1, 1);
    for (int u = u0, buf = 0; u < u1; ++u, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        next_tile<kBuffers, 2 * TileT::kLoads>(u + 1 < u1 && words.all(tiles.at(u + 1)));
        after = 0;
        if (u + kAhead < u1) {
            const uint64_t x = load(u + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
            if (kAhead > 1) after = x;
            else next = x;
        }
        const uint32_t at = buf * 2 * TileT::kBytes;
        const int j0 = tiles.at(u) * KT;
        const bool far = u < tiles.sinks;
        const WaveBlocks::Range some = far ? blocks.any_far : blocks.any, every = far ? blocks.every_far : blocks.every;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const uint32_t part = (uint32_t)(word >> (32 * kb));
            const int jb = j0 + 32 * kb;
            if (!some.has(jb) || !part) continue;
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 fk[NP], fv[NP];
#pragma unroll
                for (int pl = 0; pl < NP; ++pl) {
                    fk[pl] = frags.rows(at, pl * KT * DP * 2, kb, ks);
                    fv[pl] = frags.rows(at, TileT::kBytes + pl * KT * DP * 2, kb, ks);
                }
                s = mma(fk, q[ks], s);
                dp = mma(fv, g[ks], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = exp2_fast(fmaf(s[i], a.c, -lse)) * fmaf(dp[i], a.scale, delta);   // scale dS
            if (!every.has(jb) || part != ~0u) {
                const uint32_t x = (seen_bits(see, a.win.sinks, jb) & part) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = or_zero(spread_bit(x, 8 * (i >> 2) + (i & 3)), s[i]);
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                bf16x8 p[NS];
                to_operand(s, st, p);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    bf16x8 f[NP];
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl) f[pl] = frags.cols(at, pl * KT * DP * 2, kb, st, d);
                    dq[d] = mma(f, p, dq[d]);
                }
            }
        }
        word = next;
        next = after;
    }
    if (r >= rows) return;
    // one key: its probability is 1 whatever q is
    const bool one = see.hi - see.lo + min(a.win.sinks, see.lo) < 2;
    if (one)
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[d][i] = 0.0f;
    if (w.splits > 1) {
        const PartRow pr = part_row(a.parts, a.bhs, w.bh, rows, r);
        float* out = a.part + (pr.at + w.split * pr.step) * DP;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(out + 32 * d + reg_row(i)) =
                    f32x4{dq[d][i], dq[d][i + 1], dq[d][i + 2], dq[d][i + 3]};
        return;
    }
    T* row = static_cast<T*>(a.dq) + (((int64_t)w.b * a.nq + tok) * a.hq + head) * a.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = dq[d][i];
        store_block<T>(row, 32 * d, a.dim, x);
    }
}

// Two workgroups a CU from 64 channels on: three spill where P and dS are in one plane (18,000 x 16 x 64, 1025 keys a window, 266 us
// for 176).  At 32 channels four, or three where they are in two planes, with which four spill (60,000 x 16 x 32, 513 keys, 323 us for
// 296).  The sinks' one-wave workgroups: as many as their tiles' LDS allows.
constexpr int window_dkv_per_cu(int np, int ns, int dp, int nw) {
    if (nw > 1) return np > 1 ? dkv_per_cu(np, ns, dp) : dp >= 64 ? 2 : ns > 1 ? 3 : 4;
    if (np > 1) return dp > 96 ? 1 : dp > 64 ? 2 : dp > 32 ? 3 : 6;
    return dp > 64 ? 3 : dp > 32 ? 6 : 8;
}
constexpr int dkv_bound(int np, int ns, int dp, int nw) { return nw > 1 ? window_dkv_per_cu(np, ns, dp, nw) : np > 1 && dp > 32 ? 1 : 2; }

// As k_attn_dkv: keys in the lanes, the queries that see any of the workgroup's keys pass by, head after head.  NS: planes of P and dS,
// as there.  (P in one plane throughout is less work, 200,000 x 8 heads x 64, 513 keys a window 820 -> 706 us, and puts dV 2.3e-3 off
// where its own rounding is 1.7e-3.)
template <int NP, int NS, int DP, int KS, int NW, int QT, typename T>
__global__ void __launch_bounds__(NW * 64, dkv_bound(NP, NS, DP, NW)) k_window_dkv(WinBwd a) {
    static_assert(NW == 1 || NW % 2 == 0, "waves in pairs load the statistics, or one does");
    constexpr int NT = NW * 64, QB = QT / 32, DB = DP / 32;
    typedef WinTile<NP, DP, QT, NT> TileT;
    constexpr int kBuffers = NP > 1 && NW == 1 ? 2 : buffers(2, TileT::kBytes), kAhead = kBuffers - 1;
    constexpr int kStats = NW == 1 ? 2 : 1;    // loads of statistics a wave
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    __shared__ __attribute__((aligned(16))) float stat[kBuffers][2][64];   // lse and -delta of the tile's rows
    static_assert(window_dkv_per_cu(NP, NS, DP, NW) * (sizeof(lds) + sizeof(stat)) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int wave = g2v::uniform(threadIdx.x >> 6), half = (threadIdx.x >> 5) & 1;
    const int n = a.all_queries ? min(a.win.sinks, a.nk) : a.nk;
    const int g0 = w.tile * (NW * 32), g1 = min(g0 + NW * 32, n) - 1;    // the workgroup's keys, the wave's and the lane's
    const int first = g0 + wave * 32, last = min(first + 32, n) - 1, j = first + (threadIdx.x & 31);
    auto from = [&](int key) { return min(max(key - a.win.right - a.win.shift, 0), a.nq); };    // queries [from, to) see a key
    auto to = [&](int key) {
        return a.all_queries ? a.nq : min(max(key + a.win.left - a.win.shift + 1, 0), a.nq);
    };
    const int q0 = g2v::uniform(from(g0)), q1 = g2v::uniform(to(g1));
    const int tile0 = q0 / QT, per = q0 < q1 ? (q1 + QT - 1) / QT - tile0 : 0;     // tiles of a query head
    int u0, u1;
    split_range(per * a.group, w.split, w.splits, u0, u1);
    const int k0 = from(j), k1 = to(j);
    bool valid = j < n && k0 < k1;    // (rows that no query sees are not read either)
    if (valid && a.win.mask) valid = a.win.mask[grad_row(a, w.b, j)];
    // blocks of 32 queries of which any sees one of the wave's keys, and those that see all of them
    WaveBlocks::Range any = {0, 0u}, every = {0, 0u};
    if (__any(valid)) {
        const int w0 = g2v::uniform(from(first)), w1 = g2v::uniform(to(last)), w2 = g2v::uniform(from(last)), w3 = g2v::uniform(to(first));
        if (w1 > w0) any = {w0 - 31, (uint32_t)(w1 - w0 + 31)};
        if (w3 - 31 > w2) every = {w2, (uint32_t)(w3 - 31 - w2)};
    }
    if (a.win.mask && !__syncthreads_or(valid)) u1 = u0;    // nothing to add up

    bf16x8 k[KS][NP], v[KS][NP];
    {
        const int64_t row = j + (j >= a.win.sinks ? a.win.skip : 0);
        const char* krow = a.k.p + w.b * a.k.sb + w.h * a.k.sh + row * a.k.sn;
        const char* vrow = a.v.p + w.b * a.v.sb + w.h * a.v.sh + row * a.v.sn;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int pl = 0; pl < NP; ++pl) k[ks][pl] = v[ks][pl] = __builtin_bit_cast(bf16x8, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        if (valid) {
            load_row<DP>(krow, a.k.chunks, k);
            load_row<DP>(vrow, a.v.chunks, v);
        }
    }

    TileT qtile, gtile;
    qtile.init(a.q);
    gtile.init(a.g);
    Frags<DP> frags;
    frags.init(lds_off(lds));
    // unit u is tile `at` of the head's `per` tiles; the loads' place and the products' step through them without a division
    struct Place {
        int head, at;
    };
    auto step = [](Place& p, int per) __attribute__((always_inline)) {
        if (++p.at == per) {
            p.at = 0;
            ++p.head;
        }
    };
    const int skip = per ? g2v::uniform(u0 / per) : 0;
    Place here = {w.h * a.group + skip, u0 - skip * per}, there = here;
    auto load = [&](int buf) __attribute__((always_inline)) {
        const int t = tile0 + there.at, head = there.head;
        const char* qbase = a.q.p + w.b * a.q.sb + head * a.q.sh;
        const char* gbase = a.g.p + w.b * a.g.sb + head * a.g.sh;
        if ((t + 1) * QT <= a.nq) {
            qtile.load(a.q, qbase + (int64_t)t * QT * a.q.sn, lds_off(lds[buf][0]));
            gtile.load(a.g, gbase + (int64_t)t * QT * a.g.sn, lds_off(lds[buf][1]));
        } else {
            TileT::load_tail(a.q, qbase, t * QT, a.nq, lds_off(lds[buf][0]));
            TileT::load_tail(a.g, gbase, t * QT, a.nq, lds_off(lds[buf][1]));
        }
        step(there, per);
        // rows past the end are there in the padded statistics: lse +inf makes their probabilities 0
        const int64_t at = ((int64_t)w.b * a.hq + head) * a.nqp + t * QT;
        const uint32_t lane = threadIdx.x & 63;
        if constexpr (NW == 1) {
            if (lane < QT) {
                dma4(a.lse + at, lane * 4, lds_off(stat[buf][0]));
                dma4(a.delta + at, lane * 4, lds_off(stat[buf][1]));
            }
        } else {    // even waves load lse and odd ones delta, each pair the same values: every wave has as many loads
            if (lane < QT) dma4(((wave & 1) ? a.delta : a.lse) + at, lane * 4, lds_off(stat[buf][wave & 1]));
        }
    };

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dk[d][i] = dv[d][i] = 0.0f;
    if (u0 < u1) load(0);
    settle_row(valid, a.k.chunks, k);
    settle_row(valid, a.v.chunks, v);
    if (kAhead > 1 && u0 + 1 < u1) load(1);
    for (int u = u0, buf = 0; u < u1; ++u, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        next_tile<kBuffers, TileT::kLoads ? 2 * TileT::kLoads + kStats : 0>(u + 1 < u1);
        if (u + kAhead < u1) load(buf == 0 ? kBuffers - 1 : buf - 1);
        const uint32_t at = buf * 2 * TileT::kBytes;
        const int i0 = (tile0 + here.at) * QT;
        step(here, per);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const int ib = i0 + 32 * qb;
            if (!any.has(ib)) continue;
            const int g4 = 4 * half;
            f32x16 s, dp;    // dP begins at -delta
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 de = *reinterpret_cast<const f32x4*>(&stat[buf][1][qb * 32 + 2 * i + g4]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[i + e] = 0.0f;
                    dp[i + e] = de[e];
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
                s = mma(fq, k[ks], s);
                dp = mma(fg, v[ks], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4 ls = *reinterpret_cast<const f32x4*>(&stat[buf][0][qb * 32 + 2 * i + g4]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i + e] = exp2_fast(fmaf(s[i + e], a.c, -ls[e]));
            }
            if (!every.has(ib)) {
                const uint32_t x = (bits_below(k1 - ib) & ~bits_below(k0 - ib)) >> g4;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = or_zero(spread_bit(x, 8 * (i >> 2) + (i & 3)), s[i]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] *= s[i];
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                bf16x8 p[NS], ds[NS];
                to_operand(s, st, p);
                to_operand(dp, st, ds);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    bf16x8 fg[NP], fq[NP];
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl) {
                        fg[pl] = frags.cols(at, TileT::kBytes + pl * QT * DP * 2, qb, st, d);
                        fq[pl] = frags.cols(at, pl * QT * DP * 2, qb, st, d);
                    }
                    dv[d] = mma(fg, p, dv[d]);
                    dk[d] = mma(fq, ds, dk[d]);
                }
            }
        }
    }
    if (j >= n) return;
    if (!valid) {    // a masked key's gradients are zero
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) dk[d][i] = dv[d][i] = 0.0f;
    }
    if (w.splits > 1) {
        const PartRow pr = part_row(a.parts, a.bhs, w.bh, n, j);
        float* out = a.part + (pr.at + w.split * pr.step) * (2 * DP);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                *reinterpret_cast<f32x4*>(out + 32 * d + reg_row(i)) = f32x4{dk[d][i], dk[d][i + 1], dk[d][i + 2], dk[d][i + 3]};
                *reinterpret_cast<f32x4*>(out + DP + 32 * d + reg_row(i)) =
                    f32x4{dv[d][i], dv[d][i + 1], dv[d][i + 2], dv[d][i + 3]};
            }
        return;
    }
    const int64_t at = (grad_row(a, w.b, j) * a.hk + w.h) * a.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        float x[16], y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = dk[d][i] * a.scale;
            y[i] = dv[d][i];
        }
        store_block<T>(static_cast<T*>(a.dk) + at, 32 * d, a.dim, x);
        store_block<T>(static_cast<T*>(a.dv) + at, 32 * d, a.dim, y);
    }
}

// Sums of the splits of the sinks' gradients, in a fixed order (k_attn_dkv_join's way, over the first n keys).
template <int DP, typename T>
__global__ void __launch_bounds__(256) k_window_sinks_join(WinBwd a, int n, int parts) {
    constexpr int kLanes = DP / 2;    // dK, then dV
    __shared__ float red[4][256];
    const int per = 256 / (kLanes * parts), e = threadIdx.x / parts, d = e % kLanes * 4, at = blockIdx.x * per + e / kLanes;
    const bool live = e / kLanes < per && at < a.bhs * n;
    const int bh = live ? at / n : 0, j = live ? at - bh * n : 0, b = bh / a.hk;
    const PartRow pr = part_row(a.parts, a.bhs, bh, n, j);
    const f32x4 o = join_sum(a.part + pr.at * (2 * DP) + d, pr.step * (2 * DP), pr.splits, parts, live, red);
    if (!live || threadIdx.x % parts) return;
    const float f = d < DP ? a.scale : 1.0f;
    T* row = static_cast<T*>(d < DP ? a.dk : a.dv) + (grad_row(a, b, j) * a.hk + bh % a.hk) * a.dim;
    store4<T>(row, d < DP ? d : d - DP, a.dim, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
}

// Zeros in the rows of dk and dv that are no query's (grid y: which): `each` values of a scene, 16 bytes a thread at any alignment.
template <typename T>
__global__ void __launch_bounds__(256) k_window_zeros(WinBwd a, int64_t each, int64_t blocks) {
    constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    const int64_t b = blockIdx.x / blocks, at = ((blockIdx.x - b * blocks) * 256 + threadIdx.x) * N;
    T* row = static_cast<T*>(blockIdx.y ? a.dv : a.dk) + ((b * (a.nk + a.gap) + a.gap_at) * a.hk) * a.dim;
    if (at + N <= each) {
        vec zero;
#pragma unroll
        for (int j = 0; j < N; ++j) zero[j] = (T)0.0f;
        *reinterpret_cast<vec*>(row + at) = zero;
    } else {
        for (int64_t j = at; j < each; ++j) row[j] = (T)0.0f;
    }
}

template <int NP, int DP, int KS, int NW, int KT, typename T>
hipError_t dq_launch(const WinBwd& a, hipStream_t s) {
    G2V_LAUNCH((k_window_dq<NP, DP, KS, NW, KT, T>), dim3((unsigned)workgroups(a.parts, a.bhs)), dim3(NW * 64), 0, s, a);
    return a.dq ? launch_attn_dq_join(a, NP > 1, DP, s) : hipGetLastError();
}
template <int NP, int DP, int KT, typename T>
hipError_t dq_waves(const WinBwd& a, const AttnShape& g, hipStream_t s) {
    const bool full = a.dim > DP - 16;
    if constexpr (NP == 1)
        if (g.waves == 1)
            return full ? dq_launch<NP, DP, DP / 16, 1, KT, T>(a, s) : dq_launch<NP, DP, DP / 16 - 1, 1, KT, T>(a, s);
    return full ? dq_launch<NP, DP, DP / 16, 4, KT, T>(a, s) : dq_launch<NP, DP, DP / 16 - 1, 4, KT, T>(a, s);
}

template <int NP, int NS, int DP, int NW, int QT, typename T>
hipError_t dkv_launch(const WinBwd& a, hipStream_t s) {
    const dim3 grid((unsigned)workgroups(a.parts, a.bhs)), block(NW * 64);
    if (a.dim > DP - 16) G2V_LAUNCH((k_window_dkv<NP, NS, DP, DP / 16, NW, QT, T>), grid, block, 0, s, a);
    else G2V_LAUNCH((k_window_dkv<NP, NS, DP, DP / 16 - 1, NW, QT, T>), grid, block, 0, s, a);
    if (!a.all_queries) return launch_attn_dkv_join(a, NP > 1, DP, s);
    const int n = std::min(a.win.sinks, a.nk);
    if (a.parts.head_splits > 1) {
        const int64_t rows = (int64_t)a.bhs * n;
        const int parts = attn_join_parts(rows, DP / 2, a.parts.head_splits);
        G2V_LAUNCH((k_window_sinks_join<DP, T>), dim3((unsigned)ceil_div(rows, 256 / (DP / 2 * parts))), dim3(256), 0, s, a, n, parts);
    }
    return hipGetLastError();
}
// QT: tile of the four-wave workgroups; the sinks' one-wave ones take 32 rows.
template <int DP, int QT, typename T>
hipError_t dkv_planes(const WinBwd& a, int planes, hipStream_t s) {
    if constexpr (sizeof(T) == 4) {
        return a.all_queries ? dkv_launch<3, 3, DP, 1, 32, T>(a, s) : dkv_launch<3, 3, DP, 4, QT, T>(a, s);
    } else {
        if (planes == 2) return a.all_queries ? dkv_launch<1, 2, DP, 1, 32, T>(a, s) : dkv_launch<1, 2, DP, 4, QT, T>(a, s);
        return a.all_queries ? dkv_launch<1, 1, DP, 1, 32, T>(a, s) : dkv_launch<1, 1, DP, 4, QT, T>(a, s);
    }
}

}  // namespace

AttnShape window_dq_shape(bool f32, int dp, int64_t rows) {
    AttnShape g = attn_dq_shape(f32, dp, rows);
    g.per_cu = window_dq_per_cu(f32 ? 3 : 1, dp, g.waves);
    g.blocks = 1;
    return g;
}
AttnShape window_dkv_shape(bool f32, int dp, int planes, bool all_queries) {
    AttnShape g = attn_dkv_shape(f32, dp, planes);
    g.per_cu = window_dkv_per_cu(f32 ? 3 : 1, planes, dp, g.waves);
    if (all_queries) {
        g.waves = 1;
        g.tile = 32;
        g.per_cu = window_dkv_per_cu(f32 ? 3 : 1, planes, dp, 1);
    }
    return g;
}

hipError_t launch_window_dq(const WinBwd& a, bool f32, int dp, hipStream_t s) {
    const AttnShape g = window_dq_shape(f32, dp, (int64_t)a.group * a.nq);
    if (f32) {
        switch (dp) {
            case 32: return dq_waves<3, 32, 64, float>(a, g, s);
            case 64: return dq_waves<3, 64, 32, float>(a, g, s);
            case 96: return dq_waves<3, 96, 32, float>(a, g, s);
            default: return dq_waves<3, 128, 32, float>(a, g, s);
        }
    }
    switch (dp) {
        case 32: return dq_waves<1, 32, 64, __bf16>(a, g, s);
        case 64: return dq_waves<1, 64, 64, __bf16>(a, g, s);
        case 96: return dq_waves<1, 96, 64, __bf16>(a, g, s);
        default: return dq_waves<1, 128, 64, __bf16>(a, g, s);
    }
}

hipError_t launch_window_zeros(const WinBwd& a, int batch, bool f32, hipStream_t s) {
    const int64_t each = (int64_t)a.gap * a.hk * a.dim, blocks = ceil_div(each, 256 * (f32 ? 4 : 8));
    if (batch * blocks == 0) return hipSuccess;
    const dim3 grid((unsigned)(batch * blocks), 2), block(256);
    if (f32) G2V_LAUNCH((k_window_zeros<float>), grid, block, 0, s, a, each, blocks);
    else G2V_LAUNCH((k_window_zeros<__bf16>), grid, block, 0, s, a, each, blocks);
    return hipGetLastError();
}

hipError_t launch_window_dkv(const WinBwd& a, bool f32, int dp, int planes, hipStream_t s) {
    if (f32) {
        switch (dp) {
            case 32: return dkv_planes<32, 64, float>(a, planes, s);
            case 64: return dkv_planes<64, 32, float>(a, planes, s);
            case 96: return dkv_planes<96, 32, float>(a, planes, s);
            default: return dkv_planes<128, 32, float>(a, planes, s);
        }
    }
    switch (dp) {
        case 32: return dkv_planes<32, 64, __bf16>(a, planes, s);
        case 64: return dkv_planes<64, 64, __bf16>(a, planes, s);
        case 96: return dkv_planes<96, 64, __bf16>(a, planes, s);
        default: return dkv_planes<128, 32, __bf16>(a, planes, s);
    }
}

}  // namespace g2v
