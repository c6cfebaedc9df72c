// Attention within a window, forward (g2v_attention_window.h).
#include "g2v_attention_window.h"

namespace g2v {
namespace {
using namespace attn;

#ifndef V_NQB64
#define V_NQB64 1
#endif
#ifndef V_PER64
#define V_PER64 3
#endif
constexpr int window_fwd_per_cu(int np, int dp, int waves) {
    return np == 1 && dp == 64 && waves > 1 ? V_PER64 : fwd_per_cu(np, dp, waves);
}

// As k_attn_fwd (rows in the lanes, keys in the registers).
template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
__global__ void __launch_bounds__(NW * 64, launch_bound(NW, window_fwd_per_cu(NP, DP, NW))) k_window_fwd(WinFwd a) {
    constexpr int NT = NW * 64, KB = KT / 32, DB = DP / 32;
    typedef WinTile<NP, DP, KT, NT> TileT;
    typedef TileWords<KT> Words;
    constexpr int kBuffers = buffers(window_fwd_per_cu(NP, DP, NW) > 3 ? 4 : NP == 1 && NQB == 1 ? 3 : 2, TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    static_assert(window_fwd_per_cu(NP, DP, NW) * sizeof(lds) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int lane = threadIdx.x & 63, rows = a.group * a.nq, half = lane >> 5;
    const int first = (w.tile * NW + g2v::uniform(threadIdx.x >> 6)) * (NQB * 32), r0 = first + (lane & 31);
    const int g0 = w.tile * (NW * NQB * 32), g1 = min(g0 + NW * NQB * 32, rows) - 1;    // the workgroup's rows
    const char* kbase = a.k.p + w.b * a.k.sb + w.h * a.k.sh;
    const char* vbase = a.v.p + w.b * a.v.sb + w.h * a.v.sh;
    KeyTiles<KT> tiles;
    tiles.init(a.win, a.nk, g2v::uniform(g0 / a.group), g2v::uniform(g1 / a.group));
    int u0, u1;
    split_range(tiles.all, w.split, w.splits, u0, u1);
    WaveBlocks blocks;
    blocks.init(a.win, a.nk, a.group, rows, first, NQB * 32, tiles.sinks * KT);

    bf16x8 q[NQB][KS][NP];
    KeyRange see[NQB];
    float m[NQB], l[NQB];
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        const int r = r0 + 32 * b, rc = r < rows ? r : rows - 1;
        const int tok = rc / a.group, head = w.h * a.group + rc - tok * a.group;
        const char* row = a.q.p + w.b * a.q.sb + tok * a.q.sn + head * a.q.sh;
        see[b] = key_range(a.win, a.nk, tok);
        m[b] = r < rows ? -INFINITY : 0.0f;
        l[b] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int pl = 0; pl < NP; ++pl) q[b][ks][pl] = mem_frag<DP>(row, r < rows, a.q.chunks, pl, ks);
    }

    TileT ktile, vtile;
    ktile.init(a.k);
    vtile.init(a.v);
    Frags<DP> frags;
    frags.init(lds_off(lds));
    Words words;
    words.init(a.win, a.nk);
    const char* kfar = kbase + (int64_t)a.win.gap * a.k.sn;
    const char* vfar = vbase + (int64_t)a.win.gap * a.v.sn;
    auto load = [&](int u, int buf) {
        const int t = tiles.at(u), j0 = t * KT;
        if (words.all(t)) {
            ktile.load(kfar + (int64_t)j0 * a.k.sn, lds_off(lds[buf][0]));
            vtile.load(vfar + (int64_t)j0 * a.v.sn, lds_off(lds[buf][1]));
            return Words::kAll;
        }
        const uint64_t word = words.at(a.win, tiles, a.nk, w.b, u, u1);
        TileT::load_some(a.k, kbase, j0, word, a.win.sinks, a.win.gap, lds[buf][0]);
        TileT::load_some(a.v, vbase, j0, word, a.win.sinks, a.win.gap, lds[buf][1]);
        return word;
    };

    f32x16 o[DB][NQB];
#pragma unroll
    for (int b = 0; b < NQB; ++b)
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][b][i] = 0.0f;
    uint64_t word = 0, next = 0, after = 0;    // of units u, u + 1 and u + 2
    if (u0 < u1) word = load(u0, 0);
    if (kAhead > 1 && u0 + 1 < u1) next = load(u0 + 1, 1);
    for (int u = u0, buf = 0; u < u1; ++u, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        // (a partly valid tile's loads are not the same number for every wave)
        next_tile<kBuffers, 2 * TileT::kLoads>(u + 1 < u1 && words.all(tiles.at(u + 1)));
        after = 0;
        if (u + kAhead < u1) {
            const uint64_t x = load(u + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
            if (kAhead > 1) after = x;
            else next = x;
        }
        const uint32_t at = buf * 2 * TileT::kBytes;
        const int j0 = tiles.at(u) * KT;
        // blocks of 32 keys that the wave's rows see none of, or only some of
        const bool far = u < tiles.sinks;
        const WaveBlocks::Range some = far ? blocks.any_far : blocks.any, every = far ? blocks.every_far : blocks.every;
        bool on[KB], part[KB], any = false;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            on[kb] = some.has(j0 + 32 * kb);
            part[kb] = !every.has(j0 + 32 * kb);
            if (word != Words::kAll) {
                on[kb] = on[kb] && (uint32_t)(word >> (32 * kb));
                part[kb] = part[kb] || (uint32_t)(word >> (32 * kb)) != ~0u;
            }
            any = any || on[kb];
        }
        if (any) {
            bf16x8 p[KB][2][NQB][NP];
            float sum[NQB];
            bool unseen = false;
#pragma unroll
            for (int b = 0; b < NQB; ++b) unseen = unseen || m[b] == -INFINITY;    // a row's first key may be here
            for (bool fresh = __any(unseen);; fresh = true) {
                f32x16 s[KB][NQB];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    if (!on[kb]) continue;
#pragma unroll
                    for (int b = 0; b < NQB; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[kb][b][i] = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        bf16x8 f[NP];
#pragma unroll
                        for (int pl = 0; pl < NP; ++pl) f[pl] = frags.rows(at, pl * KT * DP * 2, kb, ks);
#pragma unroll
                        for (int b = 0; b < NQB; ++b) s[kb][b] = mma(f, q[b][ks], s[kb][b]);
                    }
                    if (part[kb])
#pragma unroll
                        for (int b = 0; b < NQB; ++b) {
                            const uint32_t x = (seen_bits(see[b], a.win.sinks, j0 + 32 * kb) & (uint32_t)(word >> (32 * kb))) >> (4 * half);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                s[kb][b][i] = or_lowest(spread_bit(x, 8 * (i >> 2) + (i & 3)), s[kb][b][i]);
                        }
                }
                if (fresh) {
#pragma unroll
                    for (int b = 0; b < NQB; ++b) {
                        float top = m[b];
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb)
                            if (on[kb])
#pragma unroll
                                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][b][i]);
                        top = half_max(top);
                        const float f = m[b] == -INFINITY ? 0.0f : exp2_fast((m[b] - top) * a.c);
                        m[b] = top;
                        l[b] *= f;
#pragma unroll
                        for (int d = 0; d < DB; ++d)
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[d][b][i] *= f;
                    }
                }
                bool over = false;
#pragma unroll
                for (int b = 0; b < NQB; ++b) {
                    const float mc = m[b] == -INFINITY ? 0.0f : m[b] * a.c;    // no key yet: all probabilities are 0
                    sum[b] = 0.0f;
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        if (!on[kb]) continue;
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[kb][b][i] = exp2_fast(fmaf(s[kb][b][i], a.c, -mc));
#pragma unroll
                        for (int st = 0; st < 2; ++st) {
                            to_operand(s[kb][b], st, p[kb][st][b]);
                            if constexpr (NP == 1) sum[b] = add_operand(p[kb][st][b][0], sum[b]);
                        }
                        if constexpr (NP > 1)
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum[b] += s[kb][b][i];
                    }
                    over = over || sum[b] > kFar;
                }
                if (fresh || !__any(over)) break;
            }
#pragma unroll
            for (int b = 0; b < NQB; ++b) l[b] += sum[b];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                if (!on[kb]) continue;
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        bf16x8 f[NP];
#pragma unroll
                        for (int pl = 0; pl < NP; ++pl) f[pl] = frags.cols(at, TileT::kBytes + pl * KT * DP * 2, kb, st, d);
#pragma unroll
                        for (int b = 0; b < NQB; ++b) o[d][b] = mma(f, p[kb][st][b], o[d][b]);
                    }
            }
        }
        word = next;
        next = after;
    }
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        const int r = r0 + 32 * b;
        const float total = half_sum(l[b]);
        if (r >= rows) continue;
        if (w.splits > 1) {
            const PartRow pr = part_row(a.parts, a.bhs, w.bh, rows, r);
            const int64_t at = pr.at + w.split * pr.step;
            if (lane < 32) {
                a.part_ml[2 * at] = m[b] * a.c;
                a.part_ml[2 * at + 1] = total;
            }
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<f32x4*>(a.part_o + at * DP + 32 * d + reg_row(i)) =
                        f32x4{o[d][b][i], o[d][b][i + 1], o[d][b][i + 2], o[d][b][i + 3]};
            continue;
        }
        const int tok = r / a.group, head = w.h * a.group + r - tok * a.group;
        const float inv = total > 0.0f ? 1.0f / total : 0.0f;
        if (a.lse && lane < 32)
            a.lse[((int64_t)w.b * a.hq + head) * a.nq + tok] = total > 0.0f ? fmaf(m[b], a.c, log2f(total)) : INFINITY;
        const int64_t at = (((int64_t)w.b * a.nq + tok) * a.hq + head) * a.dim;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            float x[16], lost[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = o[d][b][i] * inv;
                lost[i] = lost_by_rounding(x[i]);
            }
            store_block<T>(static_cast<T*>(a.out) + at, 32 * d, a.dim, x);
            if constexpr (sizeof(T) == 2)
                if (a.rest) store_block<T>(static_cast<T*>(a.rest) + at, 32 * d, a.dim, lost);    // see store_out
        }
    }
}

// Bits of the valid keys, a wave a word.
__global__ void __launch_bounds__(256) k_window_bits(int nk, int sinks, int gap, int words, int64_t all, const unsigned char* mask,
                                                     uint64_t* bits) {
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= all) return;
    const int64_t b = at / words;
    const int j = (int)(at - b * words) * 64 + (threadIdx.x & 63);
    const bool valid = j < nk && mask[b * (nk + gap) + j + (j >= sinks ? gap : 0)];
    const uint64_t x = __ballot(valid);
    if ((threadIdx.x & 63) == 0) bits[at] = x;
}

template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
hipError_t fwd_launch(const WinFwd& a, hipStream_t s) {
    G2V_LAUNCH((k_window_fwd<NP, DP, KS, NQB, NW, KT, T>), dim3((unsigned)workgroups(a.parts, a.bhs)), dim3(NW * 64), 0, s, a);
    return launch_attn_join(a, NP > 1, DP, s);
}
template <int NP, int DP, int NQB, int KT, typename T>
hipError_t fwd_waves(const WinFwd& a, const AttnShape& g, hipStream_t s) {
    const bool full = a.dim > DP - 16;
    if constexpr (NP == 1)
        if (g.waves == 1)
            return full ? fwd_launch<NP, DP, DP / 16, 1, 1, KT, T>(a, s) : fwd_launch<NP, DP, DP / 16 - 1, 1, 1, KT, T>(a, s);
    return full ? fwd_launch<NP, DP, DP / 16, NQB, 4, KT, T>(a, s) : fwd_launch<NP, DP, DP / 16 - 1, NQB, 4, KT, T>(a, s);
}

}  // namespace

AttnShape window_fwd_shape(bool f32, int dp, int64_t rows) {
    AttnShape g = attn_fwd_shape(f32, dp, rows);
    g.per_cu = window_fwd_per_cu(f32 ? 3 : 1, dp, g.waves);
    if (!f32 && dp == 64 && g.waves > 1) g.blocks = V_NQB64;
    return g;
}

hipError_t launch_window_fwd(const WinFwd& a, bool f32, int dp, hipStream_t s) {
    const AttnShape g = window_fwd_shape(f32, dp, (int64_t)a.group * a.nq);
    if (f32) {
        switch (dp) {
            case 32: return fwd_waves<3, 32, 1, 64, float>(a, g, s);
            case 64: return fwd_waves<3, 64, 1, 32, float>(a, g, s);
            case 96: return fwd_waves<3, 96, 1, 32, float>(a, g, s);
            default: return fwd_waves<3, 128, 1, 32, float>(a, g, s);
        }
    }
    switch (dp) {
        case 32: return fwd_waves<1, 32, 2, 64, __bf16>(a, g, s);
        case 64: return fwd_waves<1, 64, V_NQB64, 64, __bf16>(a, g, s);
        case 96: return fwd_waves<1, 96, 1, 64, __bf16>(a, g, s);
        default: return fwd_waves<1, 128, 2, 32, __bf16>(a, g, s);
    }
}

hipError_t launch_window_bits(int batch, int nk, int sinks, int gap, const unsigned char* mask, int words, uint64_t* bits,
                              hipStream_t s) {
    const int64_t all = (int64_t)batch * words;
    if (all > 0) G2V_LAUNCH(k_window_bits, dim3((unsigned)ceil_div(all, 4)), dim3(256), 0, s, nk, sinks, gap, words, all, mask, bits);
    return hipGetLastError();
}

}  // namespace g2v
