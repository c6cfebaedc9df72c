// Attention within a window, forward (g2v_attention_window.h).
#include "g2v_attention_window.h"

namespace g2v {
namespace {
using namespace attn;

// Workgroups that share a CU, as in g2v_attention.h, at one block of rows a wave.  Windows of 513 keys and 8 sinks, us: 60,000 x 16
// heads x 32, four 156 (two blocks, three workgroups, spilling: 330); 40,000 x 8 x 128, two 166 (two blocks, spilling: 937); 40,000 x 8
// x 96, three 110 and two 121; 200,000 x 8 x 64 without sinks, three 392 and four, spilling, 594.
constexpr int window_fwd_per_cu(int np, int dp, int waves) {
    return np == 1 && waves > 1 ? (dp == 32 ? 4 : dp > 96 ? 2 : 3) : fwd_per_cu(np, dp, waves);
}

// A tile of float32 rows on its way to LDS (as Tile's three planes): in registers while the tile before it is computed.
template <int DP, int ROWS, int NT>
struct FloatTile {
    static constexpr int C = DP / 8, kChunks = ROWS * C, kIter = (kChunks + NT - 1) / NT;
    f32x8 x0, x1;    // (an array of them is kept in memory by the compiler)
    __device__ __forceinline__ static bool on(int it) { return kChunks % NT == 0 || it * NT + (int)threadIdx.x < kChunks; }
    // Rows j0 .. of base, those of the word's bits, zeros in the others' place.
    __device__ __forceinline__ void fetch(const RowSrc& s, const char* base, int dim, int j0, uint64_t word, int sinks, int skip) {
        static_assert(kIter <= 2, "chunks of a thread");
        auto one = [&](int it) __attribute__((always_inline)) {
            const int L = it * NT + threadIdx.x, row = L / C, j = j0 + row;
            return load_floats(reinterpret_cast<const float*>(base + ((int64_t)j + (j >= sinks ? skip : 0)) * s.sn),
                               on(it) && (word >> row & 1), L % C, dim);
        };
        x0 = one(0);
        if constexpr (kIter > 1) x1 = one(1);
    }
    __device__ __forceinline__ void store(char* lds) const {
        auto one = [&](int it, const f32x8 x) __attribute__((always_inline)) {
            const int L = it * NT + threadIdx.x, row = L / C, c = L % C;
            if (!on(it)) return;
            bf16x8 o[3];
            split_planes(x, o);
#pragma unroll
            for (int pl = 0; pl < 3; ++pl)
                *reinterpret_cast<bf16x8*>(lds + (pl * kChunks + row * C + swz<DP>(row, c)) * 16) = o[pl];
        };
        one(0, x0);
        if constexpr (kIter > 1) one(1, x1);
    }
};

// As k_attn_fwd (rows in the lanes, keys in the registers).
// FLOATS: q, k and v are float32 rows, split into planes here; else bfloat16 rows, planes packed before.
template <int NP, bool FLOATS, int DP, int KS, int NW, int KT, typename T>
__global__ void __launch_bounds__(NW * 64, launch_bound(NW, window_fwd_per_cu(NP, DP, NW))) k_window_fwd(WinFwd a) {
    static_assert(!FLOATS || NP == 3, "planes of float32");
    constexpr int NT = NW * 64, KB = KT / 32, DB = DP / 32;
    typedef WinTile<NP, DP, KT, NT> TileT;
    typedef TileWords<KT> Words;
    constexpr int kBuffers = FLOATS ? 2 : buffers(NP > 1 ? 2 : window_fwd_per_cu(NP, DP, NW), TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    static_assert(window_fwd_per_cu(NP, DP, NW) * sizeof(lds) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int lane = threadIdx.x & 63, rows = a.group * a.nq, half = lane >> 5;
    const int first = (w.tile * NW + g2v::uniform(threadIdx.x >> 6)) * 32, r = first + (lane & 31);
    const int g0 = w.tile * (NW * 32), g1 = min(g0 + NW * 32, rows) - 1;    // the workgroup's rows
    const char* kbase = a.k.p + w.b * a.k.sb + w.h * a.k.sh;
    const char* vbase = a.v.p + w.b * a.v.sb + w.h * a.v.sh;
    KeyTiles<KT> tiles;
    tiles.init(a.win, a.nk, g2v::uniform(g0 / a.group), g2v::uniform(g1 / a.group));
    int u0, u1;
    split_range(tiles.all, w.split, w.splits, u0, u1);
    WaveBlocks blocks;
    blocks.init(a.win, a.nk, a.group, rows, first, tiles.sinks * KT);

    bf16x8 q[KS][NP];
    f32x8 qf[FLOATS ? KS : 1];
    float m = r < rows ? -INFINITY : 0.0f, l = 0.0f;
    const int rc = r < rows ? r : rows - 1, load_tok = rc / a.group, load_head = w.h * a.group + rc - load_tok * a.group;
    const char* row = a.q.p + w.b * a.q.sb + load_tok * a.q.sn + load_head * a.q.sh;
    const KeyRange see = key_range(a.win, a.nk, load_tok);
    if constexpr (FLOATS)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            qf[ks] = load_floats(reinterpret_cast<const float*>(row), r < rows, 2 * ks + half, a.dim);
    else load_row<DP>(row, a.q.chunks, q);

    TileT ktile, vtile;
    FloatTile<DP, KT, NT> kfloat, vfloat;
    if constexpr (!FLOATS) {
        ktile.init(a.k);
        vtile.init(a.v);
    }
    Frags<DP> frags;
    frags.init(lds_off(lds));
    Words words;
    words.init(a.win, a.nk);
    const char* kfar = kbase + (int64_t)a.win.skip * a.k.sn;
    const char* vfar = vbase + (int64_t)a.win.skip * a.v.sn;
    auto load = [&](int u, int buf) __attribute__((always_inline)) {
        const int t = tiles.at(u), j0 = t * KT;
        if constexpr (FLOATS) {    // into registers
            const uint64_t word = words.all(t) ? Words::kAll : words.at(a.win, tiles, a.nk, w.b, u, u1);
            kfloat.fetch(a.k, kbase, a.dim, j0, word, a.win.sinks, a.win.skip);
            vfloat.fetch(a.v, vbase, a.dim, j0, word, a.win.sinks, a.win.skip);
            return word;
        }
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

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    auto store = [&](int buf) __attribute__((always_inline)) {    // from registers to LDS
        if constexpr (FLOATS) {
            kfloat.store(lds[buf][0]);
            vfloat.store(lds[buf][1]);
        }
    };
    uint64_t word = 0, next = 0, after = 0;    // of units u, u + 1 and u + 2
    if (u0 < u1) {
        word = load(u0, 0);
        store(0);
    }
    if constexpr (FLOATS)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) split_planes(qf[ks], q[ks]);
    settle_row(FLOATS || r < rows, FLOATS ? DP / 8 : a.q.chunks, q);
    if (kAhead > 1 && u0 + 1 < u1) next = load(u0 + 1, 1);
    for (int u = u0, buf = 0; u < u1; ++u, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        // (a partly valid tile's loads are not the same number for every wave)
        next_tile<kBuffers, (FLOATS ? 0 : 2 * TileT::kLoads)>(u + 1 < u1 && words.all(tiles.at(u + 1)));
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
            bf16x8 p[KB][2][NP];
            float sum;
            for (bool fresh = __any(m == -INFINITY);; fresh = true) {    // (a row's first key may be here)
                f32x16 s[KB];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    if (!on[kb]) continue;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        bf16x8 f[NP];
#pragma unroll
                        for (int pl = 0; pl < NP; ++pl) f[pl] = frags.rows(at, pl * KT * DP * 2, kb, ks);
                        s[kb] = mma(f, q[ks], s[kb]);
                    }
                    if (part[kb]) {
                        const uint32_t x = (seen_bits(see, a.win.sinks, j0 + 32 * kb) & (uint32_t)(word >> (32 * kb))) >> (4 * half);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[kb][i] = or_lowest(spread_bit(x, 8 * (i >> 2) + (i & 3)), s[kb][i]);
                    }
                }
                if (fresh) {
                    float top = m;
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
                        if (on[kb])
#pragma unroll
                            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
                    top = half_max(top);
                    const float f = m == -INFINITY ? 0.0f : exp2_fast((m - top) * a.c);
                    m = top;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] *= f;
                }
                const float mc = m == -INFINITY ? 0.0f : m * a.c;    // no key yet: all probabilities are 0
                sum = 0.0f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    if (!on[kb]) continue;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[kb][i] = exp2_fast(fmaf(s[kb][i], a.c, -mc));
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        to_operand(s[kb], st, p[kb][st]);
                        if constexpr (NP == 1) sum = add_operand(p[kb][st][0], sum);
                    }
                    if constexpr (NP > 1)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum += s[kb][i];
                }
                if (fresh || !__any(sum > kFar)) break;
            }
            l += sum;
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
                        o[d] = mma(f, p[kb][st], o[d]);
                    }
            }
        }
        if (u + 1 < u1) store(buf ^ 1);
        word = next;
        next = after;
    }
    const float total = half_sum(l);
    if (r >= rows) return;
    if (w.splits > 1) {
        const PartRow pr = part_row(a.parts, a.bhs, w.bh, rows, r);
        const int64_t at = pr.at + w.split * pr.step;
        if (lane < 32) {
            a.part_ml[2 * at] = m * a.c;
            a.part_ml[2 * at + 1] = total;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(a.part_o + at * DP + 32 * d + reg_row(i)) =
                    f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        return;
    }
    // (made again from r: kept over the loop, they spill at 96 channels, 134 -> 153 us)
    const int tok = r / a.group, head = w.h * a.group + r - tok * a.group;
    const float inv = total > 0.0f ? 1.0f / total : 0.0f;
    if (a.lse && lane < 32)
        a.lse[((int64_t)w.b * a.hq + head) * a.nq + tok] = total > 0.0f ? fmaf(m, a.c, log2f(total)) : INFINITY;
    const int64_t at = (((int64_t)w.b * a.nq + tok) * a.hq + head) * a.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        float x[16], lost[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = o[d][i] * inv;
            lost[i] = lost_by_rounding(x[i]);
        }
        store_block<T>(static_cast<T*>(a.out) + at, 32 * d, a.dim, x);
        if constexpr (sizeof(T) == 2)
            if (a.rest) store_block<T>(static_cast<T*>(a.rest) + at, 32 * d, a.dim, lost);    // see store_out of g2v_attention_fwd.hip
    }
}

template <int NP, int DP, int KS, int NW, int KT, typename T>
hipError_t fwd_launch(const WinFwd& a, hipStream_t s) {
    const dim3 grid((unsigned)workgroups(a.parts, a.bhs)), block(NW * 64);
    if constexpr (NP > 1) {
        if (a.floats) G2V_LAUNCH((k_window_fwd<NP, true, DP, KS, NW, KT, T>), grid, block, 0, s, a);
        else G2V_LAUNCH((k_window_fwd<NP, false, DP, KS, NW, KT, T>), grid, block, 0, s, a);
    } else {
        G2V_LAUNCH((k_window_fwd<NP, false, DP, KS, NW, KT, T>), grid, block, 0, s, a);
    }
    return launch_attn_join(a, NP > 1, DP, s);
}
template <int NP, int DP, int KT, typename T>
hipError_t fwd_waves(const WinFwd& a, const AttnShape& g, hipStream_t s) {
    const bool full = a.dim > DP - 16;
    if constexpr (NP == 1)
        if (g.waves == 1)
            return full ? fwd_launch<NP, DP, DP / 16, 1, KT, T>(a, s) : fwd_launch<NP, DP, DP / 16 - 1, 1, KT, T>(a, s);
    return full ? fwd_launch<NP, DP, DP / 16, 4, KT, T>(a, s) : fwd_launch<NP, DP, DP / 16 - 1, 4, KT, T>(a, s);
}

}  // namespace

// Waves as there.  float32 rows take four however few they are: those without a row load and split tiles with the others (one query, 4097
// keys x 16 heads x 64, 18 us and 10 with its join's).
AttnShape window_fwd_shape(bool f32, int dp, int64_t rows) {
    AttnShape g = attn_fwd_shape(f32, dp, rows);
    g.per_cu = window_fwd_per_cu(f32 ? 3 : 1, dp, g.waves);
    g.blocks = 1;
    return g;
}

hipError_t launch_window_fwd(const WinFwd& a, bool f32, int dp, hipStream_t s) {
    const AttnShape g = window_fwd_shape(f32, dp, (int64_t)a.group * a.nq);
    if (f32) {
        switch (dp) {
            case 32: return fwd_waves<3, 32, 64, float>(a, g, s);
            case 64: return fwd_waves<3, 64, 32, float>(a, g, s);
            case 96: return fwd_waves<3, 96, 32, float>(a, g, s);
            default: return fwd_waves<3, 128, 32, float>(a, g, s);
        }
    }
    switch (dp) {
        case 32: return fwd_waves<1, 32, 64, __bf16>(a, g, s);
        case 64: return fwd_waves<1, 64, 64, __bf16>(a, g, s);
        case 96: return fwd_waves<1, 96, 64, __bf16>(a, g, s);
        default: return fwd_waves<1, 128, 32, __bf16>(a, g, s);
    }
}

}  // namespace g2v
