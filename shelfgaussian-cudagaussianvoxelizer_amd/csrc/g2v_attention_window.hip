// Attention within a window: query i, at key place p = i + shift, sees the keys
//
//   [0, min(sinks, p + right + 1))  and  [p - left, p + right],
//
// those among them whose bit is set, and O, dQ, dK and dV are those of g2v_attention_fwd.hip and g2v_attention_bwd.hip over
// these keys.  A wave's 32 or 64 rows see a range of keys little longer than a window, so a workgroup walks the tiles of the
// sinks and then those of its rows' ranges, and a wave skips the tiles that none of its rows sees.  Where a tile lies inside
// every row's range no score is looked at; at the range's ends a lane makes 32 bits of what its row sees of a block of 32 keys, and
// an operation spreads one of them over a register (v_bfe) and another lets the score through or not (v_bfi).  Masked keys are
// not packed away: the word of a tile's 64 valid keys is in a scalar register, their rows alone are loaded, and zeros stand in
// the other rows' place, as what they hold may be NaN.
//
// For dK and dV keys are in the lanes and a key's queries are a range, too: p - right .. p + left, and for a sink all from
// p - right on.  As that would have one workgroup walk all queries, the sinks' gradients are computed again by one-wave
// workgroups that share out the queries, and joined.
#include <algorithm>

#include "g2v_attention.h"

namespace g2v {
namespace {
using namespace attn;

// Keys [lo, hi) that a query sees beside the sinks.
struct KeyRange {
    int lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const AttnWindow& w, int nk, int tok) {
    const int p = tok + w.shift;
    KeyRange r;
    r.hi = min(max(p + w.right + 1, 0), nk);
    r.lo = min(max(p - w.left, 0), r.hi);
    return r;
}

// The lowest x of 32 bits, none to all.
__device__ __forceinline__ uint32_t bits_below(int x) { return (uint32_t)((1ull << min(max(x, 0), 32)) - 1); }
// Bit j: whether a row sees key base + j.
__device__ __forceinline__ uint32_t seen_bits(const KeyRange& r, int sinks, int base) {
    return bits_below(r.hi - base) & (~bits_below(r.lo - base) | bits_below(sinks - base));
}
// Bit j of x in all bits.
__device__ __forceinline__ uint32_t spread_bit(uint32_t x, int j) { return (uint32_t)((int32_t)(x << (31 - j)) >> 31); }
// x where the mask's bits are set, else -inf; or else 0.
__device__ __forceinline__ float or_lowest(uint32_t mask, float x) {
    return __uint_as_float((mask & __float_as_uint(x)) | (~mask & 0xff800000u));
}
__device__ __forceinline__ float or_zero(uint32_t mask, float x) { return __uint_as_float(mask & __float_as_uint(x)); }

// The tiles of KT keys that a workgroup's tokens [first, last] see: those of the sinks, then those of the ranges.
template <int KT>
struct KeyTiles {
    int sinks, from, all;
    __device__ __forceinline__ void init(const AttnWindow& w, int nk, int first, int last) {
        const int hi = key_range(w, nk, last).hi, lo = key_range(w, nk, first).lo;
        sinks = (min(w.sinks, hi) + KT - 1) / KT;
        from = max(sinks, lo / KT);
        all = sinks + max(0, (hi + KT - 1) / KT - from);
    }
    __device__ __forceinline__ int at(int u) const { return u < sinks ? u : from + u - sinks; }
};

// The words of a workgroup's units [u0, u1): bit j for key j of the unit's tile.  A lane holds one of 64 units at a time, so that
// the loop over the units reads no memory for them.
template <int KT>
struct TileWords {
    static constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << KT) - 1;
    uint64_t held;
    int from;
    __device__ __forceinline__ void init() { from = -64; }
    __device__ __forceinline__ uint64_t at(const AttnWindow& w, const KeyTiles<KT>& tiles, int nk, int b, int u, int u1) {
        const int t = tiles.at(u), left = nk - t * KT;
        uint64_t x = left >= KT ? kAll : (1ull << left) - 1;
        // what lies between the sinks and the first query's window no query sees
        const int unseen = min(w.shift - w.left - t * KT, KT), sinks = min(max(w.sinks - t * KT, 0), KT);
        if (unseen > sinks) x &= ~((unseen == 64 ? ~0ull : (1ull << unseen) - 1) & ~((1ull << sinks) - 1));
        if (w.bits) {
            if (u >= from + 64 || u < from) {
                from = u;
                const int mine = u + (int)(threadIdx.x & 63);
                held = 0;
                if (mine < u1) {
                    const int tm = tiles.at(mine);
                    const uint64_t* row = w.bits + (int64_t)b * w.words;
                    held = KT == 64 ? row[tm] : (row[tm >> 1] >> (32 * (tm & 1))) & kAll;
                }
            }
            const int lane = u - from;
            const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)held, lane);
            const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(held >> 32), lane);
            x &= (uint64_t)hi << 32 | lo;
        }
        return x;
    }
};

// Whether a whole tile's keys are loaded by as many loads of every wave.
template <int KT>
__device__ __forceinline__ bool whole_loads(const AttnWindow& w, int j0) { return w.gap == 0 || j0 + KT <= w.sinks || j0 >= w.sinks; }

// Loads rows [j0, j0 + KT) of base, those of the word's bits; zeros in the others' place, nothing where there are none.  Rows
// from `sinks` on are `gap` rows further.
template <int KT, typename TileT>
__device__ __forceinline__ void load_keys(const TileT& tile, const char* base, int64_t sn, int j0, uint64_t word, const AttnWindow& w,
                                          char* lds) {
    if (word == 0) return;
    if (word == TileWords<KT>::kAll && whole_loads<KT>(w, j0)) {
        tile.load(base, sn, (int64_t)j0 + (j0 >= w.sinks ? w.gap : 0), lds_off(lds));
        return;
    }
#pragma unroll
    for (int it = 0; it < TileT::kIter; ++it) {
        if (!tile.on[it]) continue;
        const int j = j0 + tile.row[it];
        if (word >> tile.row[it] & 1) dma16(base + ((int64_t)j + (j >= w.sinks ? w.gap : 0)) * sn + tile.off[it], tile.dst(lds_off(lds), it));
        else *reinterpret_cast<f32x4*>(lds + (it * TileT::kThreads + threadIdx.x) * 16) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// A wave's rows, as what they see of a tile.
struct WaveRange {
    int lo0, lo1, hi0, hi1;    // of its first and its last row
    __device__ __forceinline__ void init(const AttnWindow& w, int nk, int group, int rows, int first, int count) {
        lo0 = lo1 = hi0 = hi1 = 0;
        if (first >= rows) return;
        const KeyRange a = key_range(w, nk, first / group), b = key_range(w, nk, (min(first + count, rows) - 1) / group);
        lo0 = g2v::uniform(a.lo);
        lo1 = g2v::uniform(b.lo);
        hi0 = g2v::uniform(a.hi);
        hi1 = g2v::uniform(b.hi);
    }
    // Whether any row sees a key of [j0, j0 + n); whether every row sees all of them.
    __device__ __forceinline__ bool any(int j0, int n, int sinks) const { return j0 < hi1 && (j0 + n > lo0 || j0 < sinks); }
    __device__ __forceinline__ bool every(int j0, int n, int sinks) const {
        return j0 + n <= hi0 && (j0 >= lo1 || j0 + n <= sinks);
    }
};

// As k_attn_fwd (rows in the lanes, keys in the registers).
template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
__global__ void __launch_bounds__(NW * 64, launch_bound(NW, fwd_per_cu(NP, DP, NW))) k_window_fwd(WinFwd a) {
    constexpr int NT = NW * 64, KB = KT / 32, DB = DP / 32;
    typedef Tile<NP, DP, KT, NT> TileT;
    typedef TileWords<KT> Words;
    constexpr int kBuffers = buffers(NP == 1 && NQB == 1 ? 3 : 2, TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    static_assert(fwd_per_cu(NP, DP, NW) * sizeof(lds) <= kLdsBytes, "planned by more workgroups than fit");
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
    WaveRange range;
    range.init(a.win, a.nk, a.group, rows, first, NQB * 32);

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

    TileT tile;
    tile.init(a.k);
    Frags<DP> frags;
    frags.init(lds_off(lds));
    if (a.k.chunks < TileT::C) clear_lds<NT>(&lds[0][0][0], sizeof(lds));
    Words words;
    words.init();
    auto load = [&](int u, int buf) {
        const uint64_t word = words.at(a.win, tiles, a.nk, w.b, u, u1);
        const int j0 = tiles.at(u) * KT;
        load_keys<KT>(tile, kbase, a.k.sn, j0, word, a.win, lds[buf][0]);
        load_keys<KT>(tile, vbase, a.v.sn, j0, word, a.win, lds[buf][1]);
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
        next_tile<kBuffers, 2 * TileT::kLoads>(next == Words::kAll && whole_loads<KT>(a.win, tiles.at(u + 1) * KT));
        after = 0;
        if (u + kAhead < u1) {
            const uint64_t x = load(u + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
            if (kAhead > 1) after = x;
            else next = x;
        }
        const uint32_t at = buf * 2 * TileT::kBytes;
        const int j0 = tiles.at(u) * KT;
        if (word && range.any(j0, KT, a.win.sinks)) {
            const bool whole = word == Words::kAll && range.every(j0, KT, a.win.sinks);
            bf16x8 p[KB][2][NQB][NP];
            float sum[NQB];
            bool unseen = false;
#pragma unroll
            for (int b = 0; b < NQB; ++b) unseen = unseen || m[b] == -INFINITY;    // a row's first key may be here
            for (bool fresh = __any(unseen);; fresh = true) {
                f32x16 s[KB][NQB];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
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
                }
                if (!whole) {
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
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
            for (int kb = 0; kb < KB; ++kb)
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
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                store_out<T>(a, at, 32 * d + reg_row(i), o[d][b][i] * inv, o[d][b][i + 1] * inv, o[d][b][i + 2] * inv,
                             o[d][b][i + 3] * inv);
    }
}

// As k_attn_dq.
template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
__global__ void __launch_bounds__(NW * 64, launch_bound(NW, dq_per_cu(NP, DP, NW))) k_window_dq(WinBwd a) {
    constexpr int NS = NP == 1 ? 2 : NP;    // planes of dS, see k_attn_dq
    constexpr int NT = NW * 64, KB = KT / 32, DB = DP / 32;
    typedef Tile<NP, DP, KT, NT> TileT;
    typedef TileWords<KT> Words;
    constexpr int kBuffers = buffers(2, TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    static_assert(dq_per_cu(NP, DP, NW) * sizeof(lds) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int rows = a.group * a.nq, half = (threadIdx.x >> 5) & 1;
    const int first = (w.tile * NW + g2v::uniform(threadIdx.x >> 6)) * (NQB * 32), r0 = first + (threadIdx.x & 31);
    const int g0 = w.tile * (NW * NQB * 32), g1 = min(g0 + NW * NQB * 32, rows) - 1;
    const char* kbase = a.k.p + w.b * a.k.sb + w.h * a.k.sh;
    const char* vbase = a.v.p + w.b * a.v.sb + w.h * a.v.sh;
    KeyTiles<KT> tiles;
    tiles.init(a.win, a.nk, g2v::uniform(g0 / a.group), g2v::uniform(g1 / a.group));
    int u0, u1;
    split_range(tiles.all, w.split, w.splits, u0, u1);
    WaveRange range;
    range.init(a.win, a.nk, a.group, rows, first, NQB * 32);

    bf16x8 q[NQB][KS][NP], g[NQB][KS][NP];
    KeyRange see[NQB];
    float lse[NQB], delta[NQB];    // delta: negative, as it is stored, and times scale
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        const int r = r0 + 32 * b, rc = r < rows ? r : rows - 1;
        const int tok = rc / a.group, head = w.h * a.group + rc - tok * a.group;
        const char* qrow = a.q.p + w.b * a.q.sb + tok * a.q.sn + head * a.q.sh;
        const char* grow = a.g.p + w.b * a.g.sb + tok * a.g.sn + head * a.g.sh;
        see[b] = key_range(a.win, a.nk, tok);
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
    Words words;
    words.init();
    auto load = [&](int u, int buf) {
        const uint64_t word = words.at(a.win, tiles, a.nk, w.b, u, u1);
        const int j0 = tiles.at(u) * KT;
        load_keys<KT>(tile, kbase, a.k.sn, j0, word, a.win, lds[buf][0]);
        load_keys<KT>(tile, vbase, a.v.sn, j0, word, a.win, lds[buf][1]);
        return word;
    };

    f32x16 dq[DB][NQB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < NQB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) dq[d][b][i] = 0.0f;
    uint64_t word = 0, next = 0, after = 0;
    if (u0 < u1) word = load(u0, 0);
    if (kAhead > 1 && u0 + 1 < u1) next = load(u0 + 1, 1);
    for (int u = u0, buf = 0; u < u1; ++u, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        next_tile<kBuffers, 2 * TileT::kLoads>(next == Words::kAll && whole_loads<KT>(a.win, tiles.at(u + 1) * KT));
        after = 0;
        if (u + kAhead < u1) {
            const uint64_t x = load(u + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
            if (kAhead > 1) after = x;
            else next = x;
        }
        const uint32_t at = buf * 2 * TileT::kBytes;
        const int j0 = tiles.at(u) * KT;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const uint32_t part = (uint32_t)(word >> (32 * kb));
            const int jb = j0 + 32 * kb;
            if (!part || !range.any(jb, 32, a.win.sinks)) continue;
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
            if (part != ~0u || !range.every(jb, 32, a.win.sinks)) {
#pragma unroll
                for (int b = 0; b < NQB; ++b) {
                    const uint32_t x = (seen_bits(see[b], a.win.sinks, jb) & part) >> (4 * half);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[b][i] = or_zero(spread_bit(x, 8 * (i >> 2) + (i & 3)), s[b][i]);
                }
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
        word = next;
        next = after;
    }
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        const int r = r0 + 32 * b;
        if (r >= rows) continue;
        // one key: its probability is 1 whatever q is
        const bool one = see[b].hi - see[b].lo + min(a.win.sinks, see[b].lo) < 2;
        if (one)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) dq[d][b][i] = 0.0f;
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

// The sinks' one-wave workgroups: as many to a CU as their tiles' LDS allows.
constexpr int window_dkv_per_cu(int np, int ns, int dp, int nw) {
    return nw > 1 ? dkv_per_cu(np, ns, dp) : np > 1 ? (dp > 96 ? 1 : dp > 32 ? 2 : 4) : dp > 64 ? 3 : dp > 32 ? 6 : 8;
}
constexpr int dkv_bound(int np, int ns, int dp, int nw) { return nw > 1 ? dkv_per_cu(np, ns, dp) : np > 1 && dp > 32 ? 1 : 2; }

// As k_attn_dkv: keys in the lanes, the queries that see any of the workgroup's keys pass by, head after head.
template <int NP, int NS, int DP, int KS, int NW, int QT, typename T>
__global__ void __launch_bounds__(NW * 64, dkv_bound(NP, NS, DP, NW)) k_window_dkv(WinBwd a) {
    static_assert(NW == 1 || NW % 2 == 0, "waves in pairs load the statistics, or one does");
    constexpr int NT = NW * 64, QB = QT / 32, DB = DP / 32;
    typedef Tile<NP, DP, QT, NT> TileT;
    constexpr int kBuffers = buffers(2, TileT::kBytes), kAhead = kBuffers - 1;
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
    const int w0 = g2v::uniform(from(first)), w1 = first <= last ? g2v::uniform(to(last)) : 0;   // queries that any lane's key has
    const int w2 = g2v::uniform(from(last)), w3 = g2v::uniform(to(first));                       // and those that all have
    const int k0 = from(j), k1 = to(j);
    bool valid = j < n && k0 < k1;    // (rows that no query sees are not read either)
    if (valid && a.win.bits) valid = a.win.bits[(int64_t)w.b * a.win.words + (j >> 6)] >> (j & 63) & 1;
    const bool some = __any(valid);
    if (a.win.bits && !__syncthreads_or(valid)) u1 = u0;    // nothing to add up

    bf16x8 k[KS][NP], v[KS][NP];
    {
        const char* krow = a.k.p + w.b * a.k.sb + w.h * a.k.sh + j * a.k.sn;
        const char* vrow = a.v.p + w.b * a.v.sb + w.h * a.v.sh + j * a.v.sn;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int pl = 0; pl < NP; ++pl) {
                k[ks][pl] = mem_frag<DP>(krow, valid, a.k.chunks, pl, ks);
                v[ks][pl] = mem_frag<DP>(vrow, valid, a.v.chunks, pl, ks);
            }
    }

    TileT tile;
    tile.init(a.q);
    Frags<DP> frags;
    frags.init(lds_off(lds));
    if (a.q.chunks < TileT::C) clear_lds<NT>(&lds[0][0][0], sizeof(lds));
    auto load = [&](int u, int buf) {
        const int hd = u / per, t = tile0 + u - hd * per, head = w.h * a.group + hd;
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
    if (u0 < u1) load(u0, 0);
    if (kAhead > 1 && u0 + 1 < u1) load(u0 + 1, 1);
    for (int u = u0, buf = 0; u < u1; ++u, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        next_tile<kBuffers, TileT::kLoads ? 2 * TileT::kLoads + kStats : 0>(u + 1 < u1 &&
                                                                          (tile0 + (u + 1) % per + 1) * QT <= a.nq);
        if (u + kAhead < u1) load(u + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
        const uint32_t at = buf * 2 * TileT::kBytes;
        const int i0 = (tile0 + u % per) * QT;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const int ib = i0 + 32 * qb;
            if (!some || ib >= w1 || ib + 32 <= w0) continue;
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
            if (ib < w2 || ib + 32 > w3) {
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
    const int64_t at = (((int64_t)w.b * a.nk + j) * a.hk + w.h) * a.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            store4<T>(static_cast<T*>(a.dk) + at, 32 * d + reg_row(i), a.dim, dk[d][i] * a.scale, dk[d][i + 1] * a.scale,
                      dk[d][i + 2] * a.scale, dk[d][i + 3] * a.scale);
            store4<T>(static_cast<T*>(a.dv) + at, 32 * d + reg_row(i), a.dim, dv[d][i], dv[d][i + 1], dv[d][i + 2], dv[d][i + 3]);
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
    T* row = static_cast<T*>(d < DP ? a.dk : a.dv) + (((int64_t)b * a.nk + j) * a.hk + bh % a.hk) * a.dim;
    store4<T>(row, d < DP ? d : d - DP, a.dim, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
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

template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
hipError_t dq_launch(const WinBwd& a, hipStream_t s) {
    G2V_LAUNCH((k_window_dq<NP, DP, KS, NQB, NW, KT, T>), dim3((unsigned)workgroups(a.parts, a.bhs)), dim3(NW * 64), 0, s, a);
    return launch_attn_dq_join(a, NP > 1, DP, s);
}
template <int NP, int DP, int NQB, int KT, typename T>
hipError_t dq_waves(const WinBwd& a, const AttnShape& g, hipStream_t s) {
    const bool full = a.dim > DP - 16;
    if constexpr (NP == 1)
        if (g.waves == 1)
            return full ? dq_launch<NP, DP, DP / 16, 1, 1, KT, T>(a, s) : dq_launch<NP, DP, DP / 16 - 1, 1, 1, KT, T>(a, s);
    return full ? dq_launch<NP, DP, DP / 16, NQB, 4, KT, T>(a, s) : dq_launch<NP, DP, DP / 16 - 1, NQB, 4, KT, T>(a, s);
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

AttnShape window_fwd_shape(bool f32, int dp, int64_t rows) { return attn_fwd_shape(f32, dp, rows); }
AttnShape window_dq_shape(bool f32, int dp, int64_t rows) { return attn_dq_shape(f32, dp, rows); }
AttnShape window_dkv_shape(bool f32, int dp, int planes, bool all_queries) {
    AttnShape g = attn_dkv_shape(f32, dp, planes);
    if (all_queries) {
        g.waves = 1;
        g.tile = 32;
        g.per_cu = window_dkv_per_cu(f32 ? 3 : 1, planes, dp, 1);
    }
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
        case 64: return fwd_waves<1, 64, 2, 64, __bf16>(a, g, s);
        case 96: return fwd_waves<1, 96, 1, 64, __bf16>(a, g, s);
        default: return fwd_waves<1, 128, 2, 32, __bf16>(a, g, s);
    }
}

hipError_t launch_window_dq(const WinBwd& a, bool f32, int dp, hipStream_t s) {
    const AttnShape g = window_dq_shape(f32, dp, (int64_t)a.group * a.nq);
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

hipError_t launch_window_bits(int batch, int nk, int sinks, int gap, const unsigned char* mask, int words, uint64_t* bits,
                              hipStream_t s) {
    const int64_t all = (int64_t)batch * words;
    if (all > 0) G2V_LAUNCH(k_window_bits, dim3((unsigned)ceil_div(all, 4)), dim3(256), 0, s, nk, sinks, gap, words, all, mask, bits);
    return hipGetLastError();
}

}  // namespace g2v
