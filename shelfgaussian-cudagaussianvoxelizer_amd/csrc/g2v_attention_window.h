// Attention within a window: query i, at key place p = i + shift, sees the keys
//
//   [0, min(sinks, p + right + 1))  and  [p - left, p + right],
//
// those among them that the mask keeps, and O, dQ, dK and dV are those of g2v_attention_fwd.hip and g2v_attention_bwd.hip over
// these keys.  A wave's 32 rows see a range of keys little longer than a window, so a workgroup walks the tiles of the
// sinks and then those of its rows' ranges, and a wave skips the blocks of 32 keys that none of its rows sees.  Where a block lies
// inside every row's range no score is looked at; at the range's ends a lane makes 32 bits of what its row sees of the block, one
// operation spreads one of them over a register and another lets the score through or not.  Masked keys are not packed away: the word
// of a tile's valid keys is in scalar registers, their rows alone are loaded, and zeros stand in the other rows' place, as what they hold
// may be NaN.
//
// For dK and dV keys are in the lanes and a key's queries are a range, too: p - right .. p + left, and for a sink all from
// p - right on.  As that would have one workgroup walk all queries, the sinks' gradients are computed again by one-wave
// workgroups that share out the queries, and joined.
//
// Bound by memory at the shortest windows and then, like the attention over all keys, by matrix and vector work taking turns:
// 200,000 x 8 heads x 64 bfloat16, windows of 1 / 513 / 2049 keys, us: forward that a backward follows 257, 391, 1101 (its 1.0 GB
// take 200 at a copy's rate; from 513 keys on a key more for every query takes 0.46, 890 TFLOP/s), dQ with delta 413, 578, 1706, dK and
// dV 318, 827, 1750 (P and dS in two planes up to 1,024 keys).  A wave has one block of 32 rows and bfloat16 has more workgroups to a CU
// than the attention over all keys, as a row block's range is shorter than two blocks' together, and prologues and ends hide one another
// (with that attention's blocks and workgroups, 513 keys: forward 478 for 414, dQ 747 for 615, before rows were loaded as below).
#pragma once
#include "g2v_attention.h"

namespace g2v {
namespace attn {

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

// Which keys of a tile are valid, bit j for the tile's key j: all of them in the tiles of one range, by which most tiles are told;
// else a lane holds the word of one of 64 units, made from the
// mask's bytes, so that the loop over the units reads no memory for them and no kernel before it makes them.
template <int KT>
struct TileWords {
    static constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << KT) - 1;
    int whole0, whole;    // the range's first tile and its number of tiles
    uint64_t held;
    int from;
    __device__ __forceinline__ void init(const AttnWindow& w, int nk) {
        // keys between the sinks and the first query's window are seen by no query; and the sinks' rows may lie elsewhere
        const int unseen = w.shift - w.left;
        whole0 = unseen > w.sinks || w.skip ? (max(unseen, w.sinks) + KT - 1) / KT : 0;
        whole = w.mask ? 0 : max(0, nk / KT - whole0);
        from = -64;
    }
    __device__ __forceinline__ bool all(int t) const { return (uint32_t)(t - whole0) < (uint32_t)whole; }
    // Takes the keys that the mask does not keep out of the held words: a byte a lane for each unit, several units' loads at a time
    // (repeated past the ends, where no held word has a bit).
    __device__ __forceinline__ void keep(const AttnWindow& w, const KeyTiles<KT>& tiles, int nk, int b, int u, int u1) {
        constexpr int kUnits = 8;
        const unsigned char* row = w.mask + (int64_t)b * (nk + w.gap);
        const int lane = threadIdx.x & 63, key = min(lane, KT - 1), n = min(64, u1 - u);
        for (int i0 = 0; i0 < n; i0 += kUnits) {
            unsigned char x[kUnits];
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int j = min(tiles.at(min(u + i0 + i, u1 - 1)) * KT + key, nk - 1);
                x[i] = row[j + (j >= w.sinks ? w.gap : 0)];
            }
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const uint64_t kept = __ballot(x[i] != 0);
                if (lane == i0 + i) held &= kept;
            }
        }
    }
    // The word of unit u, tile t, which is none of the range's.
    __device__ __forceinline__ uint64_t at(const AttnWindow& w, const KeyTiles<KT>& tiles, int nk, int b, int u, int u1) {
        if ((uint32_t)(u - from) >= 64u) {
            from = u;
            const int mine = u + (int)(threadIdx.x & 63);
            held = 0;
            if (mine < u1) {
                const int t = tiles.at(mine), left = nk - t * KT, unseen = min(w.shift - w.left - t * KT, KT);
                const int sinks = min(max(w.sinks - t * KT, 0), KT);
                held = left >= KT ? kAll : (1ull << left) - 1;
                if (unseen > sinks) held &= ~((unseen == 64 ? ~0ull : (1ull << unseen) - 1) & ~((1ull << sinks) - 1));
            }
            if (w.mask) keep(w, tiles, nk, b, u, u1);
        }
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)held, u - from);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(held >> 32), u - from);
        return (uint64_t)hi << 32 | lo;
    }
};

// A tile in LDS as Tile's ([plane][row][DP], swizzled), with less to do for each load: chunks past the rows' end repeat the last
// one instead of being left out (the other operand is zero there, or the product's row is not stored), and offsets are kept.
template <int NP, int DP, int ROWS, int NT>
struct WinTile {
    static constexpr int C = DP / 8;
    static constexpr int kChunks = NP * ROWS * C;
    static constexpr int kBytes = kChunks * 16;
    static constexpr int kIter = (kChunks + NT - 1) / NT;
    static constexpr int kLoads = kChunks % NT ? 0 : kIter;    // of every wave; 0: not the same for all

    __device__ __forceinline__ static int row(int it) { return (it * NT + (int)threadIdx.x) % (ROWS * C) / C; }
    __device__ __forceinline__ static bool on(int it) { return kChunks % NT == 0 || it < kIter - 1 || it * NT + (int)threadIdx.x < kChunks; }
    // Byte offset of this thread's chunk in its row.
    __device__ __forceinline__ static uint32_t chunk(int it, int chunks) {
        const int L = it * NT + threadIdx.x, pl = L / (ROWS * C), c = swz<DP>(row(it), L % C);
        return (uint32_t)(pl * C + min(c, chunks - 1)) * 16;
    }
    __device__ __forceinline__ static uint32_t dst(uint32_t lds, int it) {
        return lds + it * NT * 16 + (uint32_t)g2v::uniform(threadIdx.x >> 6) * 1024;
    }
    static constexpr bool kKept = kIter <= 5;     // (more of them are spilled: see load)
    uint32_t off[kKept ? kIter : 1];    // of its chunk from the tile's first row
    __device__ __forceinline__ void init(const RowSrc& s) {
        if constexpr (kKept)
#pragma unroll
            for (int it = 0; it < kIter; ++it) off[it] = (uint32_t)row(it) * (uint32_t)s.sn + chunk(it, s.chunks);
    }
    // The rows from p on, all of them there.  (Many offsets are made anew for each tile: 40,000 x 8 heads in float32, dK and dV at 128
    // channels 2.01 -> 1.44 ms, what eight sinks take at 96 channels 0.31 -> 0.13.)
    __device__ __forceinline__ void load(const RowSrc& s, const char* p, uint32_t lds) const {
        int tid = threadIdx.x;
        if constexpr (!kKept) asm volatile("" : "+v"(tid));    // so that the compiler keeps no offset over the loop either
#pragma unroll
        for (int it = 0; it < kIter; ++it) {
            if (!on(it)) continue;
            if constexpr (kKept) {
                dma16(p, off[it], dst(lds, it));
            } else {
                const int L = it * NT + tid, pl = L / (ROWS * C), r = L % (ROWS * C) / C, c = swz<DP>(r, L % C);
                dma16(p, (uint32_t)r * (uint32_t)s.sn + (uint32_t)(pl * C + min(c, s.chunks - 1)) * 16, dst(lds, it));
            }
        }
    }
    // Rows j0 .. of base, those of the word's bits; zeros in the others' place, nothing where there are none.  Rows from `sinks` on
    // are `skip` rows further.
    __device__ __forceinline__ static void load_some(const RowSrc& s, const char* base, int j0, uint64_t word, int sinks, int skip, char* lds) {
        if (word == 0) return;
#pragma unroll
        for (int it = 0; it < kIter; ++it) {
            if (!on(it)) continue;
            const int j = j0 + row(it);
            if (word >> row(it) & 1) dma16(base + ((int64_t)j + (j >= sinks ? skip : 0)) * s.sn + chunk(it, s.chunks), dst(lds_off(lds), it));
            else *reinterpret_cast<f32x4*>(lds + (it * NT + threadIdx.x) * 16) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // Rows j0 .. n - 1 of base, the last one repeated.
    __device__ __forceinline__ static void load_tail(const RowSrc& s, const char* base, int j0, int n, uint32_t lds) {
#pragma unroll
        for (int it = 0; it < kIter; ++it)
            if (on(it)) dma16(base + (int64_t)min(j0 + row(it), n - 1) * s.sn + chunk(it, s.chunks), dst(lds, it));
    }
};

// A wave's rows: blocks of 32 keys of which any row sees one, and those that every row sees, as ranges of the blocks' first keys, for
// the tiles of the sinks and for those behind them (the first may hold too many blocks, the second too few).
struct WaveBlocks {
    struct Range {
        int at;
        uint32_t n;
        __device__ __forceinline__ bool has(int j) const { return (uint32_t)(j - at) < n; }
    };
    Range any, every, any_far, every_far;    // of the window; of the sinks' tiles
    __device__ __forceinline__ void init(const AttnWindow& w, int nk, int group, int rows, int first, int sinks_end) {
        any = every = any_far = every_far = {0, 0u};
        if (first >= rows) return;
        const KeyRange a = key_range(w, nk, first / group), b = key_range(w, nk, (min(first + 32, rows) - 1) / group);
        const int lo0 = g2v::uniform(a.lo), lo1 = g2v::uniform(b.lo), hi0 = g2v::uniform(a.hi), hi1 = g2v::uniform(b.hi);
        if (hi1 > lo0) any = {lo0 - 31, (uint32_t)(hi1 - lo0 + 31)};
        if (hi0 - 31 > lo1) every = {lo1, (uint32_t)(hi0 - 31 - lo1)};
        any_far = {0, (uint32_t)(lo0 < sinks_end ? hi1 : min(hi1, w.sinks))};
        every_far = {0, (uint32_t)max(0, min(hi0, w.sinks) - 31)};
    }
};

// Eight float32 values as three bfloat16 planes, exact to 24 bits.  A finite value above the largest bfloat16 starts with that (what
// is left is small); an infinity is its first plane alone.
constexpr float kMaxBf16 = 0x1.fep127f;
typedef float f32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void split_planes(const f32x8 x, bf16x8 (&o)[3]) {
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[j]));
    const bool large = most > kMaxBf16;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float r = x[j];
#pragma unroll
        for (int pl = 0; pl < 3; ++pl) {
            const __bf16 h = (__bf16)r;
            o[pl][j] = h;
            r -= (float)h;
        }
    }
    if (large) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float r = x[j], h = (float)(__bf16)r;
            if (!__builtin_isfinite(h) && __builtin_isfinite(r)) h = copysignf(kMaxBf16, r);
#pragma unroll
            for (int pl = 0; pl < 3; ++pl) {
                o[pl][j] = (__bf16)h;
                r = __builtin_isfinite(h) ? r - h : 0.0f;
                h = (float)(__bf16)r;
            }
        }
    }
}
// Values 8 c .. 8 c + 7 of a float32 row of whole chunks of 8, zeros past its end or without a row.
__device__ __forceinline__ f32x8 load_floats(const float* row, bool have, int c, int dim) {
    typedef float vec __attribute__((ext_vector_type(8), aligned(sizeof(float))));
    f32x8 x = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (have && 8 * c < dim) x = *reinterpret_cast<const vec*>(row + 8 * c);
    return x;
}
// Values of a row of dim at any alignment, as float32: 16 ks + 8 half + 0 .. 7 for every step ks, zeros past its end.
template <int KS, typename T>
struct RowValues {
    typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    vec x[KS];
    T tail[8];    // what is behind the last whole 8
    __device__ __forceinline__ void load(const T* row, int dim) {
        const int half = (threadIdx.x >> 5) & 1, whole = dim / 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) tail[j] = (T)0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[ks][j] = (T)0.0f;
        if (whole > 0)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) x[ks] = *reinterpret_cast<const vec*>(row + 8 * min(2 * ks + half, whole - 1));
        if (dim % 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) tail[j] = row[min(8 * whole + j, dim - 1)];
    }
    __device__ __forceinline__ f32x8 at(int ks, int dim) const {
        const int c = 2 * ks + ((threadIdx.x >> 5) & 1), whole = dim / 8;
        f32x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            o[j] = c < whole ? (float)x[ks][j] : c == whole && j < dim % 8 ? (float)tail[j] : 0.0f;
        return o;
    }
};

// A lane's row as B operands (mem_frag's), in two parts: the loads, which all go out before any is waited for, and what ends the wait
// for them and puts zeros where there is no row or no chunk (the last step alone may lack some).  A wait that is left to a loop's first
// use is waited for in every turn, and with it the tiles that are on their way.  Against mem_frag, dQ and dK with dV in us, windows of 513
// keys and P in one plane: 200,000 x 8 heads x 64 618 -> 586 and 734 -> 726, 40,000 x 8 x 96 206 -> 186 and 245 -> 226, x 128 245 -> 224
// and 524 -> 487.
// (Windows of one key, whose tensors pass the last cache: 200,000 x 8 x 64 377 -> 406 and 260 -> 314; 33 keys 401 -> 399 and 348 -> 348.)
template <int DP, int KS, int NP>
__device__ __forceinline__ void load_row(const char* row, int chunks, bf16x8 (&x)[KS][NP]) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int pl = 0; pl < NP; ++pl)
            x[ks][pl] = *reinterpret_cast<const bf16x8*>(row + (pl * (DP / 8) + min(2 * ks + half, chunks - 1)) * 16);
}
template <int KS, int NP>
__device__ __forceinline__ void settle_row(bool have, int chunks, bf16x8 (&x)[KS][NP]) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
            f32x4 v = __builtin_bit_cast(f32x4, x[ks][pl]);
            asm volatile("" : "+v"(v));
            const bool keep = have && (ks < KS - 1 || 2 * ks + half < chunks);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = keep ? v[e] : 0.0f;
            x[ks][pl] = __builtin_bit_cast(bf16x8, v);
        }
}

}  // namespace attn
}  // namespace g2v
