// Device side shared by the attention kernels (g2v_attention_fwd.hip, g2v_attention_bwd.hip).
//
// Matrix products run on v_mfma_f32_32x32x16_bf16.  Lane l of a wave holds, with n = l % 32 and g = l / 32,
//   A (32 x 16): row n, contraction slots 8g .. 8g+7;   B (16 x 32): column n, the same slots;
//   C (32 x 32): column n, rows 8 (i / 4) + 4 g + i % 4 in registers i = 0 .. 15.
// The contraction's order is free as long as A and B agree on it.  So a product's result C goes straight into the next
// product as B, without leaving its lane: registers 8 s .. 8 s + 7 are the slots of step s, which stand for rows
// 16 s + 4 g + {0..3} and 16 s + 8 + 4 g + {0..3}; the other operand reads its rows in that order (Frags::cols).
// Scores are computed with the long axis in the registers and the workgroup's own rows in the lanes (S^T = K Q^T for the
// forward and dQ, S = Q K^T for dK and dV): softmax statistics are one number a lane.
//
// float32 inputs are held as three bfloat16 planes, x = x0 + x1 + x2 exactly to 24 bits, and a product takes the six terms
// x_i y_j with i + j <= 2; what is dropped is below 2^-24 of each product.  At six bfloat16 products a float32 product
// runs 2.7 times as fast as on the float32 matrix instructions (1/16 of the bfloat16 rate).
#pragma once
#include "g2v_internal.h"

namespace g2v {
namespace attn {

typedef __attribute__((address_space(3))) char* lds_t;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;

// Rows of one tensor as the kernels read them: bfloat16, 16-byte chunks, byte strides of scene, token and head; a plane's
// chunks past `chunks` do not exist in memory and count as zero.  Packed tensors have their planes one after another.
struct RowSrc {
    const char* p;
    int64_t sb, sn, sh;
    int chunks;
};

// The chunk c of row r of a tile sits at slot swz(r, c): the 16 rows of an LDS cycle's A reads (one chunk each), and the
// four rows of a transposed read (four neighbouring chunks each), then fall on different banks.
template <int DP>
__device__ __forceinline__ int swz(int r, int c) {
    if constexpr (DP == 64) return c ^ ((((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1));
    else if constexpr (DP == 128) return c ^ (((r & 3) << 2) | ((r >> 2) & 3));
    else return c ^ ((r >> 2) & 3);
}

__device__ __forceinline__ uint32_t lds_off(const void* p) { return (uint32_t)(uintptr_t)(lds_t)p; }

// Direct-to-LDS loads: lane l's 16 (4) bytes land at lds + 16 l (4 l), whatever lanes are off.  Inline assembly, so that
// the compiler ties no wait to them: tile_barrier waits.
__device__ __forceinline__ const void* uniform(const void* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const void*>((uintptr_t)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ void dma16(const void* sbase, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 ::"v"(voff), "s"(uniform(sbase)), "s"(g2v::uniform((int)lds)) : "memory", "m0");
}
__device__ __forceinline__ void dma16(const void* addr, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 ::"v"(addr), "s"(g2v::uniform((int)lds)) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* sbase, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
                 ::"v"(voff), "s"(uniform(sbase)), "s"(g2v::uniform((int)lds)) : "memory", "m0");
}

// At most N loads of this wave outstanding (loads end in order) and its LDS operations done, then the other waves met.
template <int N>
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Workgroups of a kernel that share a CU: its launch bound (so that its registers fit), checked against its LDS, and what the
// splits of the long axis are planned by.  np, ns: planes of the inputs and of P and dS; waves: of a workgroup.  (Of one-wave
// workgroups at 32 channels six would fit, but the splits that fill so many places take the join longer: one query over 18000
// keys x 16 heads x 32 26.3 -> 27.3 us.  At one wave a SIMD four fit whatever their registers; their bound stays at two, with
// which the compiler keeps more of them out of the accumulation file: at 32 channels 4 queries x 9000 keys 20.3 -> 19.5 us.)
constexpr int kLdsBytes = 160 * 1024;
constexpr int launch_bound(int waves, int per_cu) { return waves == 1 ? 2 : per_cu; }
constexpr int fwd_per_cu(int np, int dp, int waves) {
    return np > 1 ? (dp > 64 ? 1 : 2) : waves == 1 || dp == 32 || dp == 96 ? 3 : 2;
}
constexpr int dq_per_cu(int np, int dp, int waves) {
    return np > 1 ? (dp > 64 ? 1 : 2) : waves == 1 && dp <= 64 ? 3 : 2;
}
constexpr int dkv_per_cu(int np, int ns, int dp) {
    return np > 1 ? (dp > 32 ? 1 : 2) : dp == 32 ? 4 : dp == 64 && ns == 1 ? 3 : dp == 128 && ns > 1 ? 1 : 2;
}

// Buffers of a kernel's tiles (pairs of `bytes`): three, loaded two tiles ahead, where the `groups` workgroups that the
// kernel's registers allow a CU fit its 160 KB so, else two, loaded one ahead.  Three for two: 9000 x 12 heads x 64 float32
// forward 1.33 -> 1.25 ms; bfloat16 at 96 channels dK and dV 0.395 -> 0.367 ms, but the forward there, whose
// workgroups come three to a CU with two buffers, 0.22 -> 0.25 ms.  The barrier before tile t lets tile t + 1's loads go
// on, if there are three buffers and that tile is whole: kLoads of them a wave (`counted`; in the last tile a wave's lanes
// may be off altogether).  It also ends every wave's reads of tile t - 1, whose buffer is loaded next.
constexpr int buffers(int groups, int bytes) { return 3 * 2 * bytes <= kLdsBytes / groups ? 3 : 2; }
template <int kBuffers, int kLoads>
__device__ __forceinline__ void next_tile(bool counted) {
    if (kBuffers == 3 && kLoads > 0 && counted) tile_barrier<kLoads>();
    else tile_barrier<0>();
}

// A tile of ROWS rows of one tensor in LDS: [plane][row][DP], swizzled, filled by NT threads.
template <int NP, int DP, int ROWS, int NT>
struct Tile {
    static constexpr int C = DP / 8;                    // chunks of a row
    static constexpr int kChunks = NP * ROWS * C;
    static constexpr int kBytes = kChunks * 16;
    static constexpr int kIter = (kChunks + NT - 1) / NT;
    static constexpr int kLoads = kChunks % NT ? 0 : kIter;    // of every wave; 0: not the same for all

    int row[kIter];         // this thread's row of each load
    uint32_t off[kIter];    // byte offset of its chunk in the row
    bool on[kIter];         // the chunk exists

    __device__ __forceinline__ void init(const RowSrc& s) {
#pragma unroll
        for (int it = 0; it < kIter; ++it) {
            const int L = it * NT + threadIdx.x;
            const int pl = L / (ROWS * C), rem = L % (ROWS * C);
            row[it] = rem / C;
            const int c = swz<DP>(row[it], rem % C);
            off[it] = (uint32_t)(pl * C + c) * 16;
            on[it] = c < s.chunks && L < kChunks;
        }
    }
    __device__ __forceinline__ uint32_t dst(uint32_t lds, int it) const {
        return lds + it * NT * 16 + (uint32_t)g2v::uniform(threadIdx.x >> 6) * 1024;
    }
    // Rows [j0, j0 + ROWS) of base, all of them there.
    __device__ __forceinline__ void load(const char* base, int64_t sn, int64_t j0, uint32_t lds) const {
        const char* p = base + j0 * sn;
#pragma unroll
        for (int it = 0; it < kIter; ++it)
            if (on[it]) dma16(p, (uint32_t)row[it] * (uint32_t)sn + off[it], dst(lds, it));
    }
    // Rows [j0, n) of base, zeros up to ROWS.
    __device__ __forceinline__ void load_tail(const char* base, int64_t sn, int64_t j0, int64_t n, char* lds) const {
#pragma unroll
        for (int it = 0; it < kIter; ++it) {
            if (!on[it]) continue;
            if (j0 + row[it] < n) dma16(base + (j0 + row[it]) * sn + off[it], dst(lds_off(lds), it));
            else *reinterpret_cast<f32x4*>(lds + (it * NT + threadIdx.x) * 16) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
};

// Chunks that do not exist are zero for the whole kernel: cleared once, before the first load.
template <int NT>
__device__ __forceinline__ void clear_lds(char* lds, int bytes) {
    for (int i = threadIdx.x * 16; i < bytes; i += NT * 16) *reinterpret_cast<f32x4*>(lds + i) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();
}

// Reading a tile.  The slots are permuted by exclusive or, so a lane's address of any chunk is its address of chunk 0 with
// bits flipped that are known when compiling (for DP = 96, whose rows are no power of two, only the lowest chunk bits are
// permuted, and the rest is an offset): two registers a lane, whatever the number of chunks.
template <int DP>
struct Frags {
    uint32_t row, tr;    // LDS offsets: row n's chunk g; the transposed reads' first row and chunk

    __device__ __forceinline__ void init(uint32_t lds) {
        const int l = threadIdx.x & 63, n = l & 31, g = l >> 5, dh = (l >> 4) & 1, i = l & 15;
        const int r = 4 * g + (i >> 2);
        row = lds + n * (DP * 2) + swz<DP>(n, g) * 16;
        tr = lds + r * (DP * 2) + swz<DP>(r, 2 * dh + ((i & 3) >> 1)) * 16 + (i & 1) * 8;
    }
    // A operand: rows 32 rb .. 32 rb + 31, contraction over d in 16 ks .. 16 ks + 15; `at` bytes into the buffer.
    __device__ __forceinline__ bf16x8 rows(uint32_t buf, int at, int rb, int ks) const {
        typedef const __attribute__((address_space(3))) bf16x8* p_t;
        const uint32_t flip = DP == 96 ? (ks & 1) * 32 : ks * 32, off = DP == 96 ? (ks >> 1) * 64 : 0;
        return *(p_t)(((row + buf) ^ flip) + at + rb * 32 * (DP * 2) + off);
    }
    // A operand of the transposed tile: rows d = 32 t .. 32 t + 31, contraction over the tile's rows 32 rb + 16 s .. + 15
    // in the order of a result's registers.  Each read transposes 4 x 16 values within 16 lanes.
    __device__ __forceinline__ bf16x8 cols(uint32_t buf, int at, int rb, int s, int t) const {
        typedef __attribute__((address_space(3))) s16x4* p_t;
        const uint32_t flip = DP == 96 ? 0 : t * 64, off = DP == 96 ? t * 64 : 0;
        const uint32_t base = at + (rb * 32 + 16 * s) * (DP * 2) + off;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p_t)(((tr + buf) ^ flip) + base));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (p_t)(((tr + buf) ^ (flip ^ (DP == 64 ? 16 : 32))) + base + 8 * (DP * 2)));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// B operand from memory: this lane's row, contraction over d in 16 ks .. + 15 of plane pl; zero where there is none.
template <int DP>
__device__ __forceinline__ bf16x8 mem_frag(const char* row, bool have, int chunks, int pl, int ks) {
    const int c = 2 * ks + ((threadIdx.x >> 5) & 1);
    if (have && c < chunks) return *reinterpret_cast<const bf16x8*>(row + (pl * (DP / 8) + c) * 16);
    return __builtin_bit_cast(bf16x8, s16x8{0, 0, 0, 0, 0, 0, 0, 0});
}

// acc += A B, with NA and NB planes: the terms of the first max(NA, NB) orders.
template <int NA, int NB>
__device__ __forceinline__ f32x16 mma(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x16 acc) {
    constexpr int N = NA > NB ? NA : NB;
#pragma unroll
    for (int o = N - 1; o >= 0; --o)
#pragma unroll
        for (int i = 0; i <= o; ++i)
            if (i < NA && o - i < NB) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[o - i], acc, 0, 0, 0);
    return acc;
}

// Registers 8 s .. 8 s + 7 of a result as the B operand of step s.  One plane rounds to nearest even (2^-9 of each
// probability or score gradient, independent errors that average out over the sum); three keep 24 bits.
template <int NP>
__device__ __forceinline__ void to_operand(const f32x16& x, int s, bf16x8 (&o)[NP]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float r = x[8 * s + j];
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
            const __bf16 h = (__bf16)r;
            o[pl][j] = h;
            r -= (float)h;
        }
    }
}

// acc + the sum of an operand's eight values.
__device__ __forceinline__ float add_operand(const bf16x8& x, float acc) {
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int j = 0; j < 8; j += 2) acc = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[j], x[j + 1]}, one, acc, false);
    return acc;
}

// Max / sum of a lane and the lane 32 away, in both.  (The swap's results are read as numbers first: __builtin_bit_cast of
// a vector's element takes element 0 with this compiler.)
__device__ __forceinline__ void half_swap(float v, float& x, float& y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const unsigned lo = r[0], hi = r[1];
    x = __uint_as_float(lo);
    y = __uint_as_float(hi);
}
__device__ __forceinline__ float half_max(float v) {
    float x, y;
    half_swap(v, x, y);
    return fmaxf(x, y);
}
__device__ __forceinline__ float half_sum(float v) {
    float x, y;
    half_swap(v, x, y);
    return x + y;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Tile row of register i of a result.
__device__ __forceinline__ int reg_row(int i) { return 8 * (i >> 2) + 4 * ((threadIdx.x >> 5) & 1) + (i & 3); }

// Four neighbouring values of a row, d of D, stored in the row's type.
template <typename T>
__device__ __forceinline__ void store4(T* row, int d, int D, float x0, float x1, float x2, float x3) {
    const float x[4] = {x0, x1, x2, x3};
    if ((D & 3) == 0) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        if (d < D) *reinterpret_cast<v4*>(row + d) = v4{(T)x0, (T)x1, (T)x2, (T)x3};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (d + j < D) row[d + j] = (T)x[j];
    }
}

// The same for what bfloat16 rounding leaves of the values.
__device__ __forceinline__ float lost_by_rounding(float x) { return x - (float)(__bf16)x; }

// Into which workgroups the tiles of the heads go: the first `head` tiles of each (row0 rows) to head_splits each, the others
// to `splits` each.  A tile's only workgroup writes its result; more write partial results, which are joined: rows [0, row0)
// as (head_splits, bhs, row0, ..) where they are split, behind them (splits, bhs, rows - row0, ..).
struct Parts {
    int tiles, head, head_splits, splits, row0;
};
inline int64_t workgroups(const Parts& p, int bhs) {
    return bhs * ((int64_t)p.head * p.head_splits + (int64_t)(p.tiles - p.head) * p.splits);
}
// Rows of a head that a join does not see, and those of all heads' partial results.
__host__ __device__ __forceinline__ int joined_from(const Parts& p, int rows) {
    return p.head_splits > 1 ? 0 : p.splits > 1 ? p.row0 : rows;
}
inline int64_t part_rows(const Parts& p, int bhs, int64_t rows) {
    return bhs * ((p.head_splits > 1 ? p.head_splits * (int64_t)p.row0 : 0) + (p.splits > 1 ? p.splits * (rows - p.row0) : 0));
}

// Where row r of head bh has its partial results: the first, and from one split to the next.
struct PartRow {
    int64_t at, step;
    int splits;
};
__device__ __forceinline__ PartRow part_row(const Parts& p, int bhs, int bh, int rows, int r) {
    PartRow o;
    if (r < p.row0) {
        o.splits = p.head_splits;
        o.step = (int64_t)bhs * p.row0;
        o.at = (int64_t)bh * p.row0 + r;
    } else {
        o.splits = p.splits;
        o.step = (int64_t)bhs * (rows - p.row0);
        o.at = (int64_t)bh * (rows - p.row0) + r - p.row0 + (p.head_splits > 1 ? (int64_t)bhs * p.head_splits * p.row0 : 0);
    }
    return o;
}

// A workgroup's item: head (scene b, key head h), tile and split of how many, heads fastest, so that with 8 heads or a
// multiple the workgroups of a head share an XCD's L2 (workgroups go to the 8 XCDs in turn).
struct Item {
    int b, h, bh, tile, split, splits;
};
__device__ __forceinline__ Item item_of(int id, int bhs, int hk, const Parts& p) {
    Item w;
    int at = g2v::uniform(id / bhs), first = 0, tiles = p.head;    // (divisions run in vector registers)
    w.bh = id - at * bhs;
    w.splits = p.head_splits;
    if (at >= p.head * p.head_splits) {
        at -= p.head * p.head_splits;
        first = p.head;
        tiles = p.tiles - p.head;
        w.splits = p.splits;
    }
    w.split = g2v::uniform(at / tiles);
    w.tile = first + at - w.split * tiles;
    w.b = g2v::uniform(w.bh / hk);
    w.h = w.bh - w.b * hk;
    return w;
}

// Units [lo, hi) of `all` that fall to a split.
__device__ __forceinline__ void split_range(int all, int split, int splits, int& lo, int& hi) {
    const int per = (all + splits - 1) / splits;
    lo = split * per;
    lo = lo < all ? lo : all;
    hi = lo + per < all ? lo + per : all;
}

}  // namespace attn

struct AttnFwd {
    attn::RowSrc q, k, v;
    const int* count;   // (batch) valid keys, the first rows of k and v; null: nk
    int nq, nk, hq, hk, group, dim, bhs;
    attn::Parts parts;
    float c;            // scale log2(e)
    void* out;          // (batch, nq, hq, dim)
    void* rest;         // like out: what rounding to bfloat16 left of it, or null
    float* lse;         // (batch, hq, nq) log2 of the sum of 2^(c s); +inf for a row without keys
    float* part_o;      // partial results, DP values each
    float* part_ml;     // and their maximum and sum
};

struct AttnBwd {
    attn::RowSrc q, k, v, g;
    const int* count;    // as in AttnFwd
    const int* list;     // (batch, nk) the keys that the rows of k and v are, valid ones first; null: in order
    int nq, nk, hq, hk, group, dim, bhs;
    attn::Parts parts;
    bool by_count;       // set by launch_attn_dkv
    int nqp;             // nq rounded up to 64: rows of lse and delta, padded with +inf and 0
    float c, scale;
    const float *lse, *delta;   // (batch, hq, nqp); -delta
    void *dq, *dk, *dv;
    float* part;         // partial results: dq: DP values each; dk and dv: 2 DP
};

}  // namespace g2v
