// Attention over sets of Gaussians, forward: O = softmax(scale Q K^T) V over the valid keys of each scene.
//
// One pass over the keys with the running reference and sum of the softmax.  The query heads that share a key head are
// rows of one problem (row r = query r / group, head r % group), so K and V are read once for all of them.  A wave owns NQB
// blocks of 32 rows: their Q stays in registers as B operands, K and V tiles come through LDS by direct loads, S^T = K Q^T
// lands with a lane per row and goes through exp2 straight into O^T += V^T P^T (no exchange of P).  Few rows, or a last
// round of workgroups that leaves most of the card idle: the keys are dealt to `splits` workgroups and k_attn_join joins.
//
// Bound by the matrix and the vector unit of a SIMD taking turns: at 64 channels a row's 64 keys are 256 cycles of
// products and, at 8.7 cycles for an exp2 of 64 lanes and 2.1 for anything else, about 220 of vector work; the counters show
// 44 and about 50 % of the kernel's cycles.  Two blocks of rows a wave halve what is read from LDS for each product (one block
// and three or four waves a SIMD: 1.54 and 1.48 ms for 1.38; at 128 channels two blocks spill 12 registers, 52 bytes a lane, and
// are faster than one all the same).  18000 x 16 heads x 64 bfloat16: 1.32 to 1.38 ms by card, 970 to 1000 TFLOP/s; 9000
// x 12 x 64 float32: 1.21 to 1.23 ms, 205 TFLOP/s, 1250 of bfloat16 terms.
#include "g2v_attention.h"

namespace g2v {
namespace {
using namespace attn;

// The maximum in use is that of a wave's first tile, and is taken anew from a tile in which a row's sum of probabilities
// passes this: any finite reference does in float32 as long as nothing overflows, so that most tiles skip the maximum
// (a tenth of the vector instructions; matrix and vector work of a SIMD take their time one after the other).
constexpr float kFar = 1048576.0f;

// The reference (times c) of a row whose scores were all -inf so far: any other one passes kFar from it
// (or, where c is so small that the reference itself is at float32's lowest values, is in its reach).
constexpr float kLowest = -1e37f;

// Four values of the output's row at `at`.  For a bfloat16 output that a backward follows, what its rounding leaves goes
// to `rest`: the backward's delta = sum_d dO O is subtracted from every dP of a row, and an output rounded to 2^-9 puts
// the same error on all of them, which their sum dS K does not average out (dQ then 3.2e-3 off instead of 2.2e-3).
template <typename T>
__device__ __forceinline__ void store_out(const AttnFwd& a, int64_t at, int d, float x0, float x1, float x2, float x3) {
    store4<T>(static_cast<T*>(a.out) + at, d, a.dim, x0, x1, x2, x3);
    if constexpr (sizeof(T) == 2)
        if (a.rest)
            store4<T>(static_cast<T*>(a.rest) + at, d, a.dim, lost_by_rounding(x0), lost_by_rounding(x1),
                      lost_by_rounding(x2), lost_by_rounding(x3));
}

// KS: steps of 16 that the head's width takes in the scores' product (the last of DP / 16 may hold nothing but padding).
template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
__global__ void __launch_bounds__(NW * 64, launch_bound(NW, fwd_per_cu(NP, DP, NW))) k_attn_fwd(AttnFwd a) {
    constexpr int NT = NW * 64, KB = KT / 32, DB = DP / 32;
    typedef Tile<NP, DP, KT, NT> TileT;
    constexpr int kBuffers = buffers(NP == 1 && NQB == 1 ? 3 : 2, TileT::kBytes), kAhead = kBuffers - 1;
    __shared__ __attribute__((aligned(1024))) char lds[kBuffers][2][TileT::kBytes];
    static_assert(fwd_per_cu(NP, DP, NW) * sizeof(lds) <= kLdsBytes, "planned by more workgroups than fit");
    const Item w = item_of(blockIdx.x, a.bhs, a.hk, a.parts);
    const int lane = threadIdx.x & 63, rows = a.group * a.nq;
    const int r0 = (w.tile * NW + g2v::uniform(threadIdx.x >> 6)) * (NQB * 32) + (lane & 31);
    const int n = a.count ? a.count[w.b] : a.nk;
    const char* kbase = a.k.p + w.b * a.k.sb + w.h * a.k.sh;
    const char* vbase = a.v.p + w.b * a.v.sb + w.h * a.v.sh;
    int t0, t1;
    split_range((n + KT - 1) / KT, w.split, w.splits, t0, t1);

    bf16x8 q[NQB][KS][NP];
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        const int r = r0 + 32 * b, rc = r < rows ? r : rows - 1;
        const int tok = rc / a.group, head = w.h * a.group + rc - tok * a.group;
        const char* row = a.q.p + w.b * a.q.sb + tok * a.q.sn + head * a.q.sh;
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
    auto load = [&](int t, int buf) {
        if ((t + 1) * KT <= n) {
            tile.load(kbase, a.k.sn, (int64_t)t * KT, lds_off(lds[buf][0]));
            tile.load(vbase, a.v.sn, (int64_t)t * KT, lds_off(lds[buf][1]));
        } else {
            tile.load_tail(kbase, a.k.sn, (int64_t)t * KT, n, lds[buf][0]);
            tile.load_tail(vbase, a.v.sn, (int64_t)t * KT, n, lds[buf][1]);
        }
    };

    f32x16 o[DB][NQB];
    float m[NQB], l[NQB];
#pragma unroll
    for (int b = 0; b < NQB; ++b) {
        m[b] = -INFINITY;
        l[b] = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][b][i] = 0.0f;
    }
    if (t0 < t1) load(t0, 0);
    if (kAhead > 1 && t0 + 1 < t1) load(t0 + 1, 1);
    for (int t = t0, buf = 0; t < t1; ++t, buf = buf == kBuffers - 1 ? 0 : buf + 1) {
        next_tile<kBuffers, 2 * TileT::kLoads>(t + 1 < t1 && (t + 2) * KT <= n);
        if (t + kAhead < t1) load(t + kAhead, buf == 0 ? kBuffers - 1 : buf - 1);
        const uint32_t at = buf * 2 * TileT::kBytes;
        bf16x8 p[KB][2][NQB][NP];
        float sum[NQB];
        for (bool fresh = t == t0;; fresh = true) {
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
            if ((t + 1) * KT > n) {   // the last tile's rows past the end
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (t * KT + kb * 32 + reg_row(i) >= n)
#pragma unroll
                            for (int b = 0; b < NQB; ++b) s[kb][b][i] = -INFINITY;
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
                    if (top == -INFINITY) top = fmaxf(kLowest / a.c, -3e38f);
                    const float f = exp2_fast((m[b] - top) * a.c);
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
                const float mc = m[b] * a.c;
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

// Joins the splits of a row: O = sum O_s 2^(m_s - M) / sum l_s 2^(m_s - M).  DP / 4 lanes and `parts` threads of each to a
// row: where rows are few their splits are many, and one thread after another's loads would take the time.  A
// fixed order.
template <int DP, typename T>
__global__ void __launch_bounds__(256) k_attn_join(AttnFwd a, int parts) {
    constexpr int kLanes = DP / 4;
    __shared__ float red[6][256];
    const int rows = a.group * a.nq, from = joined_from(a.parts, rows), own = rows - from, per = 256 / (kLanes * parts);
    const int part = threadIdx.x % parts, e = threadIdx.x / parts, d = e % kLanes * 4;
    const int row = blockIdx.x * per + e / kLanes;
    const bool live = e / kLanes < per && row < a.bhs * own;
    const int bh = live ? row / own : 0, r = live ? from + row - bh * own : from;
    const PartRow pr = part_row(a.parts, a.bhs, bh, rows, r);
    float top = -INFINITY, total = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        for (int s = part; s < pr.splits; s += parts) top = fmaxf(top, a.part_ml[2 * (pr.at + s * pr.step)]);
#pragma unroll 4
        for (int s = part; s < pr.splits; s += parts) {
            const int64_t p = pr.at + s * pr.step;
            const float l = a.part_ml[2 * p + 1];
            // a split without keys has no sum, and its maximum is the lowest value
            const float f = l == 0.0f ? 0.0f : exp2_fast(a.part_ml[2 * p] - top);
            const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + p * DP + d);
            total = fmaf(l, f, total);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(x[j], f, o[j]);
        }
    }
    if (parts > 1) {
        red[0][threadIdx.x] = top;
        red[1][threadIdx.x] = total;
#pragma unroll
        for (int j = 0; j < 4; ++j) red[2 + j][threadIdx.x] = o[j];
        __syncthreads();
        if (part > 0) return;
        for (int k = 1; k < parts; ++k) {
            const int i = threadIdx.x + k;
            const float up = fmaxf(top, red[0][i]);
            const float f = total == 0.0f ? 0.0f : exp2_fast(top - up), g = red[1][i] == 0.0f ? 0.0f : exp2_fast(red[0][i] - up);
            top = up;
            total = total * f + red[1][i] * g;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = o[j] * f + red[2 + j][i] * g;
        }
    }
    if (!live) return;
    const int b = bh / a.hk, tok = r / a.group, head = (bh % a.hk) * a.group + r % a.group;
    const float inv = total > 0.0f ? 1.0f / total : 0.0f;
    if (a.lse && d == 0) a.lse[((int64_t)b * a.hq + head) * a.nq + tok] = total > 0.0f ? top + log2f(total) : INFINITY;
    store_out<T>(a, (((int64_t)b * a.nq + tok) * a.hq + head) * a.dim, d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

// ---- what both directions prepare -----------------------------------------------------------------------------------

constexpr int kListThreads = 1024;
constexpr float kMaxBf16 = 0x1.fep127f;

// Valid keys of a scene in ascending order, then the others; their number in count.  One workgroup a scene.
__global__ void __launch_bounds__(kListThreads) k_attn_list(int nk, const unsigned char* mask, int* list, int* count) {
    __shared__ int sums[kListThreads / 64];
    const unsigned char* mk = mask + (int64_t)blockIdx.x * nk;
    int* out = list + (int64_t)blockIdx.x * nk;
    const int per = (nk + kListThreads - 1) / kListThreads;
    const int lo = min((int)threadIdx.x * per, nk), hi = min(lo + per, nk);
    int mine = 0;
    for (int j = lo; j < hi; ++j) mine += mk[j] != 0;
    int scan = mine;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(scan, d);
        if (lane >= d) scan += v;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    int before = 0, total = 0;
    for (int i = 0; i < kListThreads / 64; ++i) {
        if (i < wave) before += sums[i];
        total += sums[i];
    }
    int at = before + scan - mine;              // valid keys before lo
    int other = total + lo - at;                // the others before lo come after all valid ones
    for (int j = lo; j < hi; ++j) {
        if (mk[j]) out[at++] = j;
        else out[other++] = j;
    }
    if (threadIdx.x == 0) count[blockIdx.x] = total;
}

// Rows as NP bfloat16 planes of DP values each, contiguous (batch, heads, n): what the kernels cannot read in place
// (float32, and rows that are not whole 16-byte chunks), and the valid keys of a mask one after another (9000 keys, a
// fifth of them masked, 12 heads of 64: the forward takes 0.34 ms through an index in its loop, 0.28 ms on packed rows).
// A workgroup packs neighbouring rows of one head, a thread one chunk of every plane.  MASK: the list of valid keys is
// made here as well, each workgroup counting the mask before its rows and in all.
template <int NP, bool MASK, typename T>
__global__ void __launch_bounds__(256) k_attn_pack(AttnPack a) {
    __shared__ int counts[2][4];
    __shared__ unsigned long long bits;
    const int C = a.dp / 8, R = 256 / C;
    int64_t id = blockIdx.x;
    int k = 0;
    while (k < a.tensors - 1 && id >= a.blocks[k]) id -= a.blocks[k++];
    const int per = (a.n[k] + R - 1) / R;
    const int64_t bh = id / per, b = bh / a.heads[k];
    const int r0 = (int)(id - bh * per) * R;
    const int rr = threadIdx.x / C, c = threadIdx.x - rr * C;
    int64_t i = r0 + rr, slot = i;
    bool have = rr < R && i < a.n[k];
    if (MASK && a.keys[k]) {
        const unsigned char* mask = a.mask + b * a.n[k];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        int before = 0, total = 0;
        for (int j0 = 0; j0 < a.n[k]; j0 += 256) {      // the same for all lanes
            const int j = j0 + threadIdx.x;
            const bool valid = j < a.n[k] && mask[j];
            before += __popcll(__ballot(valid && j < r0));
            total += __popcll(__ballot(valid));
        }
        if (lane == 0) {
            counts[0][wave] = before;
            counts[1][wave] = total;
        }
        if (wave == 0) {
            const unsigned long long m = __ballot(r0 + lane < a.n[k] && mask[r0 + lane]);
            if (lane == 0) bits = m;
        }
        __syncthreads();
        before = counts[0][0] + counts[0][1] + counts[0][2] + counts[0][3];
        total = counts[1][0] + counts[1][1] + counts[1][2] + counts[1][3];
        const bool valid = have && (bits >> rr & 1);
        const int rank = before + __popcll(bits & ((1ull << rr) - 1));
        if (a.list_tensor == k && bh % a.heads[k] == 0) {    // valid keys in ascending order, then the others
            if (have && c == 0) a.list_out[b * a.n[k] + (valid ? rank : total + (int)i - rank)] = (int)i;
            if (r0 == 0 && threadIdx.x == 0) a.count_out[b] = total;
        }
        have = valid;
        slot = rank;
    } else if (a.count && a.keys[k]) {
        have = have && i < a.count[b];     // what lies behind is never read
        if (have) i = a.list[b * a.n[k] + i];
    }
    if (!have) return;
    const T* src = static_cast<const T*>(a.src[k]) + b * a.sb[k] + i * a.sn[k] + bh % a.heads[k] * a.sh[k];
    const int64_t row = bh * a.n[k] + slot;
    // a whole chunk in one access or two, at any alignment (global memory takes it); a row's last elements one by one
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    constexpr int kPer = 16 / sizeof(T);
    vec x[8 / kPer];
#pragma unroll
    for (int h = 0; h < 8 / kPer; ++h) {
        const int d = c * 8 + h * kPer;
        if (d + kPer <= a.dim) {
            x[h] = *reinterpret_cast<const vec*>(src + d);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[h][j] = d + j < a.dim ? src[d + j] : (T)0.0f;
        }
    }
    bf16x8 o[NP];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float r = (float)x[j / kPer][j % kPer];
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
            // a finite value above the largest bfloat16 starts with that (what is left is small); an infinity is its first
            // plane alone
            float h = (float)(__bf16)r;
            if (NP > 1 && pl == 0 && !__builtin_isfinite(h) && __builtin_isfinite(r)) h = copysignf(kMaxBf16, r);
            o[pl][j] = (__bf16)h;
            r = __builtin_isfinite(h) ? r - h : 0.0f;
        }
    }
#pragma unroll
    for (int pl = 0; pl < NP; ++pl)
        *reinterpret_cast<bf16x8*>(static_cast<char*>(a.dst[k]) + ((row * NP + pl) * C + c) * 16) = o[pl];
}

template <int NP, int DP, int KS, int NQB, int NW, int KT, typename T>
hipError_t fwd_launch(const AttnFwd& a, hipStream_t s) {
    G2V_LAUNCH((k_attn_fwd<NP, DP, KS, NQB, NW, KT, T>), dim3((unsigned)workgroups(a.parts, a.bhs)), dim3(NW * 64), 0, s, a);
    const int64_t rows = (int64_t)a.bhs * (a.group * a.nq - joined_from(a.parts, a.group * a.nq));
    if (rows > 0) {
        const int parts = attn_join_parts(rows, DP / 4, std::max(a.parts.head_splits, a.parts.splits));
        G2V_LAUNCH((k_attn_join<DP, T>), dim3((unsigned)ceil_div(rows, 256 / (DP / 4 * parts))), dim3(256), 0, s, a, parts);
    }
    return hipGetLastError();
}

template <int NP, int DP, int NQB, int KT, typename T>
hipError_t fwd_waves(const AttnFwd& a, const AttnShape& g, hipStream_t s) {
    const bool full = a.dim > DP - 16;
    if constexpr (NP == 1)
        if (g.waves == 1)
            return full ? fwd_launch<NP, DP, DP / 16, 1, 1, KT, T>(a, s) : fwd_launch<NP, DP, DP / 16 - 1, 1, 1, KT, T>(a, s);
    return full ? fwd_launch<NP, DP, DP / 16, NQB, 4, KT, T>(a, s) : fwd_launch<NP, DP, DP / 16 - 1, NQB, 4, KT, T>(a, s);
}

}  // namespace

AttnShape attn_fwd_shape(bool f32, int dp, int64_t rows) {
    AttnShape g;
    // Rows that fit one wave's block: workgroups of that one wave, three to a CU with tiles of their own in flight (one
    // query over 18000 keys x 16 heads x 64: 19 us; four waves, three of them idle, 29 us).  float32 keys are packed first,
    // which takes longer than either.
    g.waves = !f32 && rows <= 32 ? 1 : 4;
    g.blocks = g.waves == 4 && !f32 && dp != 96 ? 2 : 1;
    g.tile = (f32 && dp > 32) || dp > 96 ? 32 : 64;
    g.per_cu = fwd_per_cu(f32 ? 3 : 1, dp, g.waves);
    g.products = 2;
    return g;
}

hipError_t launch_attn_fwd(const AttnFwd& a, bool f32, int dp, hipStream_t s) {
    const AttnShape g = attn_fwd_shape(f32, dp, (int64_t)a.group * a.nq);
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

hipError_t launch_attn_list(int batch, int nk, const unsigned char* mask, int* list, int* count, hipStream_t s) {
    if (batch > 0) G2V_LAUNCH(k_attn_list, dim3(batch), dim3(kListThreads), 0, s, nk, mask, list, count);
    return hipGetLastError();
}

hipError_t launch_attn_pack(const AttnPack& args, bool f32, hipStream_t s) {
    AttnPack a = args;
    const int R = 256 / (a.dp / 8);
    int64_t blocks = 0;
    for (int k = 0; k < a.tensors; ++k) {
        a.blocks[k] = ceil_div(a.n[k], R) * a.batch * a.heads[k];
        blocks += a.blocks[k];
    }
    if (blocks == 0) return hipSuccess;
    const dim3 grid((unsigned)blocks), block(256);
    if (a.mask) {
        if (f32) G2V_LAUNCH((k_attn_pack<3, true, float>), grid, block, 0, s, a);
        else G2V_LAUNCH((k_attn_pack<1, true, __bf16>), grid, block, 0, s, a);
    } else {
        if (f32) G2V_LAUNCH((k_attn_pack<3, false, float>), grid, block, 0, s, a);
        else G2V_LAUNCH((k_attn_pack<1, false, __bf16>), grid, block, 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace g2v
