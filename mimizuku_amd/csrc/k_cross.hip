// Attention over an encoder's fp16 keys and values of any length (mz_cross_attention_args in mimizuku.h).
//
// One pass over the positions with the running maximum and sum of the softmax. A workgroup takes 16 QT queries of one (row, kv
// head) (its tokens times the query heads that share the kv head) and a share of the blocks of 32 positions; its waves take the
// blocks in turn, each with a state of its own, and join them at the end.
//
// Per block, with 16x16x32 products: S^T = K Q^T, the rows of tile j being positions 8 (i / 4) + 4 j + i % 4, so that lane (query
// c, group g) of the two results holds the eight positions 8 g .. 8 g + 7 of its query: in this order they are the k values of
// that lane in the product O^T = V^T P^T, so probabilities never leave their registers. Values lie by positions: lane (i, g) loads
// channels 4 i .. 4 i + 3 of those eight positions, eight bytes each, and 16 byte permutations make of them its operands of four
// products, whose row i is channel 4 i + u.
//
// P goes into its product as the sum of two fp16 numbers, both cut: one alone would add an error of the size of the output's
// rounding. The maximum of a state is moved only when a score passes it by more than 8 (in powers of two), so that most blocks need
// no exchange between lanes and no rescaling; P is carried times 2^7, at most 2^15. What is lost of it is below 2^-21 of itself, or
// where the second number would end below fp16's smallest step, 2^-24, below that: 2^-31 of the row's largest.
//
// Times here are of a call among 40 back to back, on keys and values of four layers in turn; rows are as long as stated, "unequal"
// ones 0.27 to 1 times that. Both sides of a rule are of one run. Under a profiler, which runs launches apart, they are up to 2 us
// longer.
#include <algorithm>

#include "mz_attn.h"
#include "mz_common.h"
#include "mz_kernels.h"

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int BLK = 32;
constexpr float UP = 7.f;  // log2 of what P is carried times

// what a row's queries see: positions first .. end - 1 of its slot
struct Seen {
    long slot;
    int first, end, count;
};
__device__ __forceinline__ Seen seen_of(const MzCross& a, int r) {
    // (all that there are go out together, an absent one's place being some other word: a branch around each would wait for one
    // after the other)
    int slot = 0, first = 0, len = 0, count = 0;
    const int* any = a.slot ? a.slot : a.first ? a.first : a.len ? a.len : a.count;
    if (any) {
        slot = *(a.slot ? a.slot + r : any);
        first = *(a.first ? a.first + r : any);
        len = *(a.len ? a.len + r : any);
        count = *(a.count ? a.count + r : any);
        slot = __builtin_amdgcn_readfirstlane(slot);
        first = __builtin_amdgcn_readfirstlane(first);
        len = __builtin_amdgcn_readfirstlane(len);
        count = __builtin_amdgcn_readfirstlane(count);
    }
    Seen s;
    s.slot = a.slot ? slot : r;
    s.count = a.count ? min(max(count, 0), a.tokens) : a.tokens;
    s.first = a.first ? max(first, 0) : 0;
    s.end = a.len ? min(max(len, 0), a.positions) : a.positions;
    if (s.slot < 0 || s.slot >= a.slots) s.slot = s.end = 0;
    s.end = max(s.end, s.first);  // (nothing: first .. first)
    return s;
}

struct Launch {
    int qt, tiles, splits;  // queries of a workgroup / 16, such tiles of a (row, kv head), workgroups that share the blocks
    int waves, own;         // waves of a workgroup; whether each has 16 qt queries of its own
    int per;                // most blocks of a share
    int kept;               // alignment rows: scores that a workgroup keeps in LDS for each query, 0: in their rows
    int group;              // query heads of a kv head
    unsigned by_heads, by_group;  // for dividing by kv_heads and group (see divided)
};

// The bytes of `n` positions `step` bytes apart, as far as a buffer descriptor reaches: what lies behind reads as zeros. (A block's
// are below 2^30 + 2^7.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t positions_at(const f16* p, long step, int n) {
    const long bytes = n > 0 ? (n - 1) * step + 128 : 0;
    return rsrc(p, (unsigned)min(bytes, 0x7fffffffL));
}

// A block as it lies: keys as operands of two tiles, values by positions.
struct Raw {
    u32x4 k[2][2];
    u32x2 v[8];
};

// the four operands of values: row i of product u is channel 4 i + u
__device__ __forceinline__ void by_channels(const u32x2 (&v)[8], f16x8 (&to)[4]) {
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const unsigned sel = u & 1 ? 0x07060302u : 0x05040100u;  // the high or low halves of both
        u32x4 x;
#pragma unroll
        for (int p = 0; p < 4; p++) x[p] = __builtin_amdgcn_perm(v[2 * p + 1][u >> 1], v[2 * p][u >> 1], sel);
        to[u] = __builtin_bit_cast(f16x8, x);
    }
}

// x less the fp16 number in the low or the high half of h, in one instruction (the compiler takes a conversion and a subtraction)
__device__ __forceinline__ float less_low(float x, unsigned h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ float less_high(float x, unsigned h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}

template <int QT>
struct State {
    float m[QT], l[QT];
    f32x4 acc[QT][4];  // result u of lane (c, g) holds channels 16 g + 4 e + u of query c
};

// Four waves that take the blocks in turn, or, with OWN, that have 16 QT queries of their own each and take every block, or, eight of
// them, two such fours that have half of the blocks each (no alignment rows).
//
// Few queries (a decoder's step) are bound by the bytes of keys and values: 32 rows of 20 heads and 409 to 1500 positions, 157 MB
// in 35.9 us (4.4 TB/s, of 6.6 that a plain read reaches: each wave has the two blocks on their way that its registers hold, and rows of
// unequal lengths leave the last CUs alone); one row of 6 heads and 250 positions, 5.0 us, is a chain of launch, lengths, keys,
// values and the join. Prompts, 8 rows of 224 tokens, 20 heads, 1500 positions: 39 us (355 TFLOP/s, counted once for O although P
// has two parts), wait for each other more than for a unit: a barrier every 32 positions with a chain of S, softmax and O between,
// per 16 queries 4 products of S and 8 of O on the matrix cores and some 60 vector instructions of softmax; vector units are busy
// 47% of the time, and an eighth of the places of 224 tokens in groups of 64 are empty.
template <int QT, bool ALIGN, int NW, bool OWN>
__global__ void __launch_bounds__(64 * NW, OWN ? (NW == 8 && QT == 1 ? 4 : 2) : QT == 1 ? 4 : 2) cross_kernel(MzCross a, Launch n) {
    static_assert(OWN ? !ALIGN : NW == 4);
    __shared__ float red[OWN ? 1 : NW][16][68], ms[NW][16], ls[NW][16];
    __shared__ float lse2s[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    // x: (row, kv head), padded to a multiple of the XCDs, so that what shares keys and values shares an XCD; y: the tiles; z: the
    // shares of the blocks
    const int pairs = a.rows * a.kv_heads, pair = min((int)blockIdx.x, pairs - 1);
    const int tile = blockIdx.y, split = blockIdx.z, grp = n.group;
    const int r = divided(pair, a.kv_heads, n.by_heads), kh = pair - r * a.kv_heads;
    const Seen s = seen_of(a, r);
    constexpr int SHARE = OWN ? 4 : 1;
    const int nq = a.tokens * grp, w0 = tile * 16 * QT * SHARE;
    const int q0 = OWN ? w0 + 16 * QT * (wave & 3) : w0;  // this wave's first query
    auto token_of = [&](int x) { return divided(x, grp, n.by_group); };
    if ((int)blockIdx.x >= pairs || token_of(w0) >= s.count) return;  // none of its tokens is there
    const int nb = (s.end - s.first + BLK - 1) / BLK;
    // (shorter rows are shared by fewer)
    const int splits = OWN || n.splits == 1 ? 1 : min(n.splits, max(1, (nb + n.per - 1) / n.per));
    if (!OWN && split >= splits) return;
    const int b0 = splits == 1 ? 0 : (int)((long)nb * split / splits);
    const int b1 = splits == 1 ? nb : (int)((long)nb * (split + 1) / splits);

    const f16* kbase = a.k + s.slot * a.k_slot + kh * a.k_head + s.first * a.k_pos;
    const f16* vbase = a.v + s.slot * a.v_slot + kh * a.v_head + s.first * a.v_pos;
    const int there = s.end - s.first;  // positions

    extern __shared__ float kept[];  // [query][n.kept]
    __shared__ int index[ALIGN ? 64 : 1];
    const int mine = ALIGN && tid < a.heads ? a.head_slot[tid] : -1;
    f16x8 qf[QT][2];
    float* al[QT];
    auto align_row = [&](int t) -> float* {
        const int x = q0 + 16 * t + c, i = token_of(x), k = x < nq && i < s.count ? index[x - i * grp] : -1;
        return k >= 0 ? a.align + (((long)r * a.tokens + i) * a.align_heads + k) * a.align_cols : nullptr;
    };
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int x = q0 + 16 * t + c, i = token_of(x), h = kh * grp + x - i * grp;
        const bool on = x < nq && i < s.count;
        const f16* q = a.q + r * a.q_row + (on ? i * a.q_token + h * a.q_head : 0) + 16 * g;
        qf[t][0] = on ? ld8(q) : f16x8{};
        qf[t][1] = on ? ld8(q + 8) : f16x8{};
        al[t] = nullptr;
    }

    // Blocks past the last read as zeros, without a memory access: the loads need no branches, around which the compiler would
    // wait for all that is on its way.
    const unsigned kstep = (unsigned)(a.k_pos * 2), vstep = (unsigned)(a.v_pos * 2);
    const unsigned kat = (8 * (c >> 2) + (c & 3)) * kstep + 32 * g, vat = 8 * g * vstep + 8 * c;
    auto fetch = [&](int b, Raw& w) {
        const int left = b < b1 ? there - b * BLK : 0;
        const auto rk = positions_at(kbase + (long)b * BLK * a.k_pos, kstep, left);
        const auto rv = positions_at(vbase + (long)b * BLK * a.v_pos, vstep, left);
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int z = 0; z < 2; z++) w.k[j][z] = __builtin_amdgcn_raw_buffer_load_b128(rk, kat + 4 * j * kstep + 16 * z, 0, 0);
#pragma unroll
        for (int e = 0; e < 8; e++) w.v[e] = __builtin_amdgcn_raw_buffer_load_b64(rv, vat + e * vstep, 0, 0);
    };

    State<QT> st;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        st.m[t] = NOTHING;
        st.l[t] = 0.f;
#pragma unroll
        for (int u = 0; u < 4; u++) st.acc[t][u] = f32x4{};
    }
    const float scale2 = a.scale * LOG2E;
    float inf = INFINITY;
    asm("" : "+s"(inf));
    auto products = [&](int b, const f16x8 (&kf)[2][2], const f16x8 (&vf)[4]) {
        const int p0 = b * BLK + 8 * g;  // this lane's positions
        const bool whole = (b + 1) * BLK <= there;
#pragma unroll
        for (int t = 0; t < QT; t++) {
            f32x4 d[2];
#pragma unroll
            for (int j = 0; j < 2; j++) d[j] = mfma16(kf[j][1], qf[t][1], mfma16(kf[j][0], qf[t][0], f32x4{}));
            if (!whole) {
                asm volatile("");  // (a branch: selections would be made for every block)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (p0 + e >= there) d[e >> 2][e & 3] = -INFINITY;
            }
            if (ALIGN && al[t] != nullptr) {
                const f32x4 x[2] = {d[0] * scale2, d[1] * scale2};
                if (n.kept) {
                    f32x4* o = (f32x4*)(kept + (16 * t + c) * n.kept + p0 - b0 * BLK);
                    o[0] = x[0];
                    o[1] = x[1];
                } else {
                    for (int e = 0; e < 8; e++)
                        if (p0 + e < there && s.first + p0 + e < a.align_cols) {
                            float* o = al[t] + s.first + p0 + e;
                            if (splits > 1) shared_store(o, x[e >> 2][e & 3]);
                            else *o = x[e >> 2][e & 3];
                        }
                }
            }
            const float top = scale2 * fmaxf(fmaxf(larger(d[0][0], d[0][1], inf), larger(d[0][2], d[0][3], inf)),
                                             fmaxf(larger(d[1][0], d[1][1], inf), larger(d[1][2], d[1][3], inf)));
            if (__ballot(top > st.m[t] + 8.f)) {
                const float mn = fmaxf(st.m[t], column_max(top)), f = __builtin_amdgcn_exp2f(st.m[t] - mn);
                st.m[t] = mn;
                st.l[t] *= f;
#pragma unroll
                for (int u = 0; u < 4; u++) st.acc[t][u] *= f;
            }
            const float less = UP - st.m[t];
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __builtin_amdgcn_exp2f(fmaf(d[e >> 2][e & 3], scale2, less));
            st.l[t] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
            u32x4 high, rest;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                high[e] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(x[2 * e], x[2 * e + 1]));
                rest[e] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(less_low(x[2 * e], high[e]), less_high(x[2 * e + 1], high[e])));
            }
            const f16x8 p = __builtin_bit_cast(f16x8, high), q = __builtin_bit_cast(f16x8, rest);
#pragma unroll
            for (int u = 0; u < 4; u++) st.acc[t][u] = mfma16(vf[u], p, mfma16(vf[u], q, st.acc[t][u]));
        }
    };
    if constexpr (OWN) {
        // Each wave loads a quarter of a block, the keys' two tiles or half of each eight positions' values, and puts it as operands
        // where all find it, a block ahead; AHEAD more are on their way. What is behind the last block is that one again.
        constexpr int AHEAD = 2, FOURS = NW / 4;
        __shared__ u32x4 all_pieces[FOURS][2][8][64];
        const int four = wave >> 2, w4 = wave & 3;
        auto& pieces = all_pieces[four];
        // this four's blocks, and the most that one has
        const int from = four * ((nb + 1) / 2), to = FOURS == 1 || four ? nb : (nb + 1) / 2, steps = FOURS == 1 ? nb : (nb + 1) / 2;
        u32x4 raw[AHEAD][2];
        const bool values = w4 >= 2;
        auto take = [&](int i, u32x4 (&x)[2]) {
            const int b = min(from + i, nb - 1), left = there - b * BLK;
            if (!values) {
                const auto rk = positions_at(kbase + (long)b * BLK * a.k_pos, kstep, left);
#pragma unroll
                for (int z = 0; z < 2; z++) x[z] = __builtin_amdgcn_raw_buffer_load_b128(rk, kat + 4 * w4 * kstep + 16 * z, 0, 0);
            } else {
                const auto rv = positions_at(vbase + (long)b * BLK * a.v_pos, vstep, left);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rv, vat + (4 * (w4 - 2) + e) * vstep, 0, 0);
                    x[e >> 1][2 * (e & 1)] = v[0];
                    x[e >> 1][2 * (e & 1) + 1] = v[1];
                }
            }
        };
        auto put = [&](int i, const u32x4 (&y)[2]) {
            if (!values) {
                u32x4* o = &pieces[i & 1][2 * w4][lane];
                o[0] = y[0];
                o[64] = y[1];
            } else
#pragma unroll
                for (int u = 0; u < 4; u++) {  // channel 4 i + u of positions 4 (w4 - 2) .. + 3 of the lane's eight
                    const unsigned sel = u & 1 ? 0x07060302u : 0x05040100u;
                    u32x2 x;
#pragma unroll
                    for (int p = 0; p < 2; p++) x[p] = __builtin_amdgcn_perm(y[p][2 + (u >> 1)], y[p][u >> 1], sel);
                    ((u32x2*)&pieces[i & 1][4 + u][lane])[w4 - 2] = x;
                }
        };
        if (nb > 0) {
            take(0, raw[0]);
            put(0, raw[0]);
#pragma unroll
            for (int d = 0; d < AHEAD; d++) take(1 + d, raw[d]);
            __syncthreads();
            for (int i0 = 0; i0 < steps; i0 += AHEAD)
#pragma unroll
                for (int d = 0; d < AHEAD; d++) {
                    const int i = i0 + d;
                    if (i >= steps) break;
                    put(i + 1, raw[d]);
                    take(i + 1 + AHEAD, raw[d]);
                    f16x8 kf[2][2], vf[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        kf[k >> 1][k & 1] = __builtin_bit_cast(f16x8, pieces[i & 1][k][lane]);
                        vf[k] = __builtin_bit_cast(f16x8, pieces[i & 1][4 + k][lane]);
                    }
                    if (FOURS == 1 || from + i < to) products(from + i, kf, vf);
                    lds_barrier();
                }
        }
        if constexpr (FOURS == 2) {  // the second four's states to the first
            float* const parts = (float*)all_pieces;  // [4 QT][18][64 lanes]
            static_assert(4 * QT * 18 * 64 * 4 <= sizeof(all_pieces));
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float* o = parts + (w4 * QT + t) * 18 * 64 + lane;
                if (four) {
                    o[0] = st.m[t];
                    o[64] = st.l[t];
#pragma unroll
                    for (int e = 0; e < 16; e++) o[(2 + e) * 64] = st.acc[t][e >> 2][e & 3];
                }
            }
            __syncthreads();
            if (four) return;
#pragma unroll
            for (int t = 0; t < QT; t++) {
                const float* o = parts + (w4 * QT + t) * 18 * 64 + lane;
                const float m1 = o[0], mn = fmaxf(st.m[t], m1), f0 = __builtin_amdgcn_exp2f(st.m[t] - mn), f1 = __builtin_amdgcn_exp2f(m1 - mn);
                st.m[t] = mn;
                st.l[t] = fmaf(st.l[t], f0, o[64] * f1);
#pragma unroll
                for (int e = 0; e < 16; e++) st.acc[t][e >> 2][e & 3] = fmaf(st.acc[t][e >> 2][e & 3], f0, o[(2 + e) * 64] * f1);
            }
        }
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int x = q0 + 16 * t + c, i = token_of(x), h = kh * grp + x - i * grp;
            const float ll = column_sum(st.l[t]), f = ll == 0.f ? 0.f : 1.f / ll;
            if (x >= nq || i >= s.count) continue;
            f16* o = a.out + r * a.out_row + i * a.out_token + h * a.out_head + 16 * g;
#pragma unroll
            for (int z = 0; z < 2; z++) {
                f16x8 y;
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = (f16)(st.acc[t][e & 3][2 * z + (e >> 2)] * f);
                *(f16x8*)(o + 8 * z) = y;
            }
            if (a.lse && g == 0)
                a.lse[((long)r * a.tokens + i) * a.heads + h] = ll == 0.f ? -INFINITY : (st.m[t] - UP + __builtin_amdgcn_logf(ll)) * LN2;
        }
        return;
    } else {
        constexpr int DEPTH = 2;
        Raw w[DEPTH];
        const int head = b0 + wave;
#pragma unroll
        for (int i = 0; i < DEPTH; i++) fetch(head + NW * i, w[i]);
        if constexpr (ALIGN) {  // (while they are on their way)
            align_indices<64 * NW>(a.head_slot, a.align_heads, kh * grp, grp, mine, index);
#pragma unroll
            for (int t = 0; t < QT; t++) al[t] = align_row(t);
        }
        for (int b = head; b < b1; b += NW * DEPTH)
#pragma unroll
            for (int i = 0; i < DEPTH; i++) {
                const int bi = b + NW * i;
                if (bi < b1) {
                    f16x8 kf[2][2], vf[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) kf[j >> 1][j & 1] = __builtin_bit_cast(f16x8, w[i].k[j >> 1][j & 1]);
                    by_channels(w[i].v, vf);
                    products(bi, kf, vf);
                }
                fetch(bi + NW * DEPTH, w[i]);
            }
    }

    // the waves' states joined, 16 queries at a time
    const int col = tid >> 4, d4 = (tid & 15) * 4;
    // Alignment rows of 16 queries: their scores (in powers of two, get(query, row, position)) to probabilities, 0 where nothing
    // is seen, by all threads, eight of a row's scores a thread at a time and the first ones of four rows.
    constexpr int STRIDE = 64 * NW;
    auto rows = [&](int t) { return (unsigned)__ballot(al[t] != nullptr) & 0xffff; };
    auto row_of_query = [&](int t, int k) {
        const unsigned long at = (unsigned long)al[t];
        return (float*)((unsigned long)(unsigned)__builtin_amdgcn_readlane((int)(at >> 32), k) << 32 |
                        (unsigned)__builtin_amdgcn_readlane((int)at, k));
    };
    const int to = min(s.end, a.align_cols);
    auto scores = [&](int t, int k, int p0, float (&x)[8], auto get) {
        const float* row = row_of_query(t, k);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int p = p0 + STRIDE * j;
            x[j] = -INFINITY;
            if (p >= s.first && p < to) x[j] = get(16 * t + k, row, p);
        }
    };
    // of the first FEW of the rows `has`
    constexpr int FEW = 4;
    typedef float Few[FEW][8];
    auto few_scores = [&](int t, unsigned has, Few& x, auto get) {
#pragma unroll
        for (int u = 0; u < FEW; u++) {
            if (!has) break;
            scores(t, __ffs(has) - 1, tid, x[u], get);
            has &= has - 1;
        }
    };
    // (x: those of the first rows are on their way)
    auto probabilities = [&](int t, Few& x, auto get) {
        for (unsigned has = rows(t); has;) {
#pragma unroll
            for (int u = 0; u < FEW; u++) {
                if (!has) break;
                const int k = __ffs(has) - 1;
                has &= has - 1;
                float* const row = row_of_query(t, k);
                const float lse2 = lse2s[k];
                for (int p0 = tid; p0 < a.align_cols; p0 += 8 * STRIDE) {
                    if (p0 != tid) scores(t, k, p0, x[u], get);
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (p0 + STRIDE * j < a.align_cols)
                            row[p0 + STRIDE * j] = x[u][j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x[u][j] - lse2);
                }
            }
            few_scores(t, has, x, get);
        }
    };
    const int share0 = s.first + b0 * BLK;
    auto in_lds = [&](int q, const float*, int p) { return kept[q * n.kept + p - share0]; };
    auto in_place = [&](int, const float* row, int p) { return row[p]; };
    auto in_memory = [&](int, const float* row, int p) { return shared_load(row + p); };
    auto emit = [&](int t, float mm, float ll, f32x4 o, Few& x, auto get) {
        const int q = q0 + 16 * t + col, i = token_of(q), h = kh * grp + q - i * grp;
        const float inv = ll == 0.f ? 0.f : 1.f / ll, lse2 = ll == 0.f ? -INFINITY : mm - UP + __builtin_amdgcn_logf(ll);
        if (q < nq && i < s.count) {
            st4(a.out + r * a.out_row + i * a.out_token + h * a.out_head + d4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            if (a.lse && d4 == 0) a.lse[((long)r * a.tokens + i) * a.heads + h] = lse2 * LN2;
        }
        if (ALIGN) {
            if (d4 == 0) lse2s[col] = lse2;
            __syncthreads();
            probabilities(t, x, get);
            __syncthreads();
        }
    };
    float* const states = a.work + JOIN_COUNTERS + ((long)pair * n.tiles + tile) * n.splits * (16 * QT) * STATE;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const float lt = column_sum(st.l[t]);
#pragma unroll
        for (int e = 0; e < 4; e++)
            *(f32x4*)&red[wave][c][16 * g + 4 * e] = f32x4{st.acc[t][0][e], st.acc[t][1][e], st.acc[t][2][e], st.acc[t][3][e]};
        if (g == 0) {
            ms[wave][c] = st.m[t];
            ls[wave][c] = lt;
        }
        __syncthreads();
        float mm = ms[0][col], ll = 0.f;
#pragma unroll
        for (int k = 1; k < NW; k++) mm = fmaxf(mm, ms[k][col]);
        f32x4 o = {};
#pragma unroll
        for (int k = 0; k < NW; k++) {
            const float f = __builtin_amdgcn_exp2f(ms[k][col] - mm);
            ll = fmaf(f, ls[k][col], ll);
            const f32x4 y = *(const f32x4*)&red[k][col][d4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(f, y[e], o[e]);
        }
        if (splits == 1) {
            Few x;
            if (n.kept) {
                few_scores(t, ALIGN ? rows(t) : 0, x, in_lds);
                emit(t, mm, ll, o, x, in_lds);
            } else {
                few_scores(t, ALIGN ? rows(t) : 0, x, in_place);
                emit(t, mm, ll, o, x, in_place);
            }
        } else if (q0 + 16 * t + col < nq) {
            float* w = states + (split * (16 * QT) + 16 * t + col) * STATE;
            shared_store(w + d4, o[0], o[1]);
            shared_store(w + d4 + 2, o[2], o[3]);
            if (d4 == 0) shared_store(w + 64, mm, ll);
        }
        if (ALIGN && splits > 1 && n.kept)  // the share's scores to where the last workgroup finds them
            for (unsigned has = rows(t); has; has &= has - 1) {
                const int k = __ffs(has) - 1;
                float* const row = row_of_query(t, k);
                for (int p = share0 + tid; p < min(min(s.first + b1 * BLK, s.end), a.align_cols); p += STRIDE)
                    shared_store(row + p, in_lds(16 * t + k, row, p));
            }
        if (t + 1 < QT) __syncthreads();
    }
    if (splits == 1 || !last_of((unsigned*)a.work + (long)pair * n.tiles + tile, splits)) return;
    // the last of the workgroups that share these queries joins their states
#pragma unroll
    for (int t = 0; t < QT; t++) {
        float mm = NOTHING, ll = 0.f;
        f32x4 o = {};
        Few x;
        few_scores(t, ALIGN ? rows(t) : 0, x, in_memory);  // (they come with the states)
        if (q0 + 16 * t + col < nq)
            for (int k0 = 0; k0 < splits; k0 += 4) {
                float2 y[4][3];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float* w = states + (min(k0 + k, splits - 1) * (16 * QT) + 16 * t + col) * STATE;
                    y[k][0] = shared_load2(w + d4);
                    y[k][1] = shared_load2(w + d4 + 2);
                    y[k][2] = shared_load2(w + 64);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (k0 + k >= splits) continue;
                    const float mn = fmaxf(mm, y[k][2].x), f0 = __builtin_amdgcn_exp2f(mm - mn), f1 = __builtin_amdgcn_exp2f(y[k][2].x - mn);
                    mm = mn;
                    ll = fmaf(ll, f0, y[k][2].y * f1);
                    o = f32x4{fmaf(o[0], f0, y[k][0].x * f1), fmaf(o[1], f0, y[k][0].y * f1), fmaf(o[2], f0, y[k][1].x * f1),
                              fmaf(o[3], f0, y[k][1].y * f1)};
                }
            }
        emit(t, mm, ll, o, x, in_memory);
    }
}

// LDS for the scores of alignment rows
constexpr long KEPT_FLOATS = 8192, KEPT_FLOATS_ALONE = 24576;
long kept_queries(const Launch& n, long nq) { return std::min(nq, 16L * n.qt); }

Launch cross_shape(const MzCross& a) {
    const long grp = a.heads / a.kv_heads, nq = (long)a.tokens * grp, cus = mz_cu_count(), pairs = (long)a.rows * a.kv_heads;
    const long blocks = ((long)a.positions + BLK - 1) / BLK;
    auto inverse = [](int d) { return (unsigned)std::min((1ULL << 32) / d, 0xffffffffULL); };
    Launch n{};
    n.group = (int)grp;
    n.by_heads = inverse(a.kv_heads);
    n.by_group = inverse(n.group);
    n.waves = 4;
    n.splits = 1;
    // OWN where groups of 64 queries reach every CU. 20 heads, 1500 positions: 16 rows of 64 tokens (320 groups) 31 to 36 us, 42
    // without; 4 of 224 (320) 26.1 and 30.2, 8 of 224 (640) 38.8 and 48.8, 16 of 224 69 and 123. Of unequal rows 25.4 and 28.9, 25.3
    // and 21.9 (the one that it loses), 31.3 and 39.7, 48.7 and 78.3.
    const long groups = pairs * ((nq + 63) / 64);
    n.own = !a.align && nq > 16 && groups >= cus;
    if (n.own) {
        // Twice the queries a wave where groups of 128 fill the card five times and leave few places empty: 32 of 224 take 129 us,
        // 145 otherwise, 8 of 1500 169 and 183; but 16 of 224 (640 groups) 67 and 66, 64 of 64 126 and 95. Of unequal rows 96 and
        // 103, 124 and 129, 55 and 49, 95 and 74.
        const long wide = pairs * ((nq + 127) / 128);
        n.qt = wide >= 5 * cus && 16 * wide <= 9 * groups ? 2 : 1;
        // Eight waves where there is but one workgroup for many CUs: 16 of 64 take 31.5 us, 40.4 with four, 4 of 224 26.4 and 29.9;
        // 8 of 224 42.9 and 38.3. Of unequal rows 26.3 and 35.8, 25.6 and 29.3, 35.5 and 31.0.
        n.waves = groups < 2 * cus ? 8 : 4;
        n.tiles = (int)((nq + 64 * n.qt - 1) / (64 * n.qt));
        return n;
    }
    // (a workgroup of 16 queries reads keys and values once for them, one of 32 for twice as many)
    n.qt = nq <= 16 ? 1 : 2;
    n.tiles = (int)((nq + 16 * n.qt - 1) / (16 * n.qt));
    const long units = pairs * n.tiles;
    // Shares of at least five blocks: one row of 6 heads and 1500 positions takes 6.8 us with five, 7.1 with ten and 7.2 with three
    // (11.0 without shares), one of 20 heads 7.8, 7.6 and 9.8 (11.2).
    n.splits = (int)std::max(1L, std::min({cus / units, blocks / 5, 256L}));
    n.per = (int)((blocks + n.splits - 1) / n.splits);
    const long keep = (long)n.per * BLK;
    n.kept = a.align && keep * kept_queries(n, nq) <= (units * n.splits <= cus ? KEPT_FLOATS_ALONE : KEPT_FLOATS) ? (int)keep : 0;
    return n;
}
static_assert(JOIN_COUNTERS >= 1024, "units that are shared have a counter each: fewer than the CUs");

template <bool ALIGN>
void launch(hipStream_t s, const MzCross& a, const Launch& n) {
    const size_t lds = (size_t)n.kept * kept_queries(n, (long)a.tokens * n.group) * 4;
    const dim3 grid(((long)a.rows * a.kv_heads + 7) / 8 * 8, n.tiles, n.splits);
    if constexpr (!ALIGN)
        if (n.own) {
            if (n.qt == 2) hipLaunchKernelGGL((cross_kernel<2, false, 4, true>), grid, dim3(256), 0, s, a, n);
            else if (n.waves == 4) hipLaunchKernelGGL((cross_kernel<1, false, 4, true>), grid, dim3(256), 0, s, a, n);
            else hipLaunchKernelGGL((cross_kernel<1, false, 8, true>), grid, dim3(512), 0, s, a, n);
            return;
        }
    if (n.qt == 2) hipLaunchKernelGGL((cross_kernel<2, ALIGN, 4, false>), grid, dim3(256), lds, s, a, n);
    else hipLaunchKernelGGL((cross_kernel<1, ALIGN, 4, false>), grid, dim3(256), lds, s, a, n);
}

}  // namespace

// (a launch has fewer than 2^32 threads along x, and 2^16 workgroups along y and z; a block's positions lie within 2^30 bytes)
bool mz_cross_fits(const MzCross& a) {
    const long nq = (long)a.tokens * (a.heads / a.kv_heads);
    return (long)a.rows * a.kv_heads < (1L << 23) - 8 && nq <= 16L * 65535 && a.k_pos <= 1 << 24 && a.v_pos <= 1 << 24;
}

size_t mz_cross_work(const MzCross& a) {
    const Launch n = cross_shape(a);
    return n.splits > 1 ? ((size_t)a.rows * a.kv_heads * n.tiles * n.splits * 16 * n.qt * STATE + JOIN_COUNTERS) * 4 : 0;
}

hipError_t mz_cross_launch(hipStream_t s, const MzCross& a) {
    const Launch n = cross_shape(a);
    a.align ? launch<true>(s, a, n) : launch<false>(s, a, n);
    return hipGetLastError();
}
